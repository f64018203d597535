// tam_muon.hip -- momentum, orthogonalisation by Newton-Schulz products and
// parameter update of a list of matrices (C ABI: tam_orthogonalize).
//
// With s the smaller and l the larger side, x (s x l or, tall, l x s) and
// q = x x^T (tall: x^T x), a step is x <- (a I + b q + c q q) x (tall: from the
// right), three products; the first two are symmetric, and only the tiles on
// and below the diagonal are computed, each stored twice.
//
// Numbers.  The norm makes every singular value of x at most 1, and the step's
// polynomial keeps them near 1, so x, q and p = a I + b q + c q q are held as
// fp16 times 2^12 (p times 2^8 where the coefficients are large): entries up to 16, and 11 bits down to 1.5e-8 of x's scale,
// at the rate of bf16 with an eighth of its error.  What a step's rounding adds
// in x's small singular directions the next steps amplify like the directions
// themselves (a per step), so x keeps a low part, and x' = p x_high + diag(p)
// x_low: p x_low with p's diagonal alone, since p is near diagonal where x_low
// matters.  The low part is a byte (5 exponent and 2 fraction bits: the upper half
// of an fp16 number), 3 bits more than x_high: singular values over 5 decades
// come out 1e-3 of the result's norm off, 2e-2 without it and 7e-4 with 11 bits, and
// the products' epilogues, which all compute units reach together, move 4 bytes an
// element for 6.  Rounding a I into p, instead of adding a x, keeps the diagonal's
// rounding at the size of the result.  That is the scheme for bf16 matrices (error
// about 1e-3 of the result's norm, below bf16's own rounding 1.7e-3).  fp32 and
// fp16 matrices have high and low fp16 parts of x, q and p, and every product is
// high high + high low + low high: 22 bits, errors near those of fp32 sums.
//
// Launches (whole list each): tam_k_mu_momentum (momentum, partial squares of
// u), tam_k_mu_start (x = u / |u|, in parts), then per step tam_k_mu_square
// twice (q, p; tam_k_mu_join between them where q's sums are cut among workgroups)
// and tam_k_mu_apply (x, the last one: the output).  Small matrices take one launch
// of their own, tam_k_mu_small.
#include "tam_gemm.h"

#include <math.h>

#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

namespace {

constexpr float kScale = 4096.f;        // what fp16 entries are multiplied by (p's: see coefficients)
constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostPartials = 512; // of a matrix's squares
constexpr uint64_t kMostSide = 65536;

// A matrix as the kernels take it.  Unit counts run over the list: units of
// phase f of matrix i are first[f] .. first[f] of i + 1.
enum { MOMENTUM, START, GRAM, SQUARE, APPLY, PHASES };

struct mat {
  void* out;
  const void* grad;
  float* momentum;
  tam_f16* x[2];      // [rows][ldx] high parts, in turns; the low parts (split: fp16, else
                      // bytes) x_low elements behind
  tam_f16 *q, *p;     // [s][lds]
  float* diag;        // p's diagonal, fp32
  double* partial;    // squares of u
  uint64_t elements;
  int64_t x_low, s_low;  // elements from a high part to its low part (s_low 0: none)
  uint32_t rows, cols, s;
  uint32_t ldx, lds;  // of x, and of q and p: whole 128-byte lines
  uint32_t wx, ws;    // cols and s in whole 16 bytes: what a row holds, zeros behind the matrix
  uint32_t tall, split, dtype, flags;
  uint32_t first[PHASES];
  uint32_t partials, chunk;  // partial squares; elements of each
  float keep, one_minus_keep, eps, decay, rate;
};

struct list {
  const mat* m;
  uint32_t n;
  uint32_t units[PHASES];
  uint32_t parts;  // of the Gram products' sums, and where they go: 64 x 64 tiles
  float* sums;     // [unit][part]
};

// The matrix whose unit of phase F b is: the last one whose first unit is not
// past b.  64 matrices are looked at at once.
template <int F>
__device__ __forceinline__ uint32_t owner(const list& l, uint32_t b) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t found = 0;
  for (uint32_t i = 0; i < l.n; i += 64) {
    const bool in = i + lane < l.n && l.m[i + lane].first[F] <= b;
    const uint64_t mask = __ballot(in);
    if (!mask) break;
    found = i + 63u - (uint32_t)__builtin_clzll(mask);
    if (mask != ~0ull) break;
  }
  return __builtin_amdgcn_readfirstlane(found);
}

// A pointer of a descriptor: to global memory. (The compiler cannot know, and its
// flat stores count as LDS work too, which the epilogues' turns through LDS wait for.)
template <typename T>
__device__ __forceinline__ T* global(T* p) {
  return (T*)(__attribute__((address_space(1))) T*)(uint64_t)p;
}

// A descriptor in registers. Read where it lies, every field would be read again
// after each store (which might have changed it), behind that store: the products'
// epilogues had 300 such loads, 16 trips to memory one after another (seven matrices of
// 4096 by 14336: 15.7 ms a step, 14.4 without; one of 128 x 96: 56 us, 49 without).
__device__ __forceinline__ mat fetch(const mat& from) {
  mat d = from;
  d.out = global(d.out);
  d.grad = global(d.grad);
  d.momentum = global(d.momentum);
  d.x[0] = global(d.x[0]);
  d.x[1] = global(d.x[1]);
  d.q = global(d.q);
  d.p = global(d.p);
  d.diag = global(d.diag);
  d.partial = global(d.partial);
  return d;
}

// ---------------------------------------------------------------------------
// descriptors
// ---------------------------------------------------------------------------
constexpr int kPut = 16;  // descriptors that one launch carries as arguments
struct put_args {
  mat m[kPut];
};
static_assert(sizeof(put_args) <= 3968, "kernel arguments");

__global__ __launch_bounds__(256) void tam_k_mu_put(put_args a, mat* to, uint32_t n) {
  const uint32_t words = n * (uint32_t)(sizeof(mat) / 4);
  for (uint32_t i = threadIdx.x; i < words; i += 256)
    reinterpret_cast<uint32_t*>(to)[i] = reinterpret_cast<const uint32_t*>(&a)[i];
}

// ---------------------------------------------------------------------------
// u
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load_grad(const mat& m, uint64_t at, uint32_t count, float (&g)[8]) {
  if (m.dtype == TAM_DTYPE_F32)
    tam_load_some(static_cast<const float*>(m.grad) + at, count, g);
  else if (m.dtype == TAM_DTYPE_BF16)
    tam_load_some(static_cast<const tam_bf16*>(m.grad) + at, count, g);
  else
    tam_load_some(static_cast<const tam_f16*>(m.grad) + at, count, g);
}

// u of elements whose gradient is g and whose (new) momentum is m.
__device__ __forceinline__ void direction(const mat& d, const float (&g)[8], const float (&m)[8], float (&u)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    u[j] = !d.momentum ? g[j]
           : d.flags & TAM_MATRIX_NESTEROV ? __builtin_fmaf(d.keep, m[j], d.one_minus_keep * g[j])
                                           : m[j];
}

// The squares of u are summed in 64 bits: in 32 they leave the range where an element
// passes 2^64, or all of them stay below 2^-75 (and eps, if it is as small, does not
// take over).
typedef uint32_t halves __attribute__((ext_vector_type(2)));
template <int CTRL>
__device__ __forceinline__ double dpp_add(double x) {
  halves h = __builtin_bit_cast(halves, x);
  h.x = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)h.x, CTRL, 0xf, 0xf, true);
  h.y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)h.y, CTRL, 0xf, 0xf, true);
  return x + __builtin_bit_cast(double, h);
}
__device__ __forceinline__ double wave_sum(double x) {  // as tam_wave_sum
  x = dpp_add<0xb1>(x);
  x = dpp_add<0x4e>(x);
  x = dpp_add<0x141>(x);
  x = dpp_add<0x140>(x);
  halves h = __builtin_bit_cast(halves, x);
  const auto a = __builtin_amdgcn_permlane16_swap(h.x, h.x, false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(h.y, h.y, false, false);
  const halves l0 = {a[0], b[0]}, l1 = {a[1], b[1]};
  x = __builtin_bit_cast(double, l0) + __builtin_bit_cast(double, l1);
  h = __builtin_bit_cast(halves, x);
  const auto c = __builtin_amdgcn_permlane32_swap(h.x, h.x, false, false);
  const auto e = __builtin_amdgcn_permlane32_swap(h.y, h.y, false, false);
  const halves h0 = {c[0], e[0]}, h1 = {c[1], e[1]};
  return __builtin_bit_cast(double, h0) + __builtin_bit_cast(double, h1);
}

// Sum over the workgroup; every thread gets it.
__device__ __forceinline__ double group_sum(double x, double* lds) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// 8 squares onto a sum, in four chains.
__device__ __forceinline__ double add_squares(double sum, const float (&u)[8]) {
  double s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = __builtin_fma((double)u[j + 4], (double)u[j + 4], (double)u[j] * (double)u[j]);
  return sum + ((s[0] + s[1]) + (s[2] + s[3]));
}

// What brings u to x times 2^12: u 2^shift times `by`. (One factor for both would pass
// fp32's range, and with it 0 / eps be a NaN.)
struct normal {
  float by;
  int shift;
  __device__ __forceinline__ float operator()(float u) const { return __builtin_ldexpf(u, shift) * by; }
};

__device__ __forceinline__ normal normalise(double squares, float eps) {
  // |u| = n 2^k, n = the root of a number in [1/4, 1) (infinity and NaN stay in n)
  const int e = __builtin_amdgcn_frexp_exp(squares), k = (e + 1) >> 1;
  const float n = sqrtf((float)__builtin_ldexp(squares, -2 * k));
  if (__builtin_ldexp((double)n, k) < (double)eps) {
    const int ke = __builtin_amdgcn_frexp_exp((double)eps);
    return {kScale / __builtin_ldexpf(eps, -ke), -ke};
  }
  return {kScale / n, -k};
}

// A unit is `chunk` consecutive elements. Memory bounds it: the seven matrices of a
// layer of 4096 by 14336, 218M elements, bf16 with fp32 momentum: 448 us, 4.9 TB/s of
// 10 bytes an element (a large copy: 5.1).
__global__ __launch_bounds__(kThreads) void tam_k_mu_momentum(list l) {
  __shared__ double lds[4];
  const mat d = fetch(l.m[owner<MOMENTUM>(l, blockIdx.x)]);
  const uint32_t unit = blockIdx.x - d.first[MOMENTUM];
  const uint64_t begin = (uint64_t)unit * d.chunk, end = begin + d.chunk < d.elements ? begin + d.chunk : d.elements;
  double sum = 0.;
  for (uint64_t at = begin + threadIdx.x * 8u; at < end; at += kThreads * 8u) {
    const uint32_t count = end - at < 8 ? (uint32_t)(end - at) : 8u;
    float g[8], m[8] = {}, u[8];
    load_grad(d, at, count, g);
    if (d.momentum) {
      tam_load_some<float>(d.momentum + at, count, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = __builtin_fmaf(d.one_minus_keep, g[j], d.keep * m[j]);
      tam_store_some(d.momentum + at, count, m);
    }
    direction(d, g, m, u);
    sum = add_squares(sum, u);
  }
  sum = group_sum(sum, lds);
  if (threadIdx.x == 0) d.partial[unit] = sum;
}

__device__ __forceinline__ void store_parts(tam_f16* high, int64_t low, const float (&v)[8]) {
  float h[8], r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // The fp32 value itself: the compiler otherwise rounds a product that v is
    // straight to fp16 for one of its uses (v_fma_mixlo_f16) and by way of fp32
    // for the other, and where the two differ, high + low is off by high's last bit.
    float x = v[j];
    asm("" : "+v"(x));
    h[j] = (float)(tam_f16)x;
    r[j] = x - h[j];  // exact
  }
  tam_store8(high, h);
  if (low) tam_store8(high + low, r);
}

// Bytes of 5 exponent and 2 fraction bits: 8 of them from fp32, rounded, and back.
struct bytes8 {
  uint32_t w[2];
};
__device__ __forceinline__ bytes8 to_bytes(const float (&v)[8]) {
  bytes8 b;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_bf8_f32(v[4 * i], v[4 * i + 1], 0, false);
    b.w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(v[4 * i + 2], v[4 * i + 3], w, true);
  }
  return b;
}
__device__ __forceinline__ float from_byte(const bytes8& b, int j) {
  const uint16_t bits = (uint16_t)((b.w[j / 4] >> (8 * (j % 4)) & 255u) << 8);
  return (float)__builtin_bit_cast(tam_f16, bits);
}

__device__ __forceinline__ uint8_t* low_bytes(const mat& d, const tam_f16* x) {
  return reinterpret_cast<uint8_t*>(const_cast<tam_f16*>(x) + d.x_low);
}

// 8 elements of x (times 2^12) in its parts.
__device__ __forceinline__ void store_x(const mat& d, tam_f16* x, uint64_t at, const float (&v)[8]) {
  if (d.split) {
    store_parts(x + at, d.x_low, v);
  } else {
    float y[8], r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = v[j];
      asm("" : "+v"(y[j]));  // as in store_parts
      r[j] = y[j] - (float)(tam_f16)y[j];
    }
    tam_store8(x + at, y);
    *reinterpret_cast<bytes8*>(low_bytes(d, x) + at) = to_bytes(r);
  }
}

// x = u / max(|u|, eps) times 2^12, in parts.  A unit is 2048 elements of x's
// rows of ldx; the columns past the matrix are zeros up to wx. Memory bounds it (the
// same list: 366 us, 5.4 TB/s): u is made again from the gradient and the momentum, 6
// bytes an element, for 4 to write and 4 to read of a copy of u.
constexpr uint32_t kStart = 2048;

__global__ __launch_bounds__(kThreads) void tam_k_mu_start(list l) {
  __shared__ double lds[4];
  const mat d = fetch(l.m[owner<START>(l, blockIdx.x)]);
  double sum = 0.;
  for (uint32_t i = threadIdx.x; i < d.partials; i += kThreads) sum += d.partial[i];
  const normal to_x = normalise(group_sum(sum, lds), d.eps);
  const uint64_t at = (uint64_t)(blockIdx.x - d.first[START]) * kStart + threadIdx.x * 8u;
  if (at >= (uint64_t)d.rows * d.ldx) return;
  const uint32_t row = (uint32_t)(at / d.ldx), col = (uint32_t)(at - (uint64_t)row * d.ldx);
  if (col >= d.wx) return;
  const uint32_t count = d.cols - col < 8 ? d.cols - col : 8u;
  const uint64_t from = (uint64_t)row * d.cols + col;
  float g[8], m[8] = {}, u[8];
  load_grad(d, from, count, g);
  if (d.momentum) tam_load_some<float>(d.momentum + from, count, m);
  direction(d, g, m, u);
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] = to_x(u[j]);
  store_x(d, d.x[0], at, u);
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
__device__ __forceinline__ tam_operand operand(const tam_f16* p, uint32_t ld, uint32_t count) {
  return {reinterpret_cast<const char*>(p), (uint64_t)ld * 2u, count, nullptr};
}

// The polynomial's coefficients as p's sums take them, of q q times 2^24, q times 2^12
// and 1, for p times its scale; back: 1 / scale. p's entries reach |a| + |b| + |c|
// where x's singular values are at most 1 (a alone where they are small: a zero
// matrix's p is a I): the scale is 2^12, or 2^8 (entries up to 255) from 15 on.
struct coefficients {
  float qq, q, one, back;
};

// Tile t of the lower triangle, row by row: rows m, columns n <= m.
__device__ __forceinline__ void triangle(uint32_t t, uint32_t& m, uint32_t& n) {
  m = (uint32_t)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while (m * (m + 1) / 2 > t) --m;
  while ((m + 1) * (m + 2) / 2 <= t) ++m;
  n = t - m * (m + 1) / 2;
}

// FIRST: q = x x^T (tall: x^T x).  Otherwise p = a I + b q + c q q. Bound by the matrix
// cores: the same list's q 847 us (1020 TFLOP/s of the triangles' operations), p 378
// (915: 700 tiles are 2.7 rounds of 256 workgroups, and a tile's epilogue stores it
// twice).
template <int TILE, int WM, int WN, bool FIRST>
__global__ __launch_bounds__(64 * WM * WN, TILE == 64 ? 3 : 2) void tam_k_mu_square(
    list l, uint32_t turn, coefficients co) {
  typedef tam_tile<tam_f16, TILE, TILE, WM, WN, tam_stages<tam_f16, TILE>(), true, true> Rows;
  typedef tam_tile<tam_f16, TILE, TILE, WM, WN, tam_stages<tam_f16, TILE>(), false, false> Columns;
  __shared__ __attribute__((aligned(16))) char smem[Rows::LDS > Columns::LDS ? Rows::LDS : Columns::LDS];
  const uint32_t unit = tam_xcd_order(blockIdx.x, gridDim.x);
  const mat d = fetch(l.m[owner<FIRST ? GRAM : SQUARE>(l, unit)]);
  uint32_t tm, tn;
  triangle(unit - d.first[FIRST ? GRAM : SQUARE], tm, tn);
  const uint32_t r0 = tm * TILE, c0 = tn * TILE;
  // the part of the sum that is this workgroup's (FIRST: blockIdx.y of l.parts)
  uint64_t k0 = 0, k1 = FIRST ? (d.tall ? d.rows : d.wx) : d.ws;
  if (FIRST && l.parts > 1) {
    const uint64_t each = (k1 + l.parts * 64u - 1) / (l.parts * 64u) * 64u;
    k0 = blockIdx.y * each < k1 ? blockIdx.y * each : k1;
    k1 = k0 + each < k1 ? k0 + each : k1;
  }
  struct parts {
    tam_oct<tam_f16> high, low;
  };
  // q where p is made from it
  auto load = [&](uint32_t row, uint32_t col) {
    parts q;
    if (!FIRST && row < d.s && col < d.ws) {
      const tam_f16* from = d.q + (uint64_t)row * d.lds + col;
      q.high = *reinterpret_cast<const tam_oct<tam_f16>*>(from);
      if (d.s_low) q.low = *reinterpret_cast<const tam_oct<tam_f16>*>(from + d.s_low);
    }
    return q;
  };
  auto store = [&](uint32_t row, uint32_t col, float(&v)[8], const parts& q) {
    if (row >= d.s || col >= d.ws) return;
    if constexpr (FIRST) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= 1.f / kScale;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = (float)q.high.v[j] + (d.s_low ? (float)q.low.v[j] : 0.f);
        v[j] = __builtin_fmaf(co.q, x, co.qq * v[j]);
      }
      if (row - col < 8) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
          if (row - col == j) {
            v[j] += co.one;
            d.diag[row] = v[j] * co.back;
          }
      }
    }
    store_parts((FIRST ? d.q : d.p) + (uint64_t)row * d.lds + col, d.s_low, v);
  };
  auto finish = [&](auto& t) {
    typedef typename std::remove_reference<decltype(t)>::type Tile;
    if constexpr (FIRST && TILE == 64) {
      if (l.parts > 1) {
        float* out = l.sums + ((uint64_t)unit * l.parts + blockIdx.y) * (64 * 64);
        t.template each<TAM_AHEAD_PASS>(
            smem, [](uint32_t, uint32_t) { return 0; },
            [&](uint32_t row, uint32_t col, float(&v)[8], int) { tam_store8(out + row * 64 + col, v); },
            [](uint32_t, uint32_t, const float*, int) {});
        return;
      }
    }
    t.template each<TAM_AHEAD_ROUND>(
        smem, [&](uint32_t row, uint32_t col) { return load(row + r0, col + c0); },
        [&](uint32_t row, uint32_t col, float(&v)[8], const parts& q) { store(row + r0, col + c0, v, q); },
        [&](uint32_t row, uint32_t col, const float* turned, int pitch) {
          // off the diagonal, the mirrored tile: element (row, col) also goes to (col, row).
          // A lane takes 8 rows of one column: 4 lanes to a column's 32 rows.
          if (tm == tn) return;
          const uint32_t lane = threadIdx.x & 63, from = (lane & 3) * 8, to_col = r0 + row + from;
          constexpr int N = Tile::COLS / 16;
          parts q[N];
#pragma unroll
          for (int i = 0; i < N; ++i) q[i] = load(c0 + col + i * 16 + (lane >> 2), to_col);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint32_t c = i * 16 + (lane >> 2);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = turned[(from + j) * pitch + c];
            store(c0 + col + c, to_col, v, q[i]);
          }
        });
  };
  tam_soon soon = {};  // q, where p is made from it
  if (!FIRST)
    soon = {reinterpret_cast<const char*>(d.q + (uint64_t)r0 * d.lds + c0), (uint64_t)d.lds * 2u, d.s - r0,
            (d.ws - c0) * 2u, TILE * 2u};
  if (FIRST && d.tall) {
    Columns t;
    t.zero();
    const tam_operand x = operand((turn ? d.x[1] : d.x[0]), d.ldx, d.wx);
    t.template run<true>(x, x, c0, r0, k0, k1, smem, soon, {d.split ? 3u : 1u, d.x_low * 2, d.x_low * 2});
    finish(t);
  } else {
    Rows t;
    t.zero();
    const tam_operand x = FIRST ? operand((turn ? d.x[1] : d.x[0]), d.ldx, d.rows) : operand(d.q, d.lds, d.s);
    const int64_t low = (FIRST ? d.x_low : d.s_low) * 2;
    t.template run<true>(x, x, c0, r0, k0, k1, smem, soon, {d.split ? 3u : 1u, low, low});
    finish(t);
  }
}

// q from the parts' sums of its tiles, added in their order.
__global__ __launch_bounds__(kThreads) void tam_k_mu_join(list l) {
  __shared__ float tile[64][65];
  const mat d = fetch(l.m[owner<GRAM>(l, blockIdx.x)]);
  uint32_t tm, tn;
  triangle(blockIdx.x - d.first[GRAM], tm, tn);
  const float* from = l.sums + (uint64_t)blockIdx.x * l.parts * (64 * 64);
  const uint32_t col = (threadIdx.x & 7u) * 8u;
  for (uint32_t row = threadIdx.x >> 3; row < 64; row += kThreads / 8) {
    float v[8] = {};
    for (uint32_t p = 0; p < l.parts; ++p) {
      float s[8];
      tam_load8(from + p * (64 * 64) + row * 64 + col, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += s[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] *= 1.f / kScale;
      tile[row][col + j] = v[j];
    }
    const uint32_t r = tm * 64 + row, c = tn * 64 + col;
    if (r < d.s && c < d.ws) store_parts(d.q + (uint64_t)r * d.lds + c, d.s_low, v);
  }
  if (tm == tn) return;
  __syncthreads();
  for (uint32_t row = threadIdx.x >> 3; row < 64; row += kThreads / 8) {
    const uint32_t r = tn * 64 + row, c = tm * 64 + col;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = tile[col + j][row];
    if (r < d.s && c < d.ws) store_parts(d.q + (uint64_t)r * d.lds + c, d.s_low, v);
  }
}

// What the last product's epilogue needs of the parameter, loaded ahead.
struct held {
  bytes8 low;            // of x, where it is bytes
  float p;               // wide: p's diagonal at the row
  tam_oct<float> out;    // the parameter: 16 or 32 bytes
};

template <typename T>
__device__ __forceinline__ void hold(const mat& d, uint32_t row, uint32_t col, held& h) {
  const T* out = static_cast<const T*>(d.out) + (uint64_t)row * d.cols + col;
  const tam_oct<T> o = *reinterpret_cast<const tam_oct<T>*>(out);
  __builtin_memcpy(&h.out, &o, sizeof(o));
}

template <typename T>
__device__ __forceinline__ void write_out(const mat& d, uint32_t row, uint32_t col, float (&v)[8], const held& h) {
  T* out = static_cast<T*>(d.out) + (uint64_t)row * d.cols + col;
  const bool update = d.flags & TAM_MATRIX_UPDATE;
  if (col + 8 <= d.cols) {
    if (update) {
      tam_oct<T> p;
      __builtin_memcpy(&p, &h.out, sizeof(p));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(-d.rate, v[j], d.decay * (float)p.v[j]);
    }
    tam_store8(out, v);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      if (col + j < d.cols)
        out[j] = tam_from_f<T>(update ? __builtin_fmaf(-d.rate, v[j], d.decay * tam_to_f(out[j])) : v[j]);
  }
}

// x' = p x (tall: x p); LAST: the output instead. back: coefficients::back. Bound by the matrix cores: the same
// list 1540 us, 1127 TFLOP/s, LAST 1555 (it reads the parameter and writes it back); the
// epilogues, which all workgroups of a round reach together, are a tenth of that.
template <int TILE, int WM, int WN, bool LAST>
__global__ __launch_bounds__(64 * WM * WN, TILE == 64 ? 3 : 2) void tam_k_mu_apply(list l, uint32_t turn, float back) {
  typedef tam_tile<tam_f16, TILE, TILE, WM, WN, tam_stages<tam_f16, TILE>(), false, true> Wide;
  typedef tam_tile<tam_f16, TILE, TILE, WM, WN, tam_stages<tam_f16, TILE>(), true, true> Tall;
  __shared__ __attribute__((aligned(16))) char smem[Wide::LDS > Tall::LDS ? Wide::LDS : Tall::LDS];
  const uint32_t unit = tam_xcd_order(blockIdx.x, gridDim.x);
  const mat d = fetch(l.m[owner<APPLY>(l, unit)]);
  uint32_t tm, tn;
  tam_tile_at(unit - d.first[APPLY], (d.rows + TILE - 1) / TILE, (d.cols + TILE - 1) / TILE, tm, tn);
  const uint32_t r0 = tm * TILE, c0 = tn * TILE;
  const tam_f16* x = (turn ? d.x[1] : d.x[0]);
  auto finish = [&](auto& t) {
    typedef typename std::remove_reference<decltype(t)>::type Tile;
    float diag[8] = {};  // tall: p's diagonal at the lane's columns, the same in every row
    if (d.tall && !d.split) {
      const uint32_t lane = threadIdx.x & 63, col = c0 + ((threadIdx.x >> 6) % WN) * Tile::COLS + lane % (Tile::COLS / 8) * 8;
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) diag[j] = col + j < d.cols ? d.diag[col + j] : 0.f;
    }
    // (the last product also holds the parameter: all of it would not fit the registers)
    t.template each<LAST ? TAM_AHEAD_ROUND : TAM_AHEAD_ALL>(
        smem,
        [&](uint32_t row, uint32_t col) {
          held h;
          row += r0;
          col += c0;
          if (row >= d.rows || col >= d.cols) return h;
          if (!d.split) {
            h.low = *reinterpret_cast<const bytes8*>(low_bytes(d, x) + (uint64_t)row * d.ldx + col);
            if (!d.tall) h.p = d.diag[row];
          }
          if (LAST && (d.flags & TAM_MATRIX_UPDATE) && col + 8 <= d.cols) {
            if (d.dtype == TAM_DTYPE_F32)
              hold<float>(d, row, col, h);
            else
              hold<tam_f16>(d, row, col, h);  // 16 bytes of either 16-bit type
          }
          return h;
        },
        [&](uint32_t row, uint32_t col, float(&v)[8], const held& h) {
          row += r0;
          col += c0;
          if (row >= d.rows || col >= d.cols) return;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= back;
          if (!d.split) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(d.tall ? diag[j] : h.p, from_byte(h.low, j), v[j]);
          }
          if constexpr (LAST) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= 1.f / kScale;
            if (d.dtype == TAM_DTYPE_F32)
              write_out<float>(d, row, col, v, h);
            else if (d.dtype == TAM_DTYPE_BF16)
              write_out<tam_bf16>(d, row, col, v, h);
            else
              write_out<tam_f16>(d, row, col, v, h);
          } else {
            store_x(d, (turn ? d.x[0] : d.x[1]), (uint64_t)row * d.ldx + col, v);
          }
        },
        [](uint32_t, uint32_t, const float*, int) {});
  };
  const tam_operand p = operand(d.p, d.lds, d.s);
  const uint32_t terms = d.split ? 3u : 1u;
  // x's low bytes; with high and low products the last epilogue's parameter instead
  tam_soon soon = {};
  if (!d.split) {
    soon = {reinterpret_cast<const char*>(low_bytes(d, x)) + (uint64_t)r0 * d.ldx + c0, d.ldx, d.rows - r0, d.wx - c0, TILE};
  } else if (LAST && (d.flags & TAM_MATRIX_UPDATE)) {
    const uint32_t size = d.dtype == TAM_DTYPE_F32 ? 4u : 2u;
    const uint64_t ld = (uint64_t)d.cols * size;
    soon = {static_cast<const char*>(d.out) + r0 * ld + (uint64_t)c0 * size, ld, d.rows - r0, (d.cols - c0) * size, TILE * size};
    if (((uintptr_t)soon.base | ld) & 3u) soon.base = nullptr;
  }
  if (d.tall) {
    Tall t;
    t.zero();
    t.template run<true>(p, operand(x, d.ldx, d.rows), c0, r0, 0, d.ws, smem, soon, {terms, d.s_low * 2, d.x_low * 2});
    finish(t);
  } else {
    Wide t;
    t.zero();
    t.template run<true>(operand(x, d.ldx, d.wx), p, c0, r0, 0, d.rows, smem, soon, {terms, d.x_low * 2, d.s_low * 2});
    finish(t);
  }
}

// ---------------------------------------------------------------------------
// small matrices: everything in one workgroup
// ---------------------------------------------------------------------------
// Sides of up to 128: x, and q and then p in its place, with their low parts, lie in
// LDS (128 KB), s rows of up to 128 columns (a tall matrix transposed), and the
// three products of a step run on the 8 waves, 32 rows by half of the columns of the
// result to each, with barriers between them. One launch for any number of such matrices: 128 x 96 in
// fp32 took 110 us in 18 launches of 4 to 8 us each, most of that the way to memory
// and back between them; here it takes 49, about 7 a step. Of the 16 x 16
// blocks that a step multiplies at 128 x 96, two fifths are not needed (columns 96 to 127
// of q and p, and one triangle of each), and two of the eight waves have no rows.
constexpr uint32_t kSmall = 128;
constexpr uint32_t kSmallThreads = 512;

// Rows of 256 bytes, 16-byte chunk c of row r at place c ^ (r & 15).
__device__ __forceinline__ uint32_t small_at(uint32_t row, uint32_t col) {
  return row * 256u + (((col >> 3) ^ (row & 15u)) << 4) + (col & 7u) * 2u;
}

// Rows row0 .. + 15, k = k0 .. k0 + 31 along the row.
__device__ __forceinline__ tam_frag<tam_f16> small_rows(const tam_lds_char* m, uint32_t row0, uint32_t k0, uint32_t lane) {
  tam_frag<tam_f16> f;
  f.v = *(const tam_lds_s8*)(m + small_at(row0 + (lane & 15u), k0 + 8u * (lane >> 4)));
  return f;
}

// Columns col0 .. + 15, k = k0 .. k0 + 31 down the rows (the transposing read).
__device__ __forceinline__ tam_frag<tam_f16> small_columns(const tam_lds_char* m, uint32_t col0, uint32_t k0, uint32_t lane) {
  const uint32_t i = lane & 15u, k = k0 + 8u * (lane >> 4) + (i >> 2), col = col0 + 4u * (i & 3u);
  const tam_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tam_lds_s4*)(m + small_at(k, col)));
  const tam_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tam_lds_s4*)(m + small_at(k + 4u, col)));
  tam_frag<tam_f16> f;
  f.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return f;
}

// 4 elements (times 2^12) at row, col in both parts.
__device__ __forceinline__ void small_store(char* high, char* low, uint32_t row, uint32_t col, const tam_f4& v) {
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  f16x4 h, r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = v[j];
    asm("" : "+v"(x));  // as in store_parts
    h[j] = (tam_f16)x;
    r[j] = (tam_f16)(x - (float)h[j]);
  }
  *reinterpret_cast<f16x4*>(high + small_at(row, col)) = h;
  *reinterpret_cast<f16x4*>(low + small_at(row, col)) = r;
}

template <typename T>
__device__ __forceinline__ void small_out(const mat& d, uint32_t row, uint32_t col, float v) {
  T* out = static_cast<T*>(d.out) + (uint64_t)row * d.cols + col;
  *out = tam_from_f<T>(d.flags & TAM_MATRIX_UPDATE ? __builtin_fmaf(-d.rate, v, d.decay * tam_to_f(*out)) : v);
}

// BLOCKS: 16-column blocks of the largest matrix (2, 4 or 8); all of them are
// computed, zeros or not, so that the reads of one k run ahead of its products.
template <int BLOCKS>
__global__ __launch_bounds__(kSmallThreads) void tam_k_mu_small(mat only, const mat* list, coefficients co, uint32_t steps) {
  __shared__ __attribute__((aligned(16))) char smem[4 * 32768];
  __shared__ double lds[8];
  char *const xh = smem, *const xl = smem + 32768, *const qh = smem + 65536, *const ql = smem + 98304;
  const tam_lds_char *const Xh = (tam_lds_char*)xh, *const Xl = (tam_lds_char*)xl;
  const tam_lds_char *const Qh = (tam_lds_char*)qh, *const Ql = (tam_lds_char*)ql;
  const mat d = fetch(list ? list[blockIdx.x] : only);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t s = d.s, width = d.tall ? d.rows : d.cols;
  // elements past the matrix are zeros in every factor
  for (uint32_t i = threadIdx.x; i < sizeof(smem) / 16; i += kSmallThreads)
    reinterpret_cast<tam_i4*>(smem)[i] = tam_i4{0, 0, 0, 0};
  constexpr int GROUPS = (BLOCKS * BLOCKS * 32 + (int)kSmallThreads - 1) / (int)kSmallThreads;  // of 8 elements a thread
  float u[GROUPS][8];
  double sum = 0.;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const uint64_t at = (uint64_t)(g * kSmallThreads + threadIdx.x) * 8u;
    const uint32_t count = at >= d.elements ? 0u : (d.elements - at < 8 ? (uint32_t)(d.elements - at) : 8u);
    float gr[8], m[8] = {};
    load_grad(d, at, count, gr);
    if (d.momentum) {
      tam_load_some<float>(d.momentum + at, count, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = __builtin_fmaf(d.one_minus_keep, gr[j], d.keep * m[j]);
      tam_store_some(d.momentum + at, count, m);
    }
    direction(d, gr, m, u[g]);
    sum = add_squares(sum, u[g]);
  }
  sum = wave_sum(sum);
  if (lane == 0) lds[wave] = sum;
  __syncthreads();
  sum = 0.;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += lds[w];
  const normal to_x = normalise(sum, d.eps);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const uint32_t at = (g * kSmallThreads + threadIdx.x) * 8u;
    uint32_t row = at / d.cols, col = at - row * d.cols;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      if (at + j < d.elements) {
        float x = to_x(u[g][j]);
        asm("" : "+v"(x));  // as in store_parts
        const tam_f16 h = (tam_f16)x;
        const uint32_t to = d.tall ? small_at(col, row) : small_at(row, col);
        *reinterpret_cast<tam_f16*>(xh + to) = h;
        *reinterpret_cast<tam_f16*>(xl + to) = (tam_f16)(x - (float)h);
      }
      if (++col == d.cols) {
        col = 0;
        ++row;
      }
    }
  }
  __syncthreads();
  // A wave's part of a result: 32 rows by half of the blocks' columns.
  constexpr int CB = BLOCKS / 2;
  const uint32_t row0 = wave / 2 * 32, col0 = wave % 2 * (CB * 16);
  const uint32_t lane_row = lane & 15u, quad = (lane >> 4) * 4u;
  const bool works = row0 < s;
  tam_f4 acc[CB][2];
  const bool split = d.split;
  // acc = sum over k of left's rows (of the result) and right's columns, in parts (bf16:
  // of the high parts)
  auto product = [&](const tam_lds_char* lh, const tam_lds_char* ll, const tam_lds_char* rh, const tam_lds_char* rl,
                     uint32_t length, auto right) {
#pragma unroll
    for (int n = 0; n < CB; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m) acc[n][m] = tam_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (uint32_t k = 0; k < length; k += 32) {
      tam_frag<tam_f16> h[2], r[2], ch[CB], cr[CB];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        h[m] = small_rows(lh, row0 + m * 16, k, lane);
        if (split) r[m] = small_rows(ll, row0 + m * 16, k, lane);
      }
#pragma unroll
      for (int n = 0; n < CB; ++n) {
        ch[n] = right(rh, col0 + n * 16, k);
        if (split) cr[n] = right(rl, col0 + n * 16, k);
      }
      // term by term: a sum's next product comes after all the others'
#pragma unroll
      for (int n = 0; n < CB; ++n)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[n][m] = tam_mfma(ch[n], h[m], acc[n][m]);
      if (!split) continue;
#pragma unroll
      for (int n = 0; n < CB; ++n)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[n][m] = tam_mfma(ch[n], r[m], acc[n][m]);
#pragma unroll
      for (int n = 0; n < CB; ++n)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[n][m] = tam_mfma(cr[n], h[m], acc[n][m]);
    }
  };
  auto in_rows = [&](const tam_lds_char* m, uint32_t first, uint32_t k) { return small_rows(m, first, k, lane); };
  auto in_columns = [&](const tam_lds_char* m, uint32_t first, uint32_t k) { return small_columns(m, first, k, lane); };
  // f(row, first of 4 columns, acc) over what the wave holds
  auto each = [&](auto f) {
#pragma unroll
    for (int n = 0; n < CB; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m) f(row0 + m * 16 + lane_row, col0 + n * 16 + quad, acc[n][m]);
  };
  for (uint32_t step = 0; step < steps; ++step) {
    if (works) {  // q = x x^T
      product(Xh, Xl, Xh, Xl, width, in_rows);
      each([&](uint32_t row, uint32_t col, tam_f4& v) { small_store(qh, ql, row, col, v * (1.f / kScale)); });
    }
    __syncthreads();
    if (works) {  // p = a I + b q + c q q
      product(Qh, Ql, Qh, Ql, s, in_rows);
      each([&](uint32_t row, uint32_t col, tam_f4& v) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        const f16x4 h = *reinterpret_cast<const f16x4*>(qh + small_at(row, col));
        const f16x4 r = *reinterpret_cast<const f16x4*>(ql + small_at(row, col));
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          v[j] = __builtin_fmaf(co.q, (float)h[j] + (float)r[j], co.qq * v[j]) +
                 (col + j == row && row < s ? co.one : 0.f);
      });
    }
    __syncthreads();  // q is read
    if (works) each([&](uint32_t row, uint32_t col, tam_f4& v) { small_store(qh, ql, row, col, v); });
    __syncthreads();
    if (works) {  // p x
      product(Qh, Ql, Xh, Xl, s, in_columns);
      if (!split)
        each([&](uint32_t row, uint32_t col, tam_f4& v) {  // and p's diagonal times x's low part
          typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
          const float p = (float)*reinterpret_cast<const tam_f16*>(qh + small_at(row, row));
          const f16x4 r = *reinterpret_cast<const f16x4*>(xl + small_at(row, col));
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(p, (float)r[j], v[j]);
        });
    }
    __syncthreads();  // x is read
    if (works && step + 1 < steps)
      each([&](uint32_t row, uint32_t col, tam_f4& v) { small_store(xh, xl, row, col, v * co.back); });
    __syncthreads();
  }
  if (!works) return;
  each([&](uint32_t row, uint32_t col, tam_f4& v) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      const uint32_t r = d.tall ? col + j : row, c = d.tall ? row : col + j;
      if (r >= d.rows || c >= d.cols) continue;
      const float x = v[j] * co.back * (1.f / kScale);
      if (d.dtype == TAM_DTYPE_F32)
        small_out<float>(d, r, c, x);
      else if (d.dtype == TAM_DTYPE_BF16)
        small_out<tam_bf16>(d, r, c, x);
      else
        small_out<tam_f16>(d, r, c, x);
    }
  });
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct plan {
  std::vector<mat> m;  // `large` ones, then the small ones
  int large;
  uint64_t bytes;
  int tile[PHASES];
  uint32_t units[PHASES];
  uint32_t parts;      // of the Gram products' sums
  float* sums;
};

int check(const TamMatrix* m, int n) {
  tam_op_begin();
  if (n < 0 || (n > 0 && !m)) return tam_op_fail(TAM_E_INVALID, "null argument");
  for (int i = 0; i < n; ++i) {
    const TamMatrix& d = m[i];
    if (!d.out || !d.grad) return tam_op_fail(TAM_E_INVALID, "matrix %d: null out or grad", i);
    if (!d.rows || !d.cols) return tam_op_fail(TAM_E_INVALID, "matrix %d has no elements", i);
    if (d.rows > kMostSide || d.cols > kMostSide)
      return tam_op_fail(TAM_E_UNSUPPORTED, "matrix %d: a side of more than %llu", i, (unsigned long long)kMostSide);
    if (d.dtype > TAM_DTYPE_F16) return tam_op_fail(TAM_E_INVALID, "matrix %d: unknown dtype %u", i, d.dtype);
    if (!(d.eps > 0.f)) return tam_op_fail(TAM_E_INVALID, "matrix %d: eps must be above 0", i);
    if ((uintptr_t)d.momentum & 3u) return tam_op_fail(TAM_E_INVALID, "matrix %d: misaligned momentum", i);
  }
  return TAM_OK;
}

uint64_t tiles(uint64_t rows, uint64_t cols, int t) { return tam_div_up(rows, t) * tam_div_up(cols, t); }
uint64_t triangle_tiles(uint64_t s, int t) { return tam_div_up(s, t) * (tam_div_up(s, t) + 1) / 2; }

// The tile of a phase, and (GRAM) the parts that its sums are cut into: the least of
// what the launches take at the measured rates (tam_tiles_us), for all tiles as if of
// one k, and no less than the longest one. Parts are of 64 x 64 tiles, and their sums
// go to memory and back (about 4 TB/s) through one launch more.
struct shape {
  int tile;
  uint32_t parts;
};

shape pick(const mat* m, int n, int phase) {
  const double cus = tam_op_cus();
  shape best = {64, 1};
  double least = 1e30;
  for (const tam_tile_rate& t : tam_rates_16) {
    double count = 0, sum = 0, longest = 0;
    for (int i = 0; i < n; ++i) {
      const mat& d = m[i];
      // q's sum runs over the longer side, p's and x's over the shorter one
      const double k = (phase == GRAM ? std::max(d.rows, d.cols) : d.s) * (d.split ? 3.0 : 1.0);
      const double c = (double)(phase == APPLY ? tiles(d.rows, d.cols, t.tile) : triangle_tiles(d.s, t.tile));
      count += c;
      sum += c * k;
      longest = std::max(longest, k);
    }
    for (uint32_t parts : {1, 2, 4, 8, 16, 32}) {
      if (parts > 1 && (phase != GRAM || t.tile != 64 || longest / parts < 256)) break;
      double us = std::max(tam_tiles_us(t, count * parts, sum / count / parts, cus), t.start + longest / parts * t.half);
      if (parts > 1) us += 4.0 + count * parts * (64 * 64 * 8) / 4e6;
      if (us < least) {
        least = us;
        best = {t.tile, parts};
      }
    }
  }
  return best;
}

// Lays the list out: the largest sums first, so that no long tile starts last.
int make(const TamMatrix* in, int n, char* base, plan& out) {
  std::vector<int> order(n);
  for (int i = 0; i < n; ++i) order[i] = i;
  auto larger = [&](int i) { return std::max(in[i].rows, in[i].cols); };
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) { return larger(i) > larger(j); });
  out.m.resize(n);
  out.large = 0;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    char* p = (char*)((uintptr_t)base + at);
    at += tam_up(bytes, 256);
    return p;
  };
  take((uint64_t)n * sizeof(mat));
  for (int k = 0; k < n; ++k) {
    const TamMatrix& d = in[order[k]];
    mat& m = out.m[k];
    m = mat{};
    m.out = d.out;
    m.grad = d.grad;
    m.momentum = d.momentum;
    m.rows = (uint32_t)d.rows;
    m.cols = (uint32_t)d.cols;
    m.elements = d.rows * d.cols;
    m.tall = d.rows > d.cols;
    m.s = m.tall ? m.cols : m.rows;
    m.wx = (uint32_t)tam_up(d.cols, 8);
    m.ws = (uint32_t)tam_up(m.s, 8);
    m.ldx = (uint32_t)tam_up(d.cols, 64);
    m.lds = (uint32_t)tam_up(m.s, 64);
    m.dtype = d.dtype;
    m.flags = d.flags;
    m.split = d.dtype != TAM_DTYPE_BF16;
    m.keep = d.keep;
    m.one_minus_keep = d.one_minus_keep;
    m.eps = d.eps;
    m.decay = d.decay;
    m.rate = d.rate;
    if (std::max(m.rows, m.cols) <= kSmall) continue;  // these come last
    out.large = k + 1;
    m.x_low = (int64_t)tam_up((uint64_t)m.rows * m.ldx, 128);
    const int64_t square = (int64_t)tam_up((uint64_t)m.s * m.lds, 128);
    m.s_low = m.split ? square : 0;
    for (int i = 0; i < 2; ++i) m.x[i] = (tam_f16*)take(m.x_low * (m.split ? 4 : 3));
    m.q = (tam_f16*)take(square * (m.split ? 4 : 2));
    m.p = (tam_f16*)take(square * (m.split ? 4 : 2));
    m.diag = (float*)take((uint64_t)m.s * 4);
    m.chunk = (uint32_t)tam_up(tam_div_up(m.elements, kMostPartials), kThreads * 8);
    m.partials = (uint32_t)tam_div_up(m.elements, m.chunk);
    m.partial = (double*)take((uint64_t)m.partials * 8);
  }
  for (int f = GRAM; f < PHASES; ++f) {
    const shape s = pick(out.m.data(), out.large, f);
    out.tile[f] = s.tile;
    if (f == GRAM) out.parts = s.parts;
  }
  uint64_t units[PHASES] = {};
  for (int i = 0; i < out.large; ++i) {
    mat& m = out.m[i];
    for (int f = 0; f < PHASES; ++f) m.first[f] = (uint32_t)units[f];
    units[MOMENTUM] += m.partials;
    units[START] += tam_div_up((uint64_t)m.rows * m.ldx, kStart);
    units[GRAM] += triangle_tiles(m.s, out.tile[GRAM]);
    units[SQUARE] += triangle_tiles(m.s, out.tile[SQUARE]);
    units[APPLY] += tiles(m.rows, m.cols, out.tile[APPLY]);
  }
  for (int f = 0; f < PHASES; ++f) {
    if (units[f] >= 1ull << 31) return tam_op_fail(TAM_E_UNSUPPORTED, "matrices of too many elements for one call");
    out.units[f] = (uint32_t)units[f];
  }
  out.sums = out.parts > 1 ? (float*)take(units[GRAM] * out.parts * (64 * 64 * 4)) : nullptr;
  out.bytes = at;
  return TAM_OK;
}

template <bool FIRST>
void launch_square(int tile, const list& l, uint32_t turn, coefficients co, hipStream_t s) {
  const dim3 grid(l.units[FIRST ? GRAM : SQUARE], FIRST ? l.parts : 1);
  if (tile == 256)
    hipLaunchKernelGGL((tam_k_mu_square<256, 2, 4, FIRST>), grid, dim3(512), 0, s, l, turn, co);
  else if (tile == 128)
    hipLaunchKernelGGL((tam_k_mu_square<128, 2, 2, FIRST>), grid, dim3(256), 0, s, l, turn, co);
  else
    hipLaunchKernelGGL((tam_k_mu_square<64, 2, 2, FIRST>), grid, dim3(256), 0, s, l, turn, co);
}

template <bool LAST>
void launch_apply(int tile, const list& l, uint32_t turn, float back, hipStream_t s) {
  const dim3 grid(l.units[APPLY]);
  if (tile == 256)
    hipLaunchKernelGGL((tam_k_mu_apply<256, 2, 4, LAST>), grid, dim3(512), 0, s, l, turn, back);
  else if (tile == 128)
    hipLaunchKernelGGL((tam_k_mu_apply<128, 2, 2, LAST>), grid, dim3(256), 0, s, l, turn, back);
  else
    hipLaunchKernelGGL((tam_k_mu_apply<64, 2, 2, LAST>), grid, dim3(256), 0, s, l, turn, back);
}

int orthogonalize(const TamMatrix* in, int n, const float* c, int steps, void* workspace, size_t ws_bytes,
                  hipStream_t s, size_t* need, uint32_t* tiles) {
  int rc = check(in, n);
  if (rc != TAM_OK) return rc;
  plan p;
  p.bytes = 0;
  if (n) rc = make(in, n, (char*)workspace, p);
  if (rc != TAM_OK) return rc;
  if (need) {
    *need = (size_t)p.bytes;
    if (tiles && n && p.large) {
      const uint32_t told[4] = {(uint32_t)p.tile[GRAM], p.parts, (uint32_t)p.tile[SQUARE], (uint32_t)p.tile[APPLY]};
      std::copy(told, told + 4, tiles);
    }
    return TAM_OK;
  }
  if (!c) return tam_op_fail(TAM_E_INVALID, "null argument");
  if (!(fabsf(c[0]) < 64.f && fabsf(c[1]) < 64.f && fabsf(c[2]) < 64.f))
    return tam_op_fail(TAM_E_INVALID, "a coefficient of 64 or more, or none");
  if (steps < 1 || steps > 64) return tam_op_fail(TAM_E_INVALID, "steps must be 1 to 64");
  if (n == 0) return TAM_OK;
  if (p.bytes > ws_bytes || !workspace)
    return tam_op_fail(TAM_E_WORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)ws_bytes,
                       (unsigned long long)p.bytes);
  if ((uintptr_t)workspace & 255u) return tam_op_fail(TAM_E_INVALID, "workspace not on 256 bytes");
  mat* table = (mat*)workspace;
  const bool only = n == 1 && !p.large;  // one small matrix goes as an argument
  for (int i = 0; i < n && !only; i += kPut) {
    put_args a;
    const int k = n - i < kPut ? n - i : kPut;
    for (int j = 0; j < kPut; ++j) a.m[j] = j < k ? p.m[i + j] : mat{};
    hipLaunchKernelGGL(tam_k_mu_put, dim3(1), dim3(256), 0, s, a, table + i, (uint32_t)k);
    TAM_OP_LAUNCHED("the descriptors");
  }
  const float scale = fabsf(c[0]) + fabsf(c[1]) + fabsf(c[2]) < 15.f ? kScale : 256.f;
  const coefficients co = {c[2] * scale / (kScale * kScale), c[1] * scale / kScale, c[0] * scale, 1.f / scale};
  if (p.large < n) {
    const uint32_t side = std::max(p.m[p.large].rows, p.m[p.large].cols);  // the list's largest
    const dim3 grid((uint32_t)(n - p.large)), block(kSmallThreads);
    const mat* list = only ? nullptr : table + p.large;
    if (side <= 32)
      hipLaunchKernelGGL(tam_k_mu_small<2>, grid, block, 0, s, p.m[p.large], list, co, (uint32_t)steps);
    else if (side <= 64)
      hipLaunchKernelGGL(tam_k_mu_small<4>, grid, block, 0, s, p.m[p.large], list, co, (uint32_t)steps);
    else
      hipLaunchKernelGGL(tam_k_mu_small<8>, grid, block, 0, s, p.m[p.large], list, co, (uint32_t)steps);
    TAM_OP_LAUNCHED("the small matrices");
  }
  if (!p.large) return TAM_OK;
  list l = {table, (uint32_t)p.large, {}, p.parts, p.sums};
  for (int f = 0; f < PHASES; ++f) l.units[f] = p.units[f];
  hipLaunchKernelGGL(tam_k_mu_momentum, dim3(l.units[MOMENTUM]), dim3(kThreads), 0, s, l);
  TAM_OP_LAUNCHED("the momentum");
  hipLaunchKernelGGL(tam_k_mu_start, dim3(l.units[START]), dim3(kThreads), 0, s, l);
  TAM_OP_LAUNCHED("the normalisation");
  for (int i = 0; i < steps; ++i) {
    const uint32_t turn = i & 1;
    launch_square<true>(p.tile[GRAM], l, turn, co, s);
    TAM_OP_LAUNCHED("the Gram product");
    if (p.parts > 1) {
      hipLaunchKernelGGL(tam_k_mu_join, dim3(l.units[GRAM]), dim3(kThreads), 0, s, l);
      TAM_OP_LAUNCHED("the Gram product's sums");
    }
    launch_square<false>(p.tile[SQUARE], l, turn, co, s);
    TAM_OP_LAUNCHED("the polynomial");
    if (i + 1 < steps)
      launch_apply<false>(p.tile[APPLY], l, turn, co.back, s);
    else
      launch_apply<true>(p.tile[APPLY], l, turn, co.back, s);
    TAM_OP_LAUNCHED("the polynomial's product");
  }
  return TAM_OK;
}

// No exception leaves the library: the plan's memory is all that can fail.
int guarded(const TamMatrix* in, int n, const float* c, int steps, void* ws, size_t bytes, hipStream_t s,
            size_t* need, uint32_t* tiles = nullptr) {
  try {
    return orthogonalize(in, n, c, steps, ws, bytes, s, need, tiles);
  } catch (const std::bad_alloc&) {
    return tam_op_fail(TAM_E_INVALID, "no host memory for %d matrices", n);
  }
}

}  // namespace

extern "C" {

int tam_orthogonalize_workspace(const TamMatrix* matrices, int n, size_t* bytes) {
  if (!bytes) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  return guarded(matrices, n, nullptr, 0, nullptr, 0, nullptr, bytes);
}

int tam_orthogonalize_tiles(const TamMatrix* matrices, int n, uint32_t* tiles) {
  if (!tiles) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  std::fill(tiles, tiles + 4, 0u);
  size_t need = 0;
  return guarded(matrices, n, nullptr, 0, nullptr, 0, nullptr, &need, tiles);
}

int tam_orthogonalize(const TamMatrix* matrices, int n, const float* coefficients, int steps, void* workspace,
                      size_t ws_bytes, void* stream) {
  return guarded(matrices, n, coefficients, steps, workspace, ws_bytes, (hipStream_t)stream, nullptr);
}

}  // extern "C"
