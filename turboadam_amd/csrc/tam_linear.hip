// tam_linear.hip -- linear layer of the C ABI: y = act(x w^T + bias) + residual
// and its gradients, on the tile core of tam_gemm.h.
//
//   z = x w^T + bias,  y = act(z) + residual
//   dz = dy act'(z),   dx = dz w,  dw = dz^T x,  dbias = sum over rows of dz
//
// Kernels:
//   tam_k_gemm   one tile of a product; the forward epilogue adds the bias, keeps
//                z (rounded to the type) for the backward pass, applies the
//                activation and adds the residual, all in fp32, and rounds once;
//   tam_k_split  the same epilogue over the partial sums of a product whose k was
//                cut among workgroups (few tiles);
//   tam_k_few    the forward product of up to 32 rows: every wave reads its part
//                of 16 weight rows once, straight to the matrix cores;
//   tam_k_slope  dz and its column sums;  tam_k_column_sum: the sums' end.
#include "tam_act.h"
#include "tam_few.h"
#include "tam_products.h"

// ---------------------------------------------------------------------------
// epilogue
// ---------------------------------------------------------------------------
struct tam_epilogue {
  void* out;            // [rows][cols], contiguous
  const void* bias;     // [cols] or null
  const void* residual; // [rows][cols] or null
  void* z;              // [rows][cols] or null
  uint32_t rows, cols, act;
};

// Eight elements of the residual, loaded ahead of their use.
template <typename T>
__device__ __forceinline__ tam_oct<T> tam_residual(const tam_epilogue& e, uint32_t row, uint32_t col) {
  tam_oct<T> r;
  if (e.residual && row < e.rows && col + 8 <= e.cols)
    r = *reinterpret_cast<const tam_oct<T>*>(static_cast<const T*>(e.residual) + (uint64_t)row * e.cols + col);
  return r;
}

// Eight elements of the bias: a lane's columns are the same in every row of a tile.
// (Loaded for each row they came behind the row's stores, 16 times a tile.)
template <typename T>
__device__ __forceinline__ tam_oct<T> tam_bias(const tam_epilogue& e, uint32_t col) {
  tam_oct<T> b;
  if (e.bias && col + 8 <= e.cols) b = *reinterpret_cast<const tam_oct<T>*>(static_cast<const T*>(e.bias) + col);
  return b;
}

// v holds columns col .. col + 7 of a row of the product, r what tam_residual gave and
// b what tam_bias gave.
template <typename T>
__device__ __forceinline__ void tam_finish(const tam_epilogue& e, uint32_t row, uint32_t col, float (&v)[8],
                                           const tam_oct<T>& r, const tam_oct<T>& b) {
  const uint64_t at = (uint64_t)row * e.cols + col;
  if (col + 8 <= e.cols) {
    if (e.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += (float)b.v[j];
    }
    // rounded to the type: half of the memory of fp32, and an error of one rounding of z
    // times the activation's second derivative
    if (e.z) tam_store8(static_cast<T*>(e.z) + at, v);
    if (e.act != TAM_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tam_act<sizeof(T) == 2>(v[j], e.act);
    }
    if (e.residual) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += (float)r.v[j];
    }
    tam_store8(static_cast<T*>(e.out) + at, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (col + j >= e.cols) break;
      float x = v[j];
      if (e.bias) x += tam_to_f(static_cast<const T*>(e.bias)[col + j]);
      if (e.z) static_cast<T*>(e.z)[at + j] = tam_from_f<T>(x);
      x = tam_act<sizeof(T) == 2>(x, e.act);
      if (e.residual) x += tam_to_f(static_cast<const T*>(e.residual)[at + j]);
      static_cast<T*>(e.out)[at + j] = tam_from_f<T>(x);
    }
  }
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------
struct tam_gemm_args {
  tam_operand P, Q;   // P: the columns' operand, Q: the rows'
  uint64_t k, k_part; // of the tiles' sums; of one of the parts they are cut into
  uint64_t k_all;     // of the whole sum: what is left is the first part's
  uint32_t tm, tn;    // tiles
  float* partial;     // [part][rows][cols] fp32, or null: one part
  tam_epilogue e;
};

// Bound by the matrix cores and, beside them, by LDS (operands in, fragments out).
// 8192 x 14336 x 4096 bf16, 256 tiles (means over 200 passes, from card to card 5%
// either way): 681 us with both operands along k (1413 TFLOP/s), 715 for dx (one
// m-major), 755 for dw (both); a library product of 8192^3 reaches 1398 to 1564 TFLOP/s from card to card, and on
// operands of zeros, at the clock that they leave, this one 1900.
// 8192 x 768 x 3072, 128 tiles: 70 us for y and z (its 100 MB of stores are the second
// bound), 47 for dx and dw each. fp32 1531 x 1001 x 777, 64 tiles: 30, 34 and 39 us;
// 17 are its operations at 143 TFLOP/s, the rest is 312 to 416 tiles on 256 compute
// units and single-word reads of m-major fragments.
// REST: operands whose rows may end inside 16 bytes.
template <typename T, int BM, int BN, int WM, int WN, bool PK, bool QK, bool REST>
__global__ __launch_bounds__(64 * WM * WN, BM == 64 ? 3 : 2) void tam_k_gemm(tam_gemm_args a) {
  typedef tam_tile<T, BM, BN, WM, WN, tam_stages<T, BM>(), PK, QK, REST> Tile;
  __shared__ __attribute__((aligned(16))) char smem[Tile::LDS];
  uint32_t m, n;
  tam_tile_at(tam_xcd_order(blockIdx.x, gridDim.x), a.tm, a.tn, m, n);
  const uint64_t k0 = blockIdx.y * a.k_part;
  const uint64_t k1 = k0 + a.k_part < a.k ? k0 + a.k_part : a.k;
  Tile t;
  t.zero();
  tam_soon soon = {};
  if (a.e.residual && !a.partial) {
    const uint64_t ld = (uint64_t)a.e.cols * sizeof(T);
    soon = {static_cast<const char*>(a.e.residual) + m * BM * ld + n * BN * sizeof(T), ld, a.e.rows - m * BM,
            (a.e.cols - n * BN) * (uint32_t)sizeof(T), BN * (uint32_t)sizeof(T)};
    if (((uintptr_t)soon.base | ld) & 3u) soon.base = nullptr;
  }
  t.run(a.P, a.Q, n * BN, m * BM, k0, k1, smem, soon);
  if (REST && blockIdx.y == 0) t.tail(a.P, a.Q, n * BN, m * BM, a.k, a.k_all);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  tam_oct<T> bias;
  if (!a.partial) bias = tam_bias<T>(a.e, n * BN + wave % WN * Tile::COLS + lane % (Tile::COLS / 8) * 8);
  t.template each<TAM_AHEAD_PASS>(
      smem, [&](uint32_t row, uint32_t col) { return tam_residual<T>(a.e, row + m * BM, col + n * BN); },
      [&](uint32_t row, uint32_t col, float(&v)[8], const tam_oct<T>& r) {
        row += m * BM;
        col += n * BN;
        if (row >= a.e.rows || col >= a.e.cols) return;
        if (a.partial) {
          float* p = a.partial + ((uint64_t)blockIdx.y * a.e.rows + row) * a.e.cols + col;
          if (col + 8 <= a.e.cols) {
            tam_store8(p, v);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (col + j < a.e.cols) p[j] = v[j];
          }
        } else {
          tam_finish<T>(a.e, row, col, v, r, bias);
        }
      },
      [](uint32_t, uint32_t, const float*, int) {});
}

// The parts' sums in their order, then the epilogue: a thread takes 8 columns. Two
// parts of 1531 x 777 fp32, gelu and residual: 8.9 us, and the products they join 30 (43
// uncut).
template <typename T>
__global__ __launch_bounds__(256) void tam_k_split(const float* partial, uint32_t parts, tam_epilogue e) {
  const uint32_t per = (e.cols + 7) / 8;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (uint64_t)per * e.rows) return;
  const uint32_t row = (uint32_t)(i / per), col = (uint32_t)(i - (uint64_t)row * per) * 8;
  const uint64_t at = (uint64_t)row * e.cols + col, step = (uint64_t)e.rows * e.cols;
  float v[8] = {};
  if (col + 8 <= e.cols) {
    for (uint32_t p = 0; p < parts; ++p) {
      float t[8];
      tam_load8(partial + p * step + at, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
  } else {
    for (uint32_t p = 0; p < parts; ++p)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < e.cols) v[j] += partial[p * step + at + j];
  }
  tam_finish<T>(e, row, col, v, tam_residual<T>(e, row, col), tam_bias<T>(e, col));
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------
// One workgroup: 16 columns of y (16 weight rows) for up to 16 * MT rows of x.
// Its 8 waves take the k axis in turns of 4 chunks to a lane; a lane of fragment
// row i loads the chunks at k0 + 8 * (4 u + lane / 16), u = 0..3: a wave's four
// loads of a row are 256 consecutive bytes. Bound by reading w once; x stays in
// the caches. The waves' sums meet in LDS in wave order.
struct tam_few_args {
  const void* x;
  const void* w;
  uint64_t ldx, ldw, k;  // elements
  tam_epilogue e;
};

template <typename T, int MT>
__global__ __launch_bounds__(64 * TAM_FEW_WAVES) void tam_k_few(tam_few_args a) {
  constexpr int N = 16 / (int)sizeof(T), U = 4;
  constexpr uint64_t TURN = 4 * U * N;  // k of a wave's turn
  __shared__ float sum[TAM_FEW_WAVES][MT * 16][20];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t i = lane & 15, q = lane >> 4, n = blockIdx.x * 16 + i;
  // rows past the last one read the first one's elements; their sums go nowhere
  const T* w = static_cast<const T*>(a.w) + (n < a.e.cols ? (uint64_t)n * a.ldw : 0);
  const T* x[MT];
  tam_f4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    x[m] = static_cast<const T*>(a.x) + (m * 16 + i < a.e.rows ? (uint64_t)(m * 16 + i) * a.ldx : 0);
    acc[m] = tam_f4{0.f, 0.f, 0.f, 0.f};
  }
  auto turn = [&](uint64_t k0, auto guard) {
    constexpr bool G = decltype(guard)::value;
    tam_frag<T> fw[U], fx[MT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) tam_few_load<T, G>(fw[u], w, k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) tam_few_load<T, G>(fx[m][u], x[m], k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) acc[m] = tam_mfma(fw[u], fx[m][u], acc[m]);
  };
  uint64_t k0 = wave * TURN;
#pragma unroll 2
  for (; k0 + TURN <= a.k; k0 += TAM_FEW_WAVES * TURN) turn(k0, std::false_type());
  if (k0 < a.k) turn(k0, std::true_type());
#pragma unroll
  for (int m = 0; m < MT; ++m)  // row m * 16 + i, columns 4 q ..
    *reinterpret_cast<tam_f4*>(&sum[wave][m * 16 + i][q * 4]) = acc[m];
  __syncthreads();
  const uint32_t t = threadIdx.x, row = t / 2;
  uint32_t col = (t % 2) * 8;
  if (t < MT * 32 && row < a.e.rows && blockIdx.x * 16 + col < a.e.cols) {
    float v[8] = {};
    for (int s = 0; s < TAM_FEW_WAVES; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += sum[s][row][col + j];
    col += blockIdx.x * 16;
    tam_finish<T>(a.e, row, col, v, tam_residual<T>(a.e, row, col), tam_bias<T>(a.e, col));
  }
}

// ---------------------------------------------------------------------------
// the backward pass's elementwise part
// ---------------------------------------------------------------------------
// A workgroup takes 512 columns (8 to a lane) of a run of rows, its waves every
// fourth row; dz leaves rounded to the type, and the columns' sums of dz in fp32,
// one row of `sums` to a run. dz == null: the sums alone (of dy). The rounding is
// what dx's and dw's matrix instructions take: in bf16 it brings their errors from
// 1.7e-3 of the result (its own rounding) to 2.4e-3; two parts of dz would double both
// products. Memory bounds it: 8192 x 3072 bf16, gelu_tanh: 33 us, 4.5 TB/s.
struct tam_slope_args {
  const void* dy;
  const void* z;
  void* dz;
  float* sums;     // [runs][cols] or null
  uint64_t ld_dz;  // elements
  uint32_t rows, cols, run, act;
};

template <typename T>
__global__ __launch_bounds__(256) void tam_k_slope(tam_slope_args a) {
  __shared__ float part[3][64][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t col = blockIdx.x * 512 + lane * 8;
  const uint32_t r0 = blockIdx.y * a.run, r1 = a.rows - r0 < a.run ? a.rows : r0 + a.run;
  const uint32_t count = col < a.cols ? a.cols - col : 0;
  float s[8] = {};
  if (col < a.cols) {
    for (uint32_t r = r0 + wave; r < r1; r += 4) {
      const uint64_t at = (uint64_t)r * a.cols + col;
      float d[8], z[8];
      tam_load_some(static_cast<const T*>(a.dy) + at, count, d);
      if (a.act != TAM_ACT_NONE) tam_load_some(static_cast<const T*>(a.z) + at, count, z);
      if (a.act != TAM_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] *= tam_act_slope<sizeof(T) == 2>(z[j], a.act);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += d[j];
      // rows of dz are whole 16 bytes: columns past the last one are zeros
      if (a.dz) tam_store8(static_cast<T*>(a.dz) + (uint64_t)r * a.ld_dz + col, d);
    }
  }
  if (!a.sums) return;
  if (wave) {
#pragma unroll
    for (int j = 0; j < 8; ++j) part[wave - 1][lane][j] = s[j];
  }
  __syncthreads();
  if (wave == 0 && col < a.cols) {
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += part[w][lane][j];
    float* out = a.sums + (uint64_t)blockIdx.y * a.cols + col;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < a.cols) out[j] = s[j];
  }
}

// out[c] = sum over runs of sums[run][c]: 64 columns to a workgroup, its 16 waves
// take every 16th run (171 runs of 3072: 4.7 us, 2 of them the launch).
template <typename T>
__global__ __launch_bounds__(1024) void tam_k_column_sum(const float* sums, uint32_t runs, uint32_t cols, T* out) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (uint32_t r = wave; r < runs; r += 16) s += sums[(uint64_t)r * cols + c];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < cols) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += part[w][lane];
    out[c] = tam_from_f<T>(v);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

int check_linear(const TamLinear* d, bool backward) {
  tam_op_begin();
  if (!d) return tam_op_fail(TAM_E_INVALID, "null argument");
  if (d->dtype > TAM_DTYPE_F16) return tam_op_fail(TAM_E_INVALID, "unknown dtype %u", d->dtype);
  if (d->activation > TAM_ACT_MAX) return tam_op_fail(TAM_E_INVALID, "unknown activation %u", d->activation);
  const uint64_t most = 1ull << 31;
  if (d->rows >= most || d->inputs >= most || d->outputs >= most)
    return tam_op_fail(TAM_E_UNSUPPORTED, "a size of 2^31 or more");
  if (d->inputs && (d->ldx < d->inputs || d->ldw < (d->w_in_out ? d->outputs : d->inputs)))
    return tam_op_fail(TAM_E_INVALID, "a row stride shorter than its row");
  // a tile's offsets of up to 256 rows are 31-bit numbers of bytes
  if ((d->ldx | d->ldw | d->inputs | d->outputs) >= 1ull << 21)
    return tam_op_fail(TAM_E_UNSUPPORTED, "a row or row stride of 2^21 elements or more");
  if (d->rows == 0 || d->outputs == 0) return TAM_OK;
  if (d->inputs && (!d->x || !d->w)) return tam_op_fail(TAM_E_INVALID, "null x or w");
  if (!backward && !d->y) return tam_op_fail(TAM_E_INVALID, "null y");
  if (backward && !d->dy) return tam_op_fail(TAM_E_INVALID, "null dy");
  if (backward && d->activation != TAM_ACT_NONE && !d->z) return tam_op_fail(TAM_E_INVALID, "null z");
  return TAM_OK;
}

// ---- products ----

template <typename T, int TILE, int WM, int WN, bool REST>
void launch_tile(bool pk, bool qk, const tam_gemm_args& a, uint32_t parts, hipStream_t s) {
  const dim3 grid(a.tm * a.tn, parts), block(64 * WM * WN);
  if (pk && qk)
    hipLaunchKernelGGL((tam_k_gemm<T, TILE, TILE, WM, WN, true, true, REST>), grid, block, 0, s, a);
  else if (qk)
    hipLaunchKernelGGL((tam_k_gemm<T, TILE, TILE, WM, WN, false, true, REST>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((tam_k_gemm<T, TILE, TILE, WM, WN, false, false, REST>), grid, block, 0, s, a);
}

template <typename T>
void launch_gemm(int tile, bool pk, bool qk, bool rest, const tam_gemm_args& a, uint32_t parts, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (tile == 256) return launch_tile<T, 256, 2, 4, false>(pk, qk, a, parts, s);
  if (tile == 128)
    return rest ? launch_tile<T, 128, 2, 2, true>(pk, qk, a, parts, s) : launch_tile<T, 128, 2, 2, false>(pk, qk, a, parts, s);
  rest ? launch_tile<T, 64, 2, 2, true>(pk, qk, a, parts, s) : launch_tile<T, 64, 2, 2, false>(pk, qk, a, parts, s);
}

// Whether m is read as it lies, and not a copy whose rows are whole lines. Rows that may end inside 16 bytes
// have kernels of their own (REST), as the bound on their loads and the rest of their
// sums would cost the others 1% (x [8192, 768], w [768, 3072], bf16, both ways: 206 -> 208
// us), and a copy of [2018, 13611] fp32 would be 25 of 110 us. The 256 tile is for
// products so large that the copy is less than 3% of them.
bool readable(const matrix& m, const shape& s, uint32_t size) { return in_words(m, size) && (m.whole || s.tile != 256); }

// out[rows][cols] = sum over k of Q's row and P's row: P and Q as they lie in
// memory, p_k / q_k: rows of the matrix are the operand's rows (contiguous along k).
int product(call& c, matrix P, bool p_k, matrix Q, bool q_k, uint64_t k, const tam_epilogue& e) {
  const shape s = choose(e.rows, e.cols, k, c.dtype);
  if (c.tiles) {
    c.tiles[0] = (uint32_t)s.tile;
    c.tiles[1] = s.parts;
  }
  const uint32_t size = kSize[c.dtype];
  int rc = copy_rows(c, {readable(P, s, size) ? nullptr : &P, readable(Q, s, size) ? nullptr : &Q});
  if (rc != TAM_OK) return rc;
  float* partial = s.parts > 1 ? (float*)c.ws.take((uint64_t)s.parts * e.rows * e.cols * 4) : nullptr;
  const uint64_t tm = tam_div_up(e.rows, s.tile), tn = tam_div_up(e.cols, s.tile);
  const uint64_t joins = tam_div_up((uint64_t)tam_div_up(e.cols, 8) * e.rows, 256);
  rc = room_of_tiles(tm * tn, s.tile, false);
  if (rc == TAM_OK && s.parts > 1) rc = room(joins, 256);
  if (rc != TAM_OK || c.dry) return rc;
  tam_gemm_args a = {};
  a.P = operand_of(P, e.cols, size);
  a.Q = operand_of(Q, e.rows, size);
  a.k_all = k;
  a.k = (!p_k || P.whole) && (!q_k || Q.whole) ? k : k - k % (16 / size);
  a.k_part = s.parts > 1 ? tam_up(tam_div_up(a.k, s.parts), 64) : a.k;
  a.tm = (uint32_t)tm;
  a.tn = (uint32_t)tn;
  a.partial = partial;
  a.e = e;
  if (c.dtype == TAM_DTYPE_BF16)
    launch_gemm<tam_bf16>(s.tile, p_k, q_k, !(P.whole && Q.whole), a, s.parts, c.stream);
  else if (c.dtype == TAM_DTYPE_F16)
    launch_gemm<tam_f16>(s.tile, p_k, q_k, !(P.whole && Q.whole), a, s.parts, c.stream);
  else
    launch_gemm<float>(s.tile, p_k, q_k, !(P.whole && Q.whole), a, s.parts, c.stream);
  TAM_OP_LAUNCHED("the product");
  if (s.parts > 1) {
    const dim3 grid((uint32_t)joins), block(256);
    if (c.dtype == TAM_DTYPE_BF16)
      hipLaunchKernelGGL(tam_k_split<tam_bf16>, grid, block, 0, c.stream, partial, s.parts, e);
    else if (c.dtype == TAM_DTYPE_F16)
      hipLaunchKernelGGL(tam_k_split<tam_f16>, grid, block, 0, c.stream, partial, s.parts, e);
    else
      hipLaunchKernelGGL(tam_k_split<float>, grid, block, 0, c.stream, partial, s.parts, e);
    TAM_OP_LAUNCHED("the parts' sum");
  }
  return TAM_OK;
}

matrix x_of(const TamLinear* d) { return matrix_of(d->x, d->ldx, d->rows, d->inputs, kSize[d->dtype]); }
matrix w_of(const TamLinear* d) {
  return matrix_of(d->w, d->ldw, d->w_in_out ? d->inputs : d->outputs, d->w_in_out ? d->outputs : d->inputs,
                   kSize[d->dtype]);
}

int forward(const TamLinear* d, call& c) {
  if (d->rows == 0 || d->outputs == 0) return TAM_OK;
  tam_epilogue e = {d->y, d->bias, d->residual, d->z, (uint32_t)d->rows, (uint32_t)d->outputs, d->activation};
  if (d->rows <= 32 && !d->w_in_out) {
    if (c.dry) return TAM_OK;
    const tam_few_args a = {d->x, d->w, d->ldx, d->ldw, d->inputs, e};
    const dim3 grid((uint32_t)tam_div_up(d->outputs, 16)), block(64 * TAM_FEW_WAVES);
#define TAM_FEW(T)                                                                   \
  if (d->rows <= 16)                                                                 \
    hipLaunchKernelGGL((tam_k_few<T, 1>), grid, block, 0, c.stream, a);              \
  else                                                                               \
    hipLaunchKernelGGL((tam_k_few<T, 2>), grid, block, 0, c.stream, a)
    if (c.dtype == TAM_DTYPE_F32) {
      TAM_FEW(float);
    } else if (c.dtype == TAM_DTYPE_BF16) {
      TAM_FEW(tam_bf16);
    } else {
      TAM_FEW(tam_f16);
    }
    TAM_OP_LAUNCHED("the product of few rows");
    return TAM_OK;
  }
  return product(c, w_of(d), !d->w_in_out, x_of(d), true, d->inputs, e);
}

// Rows of one run of tam_k_slope: about four workgroups to a compute unit, at
// least 8 rows (2 to a wave; 1531 x 777 fp32, gelu: 13.2 us with 16, 9.6 with 8, and
// the sums' 4 us grow below that).
uint32_t slope_run(uint64_t rows, uint64_t cols) {
  const uint64_t across = tam_div_up(cols, 512), runs = tam_div_up(4ull * tam_op_cus(), across);
  const uint64_t run = tam_div_up(rows, runs);
  return (uint32_t)tam_up(run < 8 ? 8 : run, 4);
}

int backward(const TamLinear* d, call& c) {
  if (d->outputs == 0 && d->inputs == 0) return TAM_OK;
  const uint32_t size = kSize[c.dtype];
  matrix dz = matrix_of(d->dy, d->outputs, d->rows, d->outputs, size);
  const bool products = (d->dx || d->dw) && d->inputs;
  const bool keep = products && (d->activation != TAM_ACT_NONE || !in_words(dz, size) || (size == 2 && !dz.whole));
  if (d->rows && d->outputs && (keep || d->db)) {
    tam_slope_args a = {d->dy, d->z, nullptr, nullptr, 0, (uint32_t)d->rows, (uint32_t)d->outputs, 0, d->activation};
    if (keep) {
      dz.ld = a.ld_dz = aligned_ld((uint32_t)d->outputs, size);
      dz.p = a.dz = c.ws.take(d->rows * dz.ld * size);
      dz.whole = true;
    }
    a.run = slope_run(d->rows, d->outputs);
    const uint32_t runs = (uint32_t)tam_div_up(d->rows, a.run);
    if (d->db) a.sums = (float*)c.ws.take((uint64_t)runs * d->outputs * 4);
    if (!c.dry) {
      const dim3 grid((uint32_t)tam_div_up(d->outputs, 512), runs), block(256), sums((uint32_t)tam_div_up(d->outputs, 64));
#define TAM_SLOPE(T)                                                                                               \
  do {                                                                                                             \
    hipLaunchKernelGGL(tam_k_slope<T>, grid, block, 0, c.stream, a);                                               \
    TAM_OP_LAUNCHED("the activation's gradient");                                                                  \
    if (d->db) {                                                                                                   \
      hipLaunchKernelGGL(tam_k_column_sum<T>, sums, dim3(1024), 0, c.stream, a.sums, runs, (uint32_t)d->outputs, (T*)d->db); \
      TAM_OP_LAUNCHED("the bias's gradient");                                                                      \
    }                                                                                                              \
  } while (0)
      if (c.dtype == TAM_DTYPE_F32)
        TAM_SLOPE(float);
      else if (c.dtype == TAM_DTYPE_BF16)
        TAM_SLOPE(tam_bf16);
      else
        TAM_SLOPE(tam_f16);
    }
  } else {  // no rows
    const int rc = zeros(c, d->db, d->outputs);
    if (rc != TAM_OK) return rc;
  }
  if (!products) return TAM_OK;
  if (d->dx && d->rows) {
    const tam_epilogue e = {d->dx, nullptr, nullptr, nullptr, (uint32_t)d->rows, (uint32_t)d->inputs, TAM_ACT_NONE};
    const int rc = product(c, w_of(d), d->w_in_out != 0, dz, true, d->outputs, e);
    if (rc != TAM_OK) return rc;
  }
  if (d->dw && d->outputs) {
    if (c.tiles) c.tiles += 2;
    const matrix x = x_of(d);
    // dw lies as w does: [outputs][inputs], or [inputs][outputs]
    tam_epilogue e = {d->dw, nullptr, nullptr, nullptr, (uint32_t)d->outputs, (uint32_t)d->inputs, TAM_ACT_NONE};
    if (!d->w_in_out) return product(c, x, false, dz, false, d->rows, e);
    e.rows = (uint32_t)d->inputs;
    e.cols = (uint32_t)d->outputs;
    return product(c, dz, false, x, false, d->rows, e);
  }
  return TAM_OK;
}

int linear(const TamLinear* d, bool back, void* workspace, uint64_t ws_bytes, void* stream, uint64_t* need,
           uint32_t* tiles = nullptr) {
  int rc = check_linear(d, back);
  if (rc != TAM_OK) return rc;
  call c = {d->dtype, (hipStream_t)stream, {nullptr, 0}, true, tiles};
  rc = back ? backward(d, c) : forward(d, c);
  if (rc != TAM_OK) return rc;
  if (need) {
    *need = c.ws.used;
    return TAM_OK;
  }
  if (c.ws.used > ws_bytes || (c.ws.used && !workspace))
    return tam_op_fail(TAM_E_WORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)ws_bytes,
                       (unsigned long long)c.ws.used);
  if ((uintptr_t)workspace & 255u) return tam_op_fail(TAM_E_INVALID, "workspace not on 256 bytes");
  c = {d->dtype, (hipStream_t)stream, {(char*)workspace, 0}, false, nullptr};
  return back ? backward(d, c) : forward(d, c);
}

}  // namespace

extern "C" {

int tam_linear_workspace(const TamLinear* d, int backward_pass, size_t* bytes) {
  if (!bytes) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  uint64_t need = 0;
  const int rc = linear(d, backward_pass != 0, nullptr, 0, nullptr, &need);
  *bytes = (size_t)need;
  return rc;
}

int tam_linear_tiles(const TamLinear* d, int backward_pass, uint32_t* tiles) {
  if (!tiles) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  for (int i = 0; i < 4; ++i) tiles[i] = 0;
  uint64_t need = 0;
  return linear(d, backward_pass != 0, nullptr, 0, nullptr, &need, tiles);
}

int tam_linear(const TamLinear* d, void* workspace, size_t ws_bytes, void* stream) {
  return linear(d, false, workspace, ws_bytes, stream, nullptr);
}

int tam_linear_backward(const TamLinear* d, void* workspace, size_t ws_bytes, void* stream) {
  return linear(d, true, workspace, ws_bytes, stream, nullptr);
}

}  // extern "C"
