// tam_gated.hip -- the first half of a gated feed-forward block of the C ABI, on the tile
// core of tam_gemm.h:
//
//   g = x gate^T,  u = x up^T,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g)
//   dx = dg gate + du up,  dgate = dg^T x,  dup = du^T x
//
// Kernels:
//   tam_k_gated      one tile of both products: half of its columns are of g and half of
//                    u, the same ones, so that one lane ends up with both and the
//                    product is formed in registers (x is staged once for both);
//   tam_k_gated_few  the forward products of up to 32 rows: every wave reads its part of
//                    16 rows of either weight once, straight to the matrix cores;
//   tam_k_gated_join the same epilogue over the partial sums of products whose k was cut
//                    among workgroups (few tiles);
//   tam_k_gated_slope dg and du, side by side in one row: then dgate and dup are one
//                    product of twice the rows, and dx is one sum of twice the length
//                    (TAM_TWO_PRODUCTS);
//   tam_k_gated_products, tam_k_gated_sum  those two products, in one launch.
#include "tam_act.h"
#include "tam_few.h"
#include "tam_products.h"

namespace {

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
struct gated_epilogue {
  void* h;     // [rows][cols], contiguous
  char* kept;  // [rows][(cols + 7) / 8] records of g and u, or null
  uint32_t rows, cols, act;
};

// What the forward pass keeps of g and u: for 8 columns a record of 64 bytes in fp32, of 48 in
// 16 bits: fp32's upper 24 bits of 8 of g and 8 of u, as bf16 and, one byte each, the next 8 bits. (Rounded
// to bf16 alone, they bring dgate's, dup's and dx's errors in bf16 from 2.4e-3 of their norm to
// 3.0e-3, 1.7e-3 of it their own rounding; the bytes cost 2% of a large training pass. fp16 would have 3 digits
// more, 2^-17 being a 32nd of its rounding, but not the range: act(g) u may be one of its numbers where g or u is not.)
template <typename T>
constexpr uint32_t gated_record = sizeof(T) == 4 ? 64 : 48;

// The low byte of x past its rounding h: of the distance of their bits, in 2^-8 of bf16's last place.
__device__ __forceinline__ uint32_t gated_low(float x, tam_bf16 h) {
  const int32_t d = (int32_t)(__builtin_bit_cast(uint32_t, x) - __builtin_bit_cast(uint32_t, (float)h)) + 128;
  return (uint32_t)(d < 32767 ? d : 32767) >> 8 & 0xffu;
}
__device__ __forceinline__ float gated_value(tam_bf16 h, uint32_t low) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, (float)h) + (uint32_t)((int32_t)(low << 24) >> 16));
}

template <typename T>
__device__ __forceinline__ void gated_keep(char* at, const float (&g)[8], const float (&u)[8]) {
  if constexpr (sizeof(T) == 4) {
    tam_store8(reinterpret_cast<T*>(at), g);
    tam_store8(reinterpret_cast<T*>(at) + 8, u);
  } else {
    tam_oct<tam_bf16> hg, hu;
    uint32_t low[4] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      hg.v[j] = (tam_bf16)g[j];
      hu.v[j] = (tam_bf16)u[j];
      low[j / 4] |= gated_low(g[j], hg.v[j]) << (j % 4 * 8);
      low[2 + j / 4] |= gated_low(u[j], hu.v[j]) << (j % 4 * 8);
    }
    *reinterpret_cast<tam_oct<tam_bf16>*>(at) = hg;
    *reinterpret_cast<tam_oct<tam_bf16>*>(at + 16) = hu;
    *reinterpret_cast<uint4*>(at + 32) = uint4{low[0], low[1], low[2], low[3]};
  }
}
template <typename T>
__device__ __forceinline__ void gated_recall(const char* at, float (&g)[8], float (&u)[8]) {
  if constexpr (sizeof(T) == 4) {
    tam_load8(reinterpret_cast<const T*>(at), g);
    tam_load8(reinterpret_cast<const T*>(at) + 8, u);
  } else {
    const tam_oct<tam_bf16> hg = *reinterpret_cast<const tam_oct<tam_bf16>*>(at);
    const tam_oct<tam_bf16> hu = *reinterpret_cast<const tam_oct<tam_bf16>*>(at + 16);
    const uint4 l = *reinterpret_cast<const uint4*>(at + 32);
    const uint32_t low[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      g[j] = gated_value(hg.v[j], low[j / 4] >> (j % 4 * 8));
      u[j] = gated_value(hu.v[j], low[2 + j / 4] >> (j % 4 * 8));
    }
  }
}

// a, b: columns col .. col + 7 of a row of g and u. h is formed of both as they are in fp32.
template <typename T>
__device__ __forceinline__ void gated_finish(const gated_epilogue& e, uint32_t row, uint32_t col, const float (&a)[8],
                                             const float (&b)[8]) {
  if (e.kept) gated_keep<T>(e.kept + ((uint64_t)row * ((e.cols + 7) / 8) + col / 8) * gated_record<T>, a, b);
  float v[8];
  tam_act8<sizeof(T) == 2>(a, e.act, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= b[j];
  tam_store_some(static_cast<T*>(e.h) + (uint64_t)row * e.cols + col, e.cols - col, v);
}

struct gated_args {
  tam_operand_pair P;  // gate, up
  tam_operand Q;       // x
  uint64_t k, k_part;
  uint32_t tm, tn;     // tiles: BM rows, BN / 2 columns of h
  float* partial;      // [part][2][rows][cols] fp32, or null: one part
  gated_epilogue e;
};

// Bound by the matrix cores, small ones by rounds that do not fill the card. 256 tiles: a workgroup to a
// compute unit, which begins its next tile before it stores the last. 8192 x 4096 -> 14336 bf16
// with what is kept: 1572 us, 1224 TFLOP/s (0.94 GB written beside it, of it 0.7 kept); 2048 x 768 -> 2048
// fp16: 25; fp32 1531 x 777 -> 1001, 64 tiles: 47.
template <typename T, int BM, int BN, int WM, int WN, bool PK>
__global__ __launch_bounds__(64 * WM * WN, BM == 64 ? 3 : 2) void tam_k_gated(gated_args a) {
  typedef tam_tile<T, BM, BN, WM, WN, tam_stages<T, BM>(), PK, true, false, true> Tile;
  __shared__ __attribute__((aligned(16))) char smem[Tile::LDS];
  const uint32_t tiles = a.tm * a.tn;
  uint32_t m, n;
  tam_tile_at(tam_xcd_order(blockIdx.x, tiles), a.tm, a.tn, m, n);
  const uint64_t k0 = blockIdx.y * a.k_part;
  const uint64_t k1 = k0 + a.k_part < a.k ? k0 + a.k_part : a.k;
  auto put = [&](uint32_t row, uint32_t col, const float(&g)[8], const float(&u)[8]) {
    if (row >= a.e.rows || col >= a.e.cols) return;
    if (a.partial) {
      const uint64_t plane = (uint64_t)a.e.rows * a.e.cols;
      float* p = a.partial + 2 * blockIdx.y * plane + (uint64_t)row * a.e.cols + col;
      tam_store_some(p, a.e.cols - col, g);
      tam_store_some(p + plane, a.e.cols - col, u);
    } else {
      gated_finish<T>(a.e, row, col, g, u);
    }
  };
  Tile t;
  if constexpr (Tile::RING) {
    // a workgroup to a compute unit, each of which takes every gridDim.x-th tile and begins
    // the next one before it stores the last
    typename Tile::ring r;
    Tile::begin(r, a.P, a.Q, n * (BN / 2), m * BM, k0, k1, smem);
    constexpr uint32_t HALF_COLS = Tile::COLS / 2, LPR = HALF_COLS / 8, RPP = 64 / LPR;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    for (uint32_t tile = blockIdx.x;;) {
      t.zero();
      t.sum(r, smem);
      const uint32_t row0 = m * BM + wm * Tile::TM * 16 + lane / LPR, col = n * (BN / 2) + wn * HALF_COLS + lane % LPR * 8;
      tile += gridDim.x;
      if (tile < tiles) {
        tam_tile_at(tam_xcd_order(tile, tiles), a.tm, a.tn, m, n);
        Tile::begin(r, a.P, a.Q, n * (BN / 2), m * BM, k0, k1, smem);
      }
#pragma unroll
      for (int f = 0; f < Tile::TM; ++f) {
        t.turn_in(smem, f);
#pragma unroll
        for (uint32_t p = 0; p < 16; p += RPP) {
          float g[8], u[8];
          t.turn_out(smem, p + lane / LPR, lane % LPR * 8, g);
          t.turn_out(smem, p + lane / LPR, HALF_COLS + lane % LPR * 8, u);
          put(row0 + f * 16 + p, col, g, u);
        }
        Tile::turned();
      }
      if (tile >= tiles) return;
    }
  } else {
    t.zero();
    t.run(a.P, a.Q, n * (BN / 2), m * BM, k0, k1, smem, tam_soon{});
    t.pairs(smem, [&](uint32_t row, uint32_t col, const float(&g)[8], const float(&u)[8]) {
      put(row + m * BM, col + n * (BN / 2), g, u);
    });
  }
}

// The parts' sums in their order, then the epilogue: a thread takes 8 columns.
template <typename T>
__global__ __launch_bounds__(256) void tam_k_gated_join(const float* partial, uint32_t parts, gated_epilogue e) {
  const uint32_t per = (e.cols + 7) / 8;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (uint64_t)per * e.rows) return;
  const uint32_t row = (uint32_t)(i / per), col = (uint32_t)(i - (uint64_t)row * per) * 8;
  const uint64_t at = (uint64_t)row * e.cols + col, plane = (uint64_t)e.rows * e.cols;
  float g[8] = {}, u[8] = {};
  for (uint32_t p = 0; p < parts; ++p) {
    float a[8], b[8];
    tam_load_some(partial + 2 * p * plane + at, e.cols - col, a);
    tam_load_some(partial + (2 * p + 1) * plane + at, e.cols - col, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      g[j] += a[j];
      u[j] += b[j];
    }
  }
  gated_finish<T>(e, row, col, g, u);
}

struct gated_few_args {
  const void* x;
  const void* gate;
  const void* up;
  uint64_t ldx, ldw, k;  // elements
  gated_epilogue e;
};

// One workgroup: 16 columns of h for up to 16 * MT rows of x, as tam_k_few; a wave's
// turn of k is half as long, as it loads two weights. Bound by memory: 1 x 4096 -> 14336 bf16
// 41 us where the weights stay in the memory-side cache, 46 to 48 where they do not (4.9 TB/s).
template <typename T, int MT>
__global__ __launch_bounds__(64 * TAM_FEW_WAVES) void tam_k_gated_few(gated_few_args a) {
  constexpr int N = 16 / (int)sizeof(T), U = 4;
  constexpr uint64_t TURN = 4 * U * N;  // k of a wave's turn
  __shared__ float sum[2][TAM_FEW_WAVES][MT * 16][20];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t i = lane & 15, q = lane >> 4, n = blockIdx.x * 16 + i;
  // rows past the last one read the first one's elements; their sums go nowhere
  const uint64_t at = n < a.e.cols ? (uint64_t)n * a.ldw : 0;
  const T *wg = static_cast<const T*>(a.gate) + at, *wu = static_cast<const T*>(a.up) + at;
  const T* x[MT];
  tam_f4 ag[MT], au[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    x[m] = static_cast<const T*>(a.x) + (m * 16 + i < a.e.rows ? (uint64_t)(m * 16 + i) * a.ldx : 0);
    ag[m] = au[m] = tam_f4{0.f, 0.f, 0.f, 0.f};
  }
  auto turn = [&](uint64_t k0, auto guard) {
    constexpr bool G = decltype(guard)::value;
    tam_frag<T> fg[U], fu[U], fx[MT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) tam_few_load<T, G>(fg[u], wg, k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int u = 0; u < U; ++u) tam_few_load<T, G>(fu[u], wu, k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) tam_few_load<T, G>(fx[m][u], x[m], k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ag[m] = tam_mfma(fg[u], fx[m][u], ag[m]);
        au[m] = tam_mfma(fu[u], fx[m][u], au[m]);
      }
  };
  uint64_t k0 = wave * TURN;
#pragma unroll 2
  for (; k0 + TURN <= a.k; k0 += TAM_FEW_WAVES * TURN) turn(k0, std::false_type());
  if (k0 < a.k) turn(k0, std::true_type());
#pragma unroll
  for (int m = 0; m < MT; ++m) {  // row m * 16 + i, columns 4 q ..
    *reinterpret_cast<tam_f4*>(&sum[0][wave][m * 16 + i][q * 4]) = ag[m];
    *reinterpret_cast<tam_f4*>(&sum[1][wave][m * 16 + i][q * 4]) = au[m];
  }
  __syncthreads();
  const uint32_t t = threadIdx.x, row = t / 2, col = (t % 2) * 8;
  if (t < MT * 32 && row < a.e.rows && blockIdx.x * 16 + col < a.e.cols) {
    float g[8] = {}, u[8] = {};
    for (int s = 0; s < TAM_FEW_WAVES; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] += sum[0][s][row][col + j];
        u[j] += sum[1][s][row][col + j];
      }
    gated_finish<T>(a.e, row, blockIdx.x * 16 + col, g, u);
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
struct gated_slope_args {
  const void* dh;
  const char* kept;
  void* out;         // [rows][2][ld]: dg, du; up to 8 columns past the last one are zeros
  uint64_t rows;
  uint32_t cols, ld, act;
};

// A thread: one record. Bound by memory: 8192 x 14336 bf16 246 us, 5.7 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void tam_k_gated_slope(gated_slope_args a) {
  const uint32_t per = (a.cols + 7) / 8;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per * a.rows) return;
  const uint64_t row = i / per;
  const uint32_t col = (uint32_t)(i - row * per) * 8, count = a.cols - col;
  const uint64_t at = row * a.cols + col;
  float d[8], g[8], u[8];
  tam_load_some(static_cast<const T*>(a.dh) + at, count, d);
  gated_recall<T>(a.kept + i * gated_record<T>, g, u);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float s = tam_act_slope<sizeof(T) == 2>(g[j], a.act), v = tam_act<sizeof(T) == 2>(g[j], a.act);
    // past the last column the record is what a tile holds there
    g[j] = (uint32_t)j < count ? d[j] * u[j] * s : 0.0f;
    u[j] = (uint32_t)j < count ? d[j] * v : 0.0f;
  }
  T* out = static_cast<T*>(a.out) + 2 * row * a.ld + col;
  tam_store8(out, g);
  tam_store8(out + a.ld, u);
}

// Where a product goes: its rows (or columns) from `half` on are those of the second array.
struct gated_out {
  void* out[2];         // [rows][cols] each, contiguous; null: not wanted
  uint32_t rows, cols;  // of the product
  uint32_t half, each;  // and of one array's rows (columns), behind which its padding lies
  bool by_cols;
};

template <typename T>
__device__ __forceinline__ void gated_put(const gated_out& e, uint32_t row, uint32_t col, const float (&v)[8]) {
  uint32_t width = e.cols, second;
  if (e.by_cols) {
    second = col >= e.half;
    col -= second ? e.half : 0;
    width = e.each;
    if (col >= width) return;
  } else {
    second = row >= e.half;
    row -= second ? e.half : 0;
    if (row >= e.each) return;
  }
  T* out = static_cast<T*>(e.out[second]);
  if (out) tam_store_some(out + (uint64_t)row * width + col, width - col, v);
}

struct gated_product_args {
  tam_operand P, Q;
  tam_parts terms;
  uint64_t k, k_part;
  uint32_t tm, tn;
  float* partial;       // [part][rows][cols] fp32, or null
  gated_out e;
};

// The weights' gradients and dx in one launch, so that neither leaves compute units empty at its end.
struct gated_products_args {
  gated_product_args w, x;
  uint32_t w_units;     // of w.tm * w.tn and its parts
  uint32_t w_first;     // the first one's workgroup: 0, or behind dx's
};

template <typename T, typename Tile, int TILE, int TERMS>
__device__ __forceinline__ void gated_product(const gated_product_args& a, uint32_t unit, char* smem) {
  const uint32_t tiles = a.tm * a.tn, part = unit / tiles;
  uint32_t m, n;
  tam_tile_at(tam_xcd_order(unit - part * tiles, tiles), a.tm, a.tn, m, n);
  const uint64_t k0 = part * a.k_part;
  const uint64_t k1 = k0 + a.k_part < a.k ? k0 + a.k_part : a.k;
  Tile t;
  t.zero();
  t.template run<TERMS>(a.P, a.Q, n * TILE, m * TILE, k0, k1, smem, tam_soon{}, a.terms);
  t.template each<TAM_AHEAD_PASS>(
      smem, [](uint32_t, uint32_t) { return 0; },
      [&](uint32_t row, uint32_t col, const float(&v)[8], int) {
        row += m * TILE;
        col += n * TILE;
        if (row >= a.e.rows || col >= a.e.cols) return;
        if (a.partial)
          tam_store_some(a.partial + ((uint64_t)part * a.e.rows + row) * a.e.cols + col, a.e.cols - col, v);
        else
          gated_put<T>(a.e, row, col, v);
      },
      [](uint32_t, uint32_t, const float*, int) {});
}

// One launch for both products, the longer sums first (dx's, where 2 outputs in its parts are more than the rows
// in theirs), so that the second fills the places that the first leaves empty in its last round (2048 x 2048 -> 8192 bf16
// both ways 387 us, 427 with dx behind). Bound by the matrix cores: 8192 x 4096 -> 14336 bf16 2765 us
// for 3.85 Tflop, 1392 TFLOP/s; 2048 x 768 -> 2048 fp16 46, fp32 1531 x 777 -> 1001 101.
// IN_OUT: of weights stored [inputs][outputs], along which dx's sums run.
template <typename T, int TILE, int WM, int WN, bool IN_OUT>
__global__ __launch_bounds__(64 * WM * WN, TILE == 64 ? 3 : 2) void tam_k_gated_products(gated_products_args a) {
  typedef tam_tile<T, TILE, TILE, WM, WN, tam_stages<T, TILE>(), false, false> Weight;
  typedef tam_tile<T, TILE, TILE, WM, WN, tam_stages<T, TILE>(), IN_OUT, true> Input;
  static_assert(Weight::LDS == Input::LDS, "one size");
  __shared__ __attribute__((aligned(16))) char smem[Weight::LDS];
  if (blockIdx.x - a.w_first < a.w_units)
    gated_product<T, Weight, TILE, TAM_ONE_TERM>(a.w, blockIdx.x - a.w_first, smem);
  else
    gated_product<T, Input, TILE, TAM_TWO_PRODUCTS>(a.x, blockIdx.x < a.w_first ? blockIdx.x : blockIdx.x - a.w_units, smem);
}

// The parts' sums in their order: 8 columns to a thread.
template <typename T>
__global__ __launch_bounds__(256) void tam_k_gated_sum(const float* partial, uint32_t parts, gated_out e) {
  const uint32_t per = (e.cols + 7) / 8;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (uint64_t)per * e.rows) return;
  const uint32_t row = (uint32_t)(i / per), col = (uint32_t)(i - (uint64_t)row * per) * 8;
  const uint64_t at = (uint64_t)row * e.cols + col, step = (uint64_t)e.rows * e.cols;
  float v[8] = {};
  for (uint32_t p = 0; p < parts; ++p) {
    float t[8];
    tam_load_some(partial + p * step + at, e.cols - col, t);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += t[j];
  }
  gated_put<T>(e, row, col, v);
}


// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int check_gated(const TamGated* d, bool back) {
  tam_op_begin();
  if (!d) return tam_op_fail(TAM_E_INVALID, "null argument");
  if (d->dtype > TAM_DTYPE_F16) return tam_op_fail(TAM_E_INVALID, "unknown dtype %u", d->dtype);
  if (d->activation > TAM_ACT_MAX) return tam_op_fail(TAM_E_INVALID, "unknown activation %u", d->activation);
  const uint64_t most = 1ull << 31;
  if (d->rows >= most || d->inputs >= most || d->outputs >= most)
    return tam_op_fail(TAM_E_UNSUPPORTED, "a size of 2^31 or more");
  if (d->inputs && (d->ldx < d->inputs || d->ldw < (d->w_in_out ? d->outputs : d->inputs)))
    return tam_op_fail(TAM_E_INVALID, "a row stride shorter than its row");
  // a tile's offsets of up to 256 rows are 31-bit numbers of bytes, of dg and du side by side too
  if ((d->ldx | d->ldw | d->inputs) >= 1ull << 21 || d->outputs >= (1ull << 20) - 64)
    return tam_op_fail(TAM_E_UNSUPPORTED, "a row or row stride of 2^21 elements or more, or 2^20 - 64 outputs or more");
  if (d->rows == 0 || d->outputs == 0) return TAM_OK;
  if (d->inputs && (!d->x || !d->gate || !d->up)) return tam_op_fail(TAM_E_INVALID, "null x, gate or up");
  if (!back && !d->h) return tam_op_fail(TAM_E_INVALID, "null h");
  if (back && (!d->dh || !d->kept)) return tam_op_fail(TAM_E_INVALID, "null dh, or what the forward pass kept");
  if ((uintptr_t)d->kept & 15u) return tam_op_fail(TAM_E_INVALID, "kept memory not on 16 bytes");
  return TAM_OK;
}

matrix x_of(const TamGated* d) { return matrix_of(d->x, d->ldx, d->rows, d->inputs, kSize[d->dtype]); }
matrix w_of(const TamGated* d, const void* w) {
  return matrix_of(w, d->ldw, d->w_in_out ? d->inputs : d->outputs, d->w_in_out ? d->outputs : d->inputs, kSize[d->dtype]);
}

template <typename T>
void launch_gated(int tile, bool pk, const gated_args& a, uint32_t parts, hipStream_t s) {
  const uint32_t tiles = a.tm * a.tn, cus = tam_op_cus();
  const dim3 grid(tile == 256 && tiles > cus ? cus : tiles, parts);
#define TAM_TILE(TILE, WM, WN)                                                                                      \
  do {                                                                                                              \
    if (pk)                                                                                                         \
      hipLaunchKernelGGL((tam_k_gated<T, TILE, TILE, WM, WN, true>), grid, dim3(64 * WM * WN), 0, s, a);            \
    else                                                                                                            \
      hipLaunchKernelGGL((tam_k_gated<T, TILE, TILE, WM, WN, false>), grid, dim3(64 * WM * WN), 0, s, a);           \
  } while (0)
  if constexpr (sizeof(T) == 2)
    if (tile == 256) {
      TAM_TILE(256, 2, 4);
      return;
    }
  if (tile == 128)
    TAM_TILE(128, 2, 2);
  else
    TAM_TILE(64, 2, 2);
#undef TAM_TILE
}

template <typename T, int TILE, int WM, int WN>
void launch_products_tile(bool in_out, const gated_products_args& a, uint32_t units, hipStream_t s) {
  if (in_out)
    hipLaunchKernelGGL((tam_k_gated_products<T, TILE, WM, WN, true>), dim3(units), dim3(64 * WM * WN), 0, s, a);
  else
    hipLaunchKernelGGL((tam_k_gated_products<T, TILE, WM, WN, false>), dim3(units), dim3(64 * WM * WN), 0, s, a);
}

template <typename T>
void launch_products(int tile, bool in_out, const gated_products_args& a, uint32_t units, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (tile == 256) return launch_products_tile<T, 256, 2, 4>(in_out, a, units, s);
  tile == 128 ? launch_products_tile<T, 128, 2, 2>(in_out, a, units, s) : launch_products_tile<T, 64, 2, 2>(in_out, a, units, s);
}

// A product's rows, columns and sum; parts of its sum.
struct extent {
  uint64_t rows, cols, k;
  uint32_t parts;
  bool wanted;
};

// The tile of both products of the backward pass, and the parts of each: the least of the estimated times.
int choose_both(extent& w, extent& x, uint32_t dtype) {
  const double cus = tam_op_cus();
  const bool f32 = dtype == TAM_DTYPE_F32;
  const tam_tile_rate* rate = f32 ? tam_rates_32 : tam_rates_16;
  int best = 64;
  double least = 1e30;
  uint32_t w_parts = 1, x_parts = 1;
  auto units = [](const extent& e, uint64_t t, uint32_t parts) {
    return e.wanted ? tam_div_up(e.rows, t) * tam_div_up(e.cols, t) * parts : 0;
  };
  auto join = [](const extent& e, uint32_t parts) {  // the sums' way to memory and back (about 4 TB/s) and a launch
    return e.wanted && parts > 1 ? 3.0 + (double)e.rows * e.cols * 8.0 * parts / 4e6 : 0.0;
  };
  for (int i = 0; i < (f32 ? 2 : 3); ++i)
    for (uint32_t wp : {1, 2, 3, 4, 8, 16, 32}) {
      if (wp > 1 && (!w.wanted || w.k / wp < 128)) break;
      for (uint32_t xp : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (xp > 1 && (!x.wanted || x.k / xp < 128)) break;
        const double us = units_us(rate[i], units(w, rate[i].tile, wp), (double)w.k / wp, units(x, rate[i].tile, xp),
                                   (double)x.k / xp, cus) + join(w, wp) + join(x, xp);
        if (us < least) {
          least = us;
          best = rate[i].tile;
          w_parts = wp;
          x_parts = xp;
        }
      }
    }
  w.parts = w_parts;
  x.parts = x_parts;
  return best;
}

int forward(const TamGated* d, call& c) {
  if (d->rows == 0 || d->outputs == 0) return TAM_OK;
  const gated_epilogue e = {d->h, (char*)d->kept, (uint32_t)d->rows, (uint32_t)d->outputs, d->activation};
  if (d->rows <= 32 && !d->w_in_out) {
    if (c.dry) return TAM_OK;
    const gated_few_args a = {d->x, d->gate, d->up, d->ldx, d->ldw, d->inputs, e};
    const dim3 grid((uint32_t)tam_div_up(d->outputs, 16)), block(64 * TAM_FEW_WAVES);
#define TAM_FEW(T)                                                              \
  if (d->rows <= 16)                                                            \
    hipLaunchKernelGGL((tam_k_gated_few<T, 1>), grid, block, 0, c.stream, a);   \
  else                                                                          \
    hipLaunchKernelGGL((tam_k_gated_few<T, 2>), grid, block, 0, c.stream, a)
    TAM_OF_TYPE(c, TAM_FEW);
    TAM_OP_LAUNCHED("the products of few rows");
    return TAM_OK;
  }
  const uint32_t size = kSize[c.dtype];
  const shape s = choose(d->rows, 2 * d->outputs, d->inputs, c.dtype);
  if (c.tiles) {
    c.tiles[0] = (uint32_t)s.tile;
    c.tiles[1] = s.parts;
  }
  matrix x = x_of(d), gate = w_of(d, d->gate), up = w_of(d, d->up);
  int rc = whole_rows(c, &x, &gate, &up);
  if (rc != TAM_OK) return rc;
  gated_args a = {};
  if (s.parts > 1) a.partial = (float*)c.ws.take(2ull * s.parts * e.rows * e.cols * 4);
  const uint64_t tm = tam_div_up(e.rows, s.tile), tn = tam_div_up(e.cols, s.tile / 2);
  const uint64_t joins = tam_div_up((uint64_t)tam_div_up(e.cols, 8) * e.rows, 256);
  rc = room_of_tiles(tm * tn, s.tile, true);
  if (rc == TAM_OK && s.parts > 1) rc = room(joins, 256);
  if (rc != TAM_OK || c.dry) return rc;
  a.P = {operand_of(gate, e.cols, size), operand_of(up, e.cols, size)};
  a.Q = operand_of(x, e.rows, size);
  a.k = d->inputs;
  a.k_part = s.parts > 1 ? tam_up(tam_div_up(a.k, s.parts), 64) : a.k;
  a.tm = (uint32_t)tm;
  a.tn = (uint32_t)tn;
  a.e = e;
#define TAM_GATED(T) launch_gated<T>(s.tile, !d->w_in_out, a, s.parts, c.stream)
  TAM_OF_TYPE(c, TAM_GATED);
  TAM_OP_LAUNCHED("the gated products");
  if (s.parts > 1) {
    const dim3 grid((uint32_t)joins), block(256);
#define TAM_JOIN(T) hipLaunchKernelGGL(tam_k_gated_join<T>, grid, block, 0, c.stream, a.partial, s.parts, e)
    TAM_OF_TYPE(c, TAM_JOIN);
    TAM_OP_LAUNCHED("the parts' sum");
  }
  return TAM_OK;
}

// a's tiles and parts; the partial sums' memory, if there are parts. Returns its units.
uint64_t lay_out(call& c, gated_product_args& a, const matrix& P, const matrix& Q, tam_parts terms, const extent& of, int tile,
                 const gated_out& e) {
  const uint32_t size = kSize[c.dtype];
  if (of.parts > 1) a.partial = (float*)c.ws.take((uint64_t)of.parts * e.rows * e.cols * 4);
  a.P = operand_of(P, e.cols, size);
  a.Q = operand_of(Q, e.rows, size);
  a.terms = terms;
  a.k = of.k / terms.terms;
  a.k_part = of.parts > 1 ? tam_up(tam_div_up(a.k, of.parts), 64) : a.k;
  a.tm = (uint32_t)tam_div_up(e.rows, tile);
  a.tn = (uint32_t)tam_div_up(e.cols, tile);
  a.e = e;
  return (uint64_t)a.tm * a.tn * of.parts;
}

uint64_t joins_of(const gated_out& e) { return tam_div_up((uint64_t)tam_div_up(e.cols, 8) * e.rows, 256); }

int join(call& c, const gated_product_args& a, uint32_t parts) {
  if (parts == 1) return TAM_OK;
  const dim3 grid((uint32_t)joins_of(a.e)), block(256);
#define TAM_SUM(T) hipLaunchKernelGGL(tam_k_gated_sum<T>, grid, block, 0, c.stream, a.partial, parts, a.e)
  TAM_OF_TYPE(c, TAM_SUM);
  TAM_OP_LAUNCHED("the parts' sum");
  return TAM_OK;
}

int backward(const TamGated* d, call& c) {
  const uint32_t size = kSize[c.dtype];
  if (d->rows == 0 || d->outputs == 0 || d->inputs == 0) {  // empty sums
    int rc = zeros(c, d->dx, d->rows * d->inputs);
    if (rc == TAM_OK) rc = zeros(c, d->dgate, d->outputs * d->inputs);
    return rc == TAM_OK ? zeros(c, d->dup, d->outputs * d->inputs) : rc;
  }
  if (!d->dx && !d->dgate && !d->dup) return TAM_OK;
  const uint32_t rows = (uint32_t)d->rows, inputs = (uint32_t)d->inputs, outputs = (uint32_t)d->outputs;
  const uint32_t ld = aligned_ld(outputs, size);
  const matrix both = {c.ws.take((uint64_t)rows * 2 * ld * size), 2ull * ld, rows, 2 * ld, true};
  const uint64_t slopes = tam_div_up((uint64_t)tam_div_up(outputs, 8) * rows, 256);
  int rc = room(slopes, 256);
  if (rc != TAM_OK) return rc;
  if (!c.dry) {
    const gated_slope_args a = {d->dh, (const char*)d->kept, (void*)both.p, rows, outputs, ld, d->activation};
    const dim3 grid((uint32_t)slopes), block(256);
#define TAM_SLOPE(T) hipLaunchKernelGGL(tam_k_gated_slope<T>, grid, block, 0, c.stream, a)
    TAM_OF_TYPE(c, TAM_SLOPE);
    TAM_OP_LAUNCHED("the activation's gradient");
  }
  matrix gate = w_of(d, d->gate), up = w_of(d, d->up), x = x_of(d);
  const bool want_w = d->dgate || d->dup;
  // dx's sum goes from one weight to the other in its stride: they are copied both or not at all
  if (in_words(gate, size) != in_words(up, size)) gate.whole = up.whole = false;
  rc = d->dx && want_w ? whole_rows(c, &gate, &up, &x) : (d->dx ? whole_rows(c, &gate, &up) : whole_rows(c, &x));
  if (rc != TAM_OK) return rc;
  // dgate and dup lie as the weights do, one product: of dg's and du's columns, a row's padding between them
  gated_out ew = {{d->dgate, d->dup}, 2 * ld, inputs, ld, outputs, false};
  if (d->w_in_out) ew = {{d->dgate, d->dup}, inputs, 2 * ld, ld, outputs, true};
  const gated_out ex = {{d->dx, nullptr}, rows, inputs, rows, rows, false};
  extent w = {ew.rows, ew.cols, rows, 1, want_w}, in = {rows, inputs, 2ull * outputs, 1, d->dx != nullptr};
  const int tile = choose_both(w, in, c.dtype);
  if (c.tiles) {
    if (d->dx) c.tiles[0] = (uint32_t)tile, c.tiles[1] = in.parts;
    if (want_w) c.tiles[2] = (uint32_t)tile, c.tiles[3] = w.parts;
  }
  gated_products_args a = {};
  uint64_t units = 0;
  if (want_w) {
    units = lay_out(c, a.w, d->w_in_out ? both : x, d->w_in_out ? x : both, {1, 0, 0}, w, tile, ew);
    a.w_units = (uint32_t)units;
  }
  if (d->dx) {
    const uint64_t x_units =
        lay_out(c, a.x, gate, both, {2, (int64_t)((intptr_t)up.p - (intptr_t)gate.p), (int64_t)ld * size}, in, tile, ex);
    if (units && in.k / in.parts > w.k / w.parts) a.w_first = (uint32_t)x_units;
    units += x_units;
  }
  rc = room_of_tiles(units, tile, false);
  if (rc == TAM_OK && want_w && w.parts > 1) rc = room(joins_of(ew), 256);
  if (rc == TAM_OK && d->dx && in.parts > 1) rc = room(joins_of(ex), 256);
  if (rc != TAM_OK || c.dry) return rc;
#define TAM_PRODUCTS(T) launch_products<T>(tile, d->w_in_out != 0, a, (uint32_t)units, c.stream)
  TAM_OF_TYPE(c, TAM_PRODUCTS);
  TAM_OP_LAUNCHED("the gradients' products");
  if (want_w) rc = join(c, a.w, w.parts);
  return rc == TAM_OK && d->dx ? join(c, a.x, in.parts) : rc;
}

int gated(const TamGated* d, bool back, void* workspace, uint64_t ws_bytes, void* stream, uint64_t* need,
          uint32_t* tiles = nullptr) {
  int rc = check_gated(d, back);
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

size_t tam_gated_kept(uint64_t rows, uint64_t outputs, uint32_t dtype) {
  return (size_t)(rows * tam_div_up(outputs, 8) * (dtype == TAM_DTYPE_F32 ? gated_record<float> : gated_record<tam_f16>));
}

int tam_gated_workspace(const TamGated* d, int backward_pass, size_t* bytes) {
  if (!bytes) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  uint64_t need = 0;
  const int rc = gated(d, backward_pass != 0, nullptr, 0, nullptr, &need);
  *bytes = (size_t)need;
  return rc;
}

int tam_gated_tiles(const TamGated* d, int backward_pass, uint32_t* tiles) {
  if (!tiles) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  for (int i = 0; i < 4; ++i) tiles[i] = 0;
  uint64_t need = 0;
  return gated(d, backward_pass != 0, nullptr, 0, nullptr, &need, tiles);
}

int tam_gated(const TamGated* d, void* workspace, size_t ws_bytes, void* stream) {
  return gated(d, false, workspace, ws_bytes, stream, nullptr);
}

int tam_gated_backward(const TamGated* d, void* workspace, size_t ws_bytes, void* stream) {
  return gated(d, true, workspace, ws_bytes, stream, nullptr);
}

}  // extern "C"
