// tam_norm.hip -- layer norm of the C ABI and its gradients.
//
//   mean, var over a row's n elements; rstd = 1 / sqrt(var + eps)
//   h = (x - mean) rstd,  y = h w + b
//   t = dy w,  dx = rstd (t - mean(t) - h mean(t h)),
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// A row lies in the registers of WPR waves, CH chunks of 8 elements to a lane
// (chunk c of lane l of wave w of the row: elements 8 * ((c * WPR + w) * 64 + l)
// ..), so x is read once, the variance is the mean of the squared distances from
// the mean, and dy and x are read once in the backward pass. Workgroups stride
// over the rows with w (and b) in registers; the weight's and bias's gradients
// are summed in registers over a workgroup's rows, one fp32 row of `sums` each,
// and tam_k_norm_sums adds those. Memory bounds both passes.
#include "tam_ops.h"

namespace {

struct norm_args {
  const void* x;
  const void* w;   // or null: 1
  const void* b;   // or null: 0
  void* y;
  float* stats;    // [rows][2]: mean, rstd; or null
  const void* dy;
  void* dx;        // or null
  float* sums;     // [workgroups][2][n]; or null
  uint64_t ldx;    // elements
  uint32_t rows, n;
  float eps;
};

// Elements at .. at + 7 of a row of n; zeros past its end.
template <typename T>
__device__ __forceinline__ tam_oct<T> row_raw(const T* row, uint32_t at, uint32_t n) {
  return tam_some(row + at, at < n ? n - at : 0);
}
template <typename T>
__device__ __forceinline__ void row_load(const T* row, uint32_t at, uint32_t n, float (&v)[8]) {
  tam_load_some(row + at, at < n ? n - at : 0, v);
}
template <typename T>
__device__ __forceinline__ void row_store(T* row, uint32_t at, uint32_t n, const float (&v)[8]) {
  tam_store_some(row + at, at < n ? n - at : 0, v);
}

// A workgroup's shape: at least 4 waves, WPR of them to a row.
template <int WPR, int CH>
struct norm_shape {
  static constexpr int WAVES = WPR > 4 ? WPR : 4;
  static constexpr int ROWS = WAVES / WPR;  // at a time
  static constexpr int THREADS = 64 * WAVES;
};

// Sums of N values over the waves of a row; `turn` alternates between two
// halves of the LDS, so one barrier is enough.
template <int WPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* lds, uint32_t& turn, int wave) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = tam_wave_sum(s[i]);
  if constexpr (WPR > 1) {
    constexpr int WAVES = WPR > 4 ? WPR : 4;
    float* at = lds + turn * WAVES * 2;
    turn ^= 1u;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) at[wave * 2 + i] = s[i];
    __syncthreads();
    const int first = wave / WPR * WPR;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) sum += at[(first + w) * 2 + i];
      s[i] = sum;
    }
  }
}

// Reads x and writes y, nothing else. 16384 x 4096 bf16: 50 us, 5.4 TB/s (a large copy:
// 5.1); 8192 x 768 fp32: 11 us, 4.5 TB/s; one row of 4096: 3.0 us, the way to memory
// and back and two sums over the waves.
template <typename T, int WPR, int CH>
__global__ __launch_bounds__((norm_shape<WPR, CH>::THREADS)) void tam_k_norm(norm_args a) {
  typedef norm_shape<WPR, CH> S;
  __shared__ float lds[4 * S::WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t turn = 0;
  uint32_t at[CH];
  float w[CH][8], b[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = 8u * (uint32_t)((c * WPR + wave % WPR) * 64 + lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[c][j] = 1.f;
      b[c][j] = 0.f;
    }
    if (a.w && at[c] < a.n) row_load(static_cast<const T*>(a.w), at[c], a.n, w[c]);
    if (a.b && at[c] < a.n) row_load(static_cast<const T*>(a.b), at[c], a.n, b[c]);
  }
  const float inv = 1.f / (float)a.n;
  // every wave of a workgroup takes the same number of turns (they share barriers)
  for (uint64_t first = (uint64_t)blockIdx.x * S::ROWS; first < a.rows; first += (uint64_t)gridDim.x * S::ROWS) {
    const uint64_t row = first + wave / WPR;
    const uint32_t n = row < a.rows ? a.n : 0;
    const T* x = static_cast<const T*>(a.x) + (row < a.rows ? row : 0) * a.ldx;
    float v[CH][8];
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      row_load(x, at[c], n, v[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += v[c][j];
    }
    row_sum<WPR>(s, lds, turn, wave);
    const float mean = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[c][j] -= mean;
        s[0] += at[c] + j < n ? v[c][j] * v[c][j] : 0.f;
      }
    row_sum<WPR>(s, lds, turn, wave);
    const float rstd = 1.f / sqrtf(s[0] * inv + a.eps);
    if (row >= a.rows) continue;
    if (a.stats && lane == 0 && wave % WPR == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (at[c] >= a.n) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = __builtin_fmaf(v[c][j] * rstd, w[c][j], b[c][j]);
      row_store(y, at[c], a.n, v[c]);
    }
  }
}

// Reads x and dy and writes dx. Two workgroups to a compute unit: their rows of `sums`
// are few (the weight's and bias's gradients stay in registers over all of a
// workgroup's rows), and the row fetched ahead hides what more of them would.
// 16384 x 4096 bf16: 80 us, 5.0 TB/s; 8192 x 768 fp32: 17 us, 4.4 TB/s.
template <typename T, int WPR, int CH>
__global__ __launch_bounds__((norm_shape<WPR, CH>::THREADS)) void tam_k_norm_backward(norm_args a) {
  typedef norm_shape<WPR, CH> S;
  __shared__ float lds[4 * S::WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t turn = 0;
  uint32_t at[CH];
  float w[CH][8], dw[CH][8], db[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = 8u * (uint32_t)((c * WPR + wave % WPR) * 64 + lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[c][j] = 1.f;
      dw[c][j] = db[c][j] = 0.f;
    }
    if (a.w && at[c] < a.n) row_load(static_cast<const T*>(a.w), at[c], a.n, w[c]);
  }
  const float inv = 1.f / (float)a.n;
  // the next row's elements are on their way while a row's sums go through the waves
  const uint64_t stride = (uint64_t)gridDim.x * S::ROWS;
  tam_oct<T> rx[CH], rdy[CH];
  float mean, rstd;
  auto fetch = [&](uint64_t row) {
    const uint64_t safe = row < a.rows ? row : 0;
    const uint32_t n = row < a.rows ? a.n : 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      rx[c] = row_raw(static_cast<const T*>(a.x) + safe * a.ldx, at[c], n);
      rdy[c] = row_raw(static_cast<const T*>(a.dy) + safe * a.n, at[c], n);
    }
    mean = a.stats[2 * safe];
    rstd = a.stats[2 * safe + 1];
  };
  fetch((uint64_t)blockIdx.x * S::ROWS + wave / WPR);
  for (uint64_t first = (uint64_t)blockIdx.x * S::ROWS; first < a.rows; first += stride) {
    const uint64_t row = first + wave / WPR;
    const uint32_t n = row < a.rows ? a.n : 0;
    const float mu = mean, rs = rstd;
    float h[CH][8], t[CH][8];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[c][j] = (float)rx[c].v[j];
        t[c][j] = (float)rdy[c].v[j];
      }
    if (first + stride < a.rows) fetch(row + stride);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // past the row's end dy is 0 and h is not used
        h[c][j] = (h[c][j] - mu) * rs;
        db[c][j] += t[c][j];
        if (at[c] + j < n) dw[c][j] = __builtin_fmaf(t[c][j], h[c][j], dw[c][j]);
        t[c][j] *= w[c][j];
        s[0] += t[c][j];
        if (at[c] + j < n) s[1] = __builtin_fmaf(t[c][j], h[c][j], s[1]);
      }
    row_sum<WPR>(s, lds, turn, wave);
    if (row >= a.rows || !a.dx) continue;
    const float m0 = s[0] * inv, m1 = s[1] * inv;
    T* dx = static_cast<T*>(a.dx) + row * a.n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (at[c] >= a.n) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[c][j] = rs * (t[c][j] - m0 - h[c][j] * m1);
      row_store(dx, at[c], a.n, t[c]);
    }
  }
  if (!a.sums) return;
  // the workgroup's waves that hold the same columns, in wave order
  float* out = a.sums + (uint64_t)blockIdx.x * 2 * a.n;
  if constexpr (S::ROWS == 1) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (at[c] < a.n) {
        row_store(out, at[c], a.n, dw[c]);
        row_store(out + a.n, at[c], a.n, db[c]);
      }
  } else {
    static_assert(WPR == 1, "rows of one wave");
    __shared__ float part[S::WAVES][2][512];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        part[wave][0][j * 64 + lane] = dw[c][j];
        part[wave][1][j * 64 + lane] = db[c][j];
      }
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < 1024; i += 64 * S::WAVES) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < S::WAVES; ++k) v += part[k][i >> 9][i & 511];
        const uint32_t col = c * 512u + (i & 63u) * 8u + (i >> 6 & 7u);
        if (col < a.n) out[(i >> 9) * a.n + col] = v;
      }
    }
  }
}

// dw and db: the column sums of `groups` rows of [2][n]. A workgroup takes 64
// columns; its 16 waves every 16th row, 8 loads on their way each. 512 rows of 2 x
// 4096: 5.0 us, of 2 x 768: 3.9, of which a launch is about 2.
template <typename T>
__global__ __launch_bounds__(1024) void tam_k_norm_sums(const float* sums, uint32_t groups, uint32_t n, T* dw, T* db) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t c = (uint64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < 2ull * n) {
#pragma unroll 8
    for (uint32_t g = wave; g < groups; g += 16) s += sums[(uint64_t)g * 2 * n + c];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < 2ull * n) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += part[w][lane];
    if (c < n) {
      if (dw) dw[c] = tam_from_f<T>(v);
    } else if (db) {
      db[c - n] = tam_from_f<T>(v);
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Waves of a row and chunks of a lane. The fewest lanes without work first; one
// wave where a row fits 16 elements a lane (no barriers), 16 elements a lane
// beyond as far as the waves go, but 8 waves of 32 elements for the backward pass of
// rows past 8192: 16 waves leave a lane 128 registers, and its six rows of 16 elements
// spill (4096 x 16384 bf16: 523 us, 135 with 8 waves; forward 49 with 16 waves, 62
// with 8). 8 waves spill less, not nothing: 30 registers of 256 in 16 bits and 105 in
// fp32, 3.0 and 3.2 TB/s there. Past 16384 the rows fit neither: the backward pass
// spills 514 to 705 registers and the forward pass 114 to 168 (4096 x 32768 bf16: 2160 us,
// 0.4 TB/s, and 248, 2.2).
struct pick {
  int wpr, ch;
};
constexpr uint32_t kMost = 32768;

pick pick_shape(uint32_t n, bool backward) {
  if (n <= 512) return {1, 1};
  if (n <= 1024) return {1, 2};
  if (n <= 2048) return {4, 1};
  if (n <= 4096) return {4, 2};
  if (n <= 8192) return {4, 4};
  if (n <= 16384) return backward ? pick{8, 4} : pick{16, 2};
  return {16, 4};
}

uint32_t norm_grid(const TamNorm* d, bool backward) {
  const pick p = pick_shape((uint32_t)d->n, backward);
  const uint64_t rows = p.wpr >= 4 ? 1 : 4, need = tam_div_up(d->rows, rows);
  const uint64_t most = (uint64_t)tam_op_cus() * (p.wpr == 16 ? 2 : (backward ? 2 : 8));
  return (uint32_t)(need < most ? need : most);
}

template <typename T>
void launch_norm(const norm_args& a, pick p, uint32_t grid, bool backward, hipStream_t s) {
#define TAM_NORM(KERNEL, W, C)  \
  if (p.wpr == W && p.ch == C)  \
  hipLaunchKernelGGL((KERNEL<T, W, C>), dim3(grid), dim3(norm_shape<W, C>::THREADS), 0, s, a)
  if (backward) {
    TAM_NORM(tam_k_norm_backward, 1, 1);
    TAM_NORM(tam_k_norm_backward, 1, 2);
    TAM_NORM(tam_k_norm_backward, 4, 1);
    TAM_NORM(tam_k_norm_backward, 4, 2);
    TAM_NORM(tam_k_norm_backward, 4, 4);
    TAM_NORM(tam_k_norm_backward, 8, 4);
    TAM_NORM(tam_k_norm_backward, 16, 4);
  } else {
    TAM_NORM(tam_k_norm, 1, 1);
    TAM_NORM(tam_k_norm, 1, 2);
    TAM_NORM(tam_k_norm, 4, 1);
    TAM_NORM(tam_k_norm, 4, 2);
    TAM_NORM(tam_k_norm, 4, 4);
    TAM_NORM(tam_k_norm, 16, 2);
    TAM_NORM(tam_k_norm, 16, 4);
  }
#undef TAM_NORM
}

template <typename T>
void launch_sums(const float* sums, uint32_t groups, uint32_t n, void* dw, void* db, hipStream_t s) {
  hipLaunchKernelGGL(tam_k_norm_sums<T>, dim3((uint32_t)tam_div_up(2ull * n, 64)), dim3(1024), 0, s, sums, groups, n,
                     (T*)dw, (T*)db);
}

int check_norm(const TamNorm* d, bool backward) {
  tam_op_begin();
  if (!d) return tam_op_fail(TAM_E_INVALID, "null argument");
  if (d->dtype > TAM_DTYPE_F16) return tam_op_fail(TAM_E_INVALID, "unknown dtype %u", d->dtype);
  if (d->n == 0) return tam_op_fail(TAM_E_INVALID, "rows of no elements");
  if (d->n > kMost) return tam_op_fail(TAM_E_UNSUPPORTED, "rows of more than %u elements", kMost);
  if (d->rows >= 1ull << 31) return tam_op_fail(TAM_E_UNSUPPORTED, "2^31 rows or more");
  if (!(d->eps >= 0.f)) return tam_op_fail(TAM_E_INVALID, "eps must be 0 or more");
  if (d->ldx < d->n) return tam_op_fail(TAM_E_INVALID, "a row stride shorter than its row");
  if (d->rows && (!d->x || (!backward && !d->y) || (backward && (!d->dy || !d->stats))))
    return tam_op_fail(TAM_E_INVALID, "null argument");
  return TAM_OK;
}

uint64_t norm_need(const TamNorm* d, bool backward) {
  if (!backward || !(d->dw || d->db)) return 0;
  return tam_up((uint64_t)norm_grid(d, true) * 2 * d->n * 4, 256);
}

int norm(const TamNorm* d, bool backward, void* workspace, size_t ws_bytes, hipStream_t s) {
  const int rc = check_norm(d, backward);
  if (rc != TAM_OK) return rc;
  const uint64_t need = norm_need(d, backward);
  if (need > ws_bytes || (need && !workspace))
    return tam_op_fail(TAM_E_WORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)ws_bytes,
                       (unsigned long long)need);
  const uint32_t grid = norm_grid(d, backward);
  const bool sums = backward && (d->dw || d->db);
  const norm_args a = {d->x,  d->w, d->b, d->y, d->stats, d->dy, d->dx, sums ? (float*)workspace : nullptr, d->ldx,
                       (uint32_t)d->rows, (uint32_t)d->n, d->eps};
  const pick p = pick_shape((uint32_t)d->n, backward);
  if (grid) {
    if (d->dtype == TAM_DTYPE_F32)
      launch_norm<float>(a, p, grid, backward, s);
    else if (d->dtype == TAM_DTYPE_BF16)
      launch_norm<tam_bf16>(a, p, grid, backward, s);
    else
      launch_norm<tam_f16>(a, p, grid, backward, s);
    TAM_OP_LAUNCHED("layer norm");
  }
  if (sums) {  // of no rows: zeros
    if (d->dtype == TAM_DTYPE_F32)
      launch_sums<float>(a.sums, grid, a.n, d->dw, d->db, s);
    else if (d->dtype == TAM_DTYPE_BF16)
      launch_sums<tam_bf16>(a.sums, grid, a.n, d->dw, d->db, s);
    else
      launch_sums<tam_f16>(a.sums, grid, a.n, d->dw, d->db, s);
    TAM_OP_LAUNCHED("layer norm's column sums");
  }
  return TAM_OK;
}

}  // namespace

extern "C" {

int tam_norm_workspace(const TamNorm* d, int backward_pass, size_t* bytes) {
  const int rc = check_norm(d, backward_pass != 0);
  if (rc != TAM_OK) return rc;
  if (!bytes) return tam_op_fail(TAM_E_INVALID, "null argument");
  *bytes = (size_t)norm_need(d, backward_pass != 0);
  return TAM_OK;
}

int tam_norm(const TamNorm* d, void* stream) { return norm(d, false, nullptr, 0, (hipStream_t)stream); }

int tam_norm_backward(const TamNorm* d, void* workspace, size_t ws_bytes, void* stream) {
  return norm(d, true, workspace, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
