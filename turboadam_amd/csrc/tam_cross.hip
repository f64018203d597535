// tam_cross.hip -- output projection with softmax cross entropy of the C ABI, on the tile
// core of tam_gemm.h:
//
//   z = x w^T,  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,target_i
//   dz = (exp(z - lse) - onehot) dloss_i,  dx = dz w,  dw = dz^T x
//
// z (rows x vocabulary) is never in memory as a whole, but for up to 64 words.
//
// Forward.  A tile of z stays in the matrix cores' registers and leaves a maximum and a sum
// of exponentials of each of its rows, 8 bytes for its 64 to 256 columns
// (tam_k_cross_logits); tam_k_cross_join makes lse and the loss of them.  Up to 32 rows read the
// weight straight to the matrix cores (tam_k_cross_few); up to 64 words are a row's end in one workgroup,
// and their z, which is small beside x, is kept for the backward pass (tam_k_cross_words).
//
// Backward.  Pieces of the vocabulary: z again, and dz of a piece, rounded to the type, goes
// to memory (tam_k_cross_logits); then the piece's rows of dw, whole sums, and its share of
// dx, added to fp32 sums that tam_k_cross_out rounds at the end.  To make z again costs a
// third of the gradients' products; to keep it would cost rows * vocabulary.
//
// Rows that do not count take no part: tam_k_cross_rows numbers the others, x is gathered
// into rows of whole lines (22 us of 24 ms for 8192 x 4096; the backward pass reads the same), and every
// later kernel reads their number from the device: its tiles of rows past it return at once, and
// sums over rows end there.  So NaN in a padded row reaches nothing.
//
// dz is held as (exp(z - lse) - onehot) * w, |w| < 2 (fp16: times 2^14, as a softmax
// over 10^5 words lies below fp16's numbers otherwise), and the results are multiplied by
// the power of two or the factor that is missing (scale) when they are rounded.
#include "tam_few.h"
#include "tam_products.h"

#include <math.h>

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// With the hardware's 2^x and the rounding of its argument off by up to 2^-23 (1 + |x|) of the result. That is below
// 2^-16 for dz, which is rounded to 16 bits, wherever it is not 0; a sum's terms of a large |x| are as small as e^-|x|.
template <typename T>
__device__ __forceinline__ float cross_exp(float x) {
  if constexpr (sizeof(T) == 2)
    return __builtin_amdgcn_exp2f(kLog2e * x);
  else
    return expf(x);
}

// What multiplies 16-bit types' logits ahead of the hardware's 2^x. Past 2^30 they are 64 or more apart, and any base
// tells the largest from the others; log2e times them may be infinite.
__device__ __forceinline__ float cross_rate(float at) { return fabsf(at) < 1073741824.0f ? kLog2e : 1.0f; }

// The sum of exp(z - top) over a lane's values, top their maximum or more, but in 16-bit types for the
// factor that cross_settled takes out. A top of -inf (words that cannot be, or columns past the last one) counts as
// 0: exp(-inf) is 0; a NaN or an infinity makes the sum NaN.
template <typename T, int N>
__device__ __forceinline__ float cross_terms(const float (&z)[N], float top) {
  const float at = top == -INFINITY ? 0.0f : top;
  float sum = 0.f;
  if constexpr (sizeof(T) == 2) {  // one multiplication and addition ahead of the hardware's 2^x
    const float rate = cross_rate(at), shift = -rate * at;
#pragma unroll
    for (int j = 0; j < N; ++j) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(z[j], rate, shift));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) sum += expf(z[j] - at);
  }
  return sum;
}

// The sum without the rounding of log2e top, which all of its terms have alike: 2^-24 |top| of it, 6e-5 at logits of
// 1000. Once for a row of a wave's or a workgroup's columns.
template <typename T>
__device__ __forceinline__ float cross_settled(float sum, float top) {
  if constexpr (sizeof(T) == 2) {
    const float at = top == -INFINITY ? 0.0f : top, rate = cross_rate(at);
    sum *= __builtin_amdgcn_exp2f(__builtin_fmaf(-rate, at, rate * at));
  }
  return sum;
}

// log(sum of exp) - z of the target: the large numbers meet first, so that a loss is as exact at logits of 1000 as of 1.
__device__ __forceinline__ float cross_loss(float top, float sum, float hit) { return (top - hit) + logf(sum); }

// What the forward pass keeps, and what every kernel reads: all by the row's own number but
// `index` and `target`, which are by its number among those that count.
struct cross_rows {
  uint32_t* count;
  uint32_t* index;   // -> row
  int32_t* place;    // of a row -> number, or -1
  int32_t* target;   // -1: outside the vocabulary
  float* lse;
};

struct cross_rows_args {
  cross_rows r;
  const int64_t* targets;
  float* loss;       // zeros for rows that do not count, or null
  int64_t ignored;
  uint32_t rows;
  int64_t vocabulary;
};

// One workgroup numbers the rows that count, 8192 a turn in their order: 8 rows to a
// thread, sums of the threads' numbers over waves and workgroup. Bound by its trips to memory: 8192
// rows 14 us, of 8 to 24 ms; several workgroups would have to wait for each other, or be two launches.
__global__ __launch_bounds__(1024) void tam_k_cross_rows(cross_rows_args a) {
  __shared__ uint32_t part[16];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t base = 0;
  for (uint64_t first = 0; first < a.rows; first += 8192) {
    const uint64_t row0 = first + threadIdx.x * 8;
    int64_t t[8];
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = row0 + i < a.rows ? a.targets[row0 + i] : a.ignored;
      n += t[i] != a.ignored;
    }
    uint32_t upto = n;  // of the wave's lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t v = __shfl_up(upto, d);
      upto += lane >= (uint32_t)d ? v : 0;
    }
    __syncthreads();
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    uint32_t at = base + upto - n;
    for (uint32_t w = 0; w < 16; ++w) {
      at += w < wave ? part[w] : 0;
      base += part[w];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row0 + i < a.rows) {
        const bool counts = t[i] != a.ignored;
        if (counts) {
          a.r.index[at] = (uint32_t)(row0 + i);
          a.r.target[at] = t[i] >= 0 && t[i] < a.vocabulary ? (int32_t)t[i] : -1;
        } else if (a.loss) {
          a.loss[row0 + i] = 0.f;
        }
        a.r.place[row0 + i] = counts ? (int32_t)at : -1;
        at += counts;
      }
  }
  if (threadIdx.x == 0) *a.r.count = base;
}

// to[j] = the j-th row of x that counts, zeros behind it: 8 16-bit units to a thread. Bound by
// memory: 7680 of 8192 rows of 4096 bf16 22 us, 5.7 TB/s.
__global__ __launch_bounds__(256) void tam_k_cross_gather(const tam_f16* x, uint64_t ldx, uint32_t cols, cross_rows r,
                                                          uint32_t rows, tam_f16* to, uint32_t ld) {
  const uint32_t per = ld / 8, count = *r.count;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t j = i / per;
  if (j >= count || j >= rows) return;
  const uint32_t c = (uint32_t)(i - j * per) * 8;
  *reinterpret_cast<tam_oct<tam_f16>*>(to + j * ld + c) =
      tam_some(x + (uint64_t)r.index[j] * ldx + c, c < cols ? cols - c : 0);
}

// ---------------------------------------------------------------------------
// z
// ---------------------------------------------------------------------------
struct cross_logits_args {
  tam_operand P, Q;    // rows of w of the piece; gathered rows of x
  uint64_t k;
  uint32_t tm, tn;
  cross_rows r;
  uint32_t first;      // column of the piece's first one
  uint32_t cols;       // of the piece
  uint64_t rows;       // of every array here
  float2* parts;       // forward: [tn][rows] maximum and sum of a tile's row
  float* hit;          // forward: [rows] z of the target
  const struct cross_row* row;  // backward: [rows]
  void* dz;            // backward: [rows][ld]
  uint64_t ld;
};

// A row that counts, by its number, as dz takes it.
struct cross_row {
  float lse, w;
  int32_t target;
  uint32_t unused;
};

// Over the four lanes whose numbers agree in their last four bits; all get the same bits.
template <typename F>
__device__ __forceinline__ float cross_rows4(float x, F f) {
  const uint32_t i = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  const uint32_t j = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(j, j, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// A lane holds 4 consecutive columns of a row in each of its fragments. Forward: the maximum
// and the sum over its 4 TN columns, then the row's 4 lanes, then the tile's waves side by side
// (`at`: [TILE][WN] in LDS), and the target's z if it is here.
template <typename T, typename Tile, int TILE, int WN, typename Sync>
__device__ __forceinline__ void cross_forward(const cross_logits_args& a, Tile& t, const int32_t (&target)[Tile::TM],
                                              uint32_t m, uint32_t n, uint32_t count, float2* at, Sync sync) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const uint32_t col0 = n * TILE + wn * Tile::TN * 16 + (lane >> 4) * 4;  // the lane's first column
  if (n * TILE + TILE > a.cols)
#pragma unroll
    for (uint32_t c = 0; c < Tile::TN; ++c)
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        if (col0 + c * 16 + j >= a.cols)
#pragma unroll
          for (int f = 0; f < Tile::TM; ++f) t.acc[c][f][j] = -INFINITY;
  bool here = false;  // a row's target is in its lane's columns: of 128 rows and 64 of 50257 columns, one wave in six
#pragma unroll
  for (int f = 0; f < Tile::TM; ++f) here |= target[f] >= 0 && (uint32_t)target[f] - col0 < Tile::TN * 16u;
  if (__any(here))
#pragma unroll
    for (int f = 0; f < Tile::TM; ++f)
#pragma unroll
      for (uint32_t c = 0; c < Tile::TN; ++c)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          if (target[f] == (int32_t)(col0 + c * 16 + j))
            a.hit[m * TILE + (wm * Tile::TM + f) * 16 + (lane & 15)] = t.acc[c][f][j];
#pragma unroll
  for (int f = 0; f < Tile::TM; ++f) {
    float z[4 * Tile::TN];
#pragma unroll
    for (int c = 0; c < Tile::TN; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) z[4 * c + j] = t.acc[c][f][j];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * Tile::TN; ++i) top = fmaxf(top, z[i]);
    top = cross_rows4(top, [](float x, float y) { return fmaxf(x, y); });
    const float sum = cross_rows4(cross_terms<T>(z, top), [](float x, float y) { return x + y; });
    if (lane < 16) at[((wm * Tile::TM + f) * 16 + lane) * WN + wn] = float2{top, sum};
  }
  sync();
  const uint32_t row = m * TILE + threadIdx.x;
  if (threadIdx.x < TILE && row < count) {
    float2 part[WN], all = {-INFINITY, 0.f};
#pragma unroll
    for (int w = 0; w < WN; ++w) {
      part[w] = at[threadIdx.x * WN + w];
      all.x = fmaxf(all.x, part[w].x);
    }
    const float top = all.x == -INFINITY ? 0.0f : all.x;  // a part of no words is 0 times exp(-inf)
#pragma unroll
    for (int w = 0; w < WN; ++w) all.y += cross_settled<T>(part[w].y, part[w].x) * cross_exp<T>(part[w].x - top);
    a.parts[(uint64_t)n * a.rows + row] = all;
  }
}

// Backward, of a tile whose next one has begun: dz where the sums lie, in the type, and turned
// in LDS by 16 rows, so that a row's 64 columns leave as one line.
template <typename T, typename Tile, int TILE, int WN>
__device__ __forceinline__ void cross_backward(const cross_logits_args& a, Tile& t, const float (&lse)[Tile::TM],
                                               const float (&w)[Tile::TM], const int32_t (&target)[Tile::TM], uint32_t m,
                                               uint32_t n, uint32_t count, char* smem) {
  typedef T four __attribute__((ext_vector_type(4)));
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const uint32_t col0 = n * TILE + wn * Tile::TN * 16 + (lane >> 4) * 4, row = lane & 15;
  T* const out = static_cast<T*>(a.dz);
  bool some = n * TILE + TILE > a.cols;  // columns past the last one, or (a wave in six) a target in a lane's columns
#pragma unroll
  for (int f = 0; f < Tile::TM; ++f) some |= target[f] >= 0 && (uint32_t)target[f] - a.first - col0 < Tile::TN * 16u;
  auto rows = [&](auto special) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < Tile::TM; ++f) {
      tam_lds_char* const turn = t.spare(smem) + f % 2 * 2048;
      const uint32_t hit = (uint32_t)target[f] - a.first - col0;
#pragma unroll
      for (uint32_t c = 0; c < Tile::TN; ++c) {
        four v;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          float p = cross_exp<T>(t.acc[c][f][j] - lse[f]);
          if constexpr (decltype(special)::value) {
            p -= hit == c * 16 + j ? 1.0f : 0.0f;
            if (col0 + c * 16 + j >= a.cols) p = 0.0f;  // the sum over columns takes whole 16 bytes
          }
          v[j] = (T)(p * w[f]);
        }
        // 8 bytes; the 16 that they are half of lie at their place ^ row
        *(__attribute__((address_space(3))) four*)(turn + row * 128 + ((c * 2 + (lane >> 5)) ^ (row & 7)) * 16 +
                                                   (lane >> 4 & 1) * 8) = v;
      }
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t r = h * 8 + lane / 8, at = m * TILE + (wm * Tile::TM + f) * 16 + r;
        const uint32_t col = n * TILE + wn * Tile::TN * 16 + lane % 8 * 8;
        const tam_s8 v = *(const tam_lds_s8*)(turn + r * 128 + ((lane % 8) ^ (r & 7)) * 16);
        if (at < count && col < a.cols) *reinterpret_cast<tam_s8*>(out + (uint64_t)at * a.ld + col) = v;
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (__any(some))
    rows(std::true_type());
  else
    rows(std::false_type());
}

// Bound by the matrix cores and, at small k, by what follows the sums: exponentials, and
// in the backward pass the stores. 16-bit tiles of 256: a workgroup to a compute unit, which begins
// its next tile before it goes through the last one's sums. bf16, 7680 rows that count x 4096 over
// 128256 words: 6123 us (1318 TFLOP/s), in four pieces of dz 6347 (1271); 8192 x 768 over 50257 words
// 598 (1057), two pieces of dz 660 (958, 1.2 TB/s written beside it). fp32 619 x 515 over 9973 words, 64
// tiles: 68 and 69 (91 to 93 TFLOP/s).
template <typename T, int TILE, int WM, int WN, bool BACK>
__global__ __launch_bounds__(64 * WM * WN, TILE == 64 ? 3 : 2) void tam_k_cross_logits(cross_logits_args a) {
  typedef tam_tile<T, TILE, TILE, WM, WN, tam_stages<T, TILE>(), true, true> Tile;
  __shared__ __attribute__((aligned(16))) char smem[Tile::LDS];
  const uint32_t count = *a.r.count, tm = (count + TILE - 1) / TILE, tiles = tm * a.tn;
  if (blockIdx.x >= tiles) return;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN;
  uint32_t m, n;
  tam_tile_at(tam_xcd_order(blockIdx.x, tiles), tm, a.tn, m, n);
  a.Q.count = count;
  Tile t;
  if constexpr (Tile::RING) {
    typename Tile::ring r;
    Tile::begin(r, a.P, a.Q, n * TILE, m * TILE, 0, a.k, smem);
    for (uint32_t tile = blockIdx.x;;) {
      t.zero();
      t.sum(r, smem);
      // ahead of the next tile's loads, behind which they would come
      int32_t target[Tile::TM];
      float lse[Tile::TM], w[Tile::TM];
#pragma unroll
      for (int f = 0; f < Tile::TM; ++f) {
        uint32_t row = m * TILE + (wm * Tile::TM + f) * 16 + (lane & 15);
        row = row < count ? row : count - 1;  // whose sums go nowhere
        if constexpr (BACK) {
          const cross_row of = a.row[row];
          lse[f] = of.lse;
          w[f] = of.w;
          target[f] = of.target;
        } else {
          target[f] = m * TILE + (wm * Tile::TM + f) * 16 + (lane & 15) < count ? a.r.target[row] : -1;
        }
      }
#pragma unroll
      for (int f = 0; f < Tile::TM; ++f) {
        if constexpr (BACK) asm volatile("" : "+v"(lse[f]), "+v"(w[f]));
        asm volatile("" : "+v"(target[f]));
      }
      const uint32_t m0 = m, n0 = n;
      tile += gridDim.x;
      if (tile < tiles) {
        tam_tile_at(tam_xcd_order(tile, tiles), tm, a.tn, m, n);
        Tile::begin(r, a.P, a.Q, n * TILE, m * TILE, 0, a.k, smem);
      }
      if constexpr (BACK)
        cross_backward<T, Tile, TILE, WN>(a, t, lse, w, target, m0, n0, count, smem);
      else
        cross_forward<T, Tile, TILE, WN>(a, t, target, m0, n0, count, reinterpret_cast<float2*>(smem + Tile::SPARE),
                                         [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); });
      if (tile >= tiles) return;
    }
  } else {
    t.zero();
    t.run(a.P, a.Q, n * TILE, m * TILE, 0, a.k, smem, tam_soon{});
    if constexpr (BACK) {
      t.template each<TAM_AHEAD_PASS>(
          smem,
          [&](uint32_t row, uint32_t) {
            row += m * TILE;
            return a.row[row < count ? row : count - 1];
          },
          [&](uint32_t row, uint32_t col, float(&v)[8], const cross_row& of) {
            row += m * TILE;
            col += n * TILE;
            if (row >= count || col >= a.cols) return;
            const uint32_t hit = (uint32_t)of.target - a.first - col;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
              const float p = cross_exp<T>(v[j] - of.lse) - (hit == j ? 1.0f : 0.0f);
              // columns past the last one are zeros: the sum over columns takes whole 16 bytes
              v[j] = col + j < a.cols ? p * of.w : 0.0f;
            }
            tam_store8(static_cast<T*>(a.dz) + (uint64_t)row * a.ld + col, v);
          },
          [](uint32_t, uint32_t, const float*, int) {});
    } else {
      int32_t target[Tile::TM];
#pragma unroll
      for (int f = 0; f < Tile::TM; ++f) {
        const uint32_t row = m * TILE + (wm * Tile::TM + f) * 16 + (lane & 15);
        target[f] = row < count ? a.r.target[row] : -1;
      }
      cross_forward<T, Tile, TILE, WN>(a, t, target, m, n, count, reinterpret_cast<float2*>(smem), [] { __syncthreads(); });
    }
  }
}

struct cross_join_args {
  cross_rows r;
  const float2* parts;  // [tiles][rows], or of few rows [rows][tiles]
  const float* hit;
  float* loss;          // by row, or where they are added by number
  uint64_t rows;
  uint32_t tiles;
  bool by_number;
  const int64_t* targets;  // few rows: read here
  int64_t ignored, vocabulary;
};

// The sum of parts p0, p0 + step, .. with the common maximum.
__device__ __forceinline__ float2 cross_add(const float2& a, const float2& b) {
  const float top = fmaxf(a.x, b.x);
  return {top, (a.y != 0.f ? a.y * expf(a.x - top) : 0.f) + (b.y != 0.f ? b.y * expf(b.x - top) : 0.f)};
}

// 64 rows to a workgroup, 16 threads to a row, whose sums meet in their order. Bound by memory and
// its few workgroups: 7680 rows of 501 parts 17 us, 8192 of 197 8.6.
__global__ __launch_bounds__(1024) void tam_k_cross_join(cross_join_args a) {
  __shared__ float2 at[16][64];
  const uint32_t lane = threadIdx.x & 63, run = threadIdx.x >> 6, count = *a.r.count;
  const uint32_t j = blockIdx.x * 64 + lane;
  if (blockIdx.x * 64 >= count) return;
  float2 s = {-INFINITY, 0.f};
  if (j < count)
#pragma unroll 8
    for (uint32_t t = run; t < a.tiles; t += 16) s = cross_add(s, a.parts[(uint64_t)t * a.rows + j]);
  at[run][lane] = s;
  __syncthreads();
  if (run == 0 && j < count) {
    for (int w = 1; w < 16; ++w) s = cross_add(s, at[w][lane]);
    const uint32_t row = a.r.index[j];
    const bool inside = a.r.target[j] >= 0;
    a.r.lse[row] = inside ? s.x + logf(s.y) : NAN;
    a.loss[a.by_number ? j : row] = inside ? cross_loss(s.x, s.y, a.hit[j]) : NAN;
  }
}

// Few rows: a workgroup to a row. Bound by its trips to memory one after another: a row of 8016 parts
// 9.5 us (with 256 threads 10.8).
__global__ __launch_bounds__(1024) void tam_k_cross_join_few(cross_join_args a) {
  __shared__ float2 at[1024];
  const uint32_t row = blockIdx.x;
  const int64_t target = a.targets[row];
  const bool inside = target >= 0 && target < a.vocabulary;
  const float hit = inside ? a.hit[row] : 0.f;
  float2 s = {-INFINITY, 0.f};
#pragma unroll 8
  for (uint32_t t = threadIdx.x; t < a.tiles; t += 1024) s = cross_add(s, a.parts[(uint64_t)row * a.tiles + t]);
  at[threadIdx.x] = s;
  for (int half = 512; half >= 1; half /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < half) at[threadIdx.x] = cross_add(at[threadIdx.x], at[threadIdx.x + half]);
  }
  if (threadIdx.x == 0) {
    s = at[0];
    if (a.r.lse) a.r.lse[row] = inside ? s.x + logf(s.y) : NAN;
    a.loss[row] = target == a.ignored ? 0.f : (inside ? cross_loss(s.x, s.y, hit) : NAN);
  }
}

// The losses' sum in 64 bits, in a fixed order, over their number where it is a mean.
__global__ __launch_bounds__(1024) void tam_k_cross_sum(const float* losses, const uint32_t* count, const int64_t* targets,
                                                        int64_t ignored, uint32_t rows, bool mean, float* loss) {
  __shared__ double at[1024];
  __shared__ uint32_t number[1024];
  // few rows: by row, and those that count are counted here
  const uint32_t n = count ? *count : rows;
  double s = 0.;
  uint32_t c = 0;
  for (uint32_t j = threadIdx.x; j < n; j += 1024) {
    s += (double)losses[j];
    c += count || targets[j] != ignored;
  }
  at[threadIdx.x] = s;
  number[threadIdx.x] = c;
  for (int half = 512; half >= 1; half /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < half) {
      at[threadIdx.x] += at[threadIdx.x + half];
      number[threadIdx.x] += number[threadIdx.x + half];
    }
  }
  if (threadIdx.x == 0) *loss = (float)(mean ? at[0] / (double)(number[0] ? number[0] : 1u) : at[0]);
}

struct cross_few_args {
  const void* x;
  const void* w;
  uint64_t ldx, ldw, k;
  const int64_t* targets;
  float2* parts;  // [rows][groups of 16 columns]
  float* hit;
  uint32_t rows, cols, groups;
  // backward: rows by their numbers
  cross_rows r;
  const cross_row* row;
  void* dz;
  uint64_t ld;
};

// One workgroup: 16 columns of z for up to 16 * MT rows of x, as tam_k_few. BACK: dz of rows that
// count, of the whole vocabulary. Bound by memory: 1 x 4096 over 128256 words bf16 176 us, 6.0 TB/s; 8 x
// 7191 over 72376 487, 2.1, as rows that begin on odd addresses take loads of their own.
template <typename T, int MT, bool BACK>
__global__ __launch_bounds__(64 * TAM_FEW_WAVES) void tam_k_cross_few(cross_few_args a) {
  constexpr int N = 16 / (int)sizeof(T), U = 4;
  constexpr uint64_t TURN = 4 * U * N;  // k of a wave's turn
  __shared__ float sum[TAM_FEW_WAVES][MT * 16][20];
  const uint32_t column = blockIdx.x, rows = BACK ? *a.r.count : a.rows;
  if (rows == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t i = lane & 15, q = lane >> 4, n = column * 16 + i;
  // rows past the last one read the first one's elements; their sums go nowhere
  const T* w = static_cast<const T*>(a.w) + (n < a.cols ? (uint64_t)n * a.ldw : 0);
  const T* x[MT];
  tam_f4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const uint32_t at = m * 16 + i < rows ? m * 16 + i : 0;
    x[m] = static_cast<const T*>(a.x) + (uint64_t)(BACK ? a.r.index[at] : at) * a.ldx;
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
  const uint32_t t = threadIdx.x, row = t / 2, col = column * 16 + (t % 2) * 8;
  if (t < MT * 32) {
    float v[8] = {};
    for (int s = 0; s < TAM_FEW_WAVES; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += sum[s][t / 2][(t % 2) * 8 + j];
    if constexpr (BACK) {
      if (row < rows && col < a.cols) {
        const cross_row of = a.row[row];
        const uint32_t hit = (uint32_t)of.target - col;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const float p = cross_exp<T>(v[j] - of.lse) - (hit == j ? 1.0f : 0.0f);
          // columns past the last one are zeros: the sum over columns takes whole 16 bytes
          v[j] = col + j < a.cols ? p * of.w : 0.0f;
        }
        tam_store8(static_cast<T*>(a.dz) + (uint64_t)row * a.ld + col, v);
      }
    } else {
      const int64_t target = row < rows ? a.targets[row] : -1;
      float top = -INFINITY, all = 0.f;
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        if (col + j >= a.cols) v[j] = -INFINITY;
        else if (target == (int64_t)(col + j)) a.hit[row] = v[j];
        top = fmaxf(top, v[j]);
      }
      top = fmaxf(top, __shfl_xor(top, 1));
      all = cross_terms<T>(v, top);
      all += __shfl_xor(all, 1);
      if (t % 2 == 0 && row < rows) a.parts[(uint64_t)row * a.groups + column] = float2{top, cross_settled<T>(all, top)};
    }
  }
}

struct cross_words_args {
  const void* x;
  const void* w;
  uint64_t ldx, ldw, k;
  const int64_t* targets;
  int64_t ignored;
  float* loss;  // by row
  float* lse;   // or null: nothing is kept
  float* z;     // [rows][ld] or null
  uint32_t rows, words, ld;
};

// Rows of a workgroup: the weight is read once for them, which past 16 words is as much as x (12496 x 7900
// over 22 words fp32: 160 us with 32 rows, 213 with 16; 8192 x 4096 over 10 words bf16: 21 and 17).
constexpr int cross_words_rows(int nt) { return nt == 1 ? 16 : 32; }

// Up to 16 * NT words: a workgroup makes z of its rows, whose sums over k meet in LDS in the waves'
// order, their lse and their losses. Bound by the weight's way from the second cache and by x's from
// memory: 8192 x 4096 bf16 over 10 words 17 us (3.9 TB/s of x), over 50 words 25 (2.7); 12496 x 7900 over 22
// words fp32 160 (2.5). Turns' loads ahead of the products change nothing.
template <typename T, int NT>
__global__ __launch_bounds__(64 * TAM_FEW_WAVES) void tam_k_cross_words(cross_words_args a) {
  constexpr int N = 16 / (int)sizeof(T), U = NT == 4 ? 2 : 4, MT = cross_words_rows(NT) / 16;
  constexpr uint64_t TURN = 4 * U * N;  // k of a wave's turn
  __shared__ float sum[TAM_FEW_WAVES][MT * 16][NT * 16 + 4];
  const uint32_t row0 = blockIdx.x * MT * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t i = lane & 15, q = lane >> 4;
  const T *w[NT], *x[MT];
  tam_f4 acc[MT][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)  // words and rows past the last one read the first one's elements; their sums go nowhere
    w[n] = static_cast<const T*>(a.w) + (n * 16 + i < a.words ? (uint64_t)(n * 16 + i) * a.ldw : 0);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    x[m] = static_cast<const T*>(a.x) + (uint64_t)(row0 + m * 16 + i < a.rows ? row0 + m * 16 + i : row0) * a.ldx;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = tam_f4{0.f, 0.f, 0.f, 0.f};
  }
  auto turn = [&](uint64_t k0, auto guard) {
    constexpr bool G = decltype(guard)::value;
    tam_frag<T> fw[NT][U], fx[MT][U];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int u = 0; u < U; ++u) tam_few_load<T, G>(fx[m][u], x[m], k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int u = 0; u < U; ++u) tam_few_load<T, G>(fw[n][u], w[n], k0 + (u * 4 + q) * N, a.k);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int u = 0; u < U; ++u) acc[m][n] = tam_mfma(fw[n][u], fx[m][u], acc[m][n]);
  };
  uint64_t k0 = wave * TURN;
#pragma unroll 2
  for (; k0 + TURN <= a.k; k0 += TAM_FEW_WAVES * TURN) turn(k0, std::false_type());
  if (k0 < a.k) turn(k0, std::true_type());
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)  // row m * 16 + i, words n * 16 + 4 q ..
      *reinterpret_cast<tam_f4*>(&sum[wave][m * 16 + i][n * 16 + q * 4]) = acc[m][n];
  __syncthreads();
  const uint32_t t = threadIdx.x, at = t / (2 * NT), col = t % (2 * NT) * 8, row = row0 + at;  // 2 NT lanes to a row
  if (t >= MT * 16 * 2 * NT || row >= a.rows) return;
  float v[8] = {};
  for (int s = 0; s < TAM_FEW_WAVES; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += sum[s][at][col + j];
  if (a.z && col < a.ld) tam_store8(a.z + (uint64_t)row * a.ld + col, v);
  const int64_t target = a.targets[row];
  float top = -INFINITY, hit = 0.f;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    if (col + j >= a.words) v[j] = -INFINITY;
    else if (target == (int64_t)(col + j)) hit = v[j];
    top = fmaxf(top, v[j]);
  }
#pragma unroll
  for (int d = 1; d < 2 * NT; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  float all = cross_terms<T>(v, top);
#pragma unroll
  for (int d = 1; d < 2 * NT; d *= 2) {
    all += __shfl_xor(all, d);
    hit += __shfl_xor(hit, d);
  }
  if (t % (2 * NT) == 0) {
    const bool inside = target >= 0 && target < (int64_t)a.words;
    all = cross_settled<T>(all, top);
    if (a.lse) a.lse[row] = inside ? top + logf(all) : NAN;
    a.loss[row] = target == a.ignored ? 0.f : (inside ? cross_loss(top, all, hit) : NAN);
  }
}

// ---------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------
// dz of rows that count, of few words: 8 columns of the z that was kept to a thread.
template <typename T>
__global__ __launch_bounds__(256) void tam_k_cross_words_dz(const float* z, uint32_t ldz, uint32_t words, cross_rows r,
                                                            const cross_row* rows, T* dz, uint64_t ld) {
  const uint32_t per = ldz / 8, i = blockIdx.x * 256 + threadIdx.x, j = i / per, col = (i - j * per) * 8;
  if (j >= *r.count) return;
  const cross_row of = rows[j];
  float v[8];
  tam_load8(z + (uint64_t)r.index[j] * ldz + col, v);
  const uint32_t hit = (uint32_t)of.target - col;
#pragma unroll
  for (uint32_t c = 0; c < 8; ++c) {
    const float p = cross_exp<T>(v[c] - of.lse) - (hit == c ? 1.0f : 0.0f);
    // columns past the last one are zeros: the sum over columns takes whole 16 bytes
    v[c] = col + c < words ? p * of.w : 0.0f;
  }
  tam_store8(dz + j * ld + col, v);
}

struct cross_weights_args {
  cross_rows r;
  const float* dloss;
  int64_t stride;
  uint32_t reduction;
  float lift;     // of dz
  cross_row* row; // [rows]
  float* scale;   // what the products are multiplied by
};

// Each row's weight, and scale; 8192 rows 6.5 us, one workgroup's trips to memory. A gradient for
// each row: scale is the least power of two above the largest finite one, so that dividing by it
// rounds nothing; but 2^127 for those above it (a row's weight is then up to 2), and 2^-100 at least.
__global__ __launch_bounds__(1024) void tam_k_cross_weights(cross_weights_args a) {
  __shared__ float top[1024];
  const uint32_t count = *a.r.count;
  if (a.reduction != TAM_CROSS_NONE) {
    for (uint32_t j = threadIdx.x; j < count; j += 1024) a.row[j] = {a.r.lse[a.r.index[j]], a.lift, a.r.target[j], 0};
    if (threadIdx.x == 0)  // no row: the sums are zeros, and stay that
      *a.scale = count ? (a.reduction == TAM_CROSS_MEAN ? a.dloss[0] / (float)count : a.dloss[0]) / a.lift : 0.0f;
    return;
  }
  float most = 0.f;
  for (uint32_t j = threadIdx.x; j < count; j += 1024) {
    const float d = fabsf(a.dloss[(int64_t)a.r.index[j] * a.stride]);
    if (d < INFINITY) most = fmaxf(most, d);
  }
  top[threadIdx.x] = most;
  for (int half = 512; half >= 1; half /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < half) top[threadIdx.x] = fmaxf(top[threadIdx.x], top[threadIdx.x + half]);
  }
  __syncthreads();
  int power;
  frexpf(top[0], &power);
  power = power < -100 ? -100 : (power > 127 ? 127 : power);
  for (uint32_t j = threadIdx.x; j < count; j += 1024) {
    const uint32_t row = a.r.index[j];
    a.row[j] = {a.r.lse[row], ldexpf(a.dloss[(int64_t)row * a.stride], -power) * a.lift, a.r.target[j], 0};
  }
  if (threadIdx.x == 0) *a.scale = ldexpf(1.0f, power) / a.lift;
}

struct cross_product_args {
  tam_operand P, Q;
  uint64_t k, most_k;      // dx: of this piece, and of the widest one
  uint32_t tm, tn, parts;  // tiles (of all rows), and what a sum is cut into
  uint32_t rows, cols;
  float* sums;             // [part][rows][cols], or null: dw's own
  bool add;                // to what the sums hold
  void* out;               // dw's rows of the piece; dx, where one product makes it (no sums)
  const uint32_t* index;   // of dx's rows
};

// A piece's products: units of dw and units of dx's share in one launch, so that neither leaves
// compute units empty at its end: those of the longer sums first, so that the shorter fill the last round.
struct cross_products_args {
  cross_product_args w, x;
  uint32_t w_units;        // of w.tm * w.tn * w.parts
  uint32_t w_first;        // the first one's workgroup: 0, or behind dx's
  const uint32_t* count;
  const float* scale;
};

// Into how many parts dx's sums are cut where `count` of `rows` count: as many as there is room
// for, in the sums and in the launch, which were laid out for all of them.
__device__ __forceinline__ uint32_t cross_parts(uint32_t parts, uint32_t rows, uint32_t count, uint32_t tile, uint64_t k) {
  if (parts == 1 || count == 0) return parts;
  const uint32_t all = (rows + tile - 1) / tile, now = (count + tile - 1) / tile;
  const uint64_t room = (uint64_t)parts * rows / count, launch = (uint64_t)parts * all / now, least = k / 256;
  uint64_t n = room < launch ? room : launch;
  if (n > least) n = least;
  return n > parts ? (uint32_t)n : parts;
}

// dx's share of a piece (WEIGHT false: fp32 sums) or the piece's rows of dw.
template <typename T, int TILE, int WM, int WN, bool WEIGHT>
__device__ __forceinline__ void cross_product(cross_product_args& a, uint32_t unit, uint32_t count, const float* of_scale,
                                              char* smem) {
  typedef tam_tile<T, TILE, TILE, WM, WN, tam_stages<T, TILE>(), false, !WEIGHT> Tile;
  const uint32_t rows = WEIGHT ? a.rows : count, tm = (rows + TILE - 1) / TILE, tiles = tm * a.tn;
  const uint32_t parts = WEIGHT ? a.parts : cross_parts(a.parts, a.rows, count, TILE, a.most_k);
  if (unit >= tiles * parts) return;
  const uint32_t part = unit / tiles;
  uint32_t m, n;
  tam_tile_at(tam_xcd_order(unit - part * tiles, tiles), tm, a.tn, m, n);
  if (!WEIGHT) a.Q.count = count;
  const uint64_t k = WEIGHT ? count : a.k, per = parts > 1 ? (k / parts + 64) / 64 * 64 : k;
  const uint64_t k0 = part * per < k ? part * per : k, k1 = k0 + per < k ? k0 + per : k;
  float* const sums = a.sums ? a.sums + (uint64_t)part * rows * a.cols : nullptr;
  Tile t;
  t.zero();
  tam_soon soon = {};
  if (a.add) {
    const uint64_t ld = (uint64_t)a.cols * 4;
    soon = {reinterpret_cast<const char*>(sums) + m * TILE * ld + n * TILE * 4, ld, rows - m * TILE, (a.cols - n * TILE) * 4,
            TILE * 4};
  }
  t.run(a.P, a.Q, n * TILE, m * TILE, k0, k1, smem, soon);
  const float scale = sums ? 1.0f : *of_scale;
  t.template each<TAM_AHEAD_PASS>(
      smem,
      [&](uint32_t row, uint32_t col) {
        tam_oct<float> s = {};
        row += m * TILE;
        col += n * TILE;
        if (!WEIGHT && a.add && row < rows && col < a.cols)
          s = tam_some(sums + (uint64_t)row * a.cols + col, a.cols - col);
        return s;
      },
      [&](uint32_t row, uint32_t col, float(&v)[8], const tam_oct<float>& s) {
        row += m * TILE;
        col += n * TILE;
        if (row >= rows || col >= a.cols) return;
        if (!sums) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= scale;
          const uint64_t at = (uint64_t)(WEIGHT ? row : a.index[row]) * a.cols + col;
          tam_store_some(static_cast<T*>(a.out) + at, a.cols - col, v);
        } else {
          if (!WEIGHT && a.add)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += s.v[j];
          tam_store_some(sums + (uint64_t)row * a.cols + col, a.cols - col, v);
        }
      },
      [](uint32_t, uint32_t, const float*, int) {});
}

// Bound by the matrix cores: bf16, 7680 rows that count x 4096 over 128256 words, four pieces 11920 us
// for 16.1 Tflop (1354 TFLOP/s); 8192 x 768 over 50257 words, two pieces 1003 (1261). fp32 619 x 515 over 9973
// words, 64 tiles: 129 (99).
template <typename T, int TILE, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, TILE == 64 ? 3 : 2) void tam_k_cross_products(cross_products_args a) {
  typedef tam_tile<T, TILE, TILE, WM, WN, tam_stages<T, TILE>(), false, true> Tile;
  __shared__ __attribute__((aligned(16))) char smem[Tile::LDS];
  const uint32_t count = *a.count;
  if (blockIdx.x - a.w_first < a.w_units)
    cross_product<T, TILE, WM, WN, true>(a.w, blockIdx.x - a.w_first, count, a.scale, smem);
  else
    cross_product<T, TILE, WM, WN, false>(a.x, blockIdx.x < a.w_first ? blockIdx.x : blockIdx.x - a.w_units, count, a.scale, smem);
}

// out[row] = the parts' sums of the row's number in their order, times scale; zeros for
// rows that do not count. place == null: a row's number is its own. tile, k: dx's. Bound by memory: 8192 x
// 4096 bf16 of one part 32 us, 5.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void tam_k_cross_out(const float* sums, uint32_t parts, uint64_t rows, uint32_t cols,
                                                       const int32_t* place, const uint32_t* count, uint32_t tile, uint64_t k,
                                                       const float* scale, T* out) {
  uint64_t summed = rows;
  if (place) {
    summed = *count;
    parts = cross_parts(parts, (uint32_t)rows, (uint32_t)summed, tile, k);
  }
  const uint32_t per = (cols + 7) / 8;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per * rows) return;
  const uint64_t row = i / per;
  const uint32_t col = (uint32_t)(i - row * per) * 8;
  const int64_t at = place ? place[row] : (int64_t)row;
  float v[8] = {};
  if (at >= 0) {
    const float s = *scale;
    for (uint32_t p = 0; p < parts; ++p) {
      float t[8];
      tam_load_some(sums + (p * summed + at) * cols + col, cols - col, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= s;
  }
  tam_store_some(out + row * cols + col, cols - col, v);
}

// Zeros for the rows of dx that do not count: a workgroup to a row at a time.
__global__ __launch_bounds__(256) void tam_k_cross_clear(tam_f16* dx, uint64_t rows, uint32_t cols, const int32_t* place) {
  const float v[8] = {};
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    if (place[row] >= 0) continue;
    for (uint32_t col = threadIdx.x * 8; col < cols; col += 2048) tam_store_some(dx + row * cols + col, cols - col, v);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Passes that read the weight and x straight to the matrix cores: of few rows, and of so few words
// that tiles would be few, or mostly empty (fp32, both ways, tiles -> this: 12496 x 7900 over 22 words
// 1079 -> 555 us, 42 x 5424 over 6 words 232 -> 80). 16 rows have 512 threads of a launch, which
// takes fewer than 2^32.
bool few_words(const TamCross* d) { return d->vocabulary <= 64 && d->rows < 1ull << 26; }
bool few(const TamCross* d) { return d->rows <= 32 || few_words(d); }

constexpr uint64_t kPieceBytes = 512ull << 20;  // of dz
constexpr uint64_t kMostPiece = 1ull << 20;     // a tile's offsets are 31-bit numbers of bytes

int check_cross(const TamCross* d, bool back) {
  tam_op_begin();
  if (!d) return tam_op_fail(TAM_E_INVALID, "null argument");
  if (d->dtype > TAM_DTYPE_F16) return tam_op_fail(TAM_E_INVALID, "unknown dtype %u", d->dtype);
  if (d->reduction > TAM_CROSS_MEAN) return tam_op_fail(TAM_E_INVALID, "unknown reduction %u", d->reduction);
  const uint64_t most = 1ull << 31;
  if (d->rows >= most || d->inputs >= most || d->vocabulary >= most - 256)
    return tam_op_fail(TAM_E_UNSUPPORTED, "a size of 2^31 or more");
  if (d->inputs && (d->ldx < d->inputs || d->ldw < d->inputs))
    return tam_op_fail(TAM_E_INVALID, "a row stride shorter than its row");
  if ((d->ldx | d->ldw | d->inputs) >= 1ull << 21)
    return tam_op_fail(TAM_E_UNSUPPORTED, "a row or row stride of 2^21 elements or more");
  if (d->piece % 256 || d->piece > kMostPiece)
    return tam_op_fail(TAM_E_INVALID, "a piece that is no multiple of 256, or above 2^20");
  if (!d->rows && (back || d->reduction == TAM_CROSS_NONE)) return TAM_OK;
  if (d->rows && d->vocabulary == 0) return tam_op_fail(TAM_E_INVALID, "an empty vocabulary");
  if (d->rows && d->inputs && ((!d->x && (!back || few(d))) || !d->w)) return tam_op_fail(TAM_E_INVALID, "null x or w");
  if (d->rows && !back && !d->target) return tam_op_fail(TAM_E_INVALID, "null target");
  if (!back && !d->loss) return tam_op_fail(TAM_E_INVALID, "null loss");
  if (back && (!d->kept || !d->dloss)) return tam_op_fail(TAM_E_INVALID, "null dloss, or what the forward pass kept");
  if ((uintptr_t)d->kept & 255u) return tam_op_fail(TAM_E_INVALID, "kept memory not on 256 bytes");
  return TAM_OK;
}

uint64_t rows_bytes(uint64_t rows) { return 256 + tam_up(16 * rows, 256); }

uint32_t words_ld(const TamCross* d) { return (uint32_t)tam_up(d->vocabulary, 8); }

// Behind the rows' numbers the gathered rows of x: the backward pass reads them in place of x. Of few
// words z, by row.
uint64_t kept_bytes(const TamCross* d) {
  const uint32_t size = kSize[d->dtype];
  if (few(d)) return rows_bytes(d->rows) + (few_words(d) ? d->rows * words_ld(d) * 4ull : 0);
  return rows_bytes(d->rows) + d->rows * aligned_ld((uint32_t)d->inputs, size) * size;
}

cross_rows rows_in(void* kept, uint64_t rows) {
  if (!kept) return {};
  uint32_t* p = (uint32_t*)((char*)kept + 256);
  return {(uint32_t*)kept, p, (int32_t*)(p + rows), (int32_t*)(p + 2 * rows), (float*)(p + 3 * rows)};
}

int number_rows(const TamCross* d, const cross_rows& r, float* loss, hipStream_t s) {
  const cross_rows_args a = {r, d->target, loss, d->ignored, (uint32_t)d->rows, (int64_t)d->vocabulary};
  hipLaunchKernelGGL(tam_k_cross_rows, dim3(1), dim3(1024), 0, s, a);
  TAM_OP_LAUNCHED("the rows' numbers");
  return TAM_OK;
}

// The rows of x that count, and w, as the tiles read them, where a product does. kept: where the rows lie or, in
// the forward pass, are to lie (the workspace where it is null).
int operands(const TamCross* d, call& c, const cross_rows& r, void* kept, bool back, bool read_x, bool read_w, matrix& x,
             matrix& w) {
  const uint32_t size = kSize[c.dtype], halves = size / 2, inputs = (uint32_t)d->inputs, ld = aligned_ld(inputs, size);
  if (read_w) {
    w = matrix_of(d->w, d->ldw, d->vocabulary, d->inputs, size);
    const int rc = whole_rows(c, &w);
    if (rc != TAM_OK) return rc;
  }
  if (!read_x) return TAM_OK;
  x = {kept ? (char*)kept + rows_bytes(d->rows) : c.ws.take(d->rows * ld * size), ld, d->rows, inputs, true};
  const uint64_t copies = back && kept ? 0 : tam_div_up(d->rows * (ld * halves / 8), 256);
  const int rc = room(copies, 256);
  if (rc != TAM_OK) return rc;
  if (!c.dry && inputs && copies) {
    const dim3 grid((uint32_t)copies), block(256);
    hipLaunchKernelGGL(tam_k_cross_gather, grid, block, 0, c.stream, (const tam_f16*)d->x, d->ldx * halves, inputs * halves, r,
                       (uint32_t)d->rows, (tam_f16*)x.p, ld * halves);
    TAM_OP_LAUNCHED("the rows' copy");
  }
  return TAM_OK;
}

template <typename T, bool BACK>
void launch_logits(int tile, const cross_logits_args& a, hipStream_t s) {
  const uint32_t tiles = a.tm * a.tn, cus = tam_op_cus();
  const dim3 grid(tile == 256 && tiles > cus ? cus : tiles);
  if constexpr (sizeof(T) == 2)
    if (tile == 256) {
      hipLaunchKernelGGL((tam_k_cross_logits<T, 256, 2, 4, BACK>), grid, dim3(512), 0, s, a);
      return;
    }
  if (tile == 128)
    hipLaunchKernelGGL((tam_k_cross_logits<T, 128, 2, 2, BACK>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((tam_k_cross_logits<T, 64, 2, 2, BACK>), grid, dim3(256), 0, s, a);
}

template <typename T>
void launch_products(int tile, const cross_products_args& a, uint32_t units, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (tile == 256) {
      hipLaunchKernelGGL((tam_k_cross_products<T, 256, 2, 4>), dim3(units), dim3(512), 0, s, a);
      return;
    }
  if (tile == 128)
    hipLaunchKernelGGL((tam_k_cross_products<T, 128, 2, 2>), dim3(units), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((tam_k_cross_products<T, 64, 2, 2>), dim3(units), dim3(256), 0, s, a);
}

// A piece's two products in one launch: their tile and parts.
struct pair_shape {
  int tile;
  uint32_t w_parts, x_parts;
};

pair_shape choose_pair(uint64_t rows, uint64_t inputs, uint64_t words, bool dw, bool dx, uint32_t dtype) {
  const double cus = tam_op_cus();
  const bool f32 = dtype == TAM_DTYPE_F32;
  const tam_tile_rate* rate = f32 ? tam_rates_32 : tam_rates_16;
  pair_shape best = {64, 1, 1};
  double least = 1e30;
  for (int i = 0; i < (f32 ? 2 : 3); ++i) {
    const uint64_t t = rate[i].tile, across = tam_div_up(inputs, t);
    for (uint32_t wp : {1, 2, 4, 8, 16, 32}) {
      if (wp > 1 && (!dw || rows / wp < 128)) break;
      for (uint32_t xp : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (xp > 1 && (!dx || words / xp < 256)) break;
        const uint64_t nw = dw ? tam_div_up(words, t) * across * wp : 0, nx = dx ? tam_div_up(rows, t) * across * xp : 0;
        double us = units_us(rate[i], nw, (double)rows / wp, nx, (double)words / xp, cus);
        // parts' sums to memory and back (about 4 TB/s): dx's are there in any case, and added to
        us += (double)rows * inputs * 8.0 * (dx ? xp : 0) / 4e6;
        if (wp > 1) us += 3.0 + (double)words * inputs * 8.0 * wp / 4e6;
        if (us < least) {
          least = us;
          best = {rate[i].tile, wp, xp};
        }
      }
    }
  }
  return best;
}

// The tile of a product that is not cut into parts.
int tile_of(uint64_t rows, uint64_t cols, uint64_t k, uint32_t dtype) {
  const double cus = tam_op_cus();
  const bool f32 = dtype == TAM_DTYPE_F32;
  const tam_tile_rate* rate = f32 ? tam_rates_32 : tam_rates_16;
  int best = 64;
  double least = 1e30;
  for (int i = 0; i < (f32 ? 2 : 3); ++i) {
    const double us = tam_tiles_us(
        rate[i], (double)tam_div_up(rows, rate[i].tile) * (double)tam_div_up(cols, rate[i].tile), (double)k, cus);
    if (us < least) {
      least = us;
      best = rate[i].tile;
    }
  }
  return best;
}

cross_logits_args logits_of(const TamCross* d, const matrix& x, const matrix& w, const cross_rows& r, uint64_t first,
                            uint64_t cols, int tile, uint32_t size) {
  cross_logits_args a = {};
  a.P = operand_of(w, (uint32_t)cols, size);
  a.P.base += first * w.ld * size;
  a.Q = operand_of(x, (uint32_t)d->rows, size);
  a.k = d->inputs;
  a.tm = (uint32_t)tam_div_up(d->rows, tile);
  a.tn = (uint32_t)tam_div_up(cols, tile);
  a.r = r;
  a.first = (uint32_t)first;
  a.cols = (uint32_t)cols;
  a.rows = d->rows;
  return a;
}

int forward(const TamCross* d, call& c) {
  const bool reduced = d->reduction != TAM_CROSS_NONE;
  const uint32_t rows = (uint32_t)d->rows;
  if (rows == 0 && !reduced) return TAM_OK;
  cross_join_args j = {};
  j.targets = d->target;
  j.ignored = d->ignored;
  j.vocabulary = (int64_t)d->vocabulary;
  j.rows = rows;
  float* losses = d->loss;
  if (reduced) losses = (float*)c.ws.take(4ull * rows);
  const bool is_few = few(d);
  if (rows) {
    float* hit = few_words(d) ? nullptr : (float*)c.ws.take(4ull * rows);
    cross_rows r = rows_in(d->kept, rows);
    if (few_words(d)) {
      if (!c.dry) {
        if (d->kept) {
          const int rc = number_rows(d, r, nullptr, c.stream);
          if (rc != TAM_OK) return rc;
        }
        float* const z = d->kept ? (float*)((char*)d->kept + rows_bytes(rows)) : nullptr;
        const cross_words_args a = {d->x, d->w, d->ldx, d->ldw, d->inputs, d->target, d->ignored, losses, r.lse, z, rows,
                                    (uint32_t)d->vocabulary, words_ld(d)};
        const int nt = a.words <= 16 ? 1 : (a.words <= 32 ? 2 : 4);
        const dim3 grid((uint32_t)tam_div_up(rows, cross_words_rows(nt))), block(64 * TAM_FEW_WAVES);
#define TAM_WORDS(T)                                                             \
  if (nt == 1)                                                                   \
    hipLaunchKernelGGL((tam_k_cross_words<T, 1>), grid, block, 0, c.stream, a);  \
  else if (nt == 2)                                                              \
    hipLaunchKernelGGL((tam_k_cross_words<T, 2>), grid, block, 0, c.stream, a);  \
  else                                                                           \
    hipLaunchKernelGGL((tam_k_cross_words<T, 4>), grid, block, 0, c.stream, a)
        TAM_OF_TYPE(c, TAM_WORDS);
        TAM_OP_LAUNCHED("the logits of few words");
      }
    } else if (is_few) {
      const uint32_t groups = (uint32_t)tam_div_up(d->vocabulary, 16);
      float2* parts = (float2*)c.ws.take(8ull * rows * groups);
      const int rc = room(groups, 64 * TAM_FEW_WAVES);
      if (rc != TAM_OK) return rc;
      if (!c.dry) {
        if (d->kept) {
          const int rc = number_rows(d, r, nullptr, c.stream);
          if (rc != TAM_OK) return rc;
        }
        cross_few_args a = {};
        a.x = d->x;
        a.w = d->w;
        a.ldx = d->ldx;
        a.ldw = d->ldw;
        a.k = d->inputs;
        a.targets = d->target;
        a.parts = parts;
        a.hit = hit;
        a.rows = rows;
        a.cols = (uint32_t)d->vocabulary;
        a.groups = groups;
        const dim3 grid(groups), block(64 * TAM_FEW_WAVES);
#define TAM_FEW(T)                                                                    \
  if (rows <= 16)                                                                     \
    hipLaunchKernelGGL((tam_k_cross_few<T, 1, false>), grid, block, 0, c.stream, a);  \
  else                                                                                \
    hipLaunchKernelGGL((tam_k_cross_few<T, 2, false>), grid, block, 0, c.stream, a)
        TAM_OF_TYPE(c, TAM_FEW);
        TAM_OP_LAUNCHED("the logits of few rows");
        j.r = r;
        j.parts = parts;
        j.hit = hit;
        j.loss = losses;
        j.tiles = groups;
        hipLaunchKernelGGL(tam_k_cross_join_few, dim3(rows), dim3(1024), 0, c.stream, j);
        TAM_OP_LAUNCHED("the losses");
      }
    } else {
      if (!d->kept) r = rows_in(c.ws.take(rows_bytes(rows)), rows);
      if (!c.dry) {
        const int rc = number_rows(d, r, reduced ? nullptr : d->loss, c.stream);
        if (rc != TAM_OK) return rc;
      }
      const int tile = tile_of(rows, d->vocabulary, d->inputs, c.dtype);
      if (c.tiles) c.tiles[0] = (uint32_t)tile;
      matrix x, w;
      int rc = operands(d, c, r, d->kept, false, true, true, x, w);
      if (rc == TAM_OK) rc = room_of_tiles(tam_div_up(rows, tile) * tam_div_up(d->vocabulary, tile), tile, true);
      if (rc == TAM_OK) rc = room(tam_div_up(rows, 64), 1024);
      if (rc != TAM_OK) return rc;
      cross_logits_args a = logits_of(d, x, w, r, 0, d->vocabulary, tile, kSize[c.dtype]);
      a.parts = (float2*)c.ws.take(8ull * rows * a.tn);
      a.hit = hit;
      if (!c.dry) {
#define TAM_LOGITS(T) launch_logits<T, false>(tile, a, c.stream)
        TAM_OF_TYPE(c, TAM_LOGITS);
        TAM_OP_LAUNCHED("the logits");
        j.r = r;
        j.parts = a.parts;
        j.hit = hit;
        j.loss = losses;
        j.by_number = reduced;
        j.tiles = a.tn;
        hipLaunchKernelGGL(tam_k_cross_join, dim3((uint32_t)tam_div_up(rows, 64)), dim3(1024), 0, c.stream, j);
        TAM_OP_LAUNCHED("the losses");
      }
    }
    j.r = r;
  }
  if (reduced && !c.dry) {
    hipLaunchKernelGGL(tam_k_cross_sum, dim3(1), dim3(1024), 0, c.stream, losses, is_few ? nullptr : j.r.count, d->target,
                       d->ignored, rows, d->reduction == TAM_CROSS_MEAN, d->loss);
    TAM_OP_LAUNCHED("the losses' sum");
  }
  return TAM_OK;
}

// us of the backward pass in pieces of `piece` columns.
double pieces_us(const TamCross* d, uint64_t piece) {
  const double cus = tam_op_cus();
  const bool f32 = d->dtype == TAM_DTYPE_F32;
  const pair_shape p = choose_pair(d->rows, d->inputs, piece < d->vocabulary ? piece : d->vocabulary, d->dw, d->dx, d->dtype);
  const int tile = tile_of(d->rows, piece, d->inputs, d->dtype);
  const tam_tile_rate *rate = f32 ? tam_rates_32 : tam_rates_16, *z = rate, *t = rate;
  while (z->tile != tile) ++z;
  while (t->tile != p.tile) ++t;
  double us = 0;
  const uint64_t across = tam_div_up(d->inputs, t->tile);
  for (uint64_t first = 0, cols; first < d->vocabulary; first += cols) {
    cols = d->vocabulary - first < piece ? d->vocabulary - first : piece;
    us += tam_tiles_us(*z, (double)tam_div_up(d->rows, tile) * (double)tam_div_up(cols, tile), (double)d->inputs, cus);
    us += units_us(*t, d->dw ? tam_div_up(cols, t->tile) * across * p.w_parts : 0, (double)d->rows / p.w_parts,
                   d->dx ? tam_div_up(d->rows, t->tile) * across * p.x_parts : 0, (double)cols / p.x_parts, cus);
    us += 6.0 + (double)d->rows * d->inputs * 8.0 * (d->dx ? p.x_parts : 0) / 4e6;
  }
  return us;
}

// Columns of a piece, of at most kPieceBytes of dz: as even as they come, in whole tiles; or, where
// products are long enough for the choice to pay for itself, what is estimated to take the
// least time of a few numbers of pieces and of pieces whose dw fills the card's rounds. (8192 x 768 of
// 50257 bf16: two even pieces, 2.26 ms.)
uint64_t piece_of(const TamCross* d, uint32_t size) {
  if (d->piece) return d->piece;
  uint64_t most = kPieceBytes / (d->rows * size) / 256 * 256;
  most = most < 256 ? 256 : (most > kMostPiece ? kMostPiece : most);
  const uint64_t fewest = tam_div_up(d->vocabulary, most);
  uint64_t best = tam_up(tam_div_up(d->vocabulary, fewest), 256);
  if ((double)d->rows * (double)d->inputs * (double)d->vocabulary < 2e11 || (!d->dx && !d->dw)) return best;
  double least = pieces_us(d, best);
  auto consider = [&](uint64_t piece) {
    if (piece < 1024 || piece > most) return;
    const double us = pieces_us(d, piece);
    if (us < 0.98 * least) {
      least = us;
      best = piece;
    }
  };
  for (uint64_t n = fewest + 1; n < fewest + 4; ++n) consider(tam_up(tam_div_up(d->vocabulary, n), 256));
  const uint64_t across = tam_div_up(d->inputs, 256);
  for (uint64_t rounds = 1; rounds <= 4; ++rounds) consider(tam_op_cus() * rounds / across * 256);
  return best;
}

int backward(const TamCross* d, call& c) {
  if (!d->dx && !d->dw) return TAM_OK;
  const uint32_t rows = (uint32_t)d->rows, inputs = (uint32_t)d->inputs, size = kSize[c.dtype];
  if (!rows || !inputs) return zeros(c, d->dw, d->vocabulary * d->inputs);
  const cross_rows r = rows_in(d->kept, rows);
  cross_row* row = (cross_row*)c.ws.take(sizeof(cross_row) * (uint64_t)rows);
  float* scale = (float*)c.ws.take(4);
  if (!c.dry) {
    const float lift = c.dtype == TAM_DTYPE_F16 ? 16384.0f : 1.0f;
    const cross_weights_args a = {r, d->dloss, d->dloss_stride, d->reduction, lift, row, scale};
    hipLaunchKernelGGL(tam_k_cross_weights, dim3(1), dim3(1024), 0, c.stream, a);
    TAM_OP_LAUNCHED("the rows' weights");
  }
  matrix x = {}, w = {};
  const uint64_t piece = piece_of(d, size), widest = d->vocabulary < piece ? d->vocabulary : piece;
  // otherwise dz comes from the z that was kept, or straight from x and w
  const bool is_few = few(d), tiles = !few_words(d) && !(is_few && widest == d->vocabulary);
  int rc = operands(d, c, r, is_few ? nullptr : d->kept, true, tiles || d->dw, tiles || d->dx, x, w);
  if (rc != TAM_OK) return rc;
  const uint32_t ld = aligned_ld((uint32_t)widest, size);
  void* dz = c.ws.take((uint64_t)rows * ld * size);
  const int tile_z = tile_of(rows, widest, inputs, c.dtype);
  const pair_shape both = choose_pair(rows, inputs, widest, d->dw, d->dx, c.dtype);
  if (c.tiles) {
    c.tiles[0] = tiles ? (uint32_t)tile_z : 0;
    c.tiles[1] = (uint32_t)piece;
    c.tiles[2] = (uint32_t)both.tile;
    c.tiles[3] = both.x_parts << 16 | both.w_parts;
  }
  // one product makes all of dx where its sums are whole
  const bool direct = d->dx && both.x_parts == 1 && widest == d->vocabulary;
  float* dx_sums = d->dx && !direct ? (float*)c.ws.take(4ull * both.x_parts * rows * inputs) : nullptr;
  float* dw_sums = d->dw && both.w_parts > 1 ? (float*)c.ws.take(4ull * both.w_parts * widest * inputs) : nullptr;
  const uint32_t across = (uint32_t)tam_div_up(inputs, both.tile);
  const uint64_t eights = tam_div_up(inputs, 8), joins_w = tam_div_up(widest * eights, 256), joins_x = tam_div_up(rows * eights, 256);
  const uint64_t units_w = d->dw ? tam_div_up(widest, both.tile) * across * both.w_parts : 0;
  const uint64_t units_x = d->dx ? tam_div_up(rows, both.tile) * (uint64_t)across * both.x_parts : 0;
  rc = tiles ? room_of_tiles(tam_div_up(rows, tile_z) * tam_div_up(widest, tile_z), tile_z, true)
             : room(tam_div_up(widest, 16), 64 * TAM_FEW_WAVES);
  if (rc == TAM_OK) rc = room_of_tiles(units_w + units_x, both.tile, false);
  if (rc == TAM_OK && dw_sums) rc = room(joins_w, 256);
  if (rc == TAM_OK && d->dx && !direct) rc = room(joins_x, 256);
  if (rc != TAM_OK || c.dry) return rc;
  for (uint64_t first = 0; first < d->vocabulary; first += piece) {
    const uint32_t cols = (uint32_t)(d->vocabulary - first < piece ? d->vocabulary - first : piece);
    if (few_words(d)) {
      const uint32_t ldz = words_ld(d);
      const float* const kept = (const float*)((const char*)d->kept + rows_bytes(rows));
      const dim3 grid((uint32_t)tam_div_up((uint64_t)rows * (ldz / 8), 256)), block(256);
#define TAM_WORDS_DZ(T) \
  hipLaunchKernelGGL(tam_k_cross_words_dz<T>, grid, block, 0, c.stream, kept, ldz, cols, r, row, (T*)dz, (uint64_t)ld)
      TAM_OF_TYPE(c, TAM_WORDS_DZ);
    } else if (!tiles) {
      cross_few_args f = {};
      f.x = d->x;
      f.w = d->w;
      f.ldx = d->ldx;
      f.ldw = d->ldw;
      f.k = inputs;
      f.rows = rows;
      f.cols = cols;
      f.r = r;
      f.row = row;
      f.dz = dz;
      f.ld = ld;
      f.groups = (uint32_t)tam_div_up(cols, 16);
      const dim3 grid(f.groups), block(64 * TAM_FEW_WAVES);
#define TAM_FEW_DZ(T) hipLaunchKernelGGL((tam_k_cross_few<T, 2, true>), grid, block, 0, c.stream, f)
      TAM_OF_TYPE(c, TAM_FEW_DZ);
    } else {
      cross_logits_args a = logits_of(d, x, w, r, first, cols, tile_z, size);
      a.row = row;
      a.dz = dz;
      a.ld = ld;
#define TAM_DZ(T) launch_logits<T, true>(tile_z, a, c.stream)
      TAM_OF_TYPE(c, TAM_DZ);
    }
    TAM_OP_LAUNCHED("the logits' gradient");
    const matrix z = {dz, ld, rows, cols, true};
    cross_products_args p = {};
    p.count = r.count;
    p.scale = scale;
    uint64_t units = 0;
    if (d->dw) {
      p.w.P = operand_of(x, inputs, size);
      p.w.Q = operand_of(z, cols, size);
      p.w.tm = (uint32_t)tam_div_up(cols, both.tile);
      p.w.tn = across;
      p.w.parts = both.w_parts;
      p.w.rows = cols;
      p.w.cols = inputs;
      p.w.sums = dw_sums;
      p.w.out = (char*)d->dw + first * inputs * size;
      units = (uint64_t)p.w.tm * across * both.w_parts;
      p.w_units = (uint32_t)units;
    }
    if (d->dx) {
      p.x.P = operand_of(w, inputs, size);
      p.x.P.base += first * w.ld * size;
      p.x.Q = operand_of(z, rows, size);
      p.x.k = cols;
      p.x.most_k = widest;
      p.x.tm = (uint32_t)tam_div_up(rows, both.tile);
      p.x.tn = across;
      // a last piece of few words has fewer 64s to cut than parts: the others are empty sums
      p.x.parts = both.x_parts;
      p.x.rows = rows;
      p.x.cols = inputs;
      p.x.sums = dx_sums;
      p.x.out = d->dx;
      p.x.index = r.index;
      p.x.add = first != 0;
      const uint64_t x_units = (uint64_t)p.x.tm * across * both.x_parts;
      if (units && (uint64_t)cols * both.w_parts > (uint64_t)rows * both.x_parts) p.w_first = (uint32_t)x_units;
      units += x_units;
    }
#define TAM_PRODUCTS(T) launch_products<T>(both.tile, p, (uint32_t)units, c.stream)
    TAM_OF_TYPE(c, TAM_PRODUCTS);
    TAM_OP_LAUNCHED("dx and dw");
    if (dw_sums) {
      const dim3 grid((uint32_t)tam_div_up(cols * eights, 256)), block(256);
#define TAM_DW_OUT(T)                                                                                                     \
  hipLaunchKernelGGL(tam_k_cross_out<T>, grid, block, 0, c.stream, dw_sums, both.w_parts, (uint64_t)cols, inputs, nullptr, \
                     nullptr, 0u, 0ull, scale, (T*)p.w.out)
      TAM_OF_TYPE(c, TAM_DW_OUT);
      TAM_OP_LAUNCHED("dw's sum");
    }
  }
  if (direct) {
    const uint32_t halves = inputs * (size / 2);
    const dim3 grid(rows < 16384 ? rows : 16384), block(256);
    hipLaunchKernelGGL(tam_k_cross_clear, grid, block, 0, c.stream, (tam_f16*)d->dx, (uint64_t)rows, halves, r.place);
    TAM_OP_LAUNCHED("rows without a gradient");
  } else if (d->dx) {
    const dim3 grid((uint32_t)joins_x), block(256);
#define TAM_DX_OUT(T)                                                                                                        \
  hipLaunchKernelGGL(tam_k_cross_out<T>, grid, block, 0, c.stream, dx_sums, both.x_parts, (uint64_t)rows, inputs, r.place, \
                     r.count, (uint32_t)both.tile, widest, scale, (T*)d->dx)
    TAM_OF_TYPE(c, TAM_DX_OUT);
    TAM_OP_LAUNCHED("dx's sum");
  }
  return TAM_OK;
}

int cross(const TamCross* d, bool back, void* workspace, uint64_t ws_bytes, void* stream, uint64_t* need,
          uint32_t* tiles = nullptr) {
  int rc = check_cross(d, back);
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

size_t tam_cross_kept(const TamCross* d) { return d && d->dtype <= TAM_DTYPE_F16 ? (size_t)kept_bytes(d) : 0; }

int tam_cross_reads_x(const TamCross* d) { return d && few(d); }

int tam_cross_workspace(const TamCross* d, int backward_pass, size_t* bytes) {
  if (!bytes) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  uint64_t need = 0;
  const int rc = cross(d, backward_pass != 0, nullptr, 0, nullptr, &need);
  *bytes = (size_t)need;
  return rc;
}

int tam_cross_tiles(const TamCross* d, int backward_pass, uint32_t* tiles) {
  if (!tiles) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  for (int i = 0; i < 4; ++i) tiles[i] = 0;
  uint64_t need = 0;
  return cross(d, backward_pass != 0, nullptr, 0, nullptr, &need, tiles);
}

int tam_cross(const TamCross* d, void* workspace, size_t ws_bytes, void* stream) {
  return cross(d, false, workspace, ws_bytes, stream, nullptr);
}

int tam_cross_backward(const TamCross* d, void* workspace, size_t ws_bytes, void* stream) {
  return cross(d, true, workspace, ws_bytes, stream, nullptr);
}

}  // extern "C"
