// tam_rotary.hip -- rotary positions of the C ABI: each head's norm (optional) and the
// rotation of its pairs by position * frequency, and the gradients.
//
//   n = x rstd w,  rstd = 1 / sqrt(mean(x^2) + eps)          (without a weight: n = x)
//   (a, b) of n -> m (a cos - b sin, a sin + b cos), angle = position * frequency
//   backward: t = m (da cos + db sin, db cos - da sin),  dw = sum over heads' rows of
//   t x rstd,  dx = rstd (t w - x rstd^2 mean(t w x))
//
// Units.  A head's row is cut into units of 8 pairs: UR units of the rotated part (the
// last one may be short), then units of the rest of the row, which go past the rotation: with
// an angle of 0 an infinity or a NaN would reach the element that it is paired with.  L lanes,
// the next power of two, take a row, a unit each: two vectors of 8 elements, both halves
// of its pairs.  So a pair lies in one lane, whichever way pairs are laid out, and only
// the norm's sums cross lanes.  A wave takes 64 / L rows of a token at once (or several
// tokens, where they have fewer rows): a lane makes its 8 angles once a token, for all
// query and key heads.  They cost it about 300 instructions; with a row each they would
// take as long as the row's way to memory and back.
//
// Angles are 64-bit products in turns, of which the whole ones are dropped before the sine
// and cosine are taken in fp32: position 10^6 is as exact as position 1.
#include "tam_ops.h"

#include <float.h>
#include <math.h>

namespace {

struct heads_args {
  const char* x;  // or, in a backward pass without a norm, what is turned back
  const char* w;  // or null: no norm
  const char* dy;
  char* y;        // forward: the result; backward: dx
  int64_t x_b, x_t, dy_b, dy_t, y_b, y_t;  // bytes
  uint32_t x_h, dy_h, y_h;                 // bytes
  uint32_t heads, turns;                   // rows; of a wave, at a time
};

struct rotary_args {
  heads_args part[2];  // queries, keys
  const char* positions;
  const double* frequencies;
  float* sums;         // [workgroups][2][lanes * 16] or null
  int64_t pos_b, pos_t;  // bytes
  uint32_t tokens, batches;
  uint32_t dim, rotated, units, lanes;
  uint32_t at_once;    // tokens of a wave
  uint32_t bundles;    // of at_once tokens, in a batch
  uint32_t split;      // waves that share a bundle's rows
  uint32_t pos64;
  float eps, scale;    // scale: of the rotated part
  float sign;          // of the angles' sines: -1 turns back
};

// The elements of a lane's unit: two runs of up to 8.
struct unit {
  uint32_t e0, e1, n0, n1;
};

__device__ __forceinline__ uint32_t some_of(uint32_t from, uint32_t to) {
  return from >= to ? 0u : (to - from < 8u ? to - from : 8u);
}

template <bool SIDE>
__device__ __forceinline__ unit unit_at(uint32_t u, uint32_t dim, uint32_t rotated, uint32_t& rest) {
  const uint32_t half = rotated / 2, ur = (half + 7) / 8;
  unit r;
  rest = u >= ur;
  if (rest) {
    r.e0 = rotated + (u - ur) * 16;
    r.e1 = r.e0 + 8;
    r.n0 = some_of(r.e0, dim);
    r.n1 = some_of(r.e1, dim);
  } else if (SIDE) {
    r.e0 = u * 16;
    r.e1 = r.e0 + 8;
    r.n0 = some_of(r.e0, rotated);
    r.n1 = some_of(r.e1, rotated);
  } else {
    r.e0 = u * 8;
    r.e1 = half + r.e0;
    r.n0 = r.n1 = some_of(r.e0, half);
  }
  return r;
}

template <typename T>
struct two {
  tam_oct<T> lo, hi;
};

// The unit's elements of the row that lies `row` bytes behind a base that all lanes share: 32-bit
// offsets of a lane, whose sums cost one instruction.
template <typename T>
__device__ __forceinline__ two<T> fetch(const char* base, uint32_t row, const unit& u) {
  return {tam_some(reinterpret_cast<const T*>(base + (row + u.e0 * (uint32_t)sizeof(T))), u.n0),
          tam_some(reinterpret_cast<const T*>(base + (row + u.e1 * (uint32_t)sizeof(T))), u.n1)};
}

// The unit's pairs: of a[p] and b[p], whichever way they lie.
template <typename T, bool SIDE>
__device__ __forceinline__ void pairs(const two<T>& v, float (&a)[8], float (&b)[8]) {
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    if constexpr (SIDE) {
      a[p] = p < 4 ? (float)v.lo.v[2 * p] : (float)v.hi.v[2 * p - 8];
      b[p] = p < 4 ? (float)v.lo.v[2 * p + 1] : (float)v.hi.v[2 * p - 7];
    } else {
      a[p] = (float)v.lo.v[p];
      b[p] = (float)v.hi.v[p];
    }
  }
}

template <typename T, bool SIDE>
__device__ __forceinline__ void store(char* base, uint32_t row, const unit& u, const float (&a)[8], const float (&b)[8]) {
  float lo[8], hi[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    if constexpr (SIDE) {
      (p < 4 ? lo[2 * p & 7] : hi[2 * p & 7]) = a[p];
      (p < 4 ? lo[(2 * p + 1) & 7] : hi[(2 * p + 1) & 7]) = b[p];
    } else {
      lo[p] = a[p];
      hi[p] = b[p];
    }
  }
  tam_store_some(reinterpret_cast<T*>(base + (row + u.e0 * (uint32_t)sizeof(T))), u.n0, lo);
  tam_store_some(reinterpret_cast<T*>(base + (row + u.e1 * (uint32_t)sizeof(T))), u.n1, hi);
}

// Sum over a row's lanes (a power of two of them); all get the same bits.
__device__ __forceinline__ float lanes_sum(float x, uint32_t lanes) {
  if (lanes > 1) x = tam_dpp_add<0xb1>(x);   // quad_perm [1, 0, 3, 2]
  if (lanes > 2) x = tam_dpp_add<0x4e>(x);   // quad_perm [2, 3, 0, 1]
  if (lanes > 4) x = tam_dpp_add<0x141>(x);  // row_half_mirror
  if (lanes > 8) x = tam_dpp_add<0x140>(x);  // row_mirror
  if (lanes > 16) {
    const uint32_t i = __builtin_bit_cast(uint32_t, x);
    const auto s = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    const uint32_t s0 = s[0], s1 = s[1];
    x = __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
  }
  if (lanes > 32) {
    const uint32_t i = __builtin_bit_cast(uint32_t, x);
    const auto s = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    const uint32_t s0 = s[0], s1 = s[1];
    x = __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
  }
  return x;
}

// sin and cos of a number of turns: the quarter's number and what is left of it, both taken in 64
// bits; Taylor's sums on [-pi/4, pi/4], off by 2^-25 (the first terms left out: y^11 / 11!, y^10 / 10!).
__device__ __forceinline__ void sin_cos_turns(double turns, float& s, float& c) {
  turns -= rint(turns);
  const double quarters = rint(4.0 * turns);
  const float y = (float)__builtin_fma(4.0, turns, -quarters) * 1.57079632679489662f, z = y * y;
  const int q = (int)quarters;
  float a = __builtin_fmaf(z, 2.75573192239858925e-6f, -1.98412698412698413e-4f);
  a = __builtin_fmaf(z, a, 8.33333333333333322e-3f);
  a = __builtin_fmaf(z, a, -1.66666666666666657e-1f);
  a = __builtin_fmaf(y * z, a, y);
  float b = __builtin_fmaf(z, 2.48015873015873016e-5f, -1.38888888888888894e-3f);
  b = __builtin_fmaf(z, b, 4.16666666666666644e-2f);
  b = __builtin_fmaf(z, b, -0.5f);
  b = __builtin_fmaf(z, b, 1.0f);
  const float u = q & 1 ? b : a, v = q & 1 ? a : b;
  s = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, u) ^ ((uint32_t)q & 2u) << 30);
  c = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) ^ ((uint32_t)(q + 1) & 2u) << 30);
}

// 1 / sqrt of a norm: of 16-bit results by the hardware's root, 2^-22.
template <typename T>
__device__ __forceinline__ float inverse_root(float x) {
  if constexpr (sizeof(T) == 2)
    return __builtin_amdgcn_rsqf(x);
  else
    return 1.0f / sqrtf(x);
}

// A wave takes a bundle's rows in turns, queries' first; a turn's rows are all of one part, and their
// addresses a base that the lanes share and an offset that a lane keeps. Bound by memory and,
// nearly as much, by the vector unit: 16384 tokens of 32 + 8 heads of 128 bf16 with norms 74 us forward
// (4.6 TB/s), 113 backward (4.5). One token: 4.6, a launch and three trips to memory one after another
// (position, heads, results). 8192 tokens of 24 heads of 64 fp32, pairs side by side: 28 (3.6; not at a
// limit).
// NORM: both parts have a weight, or none. BACK: dx and the weights' sums of a norm's backward pass (without
// a norm it is the forward pass with the angles' sign turned).
template <typename T, bool SIDE, bool NORM, bool BACK>
__global__ __launch_bounds__(256, BACK ? 3 : (sizeof(T) == 2 ? 5 : 4)) void tam_k_rotary(rotary_args a) {
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t u = lane & (a.lanes - 1), group = lane / a.lanes, groups = 64 / a.lanes;
  uint32_t rest;
  unit at = unit_at<SIDE>(u, a.dim, a.rotated, rest);
  if (u >= a.units) at.n0 = at.n1 = 0;
  const uint32_t rows = a.at_once > 1 ? groups / a.at_once : groups;  // of a turn and token
  const uint32_t in = group / rows, first = group - in * rows;
  const float inv = 1.0f / (float)a.dim;
  const uint32_t turns = a.part[0].turns + a.part[1].turns, items = a.bundles * a.batches * a.split;
  float dw[2][16] = {};
  for (uint32_t item = blockIdx.x * 4 + wave; item < items; item += gridDim.x * 4) {
    const uint32_t bundle = __builtin_amdgcn_readfirstlane(item / a.split);
    const uint32_t batch = __builtin_amdgcn_readfirstlane(bundle / a.bundles), t0 = (bundle - batch * a.bundles) * a.at_once;
    const bool mine = in < a.at_once && t0 + in < a.tokens;
    const uint32_t t = mine ? in : 0;  // behind t0
    const char* const where = a.positions + batch * a.pos_b + t0 * a.pos_t + (uint64_t)t * a.pos_t;
    const double position = a.pos64 ? (double)*reinterpret_cast<const int64_t*>(where) : (double)*reinterpret_cast<const int32_t*>(where);
    float c[8], s[8];
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p) {
      // in turns; the frequencies stay in the caches (in registers they would be 16 of them)
      const bool turn = !rest && u * 8 + p < a.rotated / 2;
      sin_cos_turns(position * (turn ? a.frequencies[u * 8 + p] * 0.15915494309189535 : 0.0), s[p], c[p]);
      s[p] *= a.sign * a.scale;
      c[p] *= a.scale;
    }
#pragma unroll 1
    for (uint32_t turn = item - bundle * a.split; turn < turns; turn += a.split) {
      const bool key = turn >= a.part[0].turns;
      uint32_t which = __builtin_amdgcn_readfirstlane((uint32_t)key);
      asm("" : "+s"(which));  // a part's arguments are read where they are used: both in registers were too many
      const heads_args& h = a.part[which];
      const uint32_t row0 = (key ? turn - a.part[0].turns : turn) * rows;
      unit e = at;
      const bool here = mine && row0 + first < h.heads;
      if (!here) e.n0 = e.n1 = 0;
      const uint32_t row = e.n0 | e.n1 ? first : 0;
      auto from = [&](const char* base, int64_t b, int64_t of_t, uint32_t of_h) {
        return base + (batch * b + t0 * of_t + (int64_t)row0 * of_h);
      };
      two<T> xv, dv, wv;
      xv = fetch<T>(from(h.x, h.x_b, h.x_t, h.x_h), t * (uint32_t)h.x_t + row * h.x_h, e);
      if (BACK) dv = fetch<T>(from(h.dy, h.dy_b, h.dy_t, h.dy_h), t * (uint32_t)h.dy_t + row * h.dy_h, e);
      if (NORM) wv = fetch<T>(h.w, 0, at);
      char* const y = const_cast<char*>(from(h.y, h.y_b, h.y_t, h.y_h));
      const uint32_t to = t * (uint32_t)h.y_t + row * h.y_h;
      float x0[8], x1[8], d0[8], d1[8], w0[8], w1[8];
      if (NORM) pairs<T, SIDE>(wv, w0, w1);
      pairs<T, SIDE>(xv, x0, x1);
      if (BACK) {
        pairs<T, SIDE>(dv, d0, d1);
        if (!rest)
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float da = d0[p];
            d0[p] = __builtin_fmaf(da, c[p], -d1[p] * s[p]);
            d1[p] = __builtin_fmaf(da, s[p], d1[p] * c[p]);
          }
        {
          float sx = 0.f, sg = 0.f;
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            w0[p] *= d0[p];
            w1[p] *= d1[p];
            sx = __builtin_fmaf(x0[p], x0[p], __builtin_fmaf(x1[p], x1[p], sx));
            sg = __builtin_fmaf(w0[p], x0[p], __builtin_fmaf(w1[p], x1[p], sg));
          }
          sx = lanes_sum(sx, a.lanes);
          sg = lanes_sum(sg, a.lanes);
          // lanes without a row have sums of zeros, whose root may be infinite: they add nothing to dw
          const float rstd = here ? inverse_root<T>(__builtin_fmaf(sx, inv, a.eps)) : 0.0f, mean = -sg * inv * rstd * rstd * rstd;
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            d0[p] *= rstd;
            d1[p] *= rstd;
          }
          if (key)
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              dw[1][p] = __builtin_fmaf(d0[p], x0[p], dw[1][p]);
              dw[1][8 + p] = __builtin_fmaf(d1[p], x1[p], dw[1][8 + p]);
            }
          else
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              dw[0][p] = __builtin_fmaf(d0[p], x0[p], dw[0][p]);
              dw[0][8 + p] = __builtin_fmaf(d1[p], x1[p], dw[0][8 + p]);
            }
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            d0[p] = __builtin_fmaf(x0[p], mean, w0[p] * rstd);
            d1[p] = __builtin_fmaf(x1[p], mean, w1[p] * rstd);
          }
        }
        store<T, SIDE>(y, to, e, d0, d1);
      } else {
        if (NORM) {
          float sx = 0.f;
#pragma unroll
          for (int p = 0; p < 8; ++p) sx = __builtin_fmaf(x0[p], x0[p], __builtin_fmaf(x1[p], x1[p], sx));
          sx = lanes_sum(sx, a.lanes);
          const float rstd = inverse_root<T>(__builtin_fmaf(sx, inv, a.eps));
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            x0[p] *= rstd * w0[p];
            x1[p] *= rstd * w1[p];
          }
        }
        if (!rest)
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float xa = x0[p];
            x0[p] = __builtin_fmaf(xa, c[p], -x1[p] * s[p]);
            x1[p] = __builtin_fmaf(xa, s[p], x1[p] * c[p]);
          }
        store<T, SIDE>(y, to, e, x0, x1);
      }
    }
  }
  if constexpr (BACK) {
    if (!a.sums) return;
    // the workgroup's sums: over its waves' rows, in the lanes' order
    __shared__ float turn[4 * 64 * 17];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      __syncthreads();
#pragma unroll
      for (int p = 0; p < 16; ++p) turn[threadIdx.x * 17 + p] = dw[part][p];
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < a.lanes * 16; i += 256) {
        float sum = 0.f;
        for (uint32_t g = 0; g < 4 * groups; ++g) sum += turn[(g * a.lanes + i / 16) * 17 + i % 16];
        a.sums[((uint64_t)blockIdx.x * 2 + part) * a.lanes * 16 + i] = sum;
      }
    }
  }
}

// dw[e] = the workgroups' sums of the slot of element e, in their order: 16 elements to a
// workgroup, 64 threads to an element. 768 workgroups' sums of 128 elements, twice: 4.7 us, of it 2 the launch.
template <typename T, bool SIDE>
__global__ __launch_bounds__(1024) void tam_k_rotary_weight(const float* sums, uint32_t runs, uint32_t dim, uint32_t rotated,
                                                            uint32_t lanes, T* dq, T* dk) {
  __shared__ float part[64][16];
  const uint32_t e = blockIdx.x * 16 + (threadIdx.x & 15), run0 = threadIdx.x >> 4, which = blockIdx.y;
  T* out = which ? dk : dq;
  if (!out) return;
  float s = 0.f;
  if (e < dim) {
    const uint32_t half = rotated / 2, ur = (half + 7) / 8;
    uint32_t unit, slot;
    if (e >= rotated) {
      unit = ur + (e - rotated) / 16;
      slot = (e - rotated) % 16;
    } else if (SIDE) {
      unit = e / 16;
      slot = e % 16;
    } else {
      unit = (e < half ? e : e - half) / 8;
      slot = (e < half ? e : e - half) % 8 + (e < half ? 0 : 8);
    }
    // slots are pairs' a and b; elements side by side alternate between them
    if (SIDE) slot = slot / 2 + (slot % 2) * 8;
    const float* at = sums + (uint64_t)which * lanes * 16 + unit * 16 + slot;
#pragma unroll 8
    for (uint32_t r = run0; r < runs; r += 64) s += at[(uint64_t)r * 2 * lanes * 16];
  }
  part[run0][threadIdx.x & 15] = s;
  __syncthreads();
  if (run0 == 0 && e < dim) {
    float v = 0.f;
    for (int r = 0; r < 64; ++r) v += part[r][threadIdx.x & 15];
    out[e] = tam_from_f<T>(v);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr uint32_t kMostDim = 1024;  // a lane takes 16 elements of a head
constexpr uint32_t kMostGroups = 768;  // whose sums tam_k_rotary_weight adds

uint32_t power_of_two(uint32_t n) {
  uint32_t p = 1;
  while (p < n) p *= 2;
  return p;
}

uint32_t units_of(const TamRotary* d) {
  return (uint32_t)(tam_div_up(d->rotated / 2, 8) + tam_div_up(d->dim - d->rotated, 16));
}

int check_rotary(const TamRotary* d, bool back) {
  tam_op_begin();
  if (!d) return tam_op_fail(TAM_E_INVALID, "null argument");
  if (d->dtype > TAM_DTYPE_F16) return tam_op_fail(TAM_E_INVALID, "unknown dtype %u", d->dtype);
  if (d->dim == 0) return tam_op_fail(TAM_E_INVALID, "heads of no elements");
  if (d->rotated % 2 || d->rotated > d->dim)
    return tam_op_fail(TAM_E_INVALID, "a rotated part that is odd or longer than a head");
  if (!(d->eps == 0 || (d->eps >= FLT_MIN && d->eps <= FLT_MAX)))  // the hardware's root takes smaller ones for 0
    return tam_op_fail(TAM_E_INVALID, "an eps that is neither 0 nor one of fp32's normal numbers above it");
  if (d->dim > kMostDim || units_of(d) > 64)
    return tam_op_fail(TAM_E_UNSUPPORTED, "heads of more than %u elements (%u where the rotated part is no multiple of 16)",
                       kMostDim, kMostDim - 16);
  const uint64_t most = 1ull << 31;
  if (d->batch >= most || d->tokens >= most || d->batch * d->tokens >= most || d->q.heads >= most / 2 ||
      d->k.heads >= most / 2)
    return tam_op_fail(TAM_E_UNSUPPORTED, "2^31 tokens or heads or more");
  if (d->batch == 0 || d->tokens == 0 || d->q.heads + d->k.heads == 0) return TAM_OK;
  if (!d->positions || (d->rotated && !d->frequencies)) return tam_op_fail(TAM_E_INVALID, "null positions or frequencies");
  for (const TamHeads* h : {&d->q, &d->k}) {
    if (!h->heads) continue;
    if (!h->y || (!back && !h->x) || (back && (!h->dy || (h->w && !h->x))))
      return tam_op_fail(TAM_E_INVALID, "null heads");
    const uint64_t size = d->dtype == TAM_DTYPE_F32 ? 4 : 2;
    const uint64_t far = (1ull << 31) / size / (64 / power_of_two(units_of(d)));  // a lane's offsets are 32-bit numbers of bytes
    for (const int64_t stride : {h->x_h, h->y_h, h->dy_h})
      if (stride < 0 || (uint64_t)stride >= far)
        return tam_op_fail(TAM_E_UNSUPPORTED, "heads %lld elements apart", (long long)stride);
    if (back && h->dw && !h->w) return tam_op_fail(TAM_E_INVALID, "a gradient of a weight that is not given");
  }
  return TAM_OK;
}

// Workgroups of a call, and how it is laid out on them.
uint32_t plan(const TamRotary* d, bool back, rotary_args& a) {
  a.dim = (uint32_t)d->dim;
  a.rotated = (uint32_t)d->rotated;
  a.units = units_of(d);
  a.lanes = power_of_two(a.units);
  a.tokens = (uint32_t)d->tokens;
  a.batches = (uint32_t)d->batch;
  const uint32_t groups = 64 / a.lanes;
  const uint64_t most_heads = d->q.heads > d->k.heads ? d->q.heads : d->k.heads;
  // several tokens to a wave, unless they lie too far apart for a lane's 32-bit offsets
  const int64_t size = d->dtype == TAM_DTYPE_F32 ? 4 : 2, far = (1ll << 31) / size / 64;
  bool near = true;
  for (const TamHeads* h : {&d->q, &d->k})
    for (const int64_t stride : {h->x_t, h->y_t, h->dy_t}) near = near && (!h->heads || (stride >= 0 && stride < far));
  a.at_once = 1;
  if (near)
    while (2 * a.at_once * most_heads <= groups && a.at_once < a.tokens) a.at_once *= 2;
  const uint32_t rows = groups / a.at_once;
  a.bundles = (uint32_t)tam_div_up(a.tokens, a.at_once);
  a.part[0].turns = (uint32_t)tam_div_up(d->q.heads, rows);
  a.part[1].turns = (uint32_t)tam_div_up(d->k.heads, rows);
  const uint64_t bundles = (uint64_t)a.bundles * a.batches, turns = a.part[0].turns + a.part[1].turns;
  // few tokens: their heads go to waves of their own, until 16 waves are on every compute unit
  const uint64_t room = 16ull * tam_op_cus();
  a.split = (uint32_t)(bundles >= room ? 1 : (room / bundles < turns ? room / bundles : turns));
  const uint64_t wgs = tam_div_up(bundles * a.split, 4), most = back ? kMostGroups : 8ull * tam_op_cus();
  return (uint32_t)(wgs < most ? wgs : most);
}

template <typename T, bool SIDE>
int run_typed(const TamRotary* d, bool back, const rotary_args& a, uint32_t wgs, bool norm, hipStream_t s) {
  const dim3 grid(wgs), block(256);
  if (back && norm) {
    hipLaunchKernelGGL((tam_k_rotary<T, SIDE, true, true>), grid, block, 0, s, a);
    TAM_OP_LAUNCHED("the heads' gradient");
    if (a.sums) {
      const dim3 across((uint32_t)tam_div_up(a.dim, 16), 2);
      hipLaunchKernelGGL((tam_k_rotary_weight<T, SIDE>), across, dim3(1024), 0, s, a.sums, wgs, a.dim, a.rotated, a.lanes,
                         (T*)d->q.dw, (T*)d->k.dw);
      TAM_OP_LAUNCHED("the weights' gradients");
    }
  } else if (norm) {
    hipLaunchKernelGGL((tam_k_rotary<T, SIDE, true, false>), grid, block, 0, s, a);
    TAM_OP_LAUNCHED("the heads");
  } else {
    hipLaunchKernelGGL((tam_k_rotary<T, SIDE, false, false>), grid, block, 0, s, a);
    TAM_OP_LAUNCHED("the heads");
  }
  return TAM_OK;
}

template <typename T>
__global__ __launch_bounds__(256) void tam_k_rotary_zero(T* out, uint32_t n) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) out[i] = (T)0.0f;
}

int launch(const TamRotary* d, bool back, void* workspace, hipStream_t s);

bool normed(const TamHeads& h) { return h.heads && h.w; }

// One part of a call of which the other has no norm, or has one alone.
TamRotary part_of(const TamRotary* d, bool keys) {
  TamRotary one = *d;
  TamHeads& other = keys ? one.q : one.k;
  other = TamHeads{};
  return one;
}

int rotary(const TamRotary* d, bool back, void* workspace, uint64_t ws_bytes, void* stream, uint64_t* need) {
  int rc = check_rotary(d, back);
  if (rc != TAM_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  const bool empty = d->batch == 0 || d->tokens == 0 || d->q.heads + d->k.heads == 0;
  const bool apart = d->q.heads && d->k.heads && normed(d->q) != normed(d->k);
  uint64_t used = 0;
  if (!empty && back && ((normed(d->q) && d->q.dw) || (normed(d->k) && d->k.dw))) {
    rotary_args a = {};
    const TamRotary one = part_of(d, normed(d->k));
    const uint32_t wgs = plan(apart ? &one : d, back, a);
    used = (uint64_t)wgs * 2 * a.lanes * 16 * 4;
  }
  if (need) {
    *need = used;
    return TAM_OK;
  }
  if (used > ws_bytes || (used && !workspace))
    return tam_op_fail(TAM_E_WORKSPACE, "workspace of %llu bytes, %llu needed", (unsigned long long)ws_bytes,
                       (unsigned long long)used);
  if ((uintptr_t)workspace & 255u) return tam_op_fail(TAM_E_INVALID, "workspace not on 256 bytes");
  if (back)  // weights that no head uses
    for (const TamHeads* h : {&d->q, &d->k})
      if (h->dw && (empty || !h->heads)) {
        const dim3 grid((uint32_t)tam_div_up(d->dim, 256)), block(256);
        if (d->dtype == TAM_DTYPE_F32)
          hipLaunchKernelGGL(tam_k_rotary_zero<float>, grid, block, 0, s, (float*)h->dw, (uint32_t)d->dim);
        else  // zero has the same 16 bits in both types
          hipLaunchKernelGGL(tam_k_rotary_zero<tam_f16>, grid, block, 0, s, (tam_f16*)h->dw, (uint32_t)d->dim);
        TAM_OP_LAUNCHED("the weights' gradients");
      }
  if (empty) return TAM_OK;
  if (!apart) return launch(d, back, workspace, s);
  for (const bool keys : {false, true}) {
    const TamRotary one = part_of(d, keys);
    rc = launch(&one, back, workspace, s);
    if (rc != TAM_OK) return rc;
  }
  return TAM_OK;
}

int launch(const TamRotary* d, bool back, void* workspace, hipStream_t s) {
  rotary_args a = {};
  const uint32_t wgs = plan(d, back, a);
  const bool norm = normed(d->q) || normed(d->k), sums = back && norm && (d->q.dw || d->k.dw);
  const bool turned = back && !norm;  // the forward pass of dy with the angles' sign turned
  const int64_t size = d->dtype == TAM_DTYPE_F32 ? 4 : 2;
  int i = 0;
  for (const TamHeads* h : {&d->q, &d->k}) {
    heads_args& p = a.part[i++];
    p.x = (const char*)(turned ? h->dy : h->x);
    p.w = (const char*)h->w;
    p.dy = (const char*)h->dy;
    p.y = (char*)h->y;
    p.x_b = (turned ? h->dy_b : h->x_b) * size;
    p.x_t = (turned ? h->dy_t : h->x_t) * size;
    p.x_h = (uint32_t)((turned ? h->dy_h : h->x_h) * size);
    p.dy_b = h->dy_b * size;
    p.dy_t = h->dy_t * size;
    p.dy_h = (uint32_t)(h->dy_h * size);
    p.y_b = h->y_b * size;
    p.y_t = h->y_t * size;
    p.y_h = (uint32_t)(h->y_h * size);
    p.heads = (uint32_t)h->heads;
  }
  a.positions = (const char*)d->positions;
  a.frequencies = d->frequencies;
  a.pos_b = d->pos_b * (d->positions64 ? 8 : 4);
  a.pos_t = d->pos_t * (d->positions64 ? 8 : 4);
  a.pos64 = d->positions64;
  a.eps = d->eps;
  a.scale = d->magnitude;
  a.sign = back ? -1.0f : 1.0f;
  a.sums = sums ? (float*)workspace : nullptr;
#define TAM_ROTARY(T) (d->interleaved ? run_typed<T, true>(d, back, a, wgs, norm, s) : run_typed<T, false>(d, back, a, wgs, norm, s))
  if (d->dtype == TAM_DTYPE_F32) return TAM_ROTARY(float);
  if (d->dtype == TAM_DTYPE_BF16) return TAM_ROTARY(tam_bf16);
  return TAM_ROTARY(tam_f16);
}

}  // namespace

extern "C" {

int tam_rotary_workspace(const TamRotary* d, int backward_pass, size_t* bytes) {
  if (!bytes) {
    tam_op_begin();
    return tam_op_fail(TAM_E_INVALID, "null argument");
  }
  uint64_t need = 0;
  const int rc = rotary(d, backward_pass != 0, nullptr, 0, nullptr, &need);
  *bytes = (size_t)need;
  return rc;
}

int tam_rotary(const TamRotary* d, void* stream) { return rotary(d, false, nullptr, 0, stream, nullptr); }

int tam_rotary_backward(const TamRotary* d, void* workspace, size_t ws_bytes, void* stream) {
  return rotary(d, true, workspace, ws_bytes, stream, nullptr);
}

}  // extern "C"
