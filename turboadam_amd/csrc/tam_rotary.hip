// tam_rotary.hip -- rotary positions of the C ABI: each head's norm (optional) and the
// rotation of its pairs by position * frequency, and the gradients.
//
//   n = x rstd w,  rstd = 1 / sqrt(mean(x^2) + eps)          (without a weight: n = x)
//   (a, b) of n -> m (a cos - b sin, a sin + b cos), angle = position * frequency
//   backward: t = m (da cos + db sin, db cos - da sin),  dw = sum over heads' rows of
//   t x rstd,  dx = rstd (t w - x rstd^2 mean(t w x))
//
// Units.  A head's row is cut into units of 8 pairs: UR units of the rotated part (the
// last one may be short), then units of the rest of the row, whose angle is 0.  L lanes,
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

#include <math.h>

namespace {

struct heads_args {
  const void* x;      // or, in a backward pass without a norm, null
  const void* w;      // or null: no norm
  const void* dy;
  void* y;            // forward: the result; backward: dx
  int64_t x_b, x_t, x_h, dy_b, dy_t, dy_h, y_b, y_t, y_h;  // elements
};

struct rotary_args {
  heads_args part[2];  // queries, keys
  const void* positions;
  const double* frequencies;
  float* sums;         // [workgroups][2][L * 16] or null
  int64_t pos_b, pos_t;
  uint32_t tokens;     // of a batch
  uint32_t all;        // tokens of all batches
  uint32_t heads_q, heads;
  uint32_t dim, rotated, units, lanes;
  uint32_t at_once;    // tokens of a wave
  uint32_t split;      // waves that share a token's rows
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

template <typename T>
__device__ __forceinline__ two<T> fetch(const T* row, const unit& u) {
  return {tam_some(row + u.e0, u.n0), tam_some(row + u.e1, u.n1)};
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
__device__ __forceinline__ void store(T* row, const unit& u, const float (&a)[8], const float (&b)[8]) {
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
  tam_store_some(row + u.e0, u.n0, lo);
  tam_store_some(row + u.e1, u.n1, hi);
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

// NORM: of the heads whose part has a weight. BACK: dx and the weights' sums of a norm's
// backward pass (without a norm it is the forward pass with the angles' sign turned).
template <typename T, bool SIDE, bool NORM, bool BACK>
__global__ __launch_bounds__(256) void tam_k_rotary(rotary_args a) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t u = lane & (a.lanes - 1), group = lane / a.lanes, groups = 64 / a.lanes;
  uint32_t rest;
  unit at = unit_at<SIDE>(u, a.dim, a.rotated, rest);
  if (u >= a.units) at.n0 = at.n1 = 0;
  double turns[8];  // of a position step
#pragma unroll
  for (uint32_t p = 0; p < 8; ++p)
    turns[p] = !rest && u * 8 + p < a.rotated / 2 ? a.frequencies[u * 8 + p] * 0.15915494309189535 : 0.0;
  const uint32_t in = a.at_once > 1 ? group / a.heads : 0, first = a.at_once > 1 ? group - in * a.heads : group;
  const uint32_t step = groups * a.split;
  const uint32_t bundles = (a.all + a.at_once - 1) / a.at_once;
  const float inv = 1.0f / (float)a.dim;
  float dw[2][16] = {};
  for (uint64_t item = (uint64_t)blockIdx.x * 4 + wave; item < (uint64_t)bundles * a.split; item += (uint64_t)gridDim.x * 4) {
    const uint32_t bundle = (uint32_t)(item / a.split), share = (uint32_t)(item - (uint64_t)bundle * a.split);
    const uint32_t token = bundle * a.at_once + in;
    const bool mine = in < a.at_once && token < a.all;
    const uint32_t batch = mine ? token / a.tokens : 0, t = mine ? token - batch * a.tokens : 0;
    const int64_t where = batch * a.pos_b + t * a.pos_t;
    const double position =
        a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[where] : (double)static_cast<const int32_t*>(a.positions)[where];
    float c[8], s[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      double turn = position * turns[p];
      turn -= rint(turn);
      sincospif(2.0f * (float)turn, &s[p], &c[p]);
      s[p] *= a.sign * a.scale;
      c[p] *= rest ? 1.0f : a.scale;
    }
    for (uint32_t row = first + share * groups; row < a.heads; row += step) {
      if (!mine) break;
      const bool key = row >= a.heads_q;
      const uint32_t head = key ? row - a.heads_q : row;
      const heads_args& h = a.part[0];
      const heads_args& k = a.part[1];
      auto base = [&](const void* hp, const void* kp, int64_t hb, int64_t kb, int64_t ht, int64_t kt, int64_t hh, int64_t kh) {
        return (T*)(key ? kp : hp) + (batch * (key ? kb : hb) + t * (key ? kt : ht) + head * (key ? kh : hh));
      };
      float x0[8], x1[8], d0[8], d1[8], w0[8], w1[8];
      const T* w = NORM ? static_cast<const T*>(key ? k.w : h.w) : nullptr;
      two<T> xv, dv, wv;
      if (!BACK || w) xv = fetch(base(h.x, k.x, h.x_b, k.x_b, h.x_t, k.x_t, h.x_h, k.x_h), at);
      if (BACK) dv = fetch(base(h.dy, k.dy, h.dy_b, k.dy_b, h.dy_t, k.dy_t, h.dy_h, k.dy_h), at);
      if (w) wv = fetch(w, at);
      T* y = base(h.y, k.y, h.y_b, k.y_b, h.y_t, k.y_t, h.y_h, k.y_h);
      if (BACK) {
        pairs<T, SIDE>(dv, d0, d1);
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const float da = d0[p];
          d0[p] = __builtin_fmaf(da, c[p], -d1[p] * s[p]);
          d1[p] = __builtin_fmaf(da, s[p], d1[p] * c[p]);
        }
        float sx = 0.f, sg = 0.f;
        if (w) {
          pairs<T, SIDE>(xv, x0, x1);
          pairs<T, SIDE>(wv, w0, w1);
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            sx = __builtin_fmaf(x0[p], x0[p], __builtin_fmaf(x1[p], x1[p], sx));
            sg = __builtin_fmaf(d0[p] * w0[p], x0[p], __builtin_fmaf(d1[p] * w1[p], x1[p], sg));
          }
        }
        // a row's lanes are all here or none, and of one part: its sums cross no other row
        sx = lanes_sum(sx, a.lanes);
        sg = lanes_sum(sg, a.lanes);
        if (w) {
          const float rstd = 1.0f / sqrtf(__builtin_fmaf(sx, inv, a.eps)), mean = sg * inv * rstd * rstd;
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float g0 = d0[p] * x0[p] * rstd, g1 = d1[p] * x1[p] * rstd;
            dw[0][p] += key ? 0.f : g0;
            dw[0][8 + p] += key ? 0.f : g1;
            dw[1][p] += key ? g0 : 0.f;
            dw[1][8 + p] += key ? g1 : 0.f;
            d0[p] = rstd * __builtin_fmaf(-x0[p], mean, d0[p] * w0[p]);
            d1[p] = rstd * __builtin_fmaf(-x1[p], mean, d1[p] * w1[p]);
          }
        }
        store<T, SIDE>(y, at, d0, d1);
      } else {
        pairs<T, SIDE>(xv, x0, x1);
        if (NORM) {
          float sx = 0.f;
#pragma unroll
          for (int p = 0; p < 8; ++p) sx = __builtin_fmaf(x0[p], x0[p], __builtin_fmaf(x1[p], x1[p], sx));
          sx = lanes_sum(sx, a.lanes);
          if (w) {
            pairs<T, SIDE>(wv, w0, w1);
            const float rstd = 1.0f / sqrtf(__builtin_fmaf(sx, inv, a.eps));
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              x0[p] *= rstd * w0[p];
              x1[p] *= rstd * w1[p];
            }
          }
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const float xa = x0[p];
          x0[p] = __builtin_fmaf(xa, c[p], -x1[p] * s[p]);
          x1[p] = __builtin_fmaf(xa, s[p], x1[p] * c[p]);
        }
        store<T, SIDE>(y, at, x0, x1);
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
// workgroup, 64 threads to an element.
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
constexpr uint32_t kMostGroups = 512;  // whose sums tam_k_rotary_weight adds

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
  if (!(d->eps >= 0)) return tam_op_fail(TAM_E_INVALID, "eps below 0");
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
  a.all = (uint32_t)(d->batch * d->tokens);
  a.heads_q = (uint32_t)d->q.heads;
  a.heads = (uint32_t)(d->q.heads + d->k.heads);
  const uint32_t groups = 64 / a.lanes;
  a.at_once = a.heads < groups ? groups / a.heads : 1;
  const uint64_t bundles = tam_div_up(a.all, a.at_once), turns = tam_div_up(a.heads, groups);
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

int rotary(const TamRotary* d, bool back, void* workspace, uint64_t ws_bytes, void* stream, uint64_t* need) {
  const int rc = check_rotary(d, back);
  if (rc != TAM_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  const bool empty = d->batch == 0 || d->tokens == 0 || d->q.heads + d->k.heads == 0;
  rotary_args a = {};
  uint32_t wgs = 0;
  uint64_t used = 0;
  const bool norm = (d->q.w && d->q.heads) || (d->k.w && d->k.heads), sums = back && norm && (d->q.dw || d->k.dw);
  if (!empty) {
    wgs = plan(d, back, a);
    if (sums) used = (uint64_t)wgs * 2 * a.lanes * 16 * 4;
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
  const bool turned = back && !norm;  // the forward pass of dy with the angles' sign turned
  int i = 0;
  for (const TamHeads* h : {&d->q, &d->k}) {
    heads_args& p = a.part[i++];
    p.x = turned ? h->dy : h->x;
    p.w = h->w;
    p.dy = h->dy;
    p.y = h->y;
    p.x_b = turned ? h->dy_b : h->x_b;
    p.x_t = turned ? h->dy_t : h->x_t;
    p.x_h = turned ? h->dy_h : h->x_h;
    p.dy_b = h->dy_b;
    p.dy_t = h->dy_t;
    p.dy_h = h->dy_h;
    p.y_b = h->y_b;
    p.y_t = h->y_t;
    p.y_h = h->y_h;
  }
  a.positions = d->positions;
  a.frequencies = d->frequencies;
  a.pos_b = d->pos_b;
  a.pos_t = d->pos_t;
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
