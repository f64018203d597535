// tam_ops.h -- what the operators' sources (tam_norm.hip, tam_linear.hip,
// tam_muon.hip) share: error reporting, element types and launch helpers.
#ifndef TAM_OPS_H
#define TAM_OPS_H

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/turboadam_amd.h"

// The thread's message lies in tam_step.hip, which hands it out as
// tam_last_error(): 512 bytes, written here by every failing call too.
#define TAM_ERR_BYTES 512

__attribute__((format(printf, 2, 3))) static inline int tam_op_fail(int code, const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vsnprintf(const_cast<char*>(tam_last_error()), TAM_ERR_BYTES, fmt, args);
  va_end(args);
  return code;
}

static inline void tam_op_begin() { const_cast<char*>(tam_last_error())[0] = 0; }

#define TAM_OP_LAUNCHED(what)                                                                       \
  do {                                                                                              \
    const hipError_t e_ = hipGetLastError();                                                        \
    if (e_ != hipSuccess) return tam_op_fail(TAM_E_HIP, "HIP error at %s: code %d", what, (int)e_); \
  } while (0)

static inline uint64_t tam_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }
static inline uint64_t tam_div_up(uint64_t x, uint64_t by) { return (x + by - 1) / by; }

// Compute units of the current device; 256 (an MI355X) where it cannot be asked.
static inline uint32_t tam_op_cus() {
  static const uint32_t cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      return 256u;
    return n > 0 ? (uint32_t)n : 256u;
  }();
  return cus;
}

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------
typedef __bf16 tam_bf16;
typedef _Float16 tam_f16;
typedef float tam_f4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ float tam_to_f(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T tam_from_f(float x) {
  return (T)x;  // round to nearest even
}

// 8 consecutive elements at p to fp32 and back, 16 (32 for fp32) bytes at once.
// They may lie at any element's address: gfx950 moves 16 bytes at any address,
// and the alignment claimed to the compiler is the element's own.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) tam_oct {
  T v __attribute__((ext_vector_type(8)));
};

template <typename T>
__device__ __forceinline__ void tam_load8(const T* p, float (&x)[8]) {
  const tam_oct<T> o = *reinterpret_cast<const tam_oct<T>*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)o.v[i];
}
template <typename T>
__device__ __forceinline__ void tam_store8(T* p, const float (&x)[8]) {
  tam_oct<T> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o.v[i] = (T)x[i];
  *reinterpret_cast<tam_oct<T>*>(p) = o;
}

// The first `count` of 8 elements at p (all of them from 8 on), zeros behind: the
// loads of a short count do not wait for each other.
template <typename T>
__device__ __forceinline__ tam_oct<T> tam_some(const T* p, uint32_t count) {
  tam_oct<T> o;
  if (count >= 8) {
    o = *reinterpret_cast<const tam_oct<T>*>(p);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) o.v[j] = (T)0.f;
    if (count)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) o.v[j] = p[j < count ? j : 0];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      if (j >= count) o.v[j] = (T)0.f;
  }
  return o;
}
template <typename T>
__device__ __forceinline__ void tam_load_some(const T* p, uint32_t count, float (&x)[8]) {
  const tam_oct<T> o = tam_some(p, count);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)o.v[i];
}
template <typename T>
__device__ __forceinline__ void tam_store_some(T* p, uint32_t count, const float (&x)[8]) {
  if (count >= 8) {
    tam_store8(p, x);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      if (j < count) p[j] = (T)x[j];
  }
}

// Sum over the wave's 64 lanes; every lane gets the same bits.
template <int CTRL>
__device__ __forceinline__ float tam_dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float tam_wave_sum(float x) {
  x = tam_dpp_add<0xb1>(x);   // quad_perm [1, 0, 3, 2]
  x = tam_dpp_add<0x4e>(x);   // quad_perm [2, 3, 0, 1]
  x = tam_dpp_add<0x141>(x);  // row_half_mirror
  x = tam_dpp_add<0x140>(x);  // row_mirror
  const uint32_t i = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
  const uint32_t j = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(j, j, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
}

#endif  // TAM_OPS_H
