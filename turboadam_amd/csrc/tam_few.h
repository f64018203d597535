// tam_few.h -- what the products of few rows share: a fragment straight from memory.
#ifndef TAM_FEW_H
#define TAM_FEW_H

#include "tam_gemm.h"

#define TAM_FEW_WAVES 8

// Chunk k .. of a row; GUARD: elements from K on are zeros and not read.
template <typename T, bool GUARD>
__device__ __forceinline__ void tam_few_load(tam_frag<T>& f, const T* row, uint64_t k, uint64_t K) {
  constexpr int N = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
  struct __attribute__((packed, aligned(sizeof(T)))) any {
    vec v;
  };
  if (!GUARD || k + N <= K) {
    f.v = __builtin_bit_cast(decltype(f.v), reinterpret_cast<const any*>(row + k)->v);
  } else {
    vec v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = k + j < K ? row[k + j] : (T)0.0f;
    f.v = __builtin_bit_cast(decltype(f.v), v);
  }
}

#endif  // TAM_FEW_H
