// tam_gemm.h -- the matrix-product core of the operators: one workgroup's tile
// of D[r][c] = sum_k Q[r][k] * P[c][k] on the matrix cores, for bf16, fp16 and
// fp32 operands that are contiguous along k or along their own index.
//
// Stages.  The k axis is cut into stages of 64 bytes of a row: 32 16-bit or 16
// fp32 elements.  A stage of an operand is (rows * 64) bytes of LDS, written by
// buffer loads that go to LDS directly, 1 KB to a wave and instruction:
//   k-contiguous operand: [row][64 bytes], 16-byte chunk c of row r at place
//     c ^ (r >> 1 & 3): eight consecutive rows' chunks cover all 32 banks, so
//     the 16-byte fragment reads are free of conflicts;
//   operand contiguous along its own index ("m-major"): [k][rows], read with
//     the transposing LDS read (16 bits) or in single words (fp32); chunk c of
//     row k lies at c ^ 2 * (k & 3) (16 bits), c ^ 4 * (k >> 2 & 1) (fp32), so
//     that the 4 rows that a 16-lane group reads lie in different banks.
// Chunks outside the operand have an offset past the buffer's end, which the
// load returns as zeros: no size needs a tail loop, and the stages past the
// last one are zeros too, so every step issues the same loads and waits for
// the same count.
//
// Pipeline.  TAM_GEMM_STAGES buffers.  Step t: wait for stage t+1 (all but
// the youngest loads) and for the own LDS reads of stage t, barrier; issue the
// loads of stage t+3 into the buffer of stage t, whose fragments are in every
// wave's registers by then; read the fragments of stage t+1 among the matrix
// instructions of stage t.  One barrier a step, and nothing waits for a load
// issued less than two steps before.
//
// Fragments.  mfma 16x16x32 (16 bits) or four 16x16x4 (fp32), P as the left
// operand: a lane then holds 4 consecutive columns c of one row r.
#ifndef TAM_GEMM_H
#define TAM_GEMM_H

#include "tam_ops.h"

#define TAM_GEMM_STAGES 3
#define TAM_GEMM_ROW 64  // bytes of a row in a stage

typedef short tam_s4 __attribute__((ext_vector_type(4)));
typedef short tam_s8 __attribute__((ext_vector_type(8)));
typedef __bf16 tam_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 tam_h8 __attribute__((ext_vector_type(8)));
typedef int tam_i4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) void tam_lds_void;
typedef __attribute__((address_space(3))) char tam_lds_char;
typedef __attribute__((address_space(3))) tam_s4 tam_lds_s4;
typedef __attribute__((address_space(3))) tam_s8 tam_lds_s8;
typedef __attribute__((address_space(3))) float tam_lds_float;

// One operand of a product: element (i, k) at base + (i * ld + k) * size
// (k-contiguous) or base + (k * ld + i) * size (m-major).  The contiguous
// extent is a multiple of 16 bytes, and base and rows lie on 16 bytes.
struct tam_operand {
  const char* base;
  uint64_t ld;     // bytes from one row to the next
  uint32_t count;  // i < count
};

// Fragment of 16 rows by one stage: 8 16-bit or 4 fp32 elements a lane.
template <typename T>
struct tam_frag {
  tam_s8 v;
};
template <>
struct tam_frag<float> {
  tam_f4 v;
};

__device__ __forceinline__ tam_f4 tam_mfma(const tam_frag<tam_bf16>& a, const tam_frag<tam_bf16>& b, tam_f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tam_bf8, a.v), __builtin_bit_cast(tam_bf8, b.v), c,
                                                 0, 0, 0);
}
__device__ __forceinline__ tam_f4 tam_mfma(const tam_frag<tam_f16>& a, const tam_frag<tam_f16>& b, tam_f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tam_h8, a.v), __builtin_bit_cast(tam_h8, b.v), c, 0,
                                                0, 0);
}
// fp32: the lane's 4 elements are k = 4 * (lane / 16) + 0..3 of the stage; the
// j-th instruction sums k = j, 4 + j, 8 + j, 12 + j, the same for both operands.
__device__ __forceinline__ tam_f4 tam_mfma(const tam_frag<float>& a, const tam_frag<float>& b, tam_f4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// Loading and reading one operand's stages.  ROWS: its rows in the tile; NW:
// the workgroup's waves; KC: contiguous along k.
template <typename T, int ROWS, int NW, bool KC>
struct tam_stage {
  static constexpr int EPC = 16 / (int)sizeof(T);             // elements of a chunk
  static constexpr int BK = TAM_GEMM_ROW / (int)sizeof(T);    // k of a stage
  static constexpr int BYTES = ROWS * TAM_GEMM_ROW;           // of a stage
  static constexpr int LOADS = BYTES / 1024 / NW;             // a wave's loads of a stage
  static constexpr int CPR = ROWS * (int)sizeof(T) / 16;      // m-major: chunks of a k row
  static constexpr int KPL = KC ? 0 : 64 / CPR;               // m-major: k rows of a load
  static_assert(LOADS >= 1 && BYTES % (1024 * NW) == 0, "whole loads");

  const char* base;      // of the next stage to load
  uint64_t step;         // bytes from one stage to the next
  uint32_t off[LOADS];   // the lane's offsets; 2^31 where its row or column lies outside
  uint32_t lane_k[KC ? 1 : LOADS];

  __device__ __forceinline__ static uint32_t swizzle(uint32_t k) {
    return sizeof(T) == 2 ? 2u * (k & 3u) : 4u * (k >> 2 & 1u);
  }

  // first: the tile's first row; k0: the first k
  __device__ __forceinline__ void init(const tam_operand& o, uint32_t first, uint64_t k0, int wave, int lane) {
    if constexpr (KC) {
      base = o.base + (uint64_t)first * o.ld + k0 * sizeof(T);
      step = TAM_GEMM_ROW;
      const uint32_t chunk = (lane & 3u) ^ (lane >> 3 & 3u);
      lane_k[0] = chunk * EPC;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t row = (uint32_t)(wave * LOADS + i) * 16u + (uint32_t)(lane >> 2);
        off[i] = first + row < o.count ? (uint32_t)(row * o.ld) + chunk * 16u : 0x80000000u;
      }
    } else {
      base = o.base + k0 * o.ld + (uint64_t)first * sizeof(T);
      step = (uint64_t)BK * o.ld;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t k = (uint32_t)(wave * LOADS + i) * KPL + (uint32_t)lane / CPR;
        const uint32_t chunk = ((uint32_t)lane % CPR) ^ swizzle(k);
        lane_k[i] = k;
        off[i] = first + chunk * EPC < o.count ? (uint32_t)(k * o.ld) + chunk * 16u : 0x80000000u;
      }
    }
  }

  // Loads the next stage into LDS at `lds`; k_left: how many k are left from its
  // first one on (0 or less: zeros).
  __device__ __forceinline__ void load(tam_lds_char* lds, int wave, int64_t k_left) {
    const uint32_t left = k_left <= 0 ? 0u : (k_left > BK ? (uint32_t)BK : (uint32_t)k_left);
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x80000000u, 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const uint32_t voff = lane_k[KC ? 0 : i] < left ? off[i] : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (tam_lds_void*)(lds + (wave * LOADS + i) * 1024), 16, voff, 0, 0,
                                               0);
    }
    base += step;
  }

  // The fragment of rows row0 .. row0 + 15 of the stage at `lds`.
  __device__ __forceinline__ static void read(tam_frag<T>& f, const tam_lds_char* lds, int row0, int lane) {
    const uint32_t i = lane & 15u, q = (uint32_t)lane >> 4;
    if constexpr (KC) {
      const uint32_t place = q ^ (i >> 1 & 3u);
      const tam_lds_char* p = lds + (row0 + i) * TAM_GEMM_ROW + place * 16u;
      f.v = *(const __attribute__((address_space(3))) decltype(f.v)*)p;
    } else if constexpr (sizeof(T) == 2) {
      // k rows 8q + 4h + i/4, columns row0 + 4 * (i % 4): the transposing read gives
      // lane i the 4 k of column row0 + i
      const uint32_t jr = i >> 2;
      const uint32_t chunk = ((uint32_t)row0 / 8u + (i >> 1 & 1u)) ^ (2u * jr);
      const tam_lds_char* p = lds + (8u * q + jr) * (ROWS * 2u) + chunk * 16u + (i & 1u) * 8u;
      const tam_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tam_lds_s4*)p);
      const tam_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tam_lds_s4*)(p + 4u * (ROWS * 2u)));
      f.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const uint32_t col = (uint32_t)row0 + i;
      const uint32_t chunk = (col / 4u) ^ (4u * (q & 1u));
      const tam_lds_char* p = lds + 4u * q * (ROWS * 4u) + chunk * 16u + (col & 3u) * 4u;
#pragma unroll
      for (int j = 0; j < 4; ++j) f.v[j] = *(const tam_lds_float*)(p + j * (ROWS * 4u));
    }
  }
};

// A product of operands in two parts, high + low: the sum of high * high, high *
// low and low * high runs as one sum over three times k.  p, q: bytes from an
// operand's high part to its low part (the same layout).
struct tam_parts {
  uint32_t terms;  // 1 (high * high alone) or 3
  int64_t p, q;
};

// One workgroup's tile: BM rows (operand Q) by BN columns (operand P), WM by
// WN waves.
template <typename T, int BM, int BN, int WM, int WN, bool PK, bool QK>
struct tam_tile {
  static constexpr int NW = WM * WN;
  static constexpr int THREADS = 64 * NW;
  static constexpr int TM = BM / WM / 16;  // a wave's fragments of Q
  static constexpr int TN = BN / WN / 16;  // and of P
  typedef tam_stage<T, BN, NW, PK> SP;
  typedef tam_stage<T, BM, NW, QK> SQ;
  static constexpr int BK = SP::BK;
  static constexpr int STAGE = SP::BYTES + SQ::BYTES;
  static constexpr int LOADS = SP::LOADS + SQ::LOADS;
  static constexpr int ROUND = 32;                        // rows of a wave that the epilogue turns at once
  static constexpr int COLS = BN / WN;                    // a wave's columns
  static constexpr int PITCH = COLS + 4;                  // floats of a turned row
  static constexpr int TURN = NW * ROUND * PITCH * 4;
  static constexpr int LDS = TAM_GEMM_STAGES * STAGE > TURN ? TAM_GEMM_STAGES * STAGE : TURN;
  static_assert(TM % 2 == 0, "rounds of 32 rows");

  tam_f4 acc[TN][TM];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m) acc[n][m] = tam_f4{0.f, 0.f, 0.f, 0.f};
  }

  struct frags {
    tam_frag<T> p[TN], q[TM];
  };

  __device__ __forceinline__ static void read_all(frags& f, const tam_lds_char* lds, int wm, int wn, int lane) {
#pragma unroll
    for (int n = 0; n < TN; ++n) SP::read(f.p[n], lds, (wn * TN + n) * 16, lane);
#pragma unroll
    for (int m = 0; m < TM; ++m) SQ::read(f.q[m], lds + SP::BYTES, (wm * TM + m) * 16, lane);
  }

  __device__ __forceinline__ void multiply(const frags& f) {
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int n = 0; n < TN; ++n) acc[n][m] = tam_mfma(f.p[n], f.q[m], acc[n][m]);
  }

  // wait until at most N loads are in flight and every LDS read has returned; barrier
  template <int N>
  __device__ __forceinline__ static void sync() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  }

  // Adds the products of k0 <= k < k1 to the tile at rows r0, columns c0.
  template <bool PARTS = false>
  __device__ __forceinline__ void run(const tam_operand& P, const tam_operand& Q, uint32_t c0, uint32_t r0, uint64_t k0,
                                      uint64_t k1, char* smem, tam_parts parts = {1, 0, 0}) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    tam_lds_char* lds = (tam_lds_char*)smem;
    SP sp;
    SQ sq;
    sp.init(P, c0, k0, wave, lane);
    sq.init(Q, r0, k0, wave, lane);
    const char *const p0 = sp.base, *const q0 = sq.base;
    const int64_t length = k1 > k0 ? (int64_t)(k1 - k0) : 0;
    int64_t left = length;  // k from the next stage to load on
    uint32_t steps = (uint32_t)((length + BK - 1) / BK), term = 0;
    if constexpr (PARTS) steps *= parts.terms;
    const uint32_t pairs = (steps + 1) / 2;
    auto load = [&](uint32_t buf) {
      if constexpr (PARTS)
        if (left <= 0 && term + 1 < parts.terms) {
          ++term;
          left = length;
          sp.base = p0 + (term == 2 ? parts.p : 0);
          sq.base = q0 + (term == 1 ? parts.q : 0);
        }
      sp.load(lds + buf * STAGE, wave, left);
      sq.load(lds + buf * STAGE + SP::BYTES, wave, left);
      left -= BK;
    };
    __syncthreads();  // the LDS may hold what another tile's epilogue still reads
    load(0);
    load(1);
    load(2);
    frags a, b;
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
    read_all(a, lds, wm, wn, lane);
    uint32_t cur = 0;  // buffer of stage t
    for (uint32_t t = 0; t < pairs; ++t) {
      uint32_t next = cur == 2 ? 0 : cur + 1;
      sync<LOADS>();
      load(cur);
      read_all(b, lds + next * STAGE, wm, wn, lane);
      multiply(a);
      interleave();
      cur = next;
      next = cur == 2 ? 0 : cur + 1;
      sync<LOADS>();
      load(cur);
      read_all(a, lds + next * STAGE, wm, wn, lane);
      multiply(b);
      interleave();
      cur = next;
    }
    sync<0>();  // the LDS is the epilogue's
  }

  // LDS reads spread among the matrix instructions of a step
  __device__ __forceinline__ static void interleave() {
    constexpr int READS = (PK ? 1 : sizeof(T) == 2 ? 2 : 4) * TN + (QK ? 1 : sizeof(T) == 2 ? 2 : 4) * TM;
    constexpr int MFMAS = TN * TM * (sizeof(T) == 2 ? 1 : 4);
    constexpr int EACH = MFMAS / READS > 0 ? MFMAS / READS : 1;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);     // one LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);  // matrix instructions
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MFMAS, 0);  // the rest: the last reads return behind them
    __builtin_amdgcn_sched_barrier(0);
  }

  // Hands the tile to f(row, col, v): 8 consecutive columns of one row, in fp32,
  // turned through LDS so that consecutive lanes hold consecutive columns.
  // Rows and columns are the tile's own; every one is handed out once.
  // piece(rows0, cols0, lds, pitch): after each 32 rows of the wave, what it holds in LDS.
  template <typename F, typename G>
  __device__ __forceinline__ void each(char* smem, F f, G piece) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    float* turn = reinterpret_cast<float*>(smem) + wave * ROUND * PITCH;
    constexpr int LPR = COLS / 8;   // lanes of a row
    constexpr int RPP = 64 / LPR;   // rows of a pass
#pragma unroll
    for (int m = 0; m < TM; m += 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < TN; ++n)
          *reinterpret_cast<tam_f4*>(turn + (h * 16 + (lane & 15)) * PITCH + n * 16 + (lane >> 4) * 4) = acc[n][m + h];
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
      for (int r = lane / LPR; r < ROUND; r += RPP) {
        const int c = (lane % LPR) * 8;
        float v[8];
        const tam_f4 lo = *reinterpret_cast<const tam_f4*>(turn + r * PITCH + c);
        const tam_f4 hi = *reinterpret_cast<const tam_f4*>(turn + r * PITCH + c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = lo[j];
          v[4 + j] = hi[j];
        }
        f((uint32_t)((wm * TM + m) * 16 + r), (uint32_t)(wn * COLS + c), v);
      }
      piece((uint32_t)((wm * TM + m) * 16), (uint32_t)(wn * COLS), turn, PITCH);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// Workgroup b of n in the order in which one XCD's workgroups take consecutive
// tiles (workgroups go to the 8 XCDs in turn): neighbours share rows of Q or P
// in that XCD's L2.
__device__ __forceinline__ uint32_t tam_xcd_order(uint32_t b, uint32_t n) {
  const uint32_t x = b & 7u, q = n >> 3, r = n & 7u;
  return x * q + (x < r ? x : r) + (b >> 3);
}

// Tile t of tm x tn in groups of GROUP rows, column by column inside a group.
__device__ __forceinline__ void tam_tile_at(uint32_t t, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  constexpr uint32_t GROUP = 8;
  const uint32_t per = GROUP * tn, g = t / per, left = t - g * per;
  const uint32_t rows = tm - g * GROUP < GROUP ? tm - g * GROUP : GROUP;
  n = left / rows;
  m = g * GROUP + left - n * rows;
}

#endif  // TAM_GEMM_H
