// tam_gemm.h -- the matrix-product core of the operators: one workgroup's tile
// of D[r][c] = sum_k Q[r][k] * P[c][k] on the matrix cores, for bf16, fp16 and
// fp32 operands that are contiguous along k or along their own index.
//
// Stages.  The k axis is cut into stages of 128 bytes of a row, a whole cache
// line: 64 16-bit or 32 fp32 elements.  A stage of an operand is (rows * 128)
// bytes of LDS, written by buffer loads that go to LDS directly, 1 KB to a wave
// and instruction:
//   k-contiguous operand: [row][128 bytes], 16-byte chunk c of row r at place
//     c ^ (r >> 1 & 7): the 16-byte fragment reads are free of conflicts;
//   operand contiguous along its own index ("m-major"): [k][rows], read with
//     the transposing LDS read (16 bits) or in single words (fp32). LDS has 64
//     banks (256 bytes); a read's 32 (fp32: 64) lanes that go together hold 8 (4)
//     k rows, and chunk c of row k lies at c ^ swizzle(k), which puts them into
//     different banks. (With the rows of 16 lanes alone apart, each transposing
//     read took 4 cycles for 2: 1352 us for 8192 x 14336 x 4096, both operands.)
// Chunks outside the operand have an offset past the buffer's end, which the
// load returns as zeros: no size needs a tail loop, and the stages past the
// last one are zeros too, so every step issues the same loads.
//
// Pipeline of the 64 and 128 tiles (that of the 256 ones: tam_tile::ring).  STAGES
// buffers, fragments of half a stage in registers twice.  Step t: read the second half's fragments of stage t among the matrix instructions of the
// first half; wait for stage t+1 and for the own reads, barrier: nobody reads
// stage t's buffer any more; issue the loads of stage t+STAGES into it; read the first
// half of stage t+1 among the matrix instructions of the second half of t.  One
// barrier a step, and a load has STAGES-1 steps to arrive.
//
// Fragments.  mfma 16x16x32 (16 bits) or four 16x16x4 (fp32), P as the left
// operand: a lane then holds 4 consecutive columns c of one row r.
#ifndef TAM_GEMM_H
#define TAM_GEMM_H

#include <type_traits>

#include "tam_ops.h"

#define TAM_GEMM_ROW 128  // bytes of a row in a stage

typedef short tam_s4 __attribute__((ext_vector_type(4)));
typedef short tam_s8 __attribute__((ext_vector_type(8)));
typedef __bf16 tam_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 tam_h8 __attribute__((ext_vector_type(8)));
typedef int tam_i4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) char tam_lds_char;
typedef __attribute__((address_space(3))) tam_s4 tam_lds_s4;
typedef __attribute__((address_space(3))) tam_s8 tam_lds_s8;
typedef __attribute__((address_space(3))) float tam_lds_float;

// One operand of a product: element (i, k) at base + i * ld + k * size
// (k-contiguous) or base + k * ld + i * size (m-major). base and ld are multiples of
// 4. A product's k is a multiple of 16 bytes of its k-contiguous operands, or their
// rows are zeros up to one; the rest of a sum is tam_tile::tail's. Loads take 16 bytes
// from any multiple of 4; in an EXACT tile the words of an m-major operand from `end`
// on come as zeros (each word for itself).
struct tam_operand {
  const char* base;
  uint64_t ld;      // bytes from one row to the next
  uint32_t count;   // i < count
  const char* end;
};

// Fragment of 16 rows by half a stage: 8 16-bit or 4 fp32 elements a lane.
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
// fp32: the lane's 4 elements are k = 4 * (lane / 16) + 0..3 of the half; the
// j-th instruction sums k = j, 4 + j, 8 + j, 12 + j, the same for both operands.
__device__ __forceinline__ tam_f4 tam_mfma(const tam_frag<float>& a, const tam_frag<float>& b, tam_f4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// The same where a sum stays in its registers, and with a load to LDS issued behind it: m0,
// which takes a wait state before it is used, has it in the matrix instruction. The wait states
// before the sums are read are the caller's (tam_tile::settle).
#define TAM_MFMA_IN(TYPE, NAME)                                                                                      \
  __device__ __forceinline__ void tam_mfma_in(const tam_frag<TYPE>& a, const tam_frag<TYPE>& b, tam_f4& c) {         \
    asm volatile("v_mfma_f32_16x16x32_" NAME " %0, %1, %2, %0" : "+v"(c) : "v"(a.v), "v"(b.v));                      \
  }                                                                                                                  \
  __device__ __forceinline__ void tam_mfma_load(const tam_frag<TYPE>& a, const tam_frag<TYPE>& b, tam_f4& c,         \
                                                uint32_t lds, int place, uint32_t voff, tam_i4 rsrc) {               \
    asm volatile("s_add_i32 m0, %1, %2\n\tv_mfma_f32_16x16x32_" NAME " %0, %5, %6, %0\n\t"                           \
                 "buffer_load_dwordx4 %3, %4, 0 offen lds"                                                           \
                 : "+v"(c)                                                                                           \
                 : "s"(lds), "i"(place), "v"(voff), "s"(rsrc), "v"(a.v), "v"(b.v)                                    \
                 : "m0", "scc");                                                                                     \
  }
TAM_MFMA_IN(tam_bf16, "bf16")
TAM_MFMA_IN(tam_f16, "f16")
#undef TAM_MFMA_IN

// 16 bytes a lane from rsrc's base + voff to LDS at `lds` + 16 * lane.
__device__ __forceinline__ void tam_to_lds(uint32_t lds, uint32_t voff, tam_i4 rsrc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(rsrc)
               : "m0");
}

// A word a lane, to LDS at `lds` + 4 * lane.
__device__ __forceinline__ void tam_word_to_lds(uint32_t lds, uint32_t voff, tam_i4 rsrc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(rsrc)
               : "m0");
}

// Loading and reading one operand's stages.  ROWS: its rows in the tile; NW:
// the workgroup's waves; KC: contiguous along k; EXACT: nothing is read past the
// operand's end (see tam_tile).
template <typename T, int ROWS, int NW, bool KC, bool EXACT>
struct tam_stage {
  static constexpr int EPC = 16 / (int)sizeof(T);             // elements of a chunk
  static constexpr int BK = TAM_GEMM_ROW / (int)sizeof(T);    // k of a stage
  static constexpr int BYTES = ROWS * TAM_GEMM_ROW;           // of a stage
  static constexpr int LOADS = BYTES / 1024 / NW;             // a wave's loads of a stage
  static constexpr int CPR = ROWS * (int)sizeof(T) / 16;      // m-major: chunks of a k row
  static constexpr int KPL = KC ? 0 : 64 / CPR;               // m-major: k rows of a load
  static_assert(LOADS >= 1 && BYTES % (1024 * NW) == 0, "whole loads");

  const char* base;      // of the next stage to load
  const char* end;
  uint64_t step;         // bytes from one stage to the next
  uint32_t off[LOADS];   // the lane's offsets; 2^31 where its row or column lies outside
  uint32_t lane_k[LOADS];

  __device__ __forceinline__ static uint32_t swizzle(uint32_t k) {
    if constexpr (sizeof(T) == 4) return 4u * (k >> 2 & (CPR == 8 ? 1u : 3u));
    if constexpr (CPR == 4) return 2u * (k >> 3 & 1u);
    if constexpr (CPR == 8) return 2u * (k >> 1 & 1u) | 4u * (k >> 3 & 1u);
    return 2u * (k & 3u) | 8u * (k >> 3 & 1u);
  }

  // first: the tile's first row; k0: the first k
  __device__ __forceinline__ void init(const tam_operand& o, uint32_t first, uint64_t k0, int wave, int lane) {
    if constexpr (EXACT) end = o.end;
    if constexpr (KC) {
      base = o.base + (uint64_t)first * o.ld + k0 * sizeof(T);
      step = TAM_GEMM_ROW;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t row = (uint32_t)(wave * LOADS + i) * 8u + (uint32_t)(lane >> 3);
        const uint32_t chunk = (lane & 7u) ^ (row >> 1 & 7u);
        lane_k[i] = chunk * EPC;
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

  // Load `i` of the next stage into LDS at `lds`; left: how many k are left from the
  // stage's first one on, at most BK (zeros come past them).
  // The compiler does not know that the asm writes LDS, or of its count in vmcnt: the
  // pipeline waits for it (sync), and no wait is put before the reads of other
  // buffers (as a builtin load gets one before every transposing read: 1.7 times the
  // time for two m-major operands). m0 takes a wait state before it is used.
  __device__ __forceinline__ void load(int i, uint32_t lds, int wave, uint32_t left) const {
    const uint64_t b = (uint64_t)base;
    uint32_t records = 0x80000000u;
    if constexpr (EXACT) {
      const int64_t rest = end - base;
      records = rest <= 0 ? 0u : (rest < 0x80000000ll ? (uint32_t)rest : 0x80000000u);
    }
    const tam_i4 rsrc = {(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), (int)records, 0x00020000};
    const uint32_t voff = lane_k[i] < left ? off[i] : 0x80000000u, at = lds + (uint32_t)(wave * LOADS + i) * 1024u;
    tam_to_lds(at, voff, rsrc);
  }

  // The parts of load(), for loads that are issued together with a matrix instruction: load i goes to
  // wave * WAVE_BYTES + place(i) of the stage, from offset(i, left).
  static constexpr int WAVE_BYTES = LOADS * 1024;
  __device__ static constexpr int place(int i) { return i * 1024; }
  __device__ __forceinline__ tam_i4 rsrc(int) const {
    const uint64_t b = (uint64_t)base;
    return tam_i4{(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), (int)0x80000000u, 0x00020000};
  }
  __device__ __forceinline__ uint32_t offset(int i, uint32_t left) const { return lane_k[i] < left ? off[i] : 0x80000000u; }

  __device__ __forceinline__ const char* at() const { return base; }
  __device__ __forceinline__ void seek(const char* p) { base = p; }
  __device__ __forceinline__ void next() { base += step; }

  // The fragment of rows row0 .. row0 + 15 and half `h` of the stage at `lds`.
  __device__ __forceinline__ static void read(tam_frag<T>& f, const tam_lds_char* lds, int row0, int h, int lane) {
    const uint32_t i = lane & 15u, q = (uint32_t)lane >> 4;
    if constexpr (KC) {
      const uint32_t place = (4u * h + q) ^ (i >> 1 & 7u);
      const tam_lds_char* p = lds + (row0 + i) * TAM_GEMM_ROW + place * 16u;
      f.v = *(const __attribute__((address_space(3))) decltype(f.v)*)p;
    } else if constexpr (sizeof(T) == 2) {
      // k rows 8q + 4g + i/4, columns row0 + 4 * (i % 4): the transposing read gives
      // lane i the 4 k of column row0 + i
      const uint32_t jr = i >> 2;
      const uint32_t chunk = ((uint32_t)row0 / 8u + (i >> 1 & 1u)) ^ swizzle(8u * q + jr);
      const tam_lds_char* p = lds + (32u * h + 8u * q + jr) * (ROWS * 2u) + chunk * 16u + (i & 1u) * 8u;
      const tam_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tam_lds_s4*)p);
      const tam_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tam_lds_s4*)(p + 4u * (ROWS * 2u)));
      f.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const uint32_t col = (uint32_t)row0 + i;
      const uint32_t chunk = (col / 4u) ^ swizzle(4u * q);
      const tam_lds_char* p = lds + (16u * h + 4u * q) * (ROWS * 4u) + chunk * 16u + (col & 3u) * 4u;
#pragma unroll
      for (int j = 0; j < 4; ++j) f.v[j] = *(const tam_lds_float*)(p + j * (ROWS * 4u));
    }
  }
};

// Two operands that share a tile's columns: a wave's fragments are half of one's
// columns and half of the same columns of the other, so that one lane holds both products.
struct tam_operand_pair {
  tam_operand a, b;
};

// Their stages: ROWS / 2 rows of each, one behind the other. TN: a wave's fragments.
template <typename T, int ROWS, int NW, bool KC, int TN>
struct tam_pair_stage {
  typedef tam_stage<T, ROWS / 2, NW, KC, false> Half;
  static constexpr int BK = Half::BK, BYTES = 2 * Half::BYTES, LOADS = 2 * Half::LOADS;
  static_assert(TN % 2 == 0, "half of the fragments are of each operand");

  Half a, b;

  // first: the tile's first column of either operand
  __device__ __forceinline__ void init(const tam_operand_pair& o, uint32_t first, uint64_t k0, int wave, int lane) {
    a.init(o.a, first, k0, wave, lane);
    b.init(o.b, first, k0, wave, lane);
  }
  __device__ __forceinline__ void load(int i, uint32_t lds, int wave, uint32_t left) const {
    if (i < Half::LOADS)
      a.load(i, lds, wave, left);
    else
      b.load(i - Half::LOADS, lds + Half::BYTES, wave, left);
  }
  __device__ __forceinline__ static void read(tam_frag<T>& f, const tam_lds_char* lds, int row0, int h, int lane) {
    const int n = row0 / 16 % TN, row = (row0 / 16 / TN * (TN / 2) + n % (TN / 2)) * 16;
    Half::read(f, n < TN / 2 ? lds : lds + Half::BYTES, row, h, lane);
  }
  static constexpr int WAVE_BYTES = Half::WAVE_BYTES;
  __device__ static constexpr int place(int i) {
    return i < Half::LOADS ? i * 1024 : Half::BYTES + (i - Half::LOADS) * 1024;
  }
  __device__ __forceinline__ tam_i4 rsrc(int i) const { return i < Half::LOADS ? a.rsrc(i) : b.rsrc(i); }
  __device__ __forceinline__ uint32_t offset(int i, uint32_t left) const {
    return i < Half::LOADS ? a.offset(i, left) : b.offset(i - Half::LOADS, left);
  }
  __device__ __forceinline__ const char* at() const { return a.base; }
  __device__ __forceinline__ void seek(const char*) {}
  __device__ __forceinline__ void next() {
    a.next();
    b.next();
  }
};

// A product of operands in two parts, high + low: the sum of high * high, high *
// low and low * high runs as one sum over three times k.  p, q: bytes from an
// operand's high part to its low part (the same layout).
// Or the sum of two products, one behind the other: of operands p and q bytes apart.
enum tam_terms { TAM_ONE_TERM, TAM_HIGH_LOW, TAM_TWO_PRODUCTS };
struct tam_parts {
  uint32_t terms;  // 1 (high * high alone) or 3; 2 products
  int64_t p, q;
};

// How far ahead of its use the epilogue loads (tam_tile::each).
enum tam_ahead { TAM_AHEAD_PASS, TAM_AHEAD_ROUND, TAM_AHEAD_ALL };

// What the epilogue will read of an array laid out like the tile: a word of each line
// of it is fetched in the last step but one (to LDS, where nobody reads it: that takes
// no registers). Otherwise all compute units, whose tiles end together, wait for
// memory: of 45 us that a tile of k = 256 took, 11 were the wait for x's low part.
// The 256 tiles have no LDS left for it, and do without: their ring gained more than the
// fetch had (tam_k_mu_square's p 378 -> 354 us, tam_k_mu_apply 1540 -> 1422).
struct tam_soon {
  const char* base;         // of the tile's first element, on 4 bytes; null: nothing
  uint64_t ld;              // bytes, a multiple of 4
  uint32_t rows, bytes;     // from there on
  uint32_t width;           // bytes of a tile's row: a power of two from 64 to 1024
};

// Stages of a tile in LDS: two, but three of the small tiles of 16-bit types, whose
// steps are shorter than the way to memory (k = 4096, 64 tiles: 32 us with two, 18
// with three; 128-wide tiles gain nothing from more, and lose a neighbour).
template <typename T, int TILE>
constexpr int tam_stages() {
  return TILE == 64 && sizeof(T) == 2 ? 3 : 2;
}

// One workgroup's tile: BM rows (operand Q) by BN columns (operand P), WM by
// WN waves.
// EXACT: m-major operands whose rows may end inside 16 bytes: the last row's last
// load stops at the operand's `end` (a k-contiguous one never passes it).
// PAIR: the columns' operand is two (tam_operand_pair), BN / 2 columns of each.
template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool PK, bool QK, bool EXACT = false, bool PAIR = false>
struct tam_tile {
  static constexpr int NW = WM * WN;
  static constexpr int THREADS = 64 * NW;
  static constexpr bool RING = BM == 256;
  static constexpr int TM = BM / WM / 16;  // a wave's fragments of Q
  static constexpr int TN = BN / WN / 16;  // and of P
  typedef std::conditional_t<PAIR, tam_pair_stage<T, BN, NW, PK, TN>, tam_stage<T, BN, NW, PK, EXACT && !PK>> SP;
  typedef tam_stage<T, BM, NW, QK, EXACT && !QK> SQ;
  static constexpr int BK = SP::BK;
  static constexpr int STAGE = SP::BYTES + SQ::BYTES;
  static constexpr int LOADS = SP::LOADS + SQ::LOADS;
  static constexpr int ROUND = 32;                        // rows of a wave that the epilogue turns at once
  static constexpr int COLS = BN / WN;                    // a wave's columns
  static constexpr int PITCH = COLS + 4;                  // floats of a turned row
  static constexpr int TURN = NW * ROUND * PITCH * 4;
  static constexpr int DUMP = STAGES * STAGE > TURN ? STAGES * STAGE : TURN;
  static constexpr int LDS = RING ? 5 * SP::BYTES : DUMP + NW * 256;  // the words that `soon` fetches
  static_assert(TM % 2 == 0, "rounds of 32 rows");
  static_assert(!(RING && EXACT && !(PK && QK)), "the ring's loads have no bound at the operand's end");

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

  // wait until at most N loads are in flight and every LDS read has returned; barrier
  template <int N>
  __device__ __forceinline__ static void sync() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  }

  // Adds the products of k0 <= k < k1 to the tile at rows r0, columns c0.
  template <int TERMS = TAM_ONE_TERM, typename Columns = tam_operand>
  __device__ __forceinline__ void run(const Columns& P, const tam_operand& Q, uint32_t c0, uint32_t r0, uint64_t k0,
                                      uint64_t k1, char* smem, const tam_soon& soon, tam_parts parts = {1, 0, 0}) {
    if constexpr (RING) return run_ring<TERMS>(P, Q, c0, r0, k0, k1, smem, parts);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    tam_lds_char* lds = (tam_lds_char*)smem;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    SP sp;
    SQ sq;
    sp.init(P, c0, k0, wave, lane);
    sq.init(Q, r0, k0, wave, lane);
    const char *const p0 = sp.at(), *const q0 = sq.at();
    const int64_t length = k1 > k0 ? (int64_t)(k1 - k0) : 0;
    int64_t ahead = length;  // k from the next stage to load on
    uint32_t left = 0, steps = (uint32_t)((length + BK - 1) / BK), term = 0;
    if constexpr (TERMS != TAM_ONE_TERM) steps *= parts.terms;
    // load i of the next stage into buffer `buf`: the first one looks at what is left,
    // the last one moves on
    auto load = [&](int i, uint32_t buf) {
      if (i == 0) {
        if constexpr (TERMS != TAM_ONE_TERM)
          if (ahead <= 0 && term + 1 < parts.terms) {
            ++term;
            ahead = length;
            sp.seek(p0 + (TERMS == TAM_TWO_PRODUCTS || term == 2 ? parts.p : 0));
            sq.seek(q0 + (term == 1 ? parts.q : 0));
          }
        left = ahead <= 0 ? 0u : (ahead > BK ? (uint32_t)BK : (uint32_t)ahead);
        ahead -= BK;
      }
      if (i < SP::LOADS)
        sp.load(i, lds0 + buf * STAGE, wave, left);
      else
        sq.load(i - SP::LOADS, lds0 + buf * STAGE + SP::BYTES, wave, left);
      if (i == LOADS - 1) {
        sp.next();
        sq.next();
      }
    };
    auto fetch = [&]() {
      const uint32_t lines = soon.width > 128u ? soon.width / 128u : 1u;  // of a row
      const uint64_t b = (uint64_t)soon.base;
      const tam_i4 rsrc = {(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), (int)0x80000000u, 0x00020000};
      for (uint32_t i = wave * 64; i < BM * lines; i += NW * 64) {
        const uint32_t line = i + lane, row = line / lines, in = line % lines * 128u;
        const bool inside = row < soon.rows && row < BM && in + 4u <= soon.bytes;
        tam_word_to_lds(lds0 + DUMP + (uint32_t)wave * 256u, inside ? (uint32_t)(row * soon.ld) + in : 0x80000000u, rsrc);
      }
    };
    // Half a step: the fragments of half h of buffer `from` are read, and the loads into
    // buffer `to` issued (GLOBAL), among the products of `f`, whose rows take a group each
    // of about as many loads, reads and matrix instructions. Issued at once, the loads
    // would hold up every matrix instruction behind them until the address unit has taken
    // them, and the reads would queue.
    auto half = [&](const frags& f, frags& next, uint32_t from, int h, uint32_t to, auto global) {
      constexpr bool GLOBAL = decltype(global)::value;
      const tam_lds_char* src = lds + from * STAGE;
#pragma unroll
      for (int m = 0; m < TM; ++m) {
#pragma unroll
        for (int n = m * TN / TM; n < (m + 1) * TN / TM; ++n) SP::read(next.p[n], src, (wn * TN + n) * 16, h, lane);
        SQ::read(next.q[m], src + SP::BYTES, (wm * TM + m) * 16, h, lane);
        if constexpr (GLOBAL)
#pragma unroll
          for (int i = m * LOADS / TM; i < (m + 1) * LOADS / TM; ++i) load(i, to);
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[n][m] = tam_mfma(f.p[n], f.q[m], acc[n][m]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    __syncthreads();  // the LDS may hold what another tile's epilogue still reads
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load(i, s);
    frags a, b;
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * LOADS) : "memory");
#pragma unroll
    for (int n = 0; n < TN; ++n) SP::read(a.p[n], lds, (wn * TN + n) * 16, 0, lane);
#pragma unroll
    for (int m = 0; m < TM; ++m) SQ::read(a.q[m], lds + SP::BYTES, (wm * TM + m) * 16, 0, lane);
    uint32_t cur = 0;  // buffer of stage t
    const uint32_t last = steps > 2 && soon.base ? steps - 2 : ~0u;
    for (uint32_t t = 0; t < steps; ++t) {
      const uint32_t next = cur + 1 == STAGES ? 0 : cur + 1;
      half(a, b, cur, 1, 0, std::false_type());
      sync<(STAGES - 2) * LOADS>();
      if (t == last) fetch();
      half(b, a, next, 0, cur, std::true_type());
      cur = next;
    }
    sync<0>();  // the LDS is the epilogue's
  }

  // The same for the largest tiles, whose stages are 32 KB of each operand: a ring of five
  // such halves in place of two stages, so that one operand's loads are in flight while the
  // other's arrive. Step t: read the second half's fragments of stage t and issue the loads of
  // P's stage t + 2 among the matrix instructions of the first half; wait for stage t + 1 and
  // for the own reads, barrier; read the first half of stage t + 1 and issue the loads of Q's
  // stage t + 2 (into what P's stage t held) among those of the second half.
  // begin issues the first two stages into the first four halves, which nobody may be
  // reading; sum waits for them and adds the products. So a workgroup can begin its next
  // tile before it stores this one, by way of the fifth half (`spare`).
  // (8192 x 14336 x 4096 bf16, two whole stages -> this: 745 -> 681 us with both operands along k, 816 ->
  // 755 with neither. 4 waves of 128 x 128 in place of 8 of 128 x 64, which read less LDS: the same
  // with both along k, slower otherwise.)
  static constexpr int HALF = SP::BYTES, L = SP::LOADS;
  struct ring {
    SP sp;
    SQ sq;
    const char *p0, *q0;
    int64_t length, ahead;      // k of a sum; from the next stage to load on
    uint32_t steps, left, seen, term;
    uint32_t off_p[L], off_q[L];  // of a stage with `left`: it is BK in all but the last stages of a sum
    tam_parts parts;

    template <int TERMS>
    __device__ __forceinline__ void stage() {
      if constexpr (TERMS != TAM_ONE_TERM)
        if (ahead <= 0 && term + 1 < parts.terms) {
          ++term;
          ahead = length;
          sp.seek(p0 + (TERMS == TAM_TWO_PRODUCTS || term == 2 ? parts.p : 0));
          sq.seek(q0 + (term == 1 ? parts.q : 0));
        }
      left = ahead <= 0 ? 0u : (ahead > BK ? (uint32_t)BK : (uint32_t)ahead);
      ahead -= BK;
      if (left != seen) {
        seen = left;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          off_p[i] = sp.offset(i, left);
          off_q[i] = sq.offset(i, left);
        }
      }
    }
  };

  template <int TERMS = TAM_ONE_TERM, typename Columns = tam_operand>
  __device__ __forceinline__ static void begin(ring& r, const Columns& P, const tam_operand& Q, uint32_t c0, uint32_t r0,
                                               uint64_t k0, uint64_t k1, char* smem, tam_parts parts = {1, 0, 0}) {
    static_assert(SP::BYTES == SQ::BYTES && SP::LOADS == SQ::LOADS, "halves of one size");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(tam_lds_char*)smem);
    r.sp.init(P, c0, k0, wave, lane);
    r.sq.init(Q, r0, k0, wave, lane);
    r.p0 = r.sp.at();
    r.q0 = r.sq.at();
    r.length = r.ahead = k1 > k0 ? (int64_t)(k1 - k0) : 0;
    r.steps = (uint32_t)((r.length + BK - 1) / BK);
    if constexpr (TERMS != TAM_ONE_TERM) r.steps *= parts.terms;
    r.parts = parts;
    r.term = 0;
    r.seen = ~0u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      r.template stage<TERMS>();
#pragma unroll
      for (int i = 0; i < L; ++i) tam_to_lds(lds0 + 2 * s * HALF + wave * SP::WAVE_BYTES + SP::place(i), r.off_p[i], r.sp.rsrc(i));
#pragma unroll
      for (int i = 0; i < L; ++i)
        tam_to_lds(lds0 + (2 * s + 1) * HALF + wave * SQ::WAVE_BYTES + SQ::place(i), r.off_q[i], r.sq.rsrc(i));
      r.sp.next();
      r.sq.next();
    }
  }

  // LATER: vector memory operations that every wave has issued since begin, at least.
  template <int TERMS = TAM_ONE_TERM, int LATER = 0>
  __device__ __forceinline__ void sum(ring& r, char* smem) {
    constexpr int READS = TM + TN, SLOTS = TM * TN;
    constexpr int READ_EVERY = SLOTS * 3 / 4 / READS, LOAD_EVERY = SLOTS / 2 / L;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    tam_lds_char* lds = (tam_lds_char*)smem;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    const uint32_t lds_p = lds0 + (uint32_t)wave * SP::WAVE_BYTES, lds_q = lds0 + (uint32_t)wave * SQ::WAVE_BYTES;
    // Half a step: fragments of half h out of buffers bp and bq, P's first as they are used
    // first, spread over the first three quarters of the matrix instructions (their latency
    // is over at the barrier); the loads over the first half.
    auto half = [&](const frags& f, frags& next, uint32_t bp, uint32_t bq, int h, const auto& st, const uint32_t(&off)[L],
                    uint32_t to) {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        if (s % READ_EVERY == 0 && s / READ_EVERY < READS) {
          const int i = s / READ_EVERY;
          if (i < TN)
            SP::read(next.p[i], lds + bp * HALF, (wn * TN + i) * 16, h, lane);
          else
            SQ::read(next.q[i - TN], lds + bq * HALF, (wm * TM + i - TN) * 16, h, lane);
        }
        const int m = s / TN, n = s % TN, i = s / LOAD_EVERY;
        if (s % LOAD_EVERY == 1 && i < L)
          tam_mfma_load(f.p[n], f.q[m], acc[n][m], to, st.place(i), off[i], st.rsrc(i));
        else
          tam_mfma_in(f.p[n], f.q[m], acc[n][m]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    frags a, b;
    constexpr int FIRST = 2 * L + LATER < 63 ? 2 * L + LATER : 63;
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(FIRST) : "memory");
#pragma unroll
    for (int n = 0; n < TN; ++n) SP::read(a.p[n], lds, (wn * TN + n) * 16, 0, lane);
#pragma unroll
    for (int m = 0; m < TM; ++m) SQ::read(a.q[m], lds + HALF, (wm * TM + m) * 16, 0, lane);
    uint32_t bp = 0;  // buffer of P's stage t; those behind it, in the ring's order: Q's, and so on
    auto behind = [&](uint32_t n) { return bp + n >= 5 ? bp + n - 5 : bp + n; };
    for (uint32_t t = 0; t < r.steps; ++t) {
      r.template stage<TERMS>();
      half(a, b, bp, behind(1), 1, r.sp, r.off_p, lds_p + behind(4) * HALF);
      sync<L>();
      half(b, a, behind(2), behind(3), 0, r.sq, r.off_q, lds_q + bp * HALF);
      r.sp.next();
      r.sq.next();
      bp = behind(2);
    }
    sync<0>();  // the LDS is the epilogue's
    settle();
  }

  template <int TERMS = TAM_ONE_TERM, typename Columns = tam_operand>
  __device__ __forceinline__ void run_ring(const Columns& P, const tam_operand& Q, uint32_t c0, uint32_t r0, uint64_t k0,
                                           uint64_t k1, char* smem, tam_parts parts = {1, 0, 0}) {
    ring r;
    __syncthreads();  // the LDS may hold what another tile's epilogue still reads
    begin<TERMS>(r, P, Q, c0, r0, k0, k1, smem, parts);
    sum<TERMS>(r, smem);
  }

  // Behind the last of tam_mfma_in: a result may be read 11 wait states after it.
  __device__ __forceinline__ void settle() {
    asm volatile("s_nop 15\n\ts_nop 7");
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m) asm volatile("" : "+v"(acc[n][m]));
  }

  // Adds the products of k0 <= k < k1, a few of them, element by element.
  __device__ __forceinline__ void tail(const tam_operand& P, const tam_operand& Q, uint32_t c0, uint32_t r0, uint64_t k0,
                                       uint64_t k1) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    for (uint64_t k = k0; k < k1; ++k) {
      float p[TN][4], q[TM];
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const uint32_t at = r0 + (wm * TM + m) * 16 + (lane & 15u), i = at < Q.count ? at : Q.count - 1;
        q[m] = (float)*reinterpret_cast<const T*>(QK ? Q.base + i * Q.ld + k * sizeof(T) : Q.base + k * Q.ld + i * sizeof(T));
      }
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          const uint32_t at = c0 + (wn * TN + n) * 16 + (lane >> 4) * 4 + j, i = at < P.count ? at : P.count - 1;
          p[n][j] = (float)*reinterpret_cast<const T*>(PK ? P.base + i * P.ld + k * sizeof(T) : P.base + k * P.ld + i * sizeof(T));
        }
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[n][m][j] = __builtin_fmaf(p[n][j], q[m], acc[n][m][j]);
    }
  }

  // PAIR: hands the tile to finish(row, col, a, b): 8 consecutive columns of one row of
  // either product, in fp32; columns are 0 .. BN / 2 - 1.
  template <typename F>
  __device__ __forceinline__ void pairs(char* smem, F finish) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    float* turn = reinterpret_cast<float*>(smem) + wave * ROUND * PITCH;
    constexpr int HALF = COLS / 2, LPR = HALF / 8, RPP = 64 / LPR, PASSES = ROUND / RPP;
    const int r0 = lane / LPR, c0 = (lane % LPR) * 8;
#pragma unroll
    for (int m = 0; m < TM; m += 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < TN; ++n)
          *reinterpret_cast<tam_f4*>(turn + (h * 16 + (lane & 15)) * PITCH + n * 16 + (lane >> 4) * 4) = acc[n][m + h];
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const float* from = turn + (p * RPP + r0) * PITCH + c0;
        float a[8], b[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const tam_f4 x = *reinterpret_cast<const tam_f4*>(from + j), y = *reinterpret_cast<const tam_f4*>(from + HALF + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[j + i] = x[i];
            b[j + i] = y[i];
          }
        }
        finish((uint32_t)((wm * TM + m) * 16 + p * RPP + r0), (uint32_t)(wn * HALF + c0), a, b);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  }

  // Epilogue of a tile whose next one has begun: by 16 rows at a time through the fifth half,
  // where a wave has room for them; 16-byte chunk c of row r lies at place c ^ r.
  static constexpr int SPARE = 4 * HALF;
  __device__ __forceinline__ tam_lds_char* spare(char* smem) const {
    return (tam_lds_char*)smem + SPARE + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * (HALF / NW);
  }
  // Fragment m as fp32, by rows: one of its 16 rows to LPR lanes.
  __device__ __forceinline__ void turn_in(char* smem, int m) const {
    const uint32_t lane = threadIdx.x & 63, row = lane & 15;
    tam_lds_char* at = spare(smem) + row * (COLS * 4);
#pragma unroll
    for (int n = 0; n < TN; ++n)
      *(__attribute__((address_space(3))) tam_f4*)(at + ((n * 4 + (lane >> 4)) ^ row) * 16) = acc[n][m];
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // 8 columns of a row of it.
  __device__ __forceinline__ void turn_out(char* smem, uint32_t row, uint32_t col, float (&v)[8]) const {
    const tam_lds_char* at = spare(smem) + row * (COLS * 4);
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const tam_f4 x = *(const __attribute__((address_space(3))) tam_f4*)(at + ((col / 4 + j) ^ row) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * j + i] = x[i];
    }
  }
  __device__ __forceinline__ static void turned() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }

  // Hands the tile to finish(row, col, v, pre): 8 consecutive columns of one row, in
  // fp32, turned through LDS so that consecutive lanes hold consecutive columns.
  // Rows and columns are the tile's own; every one is handed out once. pre is what
  // load(row, col) returned for them earlier: the global loads that finish needs. A
  // load behind each pass's stores costs its whole latency, 16 times a tile; and as
  // loads and stores are counted in order, a load issued behind stores is not there
  // before they have reached memory. AHEAD: all (every load before the first store),
  // round (a round of 32 rows ahead), or pass (one pass; the code of one pass).
  // piece(rows0, cols0, lds, pitch): after each 32 rows of the wave, what it holds in LDS.
  template <tam_ahead AHEAD, typename L, typename F, typename G>
  __device__ __forceinline__ void each(char* smem, L load, F finish, G piece) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    float* turn = reinterpret_cast<float*>(smem) + wave * ROUND * PITCH;
    constexpr int LPR = COLS / 8;         // lanes of a row
    constexpr int RPP = 64 / LPR;         // rows of a pass
    constexpr int PASSES = ROUND / RPP;
    typedef decltype(load(0u, 0u)) Pre;
    const int r0 = lane / LPR, c0 = (lane % LPR) * 8;
    const uint32_t col = (uint32_t)(wn * COLS + c0);
    auto row = [&](int m, int pass) { return (uint32_t)((wm * TM + m) * 16 + pass * RPP + r0); };
    auto take = [&](int pass, float(&v)[8]) {
      const float* from = turn + (pass * RPP + r0) * PITCH + c0;
      const tam_f4 lo = *reinterpret_cast<const tam_f4*>(from), hi = *reinterpret_cast<const tam_f4*>(from + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = lo[j];
        v[4 + j] = hi[j];
      }
    };
    constexpr bool UNROLL = AHEAD != TAM_AHEAD_PASS;
    constexpr int ROUNDS = TM / 2, DEPTH = AHEAD == TAM_AHEAD_ALL ? ROUNDS : 2;
    Pre pre[DEPTH][UNROLL ? PASSES : 1];
    if constexpr (UNROLL) {
#pragma unroll
      for (int i = 0; i < DEPTH - (AHEAD == TAM_AHEAD_ROUND); ++i)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) pre[i][p] = load(row(2 * i, p), col);
    }
#pragma unroll
    for (int m = 0; m < TM; m += 2) {
      if constexpr (AHEAD == TAM_AHEAD_ROUND) {
        if (m + 2 < TM)
#pragma unroll
          for (int p = 0; p < PASSES; ++p) pre[(m / 2 + 1) % DEPTH][p] = load(row(m + 2, p), col);
      } else if constexpr (AHEAD == TAM_AHEAD_PASS) {
        pre[0][0] = load(row(m, 0), col);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < TN; ++n)
          *reinterpret_cast<tam_f4*>(turn + (h * 16 + (lane & 15)) * PITCH + n * 16 + (lane >> 4) * 4) = acc[n][m + h];
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (UNROLL) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          float v[8];
          take(p, v);
          finish(row(m, p), col, v, pre[m / 2 % DEPTH][p]);
        }
      } else {
#pragma unroll 1
        for (int p = 0; p < PASSES; ++p) {
          const Pre now = pre[0][0];
          if (p + 1 < PASSES) pre[0][0] = load(row(m, p + 1), col);
          float v[8];
          take(p, v);
          finish(row(m, p), col, v, now);
        }
      }
      piece((uint32_t)((wm * TM + m) * 16), (uint32_t)(wn * COLS), turn, PITCH);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// Workgroup b of n -> tile. Workgroups go to the 8 XCDs in turn; of each 256, which
// run together, an XCD takes 32 consecutive tiles: neighbours share rows of Q or P
// in its L2, and all of them in the memory-side cache. The tiles' order from one
// 256 to the next stays, longest first where their sums differ.
__device__ __forceinline__ uint32_t tam_xcd_order(uint32_t b, uint32_t n) {
  const uint32_t base = b & ~255u, in = b & 255u, count = n - base < 256u ? n - base : 256u;
  const uint32_t x = in & 7u, q = count >> 3, r = count & 7u;
  return base + x * q + (x < r ? x : r) + (in >> 3);
}

// Tile t of tm x tn in groups of GROUP rows, column by column inside a group.
__device__ __forceinline__ void tam_tile_at(uint32_t t, uint32_t tm, uint32_t tn, uint32_t& m, uint32_t& n) {
  constexpr uint32_t GROUP = 8;
  const uint32_t per = GROUP * tn, g = t / per, left = t - g * per;
  const uint32_t rows = tm - g * GROUP < GROUP ? tm - g * GROUP : GROUP;
  n = left / rows;
  m = g * GROUP + left - n * rows;
}

// ---------------------------------------------------------------------------
// host side: what a launch of tiles takes
// ---------------------------------------------------------------------------
// Measured on one MI355X, tiles of k = 256 .. 4096 in launches of 16 to 1024 tiles
// (bf16; fp32 in the second table): a launch that leaves half of the compute units
// empty takes start + k * half us; with r tiles on each unit (at most `resident`
// fit: 160, 68 and 49, fp32 33, KB of LDS) start + k * per_k[r - 1]. At k = 4096 and
// 1024 tiles that is 1430 TFLOP/s for 256, 1150 for 128 and 640 for 64 (fp32: 145 and
// 134); 16 tiles of k = 256 take 12, 6 and 4 us.
struct tam_tile_rate {
  int tile, resident;
  double start, half, per_k[4];
};
static const tam_tile_rate tam_rates_16[3] = {{256, 1, 6.0, 0.0166, {0.0225}},
                                              {128, 2, 3.9, 0.0085, {0.0095, 0.0140}},
                                              {64, 3, 2.6, 0.0038, {0.0040, 0.0056, 0.0085}}};
static const tam_tile_rate tam_rates_32[2] = {{128, 2, 6.0, 0.0600, {0.0612, 0.1155}},
                                              {64, 4, 2.8, 0.0180, {0.0184, 0.0315, 0.0470, 0.0622}}};

// us of `tiles` tiles of k: whole rounds, then what is left.
static inline double tam_tiles_us(const tam_tile_rate& t, double tiles, double k, double cus) {
  const double round = cus * t.resident;
  const double full = (double)(uint64_t)(tiles / round), rest = tiles - full * round;
  double us = full * (0.5 * t.start + k * t.per_k[t.resident - 1]);
  if (rest > 0) {
    const int r = (int)((rest + cus - 1) / cus);
    us += t.start + k * (rest <= 0.5 * cus ? t.half : t.per_k[r - 1]);
  }
  return us;
}

#endif  // TAM_GEMM_H
