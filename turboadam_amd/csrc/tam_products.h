// tam_products.h -- host side of the layers' matrix products: operands as they lie in
// memory, aligned copies of those that the tiles cannot read, workspaces, and the choice of
// tile and parts.
#ifndef TAM_PRODUCTS_H
#define TAM_PRODUCTS_H

#include <initializer_list>

#include "tam_gemm.h"

// ---------------------------------------------------------------------------
// alignment
// ---------------------------------------------------------------------------
// dst[r][0 .. ld_dst) = src[r][0 .. cols) of up to three matrices of 16-bit units, one behind the other, zeros
// behind a row: a thread moves 8 units and none of their bits.
struct tam_align_item {
  const tam_f16* src;
  tam_f16* dst;
  uint64_t ld_src, rows, first;  // first: the items' units of 8 before this one's
  uint32_t cols, ld_dst;
};
struct tam_align_args {
  tam_align_item item[3];
  uint64_t units;
  int n;
};

static __global__ __launch_bounds__(256) void tam_k_align(tam_align_args a) {
  uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.units) return;
  tam_align_item m = a.item[0];
#pragma unroll
  for (int n = 1; n < 3; ++n)
    if (n < a.n && i >= a.item[n].first) m = a.item[n];
  i -= m.first;
  const uint32_t per = m.ld_dst / 8;
  const uint64_t r = i / per;
  const uint32_t c = (uint32_t)(i - r * per) * 8;
  *reinterpret_cast<tam_oct<tam_f16>*>(m.dst + r * m.ld_dst + c) =
      tam_some(m.src + r * m.ld_src + c, c < m.cols ? m.cols - c : 0);
}

// Zeros, whose bits are the same in every type, for n 16-bit units.
static __global__ __launch_bounds__(256) void tam_k_zeros(tam_f16* out, uint64_t n) {
  const float v[8] = {};
  for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (uint64_t)gridDim.x * 2048)
    tam_store_some(out + i, n - i < 8 ? (uint32_t)(n - i) : 8u, v);
}

namespace {

constexpr uint32_t kSize[3] = {4, 2, 2};

// One matrix as the products read it: rows of `cols` contiguous elements; whole: they
// are 16 bytes, or zeros follow up to that.
struct matrix {
  const void* p;
  uint64_t ld, rows;
  uint32_t cols;
  bool whole;
};

// Whether the products' loads can take m as it lies: rows that begin and end on 4 bytes.
inline bool in_words(const matrix& m, uint32_t size) {
  return (uint64_t)m.cols * size % 4 == 0 && m.ld * size % 4 == 0 && (uintptr_t)m.p % 4 == 0;
}

inline matrix matrix_of(const void* p, uint64_t ld, uint64_t rows, uint64_t cols, uint32_t size) {
  return {p, ld, rows, (uint32_t)cols, cols * size % 16 == 0};
}

// Rows of a copy: whole 128-byte lines (a tile's row then touches no line more than it fills).
inline uint32_t aligned_ld(uint32_t cols, uint32_t size) { return (uint32_t)tam_up(cols, 128 / size); }

// The workspace is laid out by walking the call twice: once without memory, to
// learn its size, and once with it.
struct arena {
  char* base;
  uint64_t used;
  void* take(uint64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += tam_up(bytes, 256);
    return p;
  }
};

struct call {
  uint32_t dtype;
  hipStream_t stream;
  arena ws;
  bool dry;  // lay out the workspace only
  uint32_t* tiles;  // where a product's tile and parts are told (tam_linear_tiles), or null
};

// CALL(T) with the type of call c.
#define TAM_OF_TYPE(c, CALL)                               \
  do {                                                     \
    if ((c).dtype == TAM_DTYPE_F32) {                      \
      CALL(float);                                         \
    } else if ((c).dtype == TAM_DTYPE_BF16) {              \
      CALL(tam_bf16);                                      \
    } else {                                               \
      CALL(tam_f16);                                       \
    }                                                      \
  } while (0)

// A launch takes fewer than 2^32 threads. Asked on both walks, so that the workspace's size is refused already.
inline int room(uint64_t workgroups, uint32_t threads) {
  if (workgroups < (1ull << 32) / threads) return TAM_OK;
  return tam_op_fail(TAM_E_UNSUPPORTED, "a launch of 2^32 threads or more");
}

// Of tiles, whose numbers are 31 bits; the largest take turns on the compute units where there are more (`turns`).
inline int room_of_tiles(uint64_t tiles, int tile, bool turns) {
  if (tile == 256 && turns && tiles < 1ull << 31) return TAM_OK;
  return room(tiles, tile == 256 ? 512 : 256);
}

// An empty sum: p, if it is wanted, of `elements`.
inline int zeros(const call& c, void* p, uint64_t elements) {
  if (c.dry || !p || !elements) return TAM_OK;
  const uint64_t halves = elements * (kSize[c.dtype] / 2), wgs = tam_div_up(halves, 2048);
  hipLaunchKernelGGL(tam_k_zeros, dim3((uint32_t)(wgs < 65536 ? wgs : 65536)), dim3(256), 0, c.stream, (tam_f16*)p, halves);
  TAM_OP_LAUNCHED("an empty sum");
  return TAM_OK;
}

// ---- products ----

struct shape {
  int tile;        // rows and columns of a tile
  uint32_t parts;  // the sum is cut into
};

// Which tile, and into how many parts the sum is cut: the least of the measured
// times (tam_tiles_us). Parts add their sums' way to memory and back (about 4 TB/s)
// and a launch.
inline shape choose(uint64_t rows, uint64_t cols, uint64_t k, uint32_t dtype) {
  const double cus = tam_op_cus();
  const bool f32 = dtype == TAM_DTYPE_F32;
  const tam_tile_rate* rate = f32 ? tam_rates_32 : tam_rates_16;
  shape best = {64, 1};
  double least = 1e30;
  for (int i = 0; i < (f32 ? 2 : 3); ++i) {
    const double tiles = (double)tam_div_up(rows, rate[i].tile) * (double)tam_div_up(cols, rate[i].tile);
    for (uint32_t parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (parts > 1 && k / parts < 128) break;
      double us = tam_tiles_us(rate[i], tiles * parts, (double)k / parts, cus);
      if (parts > 1) us += 3.0 + (double)rows * cols * 8.0 * parts / 4e6;
      if (us < least) {
        least = us;
        best = {rate[i].tile, parts};
      }
    }
  }
  return best;
}

// us of n1 units of k1 and n2 of k2 on the places of a card, the longer first: each unit to the place that
// is free first.
inline double units_us(const tam_tile_rate& t, uint64_t n1, double k1, uint64_t n2, double k2, double cus) {
  if (k1 < k2 && n2) return units_us(t, n2, k2, n1, k1, cus);
  const uint64_t places = (uint64_t)cus * t.resident, all = n1 + n2;
  const int with = all >= places ? t.resident : (int)tam_div_up(all ? all : 1, (uint64_t)cus);  // on a compute unit
  const double per = all <= (uint64_t)(0.5 * cus) ? t.half : t.per_k[with - 1];
  const double d1 = 0.5 * t.start + k1 * per, d2 = 0.5 * t.start + k2 * per;
  // two kinds of places: `late` of them have one unit more
  uint64_t late = n1 % places, rounds = n1 / places;
  double early_at = rounds * d1, late_at = late ? early_at + d1 : early_at;
  uint64_t early = places - late;
  while (n2) {
    double& at = early_at <= late_at || !late ? early_at : late_at;
    const uint64_t here = &at == &early_at ? early : late, take = n2 < here ? n2 : here;
    if (take < here) return 0.5 * t.start + (at + d2 > late_at ? at + d2 : late_at);
    at += d2;
    n2 -= take;
  }
  return 0.5 * t.start + (late && late_at > early_at ? late_at : early_at);
}

// Copies, in rows of whole lines, in place of those matrices that are given. All are one launch (three of 5 us each
// were a tenth of a small layer's time). Matrices of no elements stay: nothing of them is read.
inline int copy_rows(call& c, std::initializer_list<matrix*> all) {
  const uint32_t size = kSize[c.dtype], halves = size / 2;
  tam_align_args a = {};
  for (matrix* m : all) {
    if (!m || !m->cols || !m->rows) continue;
    const uint32_t ld = aligned_ld(m->cols, size);
    void* p = c.ws.take(m->rows * ld * size);
    a.item[a.n] = {(const tam_f16*)m->p, (tam_f16*)p, m->ld * halves, m->rows, a.units, m->cols * halves, ld * halves};
    a.units += m->rows * (ld * halves / 8);
    ++a.n;
    *m = {p, ld, m->rows, m->cols, true};
  }
  const int rc = room(tam_div_up(a.units, 256), 256);
  if (rc != TAM_OK || c.dry || !a.n) return rc;
  hipLaunchKernelGGL(tam_k_align, dim3((uint32_t)tam_div_up(a.units, 256)), dim3(256), 0, c.stream, a);
  TAM_OP_LAUNCHED("the aligned copies");
  return TAM_OK;
}

// The matrices, or copies of them: rows of whole 16 bytes that begin on 4, for kernels without a REST form.
inline int whole_rows(call& c, matrix* m0, matrix* m1 = nullptr, matrix* m2 = nullptr) {
  const uint32_t size = kSize[c.dtype];
  for (matrix** m : {&m0, &m1, &m2})
    if (*m && in_words(**m, size) && (*m)->whole) *m = nullptr;
  return copy_rows(c, {m0, m1, m2});
}

// m as an operand of a product: `count` rows or columns of it are the operand's.
inline tam_operand operand_of(const matrix& m, uint32_t count, uint32_t size) {
  const char* base = (const char*)m.p;
  const uint64_t bytes = m.rows ? (m.rows - 1) * m.ld * size + tam_up((uint64_t)m.cols * size, m.whole ? 16 : 1) : 0;
  return {base, m.ld * size, count, base + bytes};
}

}  // namespace

#endif  // TAM_PRODUCTS_H
