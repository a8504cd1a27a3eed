// Device-side view of a paged key/value cache: which sequence a packed row belongs to, where a
// position lives, and 8-bit codes as bf16 (for reading back; the attention's conversions are in paged_units.cuh).
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "../dsb_api_paged.h"

namespace dsb {
namespace paged {

constexpr int kStatusBadPage = 4;   // a table entry or a length outside the cache

constexpr int kMostPositions = 1 << 30;   // of a sequence, and packed rows: sums of two stay in 32 bits

enum Kind { kBf16 = 0, kE4m3 = 1, kInt8 = 2 };

struct View {
  DsbPaged c;
  int shift;                        // log2(page)
};

inline View make_view(const DsbPaged* c) {
  View w;
  w.c = *c;
  w.shift = 0;
  while ((1 << w.shift) < c->page) ++w.shift;
  return w;
}

// What the launchers refuse (the kernels' vector accesses and shifts rely on it).
inline bool bad_cache(const DsbPaged* c) {
  if (c->kind < 0 || c->kind > 2 || c->dh < 16 || c->dh > 128 || c->dh % 16 != 0) return true;
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)) != 0) return true;
  if (c->H <= 0 || c->n_pages < 0 || c->B < 0 || c->width < 0 || c->N < 0) return true;
  if (c->N > kMostPositions || static_cast<long long>(c->width) * c->page > kMostPositions) return true;
  if (c->starts == nullptr && c->N != c->B) return true;
  if (c->kind != kBf16 && c->n_pages > 0 && (c->k_scale == nullptr || c->v_scale == nullptr)) return true;
  // scales are copied four at a time
  if (c->kind != kBf16 && ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 15) != 0) return true;
  return ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) != 0;
}

struct Rows { int first, count; };  // packed rows of a sequence

__device__ __forceinline__ Rows seq_rows(const View& w, int b) {
  if (w.c.starts == nullptr) return {b, 1};
  const int a = min(max(w.c.starts[b], 0), w.c.N), e = min(max(w.c.starts[b + 1], a), w.c.N);
  return {a, e - a};
}

// Positions of sequence b: what the table can hold at most.
__device__ __forceinline__ int seq_length(const View& w, int b) {
  const int len = w.c.lengths[b];
  const long long cap = static_cast<long long>(w.c.width) << w.shift;
  if (len > cap) {
    atomicExch(w.c.status, kStatusBadPage);
    return static_cast<int>(cap);
  }
  return max(len, 0);
}

// The sequence that packed row t belongs to, or -1 (rows before the first or behind the last one); by a whole warp.
__device__ __forceinline__ int seq_of_row_warp(const View& w, int t, int lane) {
  if (w.c.starts == nullptr) return t;
  int b = 0;                                       // how many sequences end at or before t
  for (int i = 0; i < w.c.B; i += 32) {
    const unsigned past = __ballot_sync(0xffffffffu, i + lane < w.c.B && w.c.starts[i + lane + 1] <= t);
    b += __popc(past);
    if (past != 0xffffffffu) break;
  }
  return b < w.c.B && w.c.starts[b] <= t ? b : -1;
}

// Page of position `pos` of sequence b, or -1 where the table names none of the pool.
__device__ __forceinline__ int page_of(const View& w, int b, int pos) {
  const int id = w.c.table[static_cast<size_t>(b) * w.c.width + (pos >> w.shift)];
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(w.c.n_pages)) {
    atomicExch(w.c.status, kStatusBadPage);
    return -1;
  }
  return id;
}

// Index of (page, head, slot of pos) among the rows of the pool: times dh for elements.
__device__ __forceinline__ size_t slot_row(const View& w, int page, int h, int pos) {
  return ((static_cast<size_t>(page) * w.c.H + h) << w.shift) + (pos & (w.c.page - 1));
}

// Four 8-bit codes -> four bf16 (two registers), exactly, without a conversion instruction.
// int8: 128 + (low seven bits) and 128 or 256 (by the sign bit) are bf16 values whose bits are the code's
// own; their difference is the number.  e4m3: exponent and fraction moved into bf16's places read as the
// value times 2^-120 (the biases differ by 120, subnormals included), so one product puts it right.  The
// NaN codes 0x7f, 0xff, which no write here makes, come out as +-480: the caller looks for them.
template <int KIND>
__device__ __forceinline__ uint2 codes_to_bf16(uint32_t x) {
  uint2 r = {__byte_perm(x, 0u, 0x4140), __byte_perm(x, 0u, 0x4342)};
  auto one = [](uint32_t p) -> uint32_t {
    if (KIND == kInt8) {
      const uint32_t a = (p & 0x007f007fu) | 0x43004300u, b = (p & 0x00800080u) | 0x43004300u;
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                       *reinterpret_cast<const __nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&d);
    }
    const uint32_t a = ((p & 0x007f007fu) << 4) | ((p & 0x00800080u) << 8), s = 0x7b807b80u;   // 2^120 twice
    const __nv_bfloat162 d = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&s));
    return *reinterpret_cast<const uint32_t*>(&d);
  };
  r.x = one(r.x);
  r.y = one(r.y);
  return r;
}

__device__ __forceinline__ void bf16x8_to_f32(const uint4& u, float* f) {
  const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(r[i] << 16);
    f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
  }
}

}  // namespace paged
}  // namespace dsb
