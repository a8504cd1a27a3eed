// Attention over pages, cut into units: a unit is a (sequence, key/value head, tile of query rows), its work the
// tiles of positions that its rows see.  Query rows of a head are (new token, query head of the group), tokens first.
#pragma once
#include "paged.cuh"

namespace dsb {
namespace paged {

struct AttnParams {
  View w;
  const __nv_bfloat16* q;           // [N, Hq, dh], strides in elements
  long long q_st, q_sh;
  __nv_bfloat16* out;               // [N, Hq, dh]
  int Hq, G;
  int window, sinks;                // window: kMostPositions without one
  float scale_log2;                 // scale * log2(e)
  float* part;                      // pieces of units that several workers share
  int4* meta;
  int workers;
};

// What of the positions a unit's rows see: [0, s_end) and [lo, hi).
struct Unit {
  int b, h, rt;                     // sequence, head, row tile
  int len, n, first;                // length, new tokens, first packed row of the sequence
  int rows;                         // rows of this tile
  int lo, hi, s_end;
  int lo_all, hi_all;               // [lo_all, hi_all): positions that every row of the tile sees (may be none)
  int st, skip, tiles;              // tile t of the unit is position tile t (t < st) or t + skip
};

template <int ROWS>
__device__ __forceinline__ int row_tiles(int n, int G) { return (n * G + ROWS - 1) / ROWS; }

// Fills in what depends on the row tile; b, h, rt, len, n, first are set.
template <int ROWS, int TP>
__device__ __forceinline__ void unit_range(const AttnParams& p, Unit& u) {
  const int r0 = u.rt * ROWS;
  u.rows = min(ROWS, u.n * p.G - r0);
  const int i0 = r0 / p.G, i1 = (r0 + u.rows - 1) / p.G;
  const int p_lo = u.len - u.n + i0, p_hi = u.len - u.n + i1;
  u.hi = max(p_hi + 1, 0);
  u.lo = max(0, p_lo - p.window + 1);             // p_lo >= -N, N and window at most 2^30: no overflow
  u.lo = min(u.lo, u.hi);
  u.s_end = min(p.sinks, u.lo);
  u.lo_all = max(0, p_hi - p.window + 1);
  u.hi_all = p_lo + 1;
  u.st = (u.s_end + TP - 1) / TP;
  const int t_lo = max(u.lo / TP, u.st), t_hi = (u.hi + TP - 1) / TP;
  u.skip = t_lo - u.st;
  u.tiles = max(u.st + max(t_hi - t_lo, 0), 1);   // a unit without positions writes its zeros
}

__device__ __forceinline__ void unit_sequence(const AttnParams& p, Unit& u, int b) {
  u.b = b;
  const Rows r = seq_rows(p.w, b);
  u.first = r.first;
  u.n = r.count;
  u.len = u.n > 0 ? seq_length(p.w, b) : 0;
}

// Tiles of all units of sequence b.
template <int ROWS, int TP>
__device__ __forceinline__ long long sequence_tiles(const AttnParams& p, int b) {
  Unit u;
  unit_sequence(p, u, b);
  long long sum = 0;
  const int nrt = row_tiles<ROWS>(u.n, p.G);
  for (u.rt = 0; u.rt < nrt; ++u.rt) {
    unit_range<ROWS, TP>(p, u);
    sum += u.tiles;
  }
  return sum * p.w.c.H;
}

// Rows of no sequence (before the first and behind the last one) are zero.
__device__ __forceinline__ void zero_other_rows(const AttnParams& p, int worker, int workers) {
  if (p.w.c.starts == nullptr) return;
  const int B = p.w.c.B, N = p.w.c.N;
  const int a = B > 0 ? min(max(p.w.c.starts[0], 0), N) : N, e = B > 0 ? min(max(p.w.c.starts[B], a), N) : N;
  const int per = p.Hq * p.w.c.dh / 8;             // 16-byte words of a row
  const long long words = static_cast<long long>(N - e + a) * per;
  for (long long i = worker; i < words; i += workers) {
    long long row = i / per;
    if (row >= a) row += e - a;
    reinterpret_cast<uint4*>(p.out)[row * per + i % per] = make_uint4(0u, 0u, 0u, 0u);
  }
}

}  // namespace paged
}  // namespace dsb
