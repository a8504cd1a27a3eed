// Attention over pages, cut into units: a unit is a (sequence, key/value head, tile of query rows), its work the
// tiles of positions that its rows see.  Query rows of a head are (new token, query head of the group), tokens first.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "paged.cuh"
#include "ptx.cuh"

namespace dsb {
namespace paged {

// A row's maximum: kFloor before it has seen a position, kSeen at least after it; scores at or below kSeen weigh nothing.
constexpr float kFloor = -3.40282347e38f, kSeen = -3.39e38f;
constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a row's result is multiplied with. No weight: zero for a row that sees nothing, NaN (nothing over nothing) for one
// whose scores are all -inf.
__device__ __forceinline__ float over_sum(float sum, float top) {
  return sum != 0.f ? 1.f / sum : top > kFloor ? __uint_as_float(0x7fc00000u) : 0.f;
}
// The largest, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Four codes as two registers of fp16 pairs: bytes 0, 1 and 2, 3 (K: neighbours of a row), or, crossed, 0, 2 and 1, 3
// (V: ldmatrix transposed pairs of columns, a register holds two columns of two positions).  int8: 0x6400 + u is the
// fp16 number 1024 + u, u = code + 128.
template <int KIND, bool CROSSED>
__device__ __forceinline__ uint2 codes_to_f16(uint32_t x) {
  uint2 r;
  if (KIND == kInt8) {
    x ^= 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, CROSSED ? 0x4240 : 0x4140), b = __byte_perm(x, 0x64646464u, CROSSED ? 0x4341 : 0x4342);
    const uint32_t off = 0x64806480u;                    // 1152 twice
    const __half2 u = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&off));
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
    r.x = *reinterpret_cast<const uint32_t*>(&u);
    r.y = *reinterpret_cast<const uint32_t*>(&v);
    return r;
  }
  if (CROSSED) x = __byte_perm(x, 0u, 0x3120);
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
      : "=r"(r.x), "=r"(r.y) : "r"(x));
  return r;
}

// Division of numbers below 2^31 by a number that the host knows: with 2^s the power of two from d on,
// m = ceil(2^(31 + s) / d) exceeds the quotient by less than 1, so that x m / 2^(31 + s) exceeds x / d by less than
// x / 2^(31 + s) < 1 / d, too little to reach the next whole number.
struct Divisor {
  uint32_t m;
  int shift;
  __device__ __forceinline__ int operator()(int x) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * m) >> shift);
  }
};
inline Divisor make_divisor(int d) {
  int s = 0;
  while ((1LL << s) < d) ++s;
  return {static_cast<uint32_t>(((1ULL << (31 + s)) + d - 1) / d), 31 + s};
}

// Rows of zeros are stored under a scale of 1, which says nothing of their size: beside rows with small scales it would set
// the measure that fp16 numbers are relative to. Where a scale of 1 is met the codes are looked at.
constexpr float kZeroRow = 1.f;
template <int KIND>
__device__ __forceinline__ bool zero_codes(uint32_t x) { return (KIND == kE4m3 ? x & 0x7f7f7f7fu : x) == 0u; }
template <int KIND>
__device__ __forceinline__ bool zero_codes(const uint4& x) { return zero_codes<KIND>(x.x | x.y | x.z | x.w); }

struct AttnParams {
  View w;
  const __nv_bfloat16* q;           // [N, Hq, dh], strides in elements
  long long q_st, q_sh;
  __nv_bfloat16* out;               // [N, Hq, dh]
  int Hq, G;
  Divisor by_g;                     // row -> token
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
  const int i0 = p.by_g(r0), i1 = p.by_g(r0 + u.rows - 1);
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
  const int len = seq_length(p.w, b);              // all loads at once
  const Rows r = seq_rows(p.w, b);
  u.first = r.first;
  u.n = r.count;
  u.len = u.n > 0 ? len : 0;
}

// Tiles of the units of one head of sequence i + lane: a lane's own arithmetic for a sequence of one row tile, the
// warp's for one of many.
template <int ROWS, int TP>
__device__ __forceinline__ long long head_tiles(const AttnParams& p, int i, int lane) {
  Unit u;
  int nrt = 0;
  long long x = 0;
  u.len = u.n = 0;
  if (i + lane < p.w.c.B) {
    unit_sequence(p, u, i + lane);
    nrt = row_tiles<ROWS>(u.n, p.G);
    if (nrt == 1) {
      u.rt = 0;
      unit_range<ROWS, TP>(p, u);
      x = u.tiles;
    }
  }
  for (unsigned many = __ballot_sync(0xffffffffu, nrt > 1); many != 0u; many &= many - 1) {
    const int k = __ffs(many) - 1, n = __shfl_sync(0xffffffffu, nrt, k);
    Unit v;
    v.len = __shfl_sync(0xffffffffu, u.len, k);
    v.n = __shfl_sync(0xffffffffu, u.n, k);
    long long sum = 0;
    for (v.rt = lane; v.rt < n; v.rt += 32) {
      unit_range<ROWS, TP>(p, v);
      sum += v.tiles;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == k) x = sum;
  }
  return x;
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

// Row `row` (token, query head of the group) of key/value head h of a sequence.
__device__ __forceinline__ __nv_bfloat16* out_row(const AttnParams& p, int first, int h, int row) {
  const int t = p.by_g(row);
  return p.out + (static_cast<size_t>(first + t) * p.Hq + h * p.G + (row - t * p.G)) * p.w.c.dh;
}
__device__ __forceinline__ __nv_bfloat16* out_row(const AttnParams& p, const Unit& u, int row) { return out_row(p, u.first, u.h, row); }

// A worker's run of tiles, among all tiles of all units in order (sequence, head, row tile), and the sequence of its
// first one: its tiles of a head, and how many tiles come before it.
struct Run { long long begin, end, per_head, before; int b; };

// Equal runs: worker i of n takes tiles [i T / n, (i + 1) T / n).
template <int ROWS, int TP>
__device__ __forceinline__ Run share(const AttnParams& p, int lane, long long worker, int least) {
  const int B = p.w.c.B;
  const long long H = p.w.c.H;
  long long total = 0, x = 0;
  for (int i = 0; i < B; i += 32) {
    x = head_tiles<ROWS, TP>(p, i, lane);
    long long sum = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    total += sum * H;
  }
  const long long most = total / least;
  const long long n = most < 1 ? 1 : most < p.workers ? most : p.workers;
  Run r = {0, 0, 0, 0, 0};
  if (worker >= n) return r;
  // i T / n = i (T / n) + i (T mod n) / n, in 32 bits where T fits them: a 64-bit division costs some 500 cycles
  if (total <= 0x7fffffffLL) {
    const uint32_t t = static_cast<uint32_t>(total), d = static_cast<uint32_t>(n), w = static_cast<uint32_t>(worker);
    const uint32_t whole = t / d, rest = t - whole * d;              // rest, w + 1 <= n: their product fits
    r.begin = static_cast<long long>(w) * whole + w * rest / d;
    r.end = static_cast<long long>(w + 1) * whole + (w + 1) * rest / d;
  } else {
    r.begin = worker * total / n;
    r.end = (worker + 1) * total / n;
  }
  for (int i = 0; i < B; i += 32) {                    // the sequence that holds tile r.begin
    if (B > 32) x = head_tiles<ROWS, TP>(p, i, lane);
    long long c = x * H;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, c, d);
      if (lane >= d) c += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, r.before + c > r.begin);
    if (past != 0u) {
      const int k = __ffs(past) - 1;
      r.b = i + k;
      r.per_head = __shfl_sync(0xffffffffu, x, k);
      r.before += __shfl_sync(0xffffffffu, c, k) - r.per_head * H;
      return r;
    }
    r.before += __shfl_sync(0xffffffffu, c, 31);
  }
  return r;
}

// A piece of a unit in the workspace: per row maximum and sum, then O.  Worker i has two: 2 i + 1 for a unit that begins
// in its run and ends in a later one, 2 i for one that began in an earlier run.
template <int ROWS>
__host__ __device__ constexpr int piece_floats(int dh) { return ROWS * (dh + 2); }

// A worker's segments: what of each unit lies in its run.
template <int ROWS, int TP>
struct Segments {
  Unit u;
  int nrt, t0, t1;                  // row tiles of the sequence; tiles [t0, t1) of the unit
  long long at, end;

  __device__ __forceinline__ bool on() const { return at < end; }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == u.tiles; }
  __device__ __forceinline__ int slot() const { return t0 == 0 ? 1 : 0; }        // of the worker's two pieces

  // Of a unit that other workers share: where it begins (x, y, z), or that it ends here (w).
  __device__ __forceinline__ void note(int4& meta) const {
    if (whole()) return;
    if (t0 == 0) {
      meta.x = u.b;
      meta.y = u.h;
      meta.z = u.rt;
    } else if (t1 == u.tiles) {
      meta.w = 1;
    }
  }

  __device__ void begin(const AttnParams& p, int lane, int worker, int least) {
    const Run run = share<ROWS, TP>(p, lane, worker, least);
    at = run.begin;
    end = run.end;
    if (!on()) return;
    unit_sequence(p, u, run.b);
    nrt = row_tiles<ROWS>(u.n, p.G);
    const long long off = at - run.before;
    u.h = off >> 31 == 0 && run.per_head >> 31 == 0
              ? static_cast<int>(static_cast<uint32_t>(off) / static_cast<uint32_t>(run.per_head))
              : static_cast<int>(off / run.per_head);
    long long left = off - u.h * run.per_head;         // tiles of the head before the first one
    u.rt = 0;
    for (int base = 0; nrt > 1 && base < nrt; base += 32) {
      Unit v = u;
      v.rt = base + lane;
      int x = 0;
      if (v.rt < nrt) {
        unit_range<ROWS, TP>(p, v);
        x = v.tiles;
      }
      int c = x;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, c, d);
        if (lane >= d) c += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, c > left);
      const int k = past != 0u ? __ffs(past) - 1 : 31;
      u.rt = base + k;
      left -= __shfl_sync(0xffffffffu, past != 0u ? c - x : c, k);
      if (past != 0u) break;
    }
    unit_range<ROWS, TP>(p, u);
    t0 = static_cast<int>(left);
    t1 = static_cast<int>(min(static_cast<long long>(u.tiles), t0 + (end - at)));
  }

  __device__ void next(const AttnParams& p) {
    at += t1 - t0;
    if (!on()) return;
    if (++u.rt >= nrt) {
      u.rt = 0;
      if (++u.h >= p.w.c.H) {
        u.h = 0;
        do {
          unit_sequence(p, u, u.b + 1);
          nrt = row_tiles<ROWS>(u.n, p.G);
        } while (nrt == 0);
      }
    }
    unit_range<ROWS, TP>(p, u);
    t0 = 0;
    t1 = static_cast<int>(min(static_cast<long long>(u.tiles), end - at));
  }
};

// ---- Units computed again.  Products of whole tiles hand a value that is no number on to rows that do not see it: a weight
// of zero times NaN or inf is NaN.  It shows in an O that is not finite beside a finite sum of weights; then the positions
// that only some of the unit's rows see are looked through, and if one holds such a value the work is done again row by row,
// position by position, without touching what a row does not see.  Hundreds of times slower (ragged prompts with one NaN, 16 heads of
// 128, 3.4 ms for 0.09; all 4099 x 6000 positions of an int8 chunk 39 ms for 0.19), and for diverged caches alone.

// NaN if x, or a term before it, is not finite.
__device__ __forceinline__ float track_odd(float odd, float x) { return fmaf(x, 0.f, odd); }

template <int KIND>
__device__ __forceinline__ bool odd_codes(uint32_t x) {
  return KIND == kBf16 ? (((x & 0x7fff7fffu) + 0x00800080u) & 0x80008000u) != 0u      // exponents of ones carry
                       : (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u;     // e4m3: and fractions
}

// Does a position that only some of the unit's rows see hold a value that is no number?  Threads `who` of `of`.
template <int KIND>
__device__ __noinline__ bool odd_values(const AttnParams& p, const Unit u, int who, int of) {
  if (KIND == kInt8) return false;
  const int words = p.w.c.dh * (KIND == kBf16 ? 2 : 1) >> 4;
  const int early = min(u.lo_all, u.hi) - u.lo, late = max(u.hi_all, u.lo);        // [lo, lo_all), [hi_all, hi)
  const long long n = static_cast<long long>(max(early, 0) + max(u.hi - late, 0)) * words;
  for (long long i = who; i < n; i += of) {
    const int x = static_cast<int>(i / words), word = static_cast<int>(i % words);
    const int pos = x < early ? u.lo + x : late + x - max(early, 0), page = page_of(p.w, u.b, pos);
    if (page < 0) continue;
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.w.c.v) +
                                                         slot_row(p.w, page, u.h, pos) * (16 * words)) + word);
    if (odd_codes<KIND>(v.x) || odd_codes<KIND>(v.y) || odd_codes<KIND>(v.z) || odd_codes<KIND>(v.w)) return true;
  }
  return false;
}

// Eight values from element `at` of a pool on, without their scale.
template <int KIND>
__device__ __forceinline__ void held8(const void* pool, size_t at, float* f) {
  if (KIND == kBf16) {
    bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(pool) + at)), f);
    return;
  }
  const uint2 x = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at));
  const uint2 a = codes_to_f16<KIND, false>(x.x), c = codes_to_f16<KIND, false>(x.y);
  const uint32_t h[4] = {a.x, a.y, c.x, c.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(h + i));
    f[2 * i] = y.x;
    f[2 * i + 1] = y.y;
  }
}

// Rows r0, r0 + r_step, .. of a unit over its tiles t0, t0 + step, .. below t1, by a warp, in fp32.  ml null: the results, in
// bf16.  Otherwise maximum and sum of row r at ml + 2 r, its columns 4 c .. at o + r * row_stride + c * col_stride, sum and O
// times `up`.
template <int KIND, int ROWS, int TP>
__device__ __noinline__ void rows_again(const AttnParams& p, const Unit u, int t0, int t1, int step, int r0, int r_step,
                                        int lane, float* ml, float* to, int row_stride, int col_stride, float up) {
  const int dh = p.w.c.dh, half = lane >> 4, col = 8 * (lane & 15);
  for (int r = r0; r < u.rows; r += r_step) {
    const int row = u.rt * ROWS + r, t = p.by_g(row), pos = u.len - u.n + t;
    const __nv_bfloat16* q = p.q + static_cast<long long>(u.first + t) * p.q_st + static_cast<long long>(u.h * p.G + row - t * p.G) * p.q_sh;
    float m = kFloor, l = 0.f, o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
    for (int tile = t0; tile < t1; tile += step)
      for (int x0 = (tile < u.st ? tile : tile + u.skip) * TP, x1 = x0 + TP; x0 < x1; x0 += 32) {
        const int j = x0 + lane;
        const int page = j < x1 && j <= pos && (j > pos - p.window || j < p.sinks) ? page_of(p.w, u.b, j) : -1;
        const bool on = page >= 0;
        const unsigned seen = __ballot_sync(0xffffffffu, on);
        if (seen == 0u) continue;
        const size_t at = on ? slot_row(p.w, page, u.h, j) : 0;
        float s = 0.f, vs = 1.f;
        if (on) {
#pragma unroll 4
          for (int c = 0; c < dh; c += 8) {
            float a[8], k[8];
            bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(q + c)), a);
            held8<KIND>(p.w.c.k, at * dh + c, k);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(a[e], k[e], s);
          }
          if (KIND != kBf16) {
            s *= __ldg(p.w.c.k_scale + at);
            vs = __ldg(p.w.c.v_scale + at);
          }
          s *= p.scale_log2;
        }
        float top = on ? max_nan(s, kSeen) : kFloor;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float m_new = max_nan(m, top), d = exp2_fast(m - m_new), w = on ? exp2_fast(s - m_new) : 0.f;
        l = fmaf(l, d, w);
        m = m_new;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] *= d;
#pragma unroll 8
        for (int k = 0; k < 32; k += 2) {              // half a warp a position
          const int from = k + half;
          const float y = __shfl_sync(0xffffffffu, w, from), z = __shfl_sync(0xffffffffu, vs, from);
          const unsigned long long at_k = __shfl_sync(0xffffffffu, static_cast<unsigned long long>(at), from);
          const bool mine = ((seen >> from) & 1u) && col < dh;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.f;
          if (mine) held8<KIND>(p.w.c.v, at_k * dh + col, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = mine ? fmaf(y, v[e] * z, o[e]) : o[e];
        }
      }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] += __shfl_xor_sync(0xffffffffu, o[k], 16);
    if (half != 0 || col >= dh) continue;
    if (ml == nullptr) {
      const float inv = over_sum(l, m);
      *reinterpret_cast<uint4*>(out_row(p, u, row) + col) =
          make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv),
                     pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
    } else {
      if (lane == 0) {
        ml[2 * r] = m;
        ml[2 * r + 1] = l * up;
      }
      float* x = to + static_cast<size_t>(r) * row_stride + static_cast<size_t>(col / 4) * col_stride;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = o[k] * up;
        x[col_stride + k] = o[4 + k] * up;
      }
    }
  }
}

constexpr int kMergeThreads = 256;
constexpr int kMergeChunk = 64;        // pieces whose weights are at hand at a time

// The unit that worker i left for others to end, and the worker that ends it (all lanes of a warp).
template <int ROWS>
__device__ __forceinline__ bool shared_unit(const AttnParams& p, int i, int lane, Unit& u, int& last) {
  const int4 meta = p.meta[i];
  if (meta.x < 0) return false;
  u.b = meta.x;
  u.h = meta.y;
  u.rt = meta.z;
  const Rows r = seq_rows(p.w, u.b);
  u.first = r.first;
  u.n = r.count;
  u.rows = min(ROWS, u.n * p.G - u.rt * ROWS);
  int j = i + 1;
  for (;; j += 32) {
    const int k = j + lane;
    const unsigned end = __ballot_sync(0xffffffffu, k >= p.workers || p.meta[k].w != 0);
    if (end != 0u) {
      j += __ffs(end) - 1;
      break;
    }
  }
  last = min(j, p.workers - 1);
  return true;
}

// Units of few rows and many pieces: a block per worker whose last unit goes on in later runs.  A few threads would
// wait for one piece after the other, so groups of threads take every n-th piece each; sums in a fixed order.
template <int ROWS>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_few_kernel(const AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s_w[kMergeChunk][ROWS];
  __shared__ float s_top[ROWS], s_inv[ROWS];
  __shared__ __align__(16) float4 s_sum[kMergeThreads];
  const int i = blockIdx.x, dh = p.w.c.dh, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Unit u;
  int last;
  if (!shared_unit<ROWS>(p, i, lane, u, last)) return;
  const int stride = piece_floats<ROWS>(dh), per = dh / 4;
  auto piece = [&](int j) { return p.part + (2 * static_cast<size_t>(j) + (j == i ? 1 : 0)) * stride; };
  for (int r = warp; r < u.rows; r += kMergeThreads / 32) {
    float top = kFloor;
    for (int j = i + lane; j <= last; j += 32) top = fmaxf(top, piece(j)[2 * r]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float sum = 0.f;
    for (int j = i + lane; j <= last; j += 32) sum = fmaf(exp2_fast(piece(j)[2 * r] - top), piece(j)[2 * r + 1], sum);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) {
      s_top[r] = top;
      s_inv[r] = over_sum(sum, top);
    }
  }
  const int tasks = u.rows * per;                      // float4s of the unit
  const int groups = tasks >= kMergeThreads ? 1 : kMergeThreads / tasks;
  const int grp = groups == 1 ? 0 : tid / tasks, at = groups == 1 ? tid : tid - grp * tasks;
  constexpr int kRounds = (ROWS * 32 + kMergeThreads - 1) / kMergeThreads;
  float4 a[kRounds];
  int row[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int task = at + k * kMergeThreads;
    row[k] = task < tasks && grp < groups && (k == 0 || groups == 1) ? task / per : -1;
  }
  for (int j0 = i; j0 <= last; j0 += kMergeChunk) {
    const int n = min(kMergeChunk, last + 1 - j0);
    __syncthreads();
    for (int x = tid; x < n * ROWS; x += kMergeThreads) {
      const int j = x / ROWS, r = x % ROWS;
      if (r < u.rows) s_w[j][r] = exp2_fast(piece(j0 + j)[2 * r] - s_top[r]);
    }
    __syncthreads();
#pragma unroll 4
    for (int j = grp; j < n; j += groups) {
      const float4* from = reinterpret_cast<const float4*>(piece(j0 + j) + 2 * ROWS) + at;
#pragma unroll
      for (int k = 0; k < kRounds; ++k) {
        if (row[k] >= 0) {
          const float4 o = __ldcg(from + k * kMergeThreads);
          const float w = s_w[j][row[k]];
          a[k].x = fmaf(w, o.x, a[k].x);
          a[k].y = fmaf(w, o.y, a[k].y);
          a[k].z = fmaf(w, o.z, a[k].z);
          a[k].w = fmaf(w, o.w, a[k].w);
        }
      }
    }
  }
  if (groups > 1) {
    s_sum[tid] = a[0];
    __syncthreads();
    if (grp != 0) return;
    for (int x = 1; x < groups; ++x) {
      const float4 o = s_sum[at + x * tasks];
      a[0].x += o.x;
      a[0].y += o.y;
      a[0].z += o.z;
      a[0].w += o.w;
    }
  }
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    if (row[k] < 0) continue;
    const int r = row[k], c = 4 * (at + k * kMergeThreads - r * per);
    *reinterpret_cast<uint2*>(out_row(p, u, u.rt * ROWS + r) + c) =
        make_uint2(pack_bf16x2(a[k].x * s_inv[r], a[k].y * s_inv[r]), pack_bf16x2(a[k].z * s_inv[r], a[k].w * s_inv[r]));
  }
}

// Launches a kernel that waits by itself (griddepcontrol.wait) for the stream's earlier work before it reads anything:
// its blocks may be set up while that work ends.
template <typename F, typename P>
int launch_early(F* kernel, dim3 grid, int threads, int smem, const P& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? 0 : 946;
}

inline long long workspace_bytes(long long workers, int rows, int dh) {
  return workers * static_cast<long long>(sizeof(int4)) + 2 * workers * rows * (dh + 2) * static_cast<long long>(sizeof(float));
}

// What a launcher asks of a device once, not in every call.
constexpr int kDevices = 64;
inline int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kDevices ? dev : 0;
}
inline int device_sms() {
  static std::atomic<int> sms[kDevices];
  const int dev = current_device();
  int n = sms[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    n = n > 0 ? n : 148;
    sms[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
// Lets a kernel have up to `bytes` of dynamic shared memory; `most` is the kernel's own memory of what it may have.
template <typename F>
int allow_smem(F* kernel, int bytes, std::atomic<int> (&most)[kDevices]) {
  const int dev = current_device();
  if (most[dev].load(std::memory_order_relaxed) >= bytes) return 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return 944;
  most[dev].store(bytes, std::memory_order_relaxed);
  return 0;
}

}  // namespace paged
}  // namespace dsb
