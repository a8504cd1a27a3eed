// Attention of a few query rows per key/value head (single tokens, drafted ones) over a paged cache.
//
// Each warp streams tiles of positions through a ring of its own in shared memory (16-byte asynchronous copies; the
// sixteen positions of a head in a page are contiguous) and multiplies with m16n8k16 instructions:
//   S^T [positions, rows] = K Q^T        K the M side: eight rows fill the N side, so that one row costs what eight do
//                                        and the scores of a tile stay in registers;
//   O^T [dh, rows]       += V^T P^T      V^T the M side, by transposing ldmatrix; P is transposed by movmatrix.
// 8-bit codes go through ldmatrix as pairs and become fp16 in registers, exactly (an instruction for two e4m3 codes;
// two and a half for two int8 ones); any order of the contraction will do as long as both operands have it, so a
// lane's queries are those of the four neighbouring codes it gets.  Queries, bf16, become fp16 by a power of two for
// each row that brings the largest to [128, 256): exact down to 2^-22 of it, off by 2^-33 of it below.  The keys'
// scales go to the scores in fp32, the values' to the exponents (see below).  Running maximum and sum stay in registers.
// Drafted tokens that do not all see a value that is no number have their rows done again (work_again).
//
// Two ways to share the work.  Where a warp has few tiles, a cluster of blocks takes a unit, its warps every n-th tile,
// and merges in (distributed) shared memory: one launch.  For long caches as many warps as the GPU holds take equal
// runs of consecutive tiles of all units, whatever the sequences' lengths; a unit that several warps share is left in
// pieces, which a second kernel adds up in order.  The lengths are read on the device, so a captured call follows them.
//
// What bounds it.  Reading the keys and values once is the floor (6.5 TB/s).  Six e4m3 sequences of 2000 to 32000, 16
// heads of 80: 54 us for 37, 4.6 TB/s: the rest is the plan, the merge of pieces (7 us together) and the conversion of
// codes, half of the instructions issued.  32 bf16 sequences of 100 to 512, 16 heads of 128: 17 us for 10; one of 290,
// 6 heads of 64: 6 us, a launch, three dependent loads (length, table, page) and a merge.  Four query heads or more per
// head of the cache cost twice the instructions of one: 16 int8 sequences under a window of 4096, 32 query heads over
// 4: 20 us for 9; five drafted tokens of 8 bf16 sequences, 16 over 8 heads of 64: 15 us for 3, the longest sequence
// (6000) being 30 times the shortest in clusters of equal size.
#include "common/paged_launch.h"
#include "common/ptx.cuh"

namespace dsb {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr float kZeroScale = 8.67361738e-19f;    // 2^-60: counts as the scale of a row of zeros, whose weight is only in the sum

template <bool F16>
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void ldmatrix(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// 16 bytes to shared memory; zeros where `on` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Shared memory of a warp: kStages tiles of keys, values and scales.  Rows are an odd number of 16-byte words
// apart, so that the eight rows of an ldmatrix fall on different banks.
template <int KIND, int KD>
struct Ring {
  static constexpr int kMT = KIND == kBf16 && KD > 4 ? 1 : 2;           // sixteens of positions in a tile
  static constexpr int kTP = 16 * kMT;
  static constexpr int kElem = KIND == kBf16 ? 2 : 1;
  static constexpr int kRowMost = ((KD * kElem) | 1) * 16;
  static constexpr int kScale = 2 * kTP * kRowMost;                     // scales behind the rows
  static constexpr int kStage = kScale + (KIND == kBf16 ? 0 : 2 * kTP * 4);
  // twelve warps fit an SM with a ring of 18.9 KB each
  static constexpr int kStages = 4 * kStage <= 18944 ? 4 : 3 * kStage <= 18944 ? 3 : 2 * kStage <= 18944 ? 2 : 1;
  static constexpr int kBytes = kStages * kStage;
  static_assert(kBytes <= 18944, "three blocks of four warps have to fit an SM");
};

// One warp's state for a unit: NT tiles of eight rows.  Lane (g, t) = (lane / 4, lane % 4) holds rows 2t and 2t + 1
// of a tile and of O^T the columns column(c, 0), column(c, 1) of sixteen c; its queries are row g's.
template <int KIND, int KD, int NT>
struct Warp {
  using R = Ring<KIND, KD>;
  static constexpr int kRows = 8 * NT, kTP = R::kTP, kMT = R::kMT;
  static constexpr bool kF16 = KIND != kBf16;
  uint32_t q[NT][KD][2];
  float o[NT][KD][4];
  float m[NT][2], l[NT][2];
  float f[NT][2];                    // scores to exponents of two: scale * log2(e) over the row's power of two

  static __device__ __forceinline__ int column(int c, int e, int g) {
    return KIND == kBf16 ? 16 * c + 8 * e + g : 16 * c + 2 * g + e;
  }

  __device__ __forceinline__ void begin(const AttnParams& p, const Unit& u, int g, int t) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = u.rt * kRows + 8 * nt + g;
      const bool live = 8 * nt + g < u.rows;
      const __nv_bfloat16* row = p.q;
      if (live) row += static_cast<long long>(u.first + p.by_g(r)) * p.q_st + static_cast<long long>(u.h * p.G + r - p.by_g(r) * p.G) * p.q_sh;
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        const bool on = live && 16 * k < p.w.c.dh;
        if (!kF16) {
          q[nt][k][0] = on ? __ldg(reinterpret_cast<const uint32_t*>(row + 16 * k + 2 * t)) : 0u;
          q[nt][k][1] = on ? __ldg(reinterpret_cast<const uint32_t*>(row + 16 * k + 8 + 2 * t)) : 0u;
        } else {
          const uint2 v = on ? __ldg(reinterpret_cast<const uint2*>(row + 16 * k + 4 * t)) : make_uint2(0u, 0u);
          q[nt][k][0] = v.x;
          q[nt][k][1] = v.y;
          top = max(top, max(max(v.x & 0x7fffu, (v.x >> 16) & 0x7fffu), max(v.y & 0x7fffu, (v.y >> 16) & 0x7fffu)));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][k][e] = 0.f;
      }
      f[nt][0] = f[nt][1] = p.scale_log2;
      if (kF16) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the row's largest value to that of 128; rows of zeros, tiny ones and non-numbers as they are
        const uint32_t e = top >> 7;
        const bool as_is = e < 16u || e == 255u;
        const float up = as_is ? 1.f : __uint_as_float((127u + 134u - e) << 23);
        const float down = as_is ? 1.f : __uint_as_float((e - 7u) << 23);
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            q[nt][k][x] = pack_f16x2(__uint_as_float(q[nt][k][x] << 16) * up, __uint_as_float(q[nt][k][x] & 0xffff0000u) * up);
#pragma unroll
        for (int x = 0; x < 2; ++x) f[nt][x] *= __shfl_sync(0xffffffffu, down, 4 * (2 * t + x));
      }
      m[nt][0] = m[nt][1] = kFloor;
      l[nt][0] = l[nt][1] = 0.f;
    }
  }

  // Tiles t0, t0 + step, .. below t1 of the unit; ring: this warp's shared memory.
  __device__ void run(const AttnParams& p, const Unit& u, int t0, int t1, int step, int lane, uint32_t ring) {
    const int g = lane >> 2, t = lane & 3, dh = p.w.c.dh, shift = p.w.shift;
    // 16-byte words of a row in memory; rows in shared memory are those of the layout's dimension
    const int wpr = dh * R::kElem >> 4, per_word = 65536 / wpr + 1;
    constexpr int row_b = R::kRowMost;
    int pos_of[NT][2];                                   // positions of this lane's rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
        pos_of[nt][e] = r < u.rows ? u.len - u.n + p.by_g(u.rt * kRows + r) : -1;
      }
    const int* table = p.w.c.table + static_cast<size_t>(u.b) * p.w.c.width;
    auto place = [&](int tile) { return (tile < u.st ? tile : tile + u.skip) * kTP; };
    // lane l: the page of sixteen positions l % kMT of this warp's tile n + l / kMT, -1 where no row sees any of them
    constexpr int kAhead = 32 / kMT;
    auto page_ids = [&](int n) {
      int id = -1;
      const int tile = t0 + (n + lane / kMT) * step, x = place(tile) + 16 * (lane % kMT);
      if (tile < t1 && x < u.hi && (x + 16 > u.lo || x < u.s_end)) {
        id = __ldg(table + (x >> shift));
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.w.c.n_pages)) {
          atomicExch(p.w.c.status, kStatusBadPage);
          id = -1;
        }
      }
      return id;
    };
    // the 16-byte words of sixteen positions that this lane copies: their row, and their place in shared memory
    constexpr int kCopies = (16 * KD * R::kElem + 31) / 32;
    uint32_t copy_row[kCopies], copy_dst[kCopies];
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const int i = lane + 32 * c;
      copy_row[c] = i < 16 * wpr ? (i * per_word) >> 16 : 99;            // i / wpr: exact for i < 256, wpr <= 16
      copy_dst[c] = copy_row[c] * row_b + ((i - copy_row[c] * wpr) << 4);
    }
    const bool exact = wpr == KD * R::kElem;             // the head dimension is the one of the layout: 32, 64, 80 or 128
    uint32_t absent[R::kStages];                         // bit mt: the sixteen positions have no page
    auto issue = [&](int tile, int slot, int ids, int from) {
      uint32_t gone = 0;
      if (tile < t1) {
        const int x0 = place(tile);
        const uint32_t kdst = ring + slot * R::kStage, vdst = kdst + kTP * row_b;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          const int id = __shfl_sync(0xffffffffu, ids, from + mt), x = x0 + 16 * mt;
          gone |= static_cast<uint32_t>(id < 0) << mt;
          const size_t base = ((static_cast<size_t>(max(id, 0)) * p.w.c.H + u.h) << shift) + (x & (p.w.c.page - 1));
          const size_t bytes = base * static_cast<uint32_t>(dh * R::kElem) + 16 * lane;
          const char* ks = static_cast<const char*>(p.w.c.k) + bytes;
          const char* vs = static_cast<const char*>(p.w.c.v) + bytes;
          const uint32_t kd = kdst + 16 * mt * row_b, vd = vdst + 16 * mt * row_b;
          if (exact && id >= 0 && x + 16 <= u.hi && x >= u.lo) {
            // all sixteen are seen: nothing to ask for a word, which is most of the work of a tile otherwise
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
              if (32 * (c + 1) <= 16 * KD * R::kElem || lane < 16 * KD * R::kElem - 32 * c) {
                copy16_all(kd + copy_dst[c], ks + 512 * c);
                copy16_all(vd + copy_dst[c], vs + 512 * c);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
              if (copy_row[c] >= 16u) continue;
              const int y = x + static_cast<int>(copy_row[c]);
              const bool on = id >= 0 && y < u.hi && (y >= u.lo || y < u.s_end);
              copy16(kd + copy_dst[c], ks + 512 * c, on);
              copy16(vd + copy_dst[c], vs + 512 * c, on);
            }
          }
          if (KIND != kBf16 && lane < 8) {
            const float* src = (lane < 4 ? p.w.c.k_scale : p.w.c.v_scale) + base + 4 * (lane & 3);
            copy16(ring + slot * R::kStage + R::kScale + ((lane < 4 ? 0 : kTP) + 16 * mt + 4 * (lane & 3)) * 4, src, id >= 0);
          }
        }
      }
      copies_commit();
      return gone;
    };
    if (!exact) {                                        // the words that no copy writes are zeros
      for (int i = lane; i < R::kBytes / 16; i += 32) st_shared_v4(ring + 16 * i, 0u, 0u, 0u, 0u);
      __syncwarp();
    }
    // as many tiles ahead as the ring holds, page ids kAhead tiles and more ahead of the copies that need them
    int n = 0, ids = page_ids(0), ids_after = page_ids(kAhead);
    auto ahead = [&](int slot) {
      const uint32_t gone = issue(t0 + n * step, slot, ids, (n % kAhead) * kMT);
      if (++n % kAhead == 0) {
        ids = ids_after;
        ids_after = page_ids(n + kAhead);
      }
      return gone;
    };
#pragma unroll
    for (int i = 0; i < R::kStages; ++i) absent[i] = ahead(i);
    // rows of an ldmatrix: K: positions (lane & 7) + 8 (bit 3), words by bit 4; V: positions by bit 4 (bf16) or 3
    const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_word = lane >> 4;
    const int v_row = (lane & 7) + (KIND == kBf16 ? (lane >> 4) * 8 : ((lane >> 3) & 1) * 8);
    const int v_word = KIND == kBf16 ? (lane >> 3) & 1 : lane >> 4;
    int slot = 0;
    for (int tile = t0; tile < t1; tile += step) {
      copies_wait<R::kStages - 1>();
      __syncwarp();
      const uint32_t gone = absent[0];
      const int x0 = place(tile);
      const uint32_t kst = ring + slot * R::kStage, vst = kst + kTP * row_b;
      const uint32_t sst = kst + R::kScale;
      // ---- scores
      float s[NT][kMT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        const uint32_t at = kst + (16 * mt + k_row) * row_b + 16 * k_word;
        if (KIND == kBf16) {
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            uint32_t a[4];
            ldmatrix(at + 32 * k, a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<false>(s[nt][mt], a[0], a[1], a[2], a[3], q[nt][k][0], q[nt][k][1]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < KD; k += 2) {
            uint32_t a[4];                               // the last word of an odd number of them: a next row's beside it
            ldmatrix(at + 16 * k, a);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (k + e < KD) {
                const uint2 lo = codes_to_f16<KIND, false>(a[2 * e]), hi = codes_to_f16<KIND, false>(a[2 * e + 1]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816<true>(s[nt][mt], lo.x, hi.x, lo.y, hi.y, q[nt][k + e][0], q[nt][k + e][1]);
              }
            }
          }
        }
      }
      // ---- weights: s[.][.][c] is position g + 8 (c / 2), row 2t + c % 2.  With scales v of the values the running
      // maximum is that of score + log2 v, so that a weight times its scale, 2^14 at most, is an fp16 number: 2^-11
      // off at most, or 2^-39 of the largest; the sum takes the scale out again.  A scale of zero counts as 2^-126.
      float ks[kMT][2], lv[kMT][2], rv[kMT][2];
      if (kF16) {
        bool ones = false;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks[mt][e]) : "r"(sst + (16 * mt + 8 * e + g) * 4) : "memory");
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(lv[mt][e]) : "r"(sst + (kTP + 16 * mt + 8 * e + g) * 4) : "memory");
            ones = ones || lv[mt][e] == kZeroRow;
          }
        if (ones) {
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              bool zero = lv[mt][e] == kZeroRow;
              for (int w = 0; zero && w < wpr; ++w) zero = zero_codes<KIND>(ld_shared_v4(vst + (16 * mt + 8 * e + g) * row_b + 16 * w));
              if (zero) lv[mt][e] = kZeroScale;
            }
        }
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float v = lv[mt][e] < kLeastScale ? kLeastScale : lv[mt][e];       // keeps NaN
            lv[mt][e] = log2_fast(v);
            rv[mt][e] = __fdividef(1.f, v);
          }
      }
      const bool open = gone == 0u && x0 >= u.lo_all && x0 + kTP <= u.hi_all;     // every row sees every position
      uint32_t pt[NT][kMT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t vis = 0xffffffffu;
        if (!open) {
          vis = 0;
#pragma unroll
          for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int x = x0 + 16 * mt + g + 8 * (c >> 1), pr = pos_of[nt][c & 1];
              const bool on = ((gone >> mt) & 1u) == 0u && x <= pr && (x > pr - p.window || x < p.sinks);
              vis |= static_cast<uint32_t>(on) << (4 * mt + c);
            }
        }
        float top[2] = {vis & 0x55555555u ? kSeen : kFloor, vis & 0xaaaaaaaau ? kSeen : kFloor};
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[nt][mt][c] = kF16 ? fmaf(s[nt][mt][c], ks[mt][c >> 1] * f[nt][c & 1], lv[mt][c >> 1]) : s[nt][mt][c] * f[nt][c & 1];
            if ((vis >> (4 * mt + c)) & 1u) top[c & 1] = fmaxf(top[c & 1], s[nt][mt][c]);
          }
        float d[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
          top[e] = fmaxf(top[e], m[nt][e]);
          d[e] = exp2_fast(m[nt][e] - top[e]);
          m[nt][e] = top[e];
          l[nt][e] *= d[e];
        }
        if (__any_sync(0xffffffffu, d[0] != 1.f || d[1] != 1.f)) {
#pragma unroll
          for (int c = 0; c < KD; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][c][e] *= d[e & 1];
        }
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            w[c] = (vis >> (4 * mt + c)) & 1u ? exp2_fast(s[nt][mt][c] - m[nt][c & 1] + (kF16 ? 14.f : 0.f)) : 0.f;
            if (kF16) l[nt][c & 1] = (vis >> (4 * mt + c)) & 1u ? fmaf(w[c], rv[mt][c >> 1], l[nt][c & 1]) : l[nt][c & 1];
            else l[nt][c & 1] += w[c];
          }
          // the one rounding of a weight: to bf16, 2^-8 at most, or to fp16 as above
          pt[nt][mt][0] = transpose8x8(kF16 ? pack_f16x2(w[0], w[1]) : pack_bf16x2(w[0], w[1]));
          pt[nt][mt][1] = transpose8x8(kF16 ? pack_f16x2(w[2], w[3]) : pack_bf16x2(w[2], w[3]));
        }
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        const uint32_t at = vst + (16 * mt + v_row) * row_b + 16 * v_word;
        if (KIND == kBf16) {
#pragma unroll
          for (int c = 0; c < KD; ++c) {
            uint32_t a[4];
            ldmatrix_t(at + 32 * c, a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<false>(o[nt][c], a[0], a[1], a[2], a[3], pt[nt][mt][0], pt[nt][mt][1]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < KD; c += 2) {
            uint32_t a[4];
            ldmatrix_t(at + 16 * c, a);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (c + e < KD) {
                const uint2 lo = codes_to_f16<KIND, true>(a[2 * e]), hi = codes_to_f16<KIND, true>(a[2 * e + 1]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816<true>(o[nt][c + e], lo.x, lo.y, hi.x, hi.y, pt[nt][mt][0], pt[nt][mt][1]);
              }
            }
          }
        }
      }
      __syncwarp();                                      // the whole warp has read the slot
#pragma unroll
      for (int i = 0; i + 1 < R::kStages; ++i) absent[i] = absent[i + 1];
      absent[R::kStages - 1] = ahead(slot);
      slot = slot + 1 == R::kStages ? 0 : slot + 1;
    }
    copies_wait<0>();
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
  }
};

// All lanes of a warp: an O is not finite although the sum of its weights is, and the unit's rows see different positions,
// one of which holds a value that is no number.
template <int KIND, int KD, int NT>
__device__ __forceinline__ bool work_again(const AttnParams& p, const Warp<KIND, KD, NT>& s, const Unit& u, int lane) {
  if (KIND == kInt8 || (u.lo == u.lo_all && u.hi == u.hi_all)) return false;            // single tokens
  bool odd = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = 0.f;
#pragma unroll
      for (int c = 0; c < KD; ++c) x = track_odd(track_odd(x, s.o[nt][c][e]), s.o[nt][c][2 + e]);
      odd = odd || (x != x && s.l[nt][e] < INFINITY);
    }
  return __any_sync(0xffffffffu, odd) && __any_sync(0xffffffffu, odd_values<KIND>(p, u, lane, 32));
}
template <int KIND> constexpr float kUp = KIND == kBf16 ? 1.f : 16384.f;   // weights here are 2^14 times those of rows_again

constexpr int kMostWarps = 12;          // of a block: what fits an SM

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// A cluster of blocks per unit, every warp every n-th tile: grid (blocks of a cluster x row tiles, heads, sequences);
// more row tiles than the grid has are taken in turn.
template <int KIND, int KD, int NT>
__global__ void __launch_bounds__(32 * kMostWarps, 1) paged_few_unit_kernel(const __grid_constant__ AttnParams p, int blocks) {
  using W = Warp<KIND, KD, NT>;
  static_assert(2 * W::kRows * (16 * KD + 4) * 4 <= W::R::kBytes, "two O fit a warp's ring");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float s_ml[kMostWarps][W::kRows][2];
  __shared__ float s_all[W::kRows][2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3, dh = p.w.c.dh;
  const int ld = dh + 4, per = dh / 4;                 // floats between rows of O: the merge's rows fall on different banks
  const int rank = blocks > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  auto o_of = [&](int w) { return reinterpret_cast<float*>(smem + w * W::R::kBytes); };      // over the ring once it is read
  float* mine = o_of(warp);
  float* both = o_of(0) + W::kRows * ld;               // the block's O, for the cluster
  if (blockIdx.x == 0 && blockIdx.y == 0) zero_other_rows(p, blockIdx.z * blockDim.x + threadIdx.x, gridDim.z * blockDim.x);
  Unit u;
  unit_sequence(p, u, blockIdx.z);
  u.h = blockIdx.y;
  const int nrt = row_tiles<W::kRows>(u.n, p.G), step = gridDim.x / blocks;
  for (u.rt = blockIdx.x / blocks; u.rt < nrt; u.rt += step) {
    unit_range<W::kRows, W::kTP>(p, u);
    W s;
    s.begin(p, u, g, t);
    s.run(p, u, rank * warps + warp, u.tiles, blocks * warps, lane, smem_u32(mine));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
#pragma unroll
        for (int c = 0; c < KD; ++c)
          if (16 * c < dh) {
            mine[r * ld + W::column(c, 0, g)] = s.o[nt][c][e];
            mine[r * ld + W::column(c, 1, g)] = s.o[nt][c][2 + e];
          }
        if (g == 0) {
          s_ml[warp][r][0] = s.m[nt][e];
          s_ml[warp][r][1] = s.l[nt][e];
        }
      }
    if (work_again(p, s, u, lane)) {
      __syncwarp();
      rows_again<KIND, W::kRows, W::kTP>(p, u, rank * warps + warp, u.tiles, blocks * warps, 0, 1, lane, &s_ml[warp][0][0], mine, ld, 4, kUp<KIND>);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < u.rows * per; i += blockDim.x) {
      const int r = i / per, c = 4 * (i - r * per);
      float top = kFloor, sum = 0.f;
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < warps; ++w) top = fmaxf(top, s_ml[w][r][0]);
      for (int w = 0; w < warps; ++w) {
        const float x = exp2_fast(s_ml[w][r][0] - top);
        const float4 v = *reinterpret_cast<const float4*>(o_of(w) + r * ld + c);
        sum = fmaf(x, s_ml[w][r][1], sum);
        f.x = fmaf(x, v.x, f.x);
        f.y = fmaf(x, v.y, f.y);
        f.z = fmaf(x, v.z, f.z);
        f.w = fmaf(x, v.w, f.w);
      }
      if (blocks > 1) {
        *reinterpret_cast<float4*>(both + r * ld + c) = f;
        if (c == 0) {
          s_all[r][0] = top;
          s_all[r][1] = sum;
        }
      } else {
        const float inv = over_sum(sum, top);
        *reinterpret_cast<uint2*>(out_row(p, u, u.rt * W::kRows + r) + c) =
            make_uint2(pack_bf16x2(f.x * inv, f.y * inv), pack_bf16x2(f.z * inv, f.w * inv));
      }
    }
    if (blocks > 1) {
      cluster_sync_all();
      for (int i = rank * blockDim.x + threadIdx.x; i < u.rows * per; i += blocks * blockDim.x) {
        const int r = i / per, c = 4 * (i - r * per);
        const uint32_t ml = smem_u32(s_all[r]), at = smem_u32(both + r * ld + c);
        float top = kFloor, sum = 0.f;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < blocks; ++k) top = fmaxf(top, ld_cluster_f32(mapa_shared(ml, k)));
        for (int k = 0; k < blocks; ++k) {
          const float x = exp2_fast(ld_cluster_f32(mapa_shared(ml, k)) - top);
          const float4 v = ld_cluster_f32x4(mapa_shared(at, k));
          sum = fmaf(x, ld_cluster_f32(mapa_shared(ml + 4, k)), sum);
          f.x = fmaf(x, v.x, f.x);
          f.y = fmaf(x, v.y, f.y);
          f.z = fmaf(x, v.z, f.z);
          f.w = fmaf(x, v.w, f.w);
        }
        const float inv = over_sum(sum, top);
        *reinterpret_cast<uint2*>(out_row(p, u, u.rt * W::kRows + r) + c) =
            make_uint2(pack_bf16x2(f.x * inv, f.y * inv), pack_bf16x2(f.z * inv, f.w * inv));
      }
      cluster_sync_all();                              // nobody goes on while its memory may still be read
    } else {
      __syncthreads();                                 // before the next unit's copies
    }
  }
}

constexpr int kLeastTiles = 8;

// Equal runs of tiles for every warp.
template <int KIND, int KD, int NT>
__global__ void __launch_bounds__(32 * kWarps, 3) paged_few_run_kernel(const __grid_constant__ AttnParams p) {
  using W = Warp<KIND, KD, NT>;
  extern __shared__ __align__(128) unsigned char smem[];
  const uint32_t ring = smem_u32(smem) + (threadIdx.x >> 5) * W::R::kBytes;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, dh = p.w.c.dh;
  const int worker = blockIdx.x * kWarps + (threadIdx.x >> 5);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  zero_other_rows(p, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
  int4 meta = make_int4(-1, 0, 0, 0);
  Segments<W::kRows, W::kTP> seg;
  for (seg.begin(p, lane, worker, kLeastTiles); seg.on(); seg.next(p)) {
    const Unit& u = seg.u;
    W s;
    s.begin(p, u, g, t);
    s.run(p, u, seg.t0, seg.t1, 1, lane, ring);
    float* piece = p.part + (2 * static_cast<size_t>(worker) + seg.slot()) * piece_floats<W::kRows>(dh);
    seg.note(meta);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
        if (r >= u.rows) continue;
        const float inv = over_sum(s.l[nt][e], s.m[nt][e]);
        if (!seg.whole() && g == 0) *reinterpret_cast<float2*>(piece + 2 * r) = make_float2(s.m[nt][e], s.l[nt][e]);
        float* row = piece + 2 * W::kRows + r * dh;
        __nv_bfloat16* dst = out_row(p, u, u.rt * W::kRows + r);
#pragma unroll
        for (int c = 0; c < KD; ++c)
          if (16 * c < dh) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float f = s.o[nt][c][2 * x + e];
              if (seg.whole()) dst[W::column(c, x, g)] = __float2bfloat16(f * inv);
              else row[W::column(c, x, g)] = f;
            }
          }
      }
    if (work_again(p, s, u, lane)) {
      __syncwarp();
      rows_again<KIND, W::kRows, W::kTP>(p, u, seg.t0, seg.t1, 1, 0, 1, lane, seg.whole() ? nullptr : piece, piece + 2 * W::kRows, dh, 4, kUp<KIND>);
    }
  }
  if (lane == 0) p.meta[worker] = meta;
}

constexpr int kBlocksPerSm = 3;

int few_workers() { return device_sms() * kBlocksPerSm * kWarps; }

// How the work is shared: `blocks` = 0: equal runs; else clusters of that many blocks of `warps` warps per unit, eight
// blocks at most (the portable size).
struct Sharing { int blocks, warps; };

// The warps that the GPU holds (twelve an SM) are dealt to the units; a unit gets as many as its tiles at most.  What a
// sequence really has is not known here, only what its table holds and a window leaves of it.  Above `longest`
// positions for a warp the differences between sequences, and between SMs, cost more than the plan, the pieces and the
// merge of equal runs.  Microseconds, clusters / equal runs:
//   96 units, 18 warps each (bf16, 80):    4096 positions 34 / 33, 8192 58 / 54, 32768 229 / 179
//   512 units, 3 warps (e4m3, 128):        512 positions 20 / 24, 1024 37 / 37, 2048 63 / 60, 8192 226 / 194
//   512 units, lengths 16 times apart:     512 positions 14 / 23, 2048 35 / 28, 8192 98 / 75
//   32 units, 48 warps (bf16, 128, G 4):   4096 positions 14 / 24, 16384 49 / 68, 32768 93 / 111
Sharing sharing(const DsbPaged* c, int window, int sinks, int max_new, long long units) {
  long long most = static_cast<long long>(c->width) * c->page;
  if (window > 0 && static_cast<long long>(window) + sinks + max_new < most) most = static_cast<long long>(window) + sinks + max_new;
  long long w = static_cast<long long>(kMostWarps) * device_sms() / (units > 0 ? units : 1);
  const long long tiles = (most + 31) / 32;
  if (w > tiles) w = tiles;
  if (w < 1) w = 1;
  if (w > 8 * kMostWarps) w = 8 * kMostWarps;
  Sharing s = {1, static_cast<int>(w)};
  if (w > kMostWarps) {
    s.warps = w / 6 <= 8 ? 6 : kMostWarps;
    s.blocks = static_cast<int>(w / s.warps);
  }
  const long long longest = s.blocks * s.warps > 36 ? 1024 : 448;
  if (most > longest * s.blocks * s.warps) s.blocks = 0;
  return s;
}

template <int KIND, int KD, int NT>
int launch(AttnParams& p, int max_rt, const Sharing& how, cudaStream_t stream) {
  using W = Warp<KIND, KD, NT>;
  if (how.blocks > 0) {
    const int bytes = how.warps * W::R::kBytes;
    static std::atomic<int> most[kDevices];
    if (allow_smem(paged_few_unit_kernel<KIND, KD, NT>, kMostWarps * W::R::kBytes, most)) return 944;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(max_rt * how.blocks, p.w.c.H, p.w.c.B);
    cfg.blockDim = dim3(32 * how.warps);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = how.blocks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = how.blocks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, paged_few_unit_kernel<KIND, KD, NT>, p, how.blocks) == cudaSuccess ? 0 : 945;
  }
  constexpr int bytes = kWarps * W::R::kBytes;
  static std::atomic<int> most[kDevices];
  if (allow_smem(paged_few_run_kernel<KIND, KD, NT>, bytes, most)) return 944;
  if (launch_early(paged_few_run_kernel<KIND, KD, NT>, dim3(p.workers / kWarps), 32 * kWarps, bytes, p, stream)) return 945;
  return launch_early(paged_merge_few_kernel<W::kRows>, dim3(p.workers), kMergeThreads, 0, p, stream);
}

// Sixteens of the head dimension that the registers are laid out for: 32, 64, 80 or 128.  Others use the next larger layout,
// its words that they lack being zeros, and ask for each word of a copy whether it is there.  Microseconds of heads of
// 64 / 80 / 96 / 112 / 128, 32 sequences of 100 to 512 (16 heads): bf16 10.0 / 13.2 / 17.6 / 19.2 / 16.8, e4m3 10.8 / 10.5 /
// 18.2 / 19.0 / 15.5; 6 of 2000 to 32000: bf16 73 / 94 / 111 / 126 / 132, e4m3 52 / 55 / 71 / 74 / 82.
template <int KIND, int NT>
int launch_dim(AttnParams& p, int max_rt, const Sharing& how, cudaStream_t stream) {
  const int dh = p.w.c.dh;
  if (dh <= 32) return launch<KIND, 2, NT>(p, max_rt, how, stream);
  if (dh <= 64) return launch<KIND, 4, NT>(p, max_rt, how, stream);
  if (dh <= 80) return launch<KIND, 5, NT>(p, max_rt, how, stream);
  return launch<KIND, 8, NT>(p, max_rt, how, stream);
}

template <int KIND>
int launch_rows(AttnParams& p, long long rows, const Sharing& how, cudaStream_t stream) {
  return rows <= 8 ? launch_dim<KIND, 1>(p, 1, how, stream) : launch_dim<KIND, 2>(p, 1, how, stream);
}

}  // namespace

long long few_workspace(const DsbPaged* c, int window, int sinks, int max_new, int rows) {
  const Sharing how = sharing(c, window, sinks, max_new, static_cast<long long>(c->B) * c->H);
  return how.blocks > 0 ? 0 : workspace_bytes(few_workers(), rows <= 8 ? 8 : 16, c->dh);
}

int launch_few(AttnParams& p, int window, int sinks, int max_new, long long rows, void* workspace, cudaStream_t stream) {
  const Sharing how = sharing(&p.w.c, window, sinks, max_new, static_cast<long long>(p.w.c.B) * p.w.c.H);
  if (how.blocks == 0) {
    p.workers = few_workers();
    p.meta = static_cast<int4*>(workspace);
    p.part = reinterpret_cast<float*>(p.meta + p.workers);
  }
  if (p.w.c.kind == kBf16) return launch_rows<kBf16>(p, rows, how, stream);
  if (p.w.c.kind == kE4m3) return launch_rows<kE4m3>(p, rows, how, stream);
  return launch_rows<kInt8>(p, rows, how, stream);
}

}  // namespace paged
}  // namespace dsb
