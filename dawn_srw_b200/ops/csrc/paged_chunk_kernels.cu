// Attention of a chunk of new tokens over a paged cache, on the tensor cores (tcgen05).
//
// A unit is 256 query rows of one key/value head: two tiles of 128 rows (one TMEM lane and one thread per row) that
// share every tile of 128 positions.  Per tile i and positions j:  S_i = Q_i K_j^T (TMEM);  P_i = exp2(S_i - m), written
// back to TMEM as the A operand of  O_i += P_i V_j.  While the softmax threads of one tile work, the tensor core
// works for the other.  m is a row's running maximum as of the last time that it had grown by more than 2^8: O is
// rescaled then only, and a weight stays below 2^8 times one of the true maximum (floating point loses nothing by it).
//
// bf16 pages come by TMA, one box per page and 64 columns, into the 128-byte-swizzled tiles that the instructions
// read: K-major for K, MN-major for V.  8-bit codes are read by four warps and go to the same layout as fp16 numbers,
// code * scale / 2^e, e the exponent of the largest scale among the 32 positions of a warp: for int8 rounded once, by
// 2^-11 at most (as a weight is, and far below the codes' own rounding; a scale per column in the softmax would cost each
// thread three shared-memory reads per column), for e4m3, whose scales are powers of two and whose codes are multiples of
// 2^-9, exact while the scale is not smaller than the largest by more than 2^15.  At 2^20 fp16's smallest step is 2^-12 of
// such a row's largest value, of int8's at 2^13 the rounding of the scale; where one is smaller still, the block's work is
// done again in fp32 (rows_again).  Rows of zeros have no part in it.  2^e of the keys goes to the scores, 2^e of the
// values, as in the few-row kernel, to the exponents and out of the sum.
//
// Rows of V that no query row sees are zeros, whatever the page holds there; a scale that is no number makes the scores
// of its position NaN; a value that is none, seen by some rows of a unit alone, has the block's work done again too.
//
// The blocks, one per SM, take equal runs of tiles of all units, so neither ragged lengths nor causal triangles leave
// SMs idle; units that several blocks share are left in pieces for the merge kernel.
//
// What bounds it.  The products alone, at the rate of a large matrix product (1.66 PFLOP/s), are a third of the time:
// five bf16 prompts of 301 to 2048 tokens, 16 heads of 128, 97 us for 31; 4099 tokens over 16000 int8 positions, 16
// heads of 64 that share 4 and a window of 6000, 187 us for 61.  128 positions of a unit take about 4000 cycles.  By
// arithmetic the exponential unit has 1700 of them to do, shared memory at 128 bytes a cycle 1800 (heads of 64) to 2800
// (heads of 128) for the products' operands and 512 for the loads; the clock inside the kernel shows some 700 cycles
// per tile and warp that are waits, and latencies of TMEM and shared memory, in the open: the two softmax warps of a
// quarter of the SM run in step.  Starting one of them later changed nothing; exponentials on the FMA units help by 3 % at most (see kPoly).
// A small call, 512 tokens over 2100 e4m3 positions, 16 heads of 80, takes 28 us for 3: its plan (2.5 us), two runs a
// block, the pieces and their merge (8 us).
#include <type_traits>

#include "common/host_utils.cuh"
#include "common/paged_launch.h"

namespace dsb {
namespace paged {
namespace {

constexpr int kTileRows = 128, kUnitRows = 2 * kTileRows;
constexpr int kAtom = kTileRows * 128;      // 128 rows x 64 16-bit columns
// Positions of a tile.  TMEM holds two O, two S and, for heads of up to 64, two P, so that the next S can be made while P
// is.  For wider heads P takes the place of S, and the next S has to have another place: two S of 64 positions per
// query tile.  Against one S of 128, whose softmax waits for the products: 512 tokens over 2100 e4m3 positions, 16
// heads of 80, 27 us for 31, ragged bf16 prompts with heads of 128 96 for 97.  For heads of 64 two S of 64 are slower than S and P beside each other: 148 heads,
// 256 tokens over 4352 positions 78 us for 67 (int8 98 for 74), since a product of 64 columns keeps the tensor core
// busy for 48 cycles where half of one of 128 takes 32: it reads Q from shared memory all the same.
template <int NA> constexpr int kTP = NA == 1 ? 128 : 64;
constexpr int kStages = 4;                  // tiles of K, and of V, in shared memory
// Slots of scales and absences: written with K, read by a softmax that may be a tile behind the last use of the stage.
constexpr int kMeta = 2 * kStages;
constexpr int kPlans = 4;                   // segments that the planning warp is ahead of the others at most
constexpr float kSlack = 8.f;               // how far (in powers of two) a maximum may grow before O is rescaled
constexpr int kLeast = 2;                   // tiles of 128 positions of a run

// Warpgroups 0 and 1: softmax of tiles 0 and 1.  Warps 8 and 9: their MMA.  Warps 10 and 11: TMA, the plan.
// Warpgroup 3, 8-bit kinds: loaders.
template <int KIND>
constexpr int kThreadsOf = KIND == kBf16 ? 384 : 512;

template <int NA>                            // 64-column atoms of a head
struct Smem {
  static constexpr int kQ = 0;                                   // [2 tiles][NA atoms]
  static constexpr int kTile = NA * kTP<NA> * 128;               // K, or V, of a tile: NA atoms of kTP rows
  static constexpr int kK = kQ + 2 * NA * kAtom;                 // [kStages]
  static constexpr int kV = kK + kStages * kTile;                // [kStages]
  static constexpr int kExp = kV + kStages * kTile;              // [kMeta][2][4] 2^e of the keys, e of the values
  static constexpr int kPlan = kExp + kMeta * 32;            // [kPlans] segments ahead
  static constexpr int kBar = kPlan + kPlans * 128;
  static constexpr int kTotal = kBar + 512 + 1024;
  static_assert(kTotal <= 227 * 1024, "shared memory of an SM");
};

struct ChunkParams {
  CUtensorMap k, v;                          // bf16 pages: [n_pages * H][page][dh]
  CUtensorMap q;                             // queries: [N][Hq][dh], boxes of 128 rows (tokens x a group)
  int q_tma;                                 // a group divides 128 rows: the queries come by TMA
  AttnParams a;
};

// D += A B with A in tensor memory (128 lanes, two 16-bit values per column).
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 64 columns of this thread's row, complete on return (loads whose values pass through a later wait cost a register
// move each).
__device__ __forceinline__ void tmem_ld64_now(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr)
      : "memory");
}
// 32 columns of this thread's row, complete on return (loads whose values pass through a later wait cost a register
// move each).
__device__ __forceinline__ void tmem_ld32_now(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
// 16 columns of this thread's row, complete on return (loads whose values pass through a later wait cost a register
// move each).
__device__ __forceinline__ void tmem_ld16_now(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
      "}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Two fp32 operations in an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.ftz.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.ftz.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// 2^x for two x below 100 on the FMA units: the exponential unit, a sixteenth of a lane per cycle, is what the softmax
// waits for, so it makes only some of them.  Cody and Waite's reduction to n + f, f in [-1/2, 1/2], and a polynomial in
// f of degree 4 with value 1 at 0, fitted here to the least relative error (3e-6); n goes into the exponent's bits.
// Below -127, and at -inf, the result is 0; at NaN it is some number.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x.x = fmaxf(x.x, -127.f);
  x.y = fmaxf(x.y, -127.f);
  const float2 magic = make_float2(12582912.f, 12582912.f);                    // 1.5 * 2^23: n in the low bits
  const float2 t = add2(x, magic), f = add2(x, make_float2(12582912.f - t.x, 12582912.f - t.y));
  float2 p = fma2(f, make_float2(0.009582813829183578f, 0.009582813829183578f), make_float2(0.055906426161527634f, 0.055906426161527634f));
  p = fma2(p, f, make_float2(0.24024099111557007f, 0.24024099111557007f));
  p = fma2(p, f, make_float2(0.6931241750717163f, 0.6931241750717163f));
  p = fma2(p, f, make_float2(1.f, 1.f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}
// How many of sixteen exponentials are made this way.  With four loading warps beside the softmax the issue slots are
// what is short, not the exponential unit: 4099 tokens over 16000 int8 positions took 183 us with none, 196 with four
// and 220 with eight.  bf16, heads of 64, 24 x 4096 tokens: 96.5 with none, 93.6 with three; heads of 128, whose softmax
// waits for other things, ragged prompts: 95.6 with none, 97.4 with three.
template <int KIND, int NA> constexpr int kPoly = KIND == kBf16 && NA == 1 ? 3 : 0;

// Instruction descriptor, kind::f16, fp32 accumulators: A and B both bf16 or both fp16.
__host__ __device__ constexpr uint32_t idesc16(bool bf16, int m, int n, int b_mn_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(b_mn_major) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ uint64_t desc_k(uint32_t tile) { return umma_desc(tile, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int atom) { return umma_desc(tile, atom, 1024); }
// 16-byte word c8 (eight columns) of a row of a tile made of swizzled atoms.
template <int ATOM = kAtom>
__device__ __forceinline__ uint32_t swz(uint32_t tile, int row, int c8) {
  return tile + (c8 >> 3) * ATOM + row * 128 + (((c8 & 7) ^ (row & 7)) << 4);
}

// How many of a unit's tiles of positions query tile i works on (its rows see none of the later ones).
template <int TP>
__device__ __forceinline__ int tiles_of(const AttnParams& p, const Unit& u, int i) {
  const int r0 = i * kTileRows, r1 = min(u.rows, r0 + kTileRows);
  if (r0 >= u.rows) return 0;
  const int last = u.len - u.n + p.by_g(u.rt * kUnitRows + r1 - 1);
  const int end = (max(last + 1, 0) + TP - 1) / TP;       // tiles of positions that begin at or before `last`
  return min(u.tiles, end <= u.st ? end : max(end - u.skip, u.st));
}

// A segment as the roles need it.  One warp works it out, ahead of them: the index arithmetic, with its divisions and
// dependent loads, took every warp some 3000 cycles a segment.
struct Plan {
  int b, h, rt;                     // b < 0: there are no more
  int len, n, first, rows;
  int lo, hi, s_end, st, skip;
  int t0, n0, n1;                   // first tile of positions; how many from there each query tile works on
  int whole, slot;
};
static_assert(sizeof(Plan) <= 128, "slot of a plan");

template <int TP>
__device__ __forceinline__ int place(const Plan& q, int j) { return (q.t0 + j < q.st ? q.t0 + j : q.t0 + j + q.skip) * TP; }

// Bit k: a row at position pos sees position x + k.
__device__ __forceinline__ uint32_t seen32(int x, int pos, int window, int sinks) {
  auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  const uint32_t by = below(pos - x + 1), old = below(pos - window + 1 - x) & ~below(sinks - x);
  return by & ~old;
}

// D = A B^T over KS steps of sixteen columns, both K-major; B's atoms are B_ATOM bytes apart.
template <int KS, int B_ATOM>
__device__ __forceinline__ void issue_qk(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) {
    mma_bf16_ss(d, a + (((kk >> 2) * kAtom + (kk & 3) * 32) >> 4), b + (((kk >> 2) * B_ATOM + (kk & 3) * 32) >> 4), idesc,
                kk > 0 ? 1u : 0u);
  }
}

// A whole sector of 32 bytes in one store.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// 16 bytes to shared memory, zeros where `on` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// mbar_wait for the waits between softmax and MMA, one after the other in every tile: no sleeping in between.
__device__ __forceinline__ bool wait_hot(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  long long t0 = 0;
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 0xff) == 0xff) {
      if (*abort_flag) return false;
      const long long now = clock64();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > kWaitLimitCycles) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}

// One lane of the warp, in a form that tells the compiler that it is one.
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(on));
  return on != 0u;
}

template <int S>
struct Bars {
  uint64_t q_full[2];       // queries of tile i are in shared memory (4 warps, or a TMA load)
  uint64_t q_raw[2];        // they are, and are to be converted
  uint64_t k_full[S];       // K, and the tile's scales and absences
  uint64_t k_empty[S];      // both tiles' S of the stage are done
  uint64_t v_full[S];
  uint64_t v_empty[S];      // both tiles' O of the stage are done
  uint64_t v_fix;           // V has landed, rows behind the end still have to be cleared
  uint64_t s_full[2][2];    // [query tile][place of S]
  uint64_t s_free[2];       // S has been read (4 warps); only where P has columns of its own
  uint64_t p_half[2];       // the first half of P is in TMEM (4 warps)
  // [query tile][place of S]  all of them.  A warp may be through with the next tile's S while another still makes this
  // one's P, so that with two places one barrier would count the first warp twice.
  uint64_t p_full[2][2];
  uint64_t o_done[2][2];    // [query tile][place of the S that became its weights]
  uint64_t plan_full[kPlans];
  uint64_t plan_empty[kPlans];  // every warp that works by the plan has read it
  uint32_t tmem;
  int abort;
  int again;                // an O is not finite although the sum of its weights is
  int apart;                // scales of 32 positions are too far apart for fp16 numbers
  uint32_t absent[2 * S];   // [kMeta] bits 8 w + i: no row sees sixteen positions 2 w + i, or they have no page
};

// The plans in order, for one warp.
struct Plans {
  const Plan* ring;
  uint64_t* full;
  uint64_t* empty;
  volatile int* abort_flag;
  uint32_t k;
  // false: no more, or the block gives up
  __device__ __forceinline__ bool next(Plan& q, int lane) {
    const uint32_t slot = k % kPlans;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], (k / kPlans) & 1, abort_flag));
    if (!ok) return false;
    q = ring[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[slot]);
    ++k;
    return q.b >= 0;
  }
};

// The scale that counts of a row's 8-bit codes: 0 of a row of zeros.
template <int KIND>
__device__ __forceinline__ float used_scale(float s, const void* pool, size_t row, int dh) {
  if (s != kZeroRow) return s;
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(pool) + row * dh);
  bool zero = true;
  for (int c = 0; c < dh / 16; ++c) zero = zero && zero_codes<KIND>(__ldg(x + c));
  return zero ? 0.f : s;
}

// Of a warp's scales: biased exponent of the largest finite one, that of 2^-107 at least, so that its products with a score's
// factor do not vanish; `none` where there is none.  apart: this lane's is less by more than 2^20 (e4m3 and a power of two) or
// 2^13.
template <int KIND>
__device__ __forceinline__ uint32_t largest_exponent(float x, uint32_t none, bool& apart) {
  const uint32_t e = (__float_as_uint(x) >> 23) & 0xffu;
  uint32_t most = __reduce_max_sync(0xffffffffu, e == 255u ? 0u : e);
  if (most == 0u) return none;
  most = max(most, 20u);
  apart = apart || (e != 0u && most > e + (KIND == kE4m3 && (__float_as_uint(x) & 0x7fffffu) == 0u ? 20u : 13u));
  return most;
}

// Are scales of 32 positions of a segment too far apart?  Warp `warp` of `warps`.
template <int KIND, int TP>
__device__ __noinline__ bool scales_apart(const AttnParams& p, const Unit u, int t0, int t1, int warp, int warps, int lane) {
  bool apart = false;
  for (int i = warp; i < (t1 - t0) * (TP / 32); i += warps) {
    const int tile = t0 + i / (TP / 32), x = (tile < u.st ? tile : tile + u.skip) * TP + i % (TP / 32) * 32 + lane;
    const int page = x < u.hi && (x >= u.lo || x < u.s_end) ? page_of(p.w, u.b, x) : -1;
    const size_t at = page >= 0 ? slot_row(p.w, page, u.h, x) : 0;
    largest_exponent<KIND>(page >= 0 ? used_scale<KIND>(__ldg(p.w.c.k_scale + at), p.w.c.k, at, p.w.c.dh) : 0.f, 0u, apart);
    largest_exponent<KIND>(page >= 0 ? used_scale<KIND>(__ldg(p.w.c.v_scale + at), p.w.c.v, at, p.w.c.dh) : 0.f, 0u, apart);
  }
  return apart;
}

// A block's segments again, where that is called for.
template <int KIND, int TP>
__device__ __noinline__ void segments_again(const AttnParams& p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Segments<kUnitRows, TP> seg;
  for (seg.begin(p, lane, blockIdx.x, kLeast * 128 / TP); seg.on(); seg.next(p)) {
    bool redo = odd_values<KIND>(p, seg.u, threadIdx.x, kThreadsOf<KIND>);
    if (KIND != kBf16) redo = scales_apart<KIND, TP>(p, seg.u, seg.t0, seg.t1, warp, kThreadsOf<KIND> / 32, lane) || redo;
    if (!__syncthreads_or(redo)) continue;
    float* piece = p.part + (2 * static_cast<size_t>(blockIdx.x) + seg.slot()) * piece_floats<kUnitRows>(p.w.c.dh);
    // the kernel's fp16 weights are 2^6 times the others
    rows_again<KIND, kUnitRows, TP>(p, seg.u, seg.t0, seg.t1, 1, warp, kThreadsOf<KIND> / 32, lane, seg.whole() ? nullptr : piece,
                                    piece + 2 * kUnitRows, 4, 4 * kUnitRows, KIND == kBf16 ? 1.f : 64.f);
  }
}

template <int KIND, int NA>
__global__ void __launch_bounds__(kThreadsOf<KIND>, 1) paged_chunk_kernel(const __grid_constant__ ChunkParams cp) {
  using L = Smem<NA>;
  constexpr bool kF16 = KIND != kBf16;
  constexpr bool kAhead = kF16;                 // columns of S loaded one step ahead (int8: 183 us for 194; bf16 lost 2 of 101)
  constexpr bool kAlias = NA > 1;               // no room for P beside S and O: it takes the place of S
  constexpr bool kKeep = kAlias && !kF16;       // a row of S stays in registers (beside loaders there are too few of them)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr int S = kStages, TP = kTP<NA>, kHalf = TP / 2, kTile = L::kTile, kKvAtom = TP * 128;
  static_assert(sizeof(Bars<S>) <= 512 && kMeta == 2 * S, "barriers");
  Bars<S>& b = *reinterpret_cast<Bars<S>*>(smem + L::kBar);
  volatile int* abort_flag = &b.abort;
  volatile uint32_t* absent = b.absent;
  const AttnParams& p = cp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dh = p.w.c.dh, ksteps = dh >> 4;
  // a scale's sign goes to the queries, so that the largest product has the largest score; a scale of zero, which would
  // turn the -inf of hidden scores into NaN, into queries of zero (a factor of the scores that underflows, of small
  // queries and small keys, is kept at 2^-126: products are below 2^25, so that their scores are 0 all the same)
  const bool as_is = !kF16 && p.scale_log2 > 0.f;      // queries as they are in memory

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b.q_full[i], as_is && cp.q_tma ? 1 : 4);
      mbar_init(&b.q_raw[i], 1);
      mbar_init(&b.s_full[i][0], 1);
      mbar_init(&b.s_full[i][1], 1);
      mbar_init(&b.s_free[i], 4);
      mbar_init(&b.p_half[i], 4);
      mbar_init(&b.p_full[i][0], 4);
      mbar_init(&b.p_full[i][1], 4);
      mbar_init(&b.o_done[i][0], 1);
      mbar_init(&b.o_done[i][1], 1);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&b.k_full[i], kF16 ? 4 : 1);
      mbar_init(&b.k_empty[i], 2);
      mbar_init(&b.v_full[i], kF16 ? 4 : 1);
      mbar_init(&b.v_empty[i], 2);
    }
    for (int i = 0; i < kMeta; ++i) b.absent[i] = 0;
    mbar_init(&b.v_fix, 1);
    for (int i = 0; i < kPlans; ++i) {
      mbar_init(&b.plan_full[i], 1);
      mbar_init(&b.plan_empty[i], kF16 ? 14 : 11);      // softmax, MMA, and TMA or loaders
    }
    b.abort = 0;
    b.again = b.apart = 0;
    fence_barrier_init();
    if (!kF16) {
      tma_prefetch_desc(&cp.k);
      tma_prefetch_desc(&cp.v);
    }
  }
  if (warp == 8) {
    tmem_alloc(&b.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = b.tmem;
  const uint32_t q_addr = smem_u32(smem + L::kQ), k_addr = smem_u32(smem + L::kK), v_addr = smem_u32(smem + L::kV);
  // S: columns 0 and 128 (two of 64 each, or one);  O: 256 and 256 + 64 NA;  P: where S is, or behind O
  auto s_col = [&](int i) { return tmem + 128 * i; };
  auto o_col = [&](int i) { return tmem + 256 + 64 * NA * i; };
  auto p_col = [&](int i) { return kAlias ? s_col(i) : tmem + 384 + 64 * i; };

  asm volatile("griddepcontrol.wait;" ::: "memory");      // the stream's earlier work: from here on its results are read
  Plan* plan_ring = reinterpret_cast<Plan*>(smem + L::kPlan);
  static_assert(kPlans * sizeof(Plan) <= kPlans * 128, "ring of plans");
  Plans plans = {plan_ring, b.plan_full, b.plan_empty, abort_flag, 0};
  Plan u;

  if (warp >= 8 && warp < 12) {
    if (warp < 10) {
      // ------------------------------------------------------------ MMA issue of tile I
      if (elect_one()) {
        // One lane does all of it, and no instruction stands under a condition of its own: a tcgen05.mma that became a
        // predicated one gave wrong results.  What does not change from tile to tile is made beforehand.
        const int I = warp - 8;
        const uint32_t idesc_s = idesc16(!kF16, kTileRows, TP, 0), idesc_o = idesc16(!kF16, kTileRows, dh, 1);
        const uint64_t q_desc = desc_k(q_addr + I * NA * kAtom), k_desc = desc_k(k_addr), v_desc = desc_mn(v_addr, kKvAtom);
        const uint32_t s_at = s_col(I), o_at = o_col(I), p_at = p_col(I);
        // uses of the stages, segments with work and tiles so far.  Whoever waits for a phase of a barrier has seen the
        // phase before it, or something later, so that no wait is two phases off.
        uint32_t nk = 0, nq = 0, nt = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t phase) { ok = ok && wait_hot(bar, phase & 1, abort_flag); };
        // S of the segment's j-th tile, the x-th of this query tile
        auto issue_s = [&](int j, uint32_t x) {
          const uint32_t st = (nk + j) % S, place = kAlias ? x & 1u : 0u;
          wait(&b.k_full[st], (nk + j) / S);
          if (!ok) return;
          tc_fence_after();
          const uint64_t ka = k_desc + st * (kTile >> 4);
          switch (ksteps - 4 * (NA - 1)) {
            case 1: issue_qk<4 * NA - 3, kKvAtom>(s_at + place * TP, q_desc, ka, idesc_s); break;
            case 2: issue_qk<4 * NA - 2, kKvAtom>(s_at + place * TP, q_desc, ka, idesc_s); break;
            case 3: issue_qk<4 * NA - 1, kKvAtom>(s_at + place * TP, q_desc, ka, idesc_s); break;
            default: issue_qk<4 * NA, kKvAtom>(s_at + place * TP, q_desc, ka, idesc_s);
          }
          mma_commit(&b.s_full[I][place]);
          mma_commit(&b.k_empty[st]);
        };
        for (uint32_t k = 0; ok; ++k) {
          const uint32_t slot = k % kPlans;
          wait(&b.plan_full[slot], k / kPlans);
          if (!ok) break;
          const int n0 = plan_ring[slot].n0, n1 = plan_ring[slot].n1, more = plan_ring[slot].b;
          mbar_arrive(&b.plan_empty[slot]);
          if (more < 0) break;
          const int n = max(n0, n1), mine = I == 0 ? n0 : n1;
          if (mine > 0) {
            wait(&b.q_full[I], nq++);
            if (ok) issue_s(0, nt);
            if (kAlias && mine > 1 && ok) issue_s(1, nt + 1);
          }
          for (int j = 0; j < mine && ok; ++j, ++nt) {
            const uint32_t st = (nk + j) % S;
            if (!kAlias && j + 1 < mine) {         // the next S while the weights of this one are still being made
              wait(&b.s_free[I], nt);
              if (ok) issue_s(j + 1, nt + 1);
            }
            wait(&b.v_full[st], (nk + j) / S);
            if (!kAlias) wait(&b.p_half[I], nt);
            if (kAlias) wait(&b.p_full[I][nt & 1u], nt >> 1);
            if (!ok) break;
            tc_fence_after();
            const uint64_t va = v_desc + st * (kTile >> 4);
            const uint32_t pa = p_at + (kAlias ? (nt & 1u) * TP : 0u);
            mma_ts(o_at, pa, va, idesc_o, j > 0);
#pragma unroll
            for (int kk = 1; kk < kHalf / 16; ++kk) mma_ts(o_at, pa + 8 * kk, va + (kk * 2048 >> 4), idesc_o, 1u);
            if (!kAlias) wait(&b.p_full[I][0], nt);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int kk = kHalf / 16; kk < TP / 16; ++kk) mma_ts(o_at, pa + 8 * kk, va + (kk * 2048 >> 4), idesc_o, 1u);
            mma_commit(&b.o_done[I][kAlias ? nt & 1u : 0u]);
            mma_commit(&b.v_empty[st]);
            if (kAlias) {                          // the S after the next takes the columns that this P is read from
              wait(&b.o_done[I][nt & 1u], nt >> 1);
              if (j + 2 < mine && ok) issue_s(j + 2, nt + 2);
            }
          }
          for (int j = mine; j < n && ok; ++j) {   // the other tile's alone
            const uint32_t st = (nk + j) % S;
            wait(&b.k_full[st], (nk + j) / S);
            if (ok) mbar_arrive(&b.k_empty[st]);
            wait(&b.v_full[st], (nk + j) / S);
            if (ok) mbar_arrive(&b.v_empty[st]);
          }
          nk += n;
        }
      }
    } else if (warp == 10 && !kF16) {
      // ------------------------------------------------------------ TMA loads of bf16 pages
      uint32_t nk = 0, fixes = 0;
      bool ok = true;
      const int shift = p.w.shift, box = min(p.w.c.page, TP);
      while (ok && plans.next(u, lane)) {
        const int n = max(u.n0, u.n1);
        const int* table = p.w.c.table + static_cast<size_t>(u.b) * p.w.c.width;
        for (int j = 0; j < n && ok; ++j, ++nk) {
          const uint32_t st = nk % S, par = ((nk / S) & 1) ^ 1;
          const int x0 = place<TP>(u, j);
          // lane i < TP / 16: the page of sixteen positions i, -1 where no row sees any of them
          int id = -1;
          const int x = x0 + 16 * lane;
          if (lane < TP / 16 && x < u.hi && (x + 16 > u.lo || x < u.s_end)) {
            id = __ldg(table + (x >> shift));
            if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.w.c.n_pages)) {
              atomicExch(p.w.c.status, kStatusBadPage);
              id = -1;
            }
          }
          const uint32_t gone = __ballot_sync(0xffffffffu, id < 0) & ((1u << TP / 16) - 1u);
          auto unseen = [&](int y) { return y >= u.hi || (y < u.lo && y >= u.s_end); };
          // rows of V to clear
          const bool cut = gone != 0u || x0 + TP > u.hi || (x0 < u.lo && min(x0 + TP, u.lo) > u.s_end);
          // lanes that start a box: the first sixteen of each that the tile has
          const int per = box >> 4;
          const bool mine = lane < TP / 16 && lane % per == 0;
          // a box is fetched if its page is there at all: its sixteens are of one page
          const uint32_t have = __ballot_sync(0xffffffffu, id >= 0);
          const uint32_t group = lane < TP / 16 ? (have >> (lane / per * per)) & ((1u << per) - 1u) : 0u;
          const int src_lane = group ? lane / per * per + __ffs(group) - 1 : 0;
          const int page = __shfl_sync(0xffffffffu, id, src_lane);
          const bool fetch = mine && group != 0u;
          const int boxes = __popc(__ballot_sync(0xffffffffu, fetch));
          const int c1 = (x0 + 16 * lane) & (p.w.c.page - 1), c2 = page * p.w.c.H + u.h;
          ok = __all_sync(0xffffffffu, mbar_wait(&b.k_empty[st], par, abort_flag));
          if (!ok) break;
          if (lane == 0) {
            absent[nk % kMeta] = (gone & 3u) | (gone & 12u) << 6 | (gone & 48u) << 12 | (gone & 192u) << 18;
            mbar_expect_tx(&b.k_full[st], boxes * NA * box * 128);
          }
          __syncwarp();
          if (fetch)
            for (int a = 0; a < NA; ++a)
              tma_load_3d(k_addr + st * kTile + a * kKvAtom + lane * 2048, &cp.k, &b.k_full[st], 64 * a, c1, c2);
          ok = __all_sync(0xffffffffu, mbar_wait(&b.v_empty[st], par, abort_flag));
          if (!ok) break;
          uint64_t* bar = cut ? &b.v_fix : &b.v_full[st];
          if (lane == 0) mbar_expect_tx(bar, boxes * NA * box * 128);
          __syncwarp();
          if (fetch)
            for (int a = 0; a < NA; ++a)
              tma_load_3d(v_addr + st * kTile + a * kKvAtom + lane * 2048, &cp.v, bar, 64 * a, c1, c2);
          if (cut) {
            ok = __all_sync(0xffffffffu, mbar_wait(&b.v_fix, fixes & 1, abort_flag));
            if (!ok) break;
            ++fixes;
            for (int w = lane; w < TP * 8; w += 32) {
              const int row = w >> 3;
              if (unseen(x0 + row) || ((gone >> (row >> 4)) & 1u))
                for (int a = 0; a < NA; ++a)
                  st_shared_v4(v_addr + st * kTile + a * kKvAtom + row * 128 + (w & 7) * 16, 0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.v_full[st]);
          }
        }
      }
    }
    else if (warp == 11) {
      // ------------------------------------------------------------ the plan, and notes for the merge
      Segments<kUnitRows, TP> seg;
      int4 meta = make_int4(-1, 0, 0, 0);
      uint32_t k = 0;
      bool ok = true;
      for (seg.begin(p, lane, blockIdx.x, kLeast * 128 / TP); ok; ++k) {
        const bool more = seg.on();
        const uint32_t slot = k % kPlans;
        ok = __all_sync(0xffffffffu, mbar_wait(&b.plan_empty[slot], ((k / kPlans) & 1) ^ 1, abort_flag));
        if (!ok) break;
        if (lane == 0) {
          Plan q = {-1};
          if (more) {
            const Unit& x = seg.u;
            q = {x.b, x.h, x.rt, x.len, x.n, x.first, x.rows, x.lo, x.hi, x.s_end, x.st, x.skip, seg.t0,
                 max(0, min(seg.t1, tiles_of<TP>(p, x, 0)) - seg.t0), max(0, min(seg.t1, tiles_of<TP>(p, x, 1)) - seg.t0),
                 seg.whole() ? 1 : 0, seg.slot()};
          }
          plan_ring[slot] = q;
          mbar_arrive(&b.plan_full[slot]);
        }
        __syncwarp();
        if (!more) break;
        seg.note(meta);
        seg.next(p);
      }
      if (lane == 0) p.meta[blockIdx.x] = meta;
      zero_other_rows(p, blockIdx.x * 32 + lane, gridDim.x * 32);
    }
  } else if (warp >= 12) {
    // -------------------------------------------------------------- loaders of 8-bit pages
    if (kF16) {
      // 128 threads per tile: kParts of them for a position, each every kParts-th word of its rows of K and V
      constexpr int kParts = kTileRows / TP, kWords = 4 * NA / kParts;
      const int tid = (threadIdx.x - 384) % TP, part = (threadIdx.x - 384) / TP, shift = p.w.shift;
      const int chunk = tid >> 5;                                        // 32 positions of this warp
      // the tile that is fetched, one ahead of the one that is stored
      int j = 0, n = 0;
      // 1: there is one, 0: none.  -1, unless `far`: the next segment has none.  Further plans come only when those who
      // work by the first have gone on, for which they may still want the values of the tile that is being stored.
      auto more = [&](bool far) {
        while (j >= n) {
          if (!plans.next(u, lane)) return 0;
          n = max(u.n0, u.n1);
          j = 0;
          if (n == 0 && !far) return -1;
        }
        return 1;
      };
      struct Row { bool on, gone; size_t at; float ks, vs; };
      auto find = [&]() {
        const int x = place<TP>(u, j) + tid, x16 = x & ~15;
        int id = -1;
        if (x16 < u.hi && (x16 + 16 > u.lo || x16 < u.s_end)) {
          id = __ldg(p.w.c.table + static_cast<size_t>(u.b) * p.w.c.width + (x >> shift));
          if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.w.c.n_pages)) {
            atomicExch(p.w.c.status, kStatusBadPage);
            id = -1;
          }
        }
        Row r;
        r.gone = id < 0;
        r.on = id >= 0 && x < u.hi && (x >= u.lo || x < u.s_end);
        r.at = r.on ? slot_row(p.w, id, u.h, x) : 0;
        r.ks = r.on ? __ldg(p.w.c.k_scale + r.at) : 0.f;
        r.vs = r.on ? __ldg(p.w.c.v_scale + r.at) : 0.f;
        return r;
      };
      auto fetch = [&](const void* pool, const Row& r, uint4 (&raw)[kWords]) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(pool) + r.at * dh) + part;
#pragma unroll
        for (int c = 0; c < kWords; ++c)
          raw[c] = r.on && kParts * c + part < ksteps ? __ldg(src + kParts * c) : make_uint4(0u, 0u, 0u, 0u);
      };
      // codes * r as fp16, r in two parts, whose second one is a multiple of 2^-24: the product is rounded once, and r, of
      // 2^-13 at least unless it is a power of two, by 2^-12 at most
      auto store = [&](const uint4 (&raw)[kWords], uint32_t tile, float r) {
        const __half hi = __float2half_rn(r), lo = __float2half_rn(r - __half2float(hi));
        const __half2 h2 = __half2half2(hi), l2 = __half2half2(lo);
        auto scaled = [&](uint32_t x) {
          const __half2 v = *reinterpret_cast<const __half2*>(&x);
          const __half2 y = __hfma2(v, h2, __hmul2(v, l2));
          return *reinterpret_cast<const uint32_t*>(&y);
        };
#pragma unroll
        for (int c = 0; c < kWords; ++c) {                                // sixteen codes: two words of eight columns
          const int word = 2 * (kParts * c + part);
          if (word < 2 * ksteps) {
            const uint2 a = codes_to_f16<KIND, false>(raw[c].x), d = codes_to_f16<KIND, false>(raw[c].y),
                        e = codes_to_f16<KIND, false>(raw[c].z), f = codes_to_f16<KIND, false>(raw[c].w);
            st_shared_v4(swz<kKvAtom>(tile, tid, word), scaled(a.x), scaled(a.y), scaled(d.x), scaled(d.y));
            st_shared_v4(swz<kKvAtom>(tile, tid, word + 1), scaled(e.x), scaled(e.y), scaled(f.x), scaled(f.y));
          }
        }
      };
      uint4 kraw[kWords], vraw[kWords];
      Row r = {false, true, 0, 0.f, 0.f};
      bool have = more(true) > 0, ok = true;
      if (have) {
        r = find();
        fetch(p.w.c.k, r, kraw);
        fetch(p.w.c.v, r, vraw);
      }
      for (uint32_t nk = 0; have && ok; ++nk) {
        const uint32_t st = nk % S, par = ((nk / S) & 1) ^ 1, slot = nk % kMeta;
        const uint32_t none = __ballot_sync(0xffffffffu, r.gone);         // two sixteens of this warp
        // where there is no scale, of keys that of 1; of values 2^-60: rows of zeros have their weight in the sum alone
        bool apart = false;
        if (r.ks == kZeroRow || r.vs == kZeroRow) {
          r.ks = used_scale<KIND>(r.ks, p.w.c.k, r.at, dh);
          r.vs = used_scale<KIND>(r.vs, p.w.c.v, r.at, dh);
        }
        const uint32_t ek = largest_exponent<KIND>(r.ks, 127u, apart), ev = largest_exponent<KIND>(r.vs, 67u, apart);
        if (apart) *static_cast<volatile int*>(&b.apart) = 1;
        // 2^(127 - e) as a float: e of 254 at most
        float rk = r.ks * __uint_as_float((254u - ek) << 23), rv = r.vs * __uint_as_float((254u - ev) << 23);
        const bool odd = !(fabsf(r.ks) < INFINITY) || !(fabsf(r.vs) < INFINITY);
        if (odd) {                                                        // NaN scores for whoever sees the position
          rk = __uint_as_float(0x7fc00000u);
          rv = 0.f;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&b.k_empty[st], par, abort_flag));
        if (!ok) break;
        if (lane == 0 && part == 0) {
          float* e = reinterpret_cast<float*>(smem + L::kExp) + slot * 8 + chunk;
          e[0] = __uint_as_float(ek << 23);
          e[4] = static_cast<float>(static_cast<int>(ev) - 127);
          reinterpret_cast<volatile uint8_t*>(absent + slot)[chunk] = (none & 0xffffu ? 1 : 0) | (none >> 16 ? 2 : 0);
        }
        store(kraw, k_addr + st * kTile, rk);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.k_full[st]);
        ++j;
        int got = more(false);
        Row next = {false, true, 0, 0.f, 0.f};
        if (got > 0) {
          next = find();
          fetch(p.w.c.k, next, kraw);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&b.v_empty[st], par, abort_flag));
        if (!ok) break;
        store(vraw, v_addr + st * kTile, rv);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.v_full[st]);
        if (got < 0) {
          got = more(true);
          if (got > 0) {
            next = find();
            fetch(p.w.c.k, next, kraw);
          }
        }
        have = got > 0;
        if (have) fetch(p.w.c.v, next, vraw);
        r = next;
      }
    }
  } else {
    // -------------------------------------------------------------- softmax, a thread per query row
    const int i = warp >> 2, row = threadIdx.x - 128 * i;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_base = s_col(i) + lanes, o_at = o_col(i) + lanes, p_base = p_col(i) + lanes;
    const uint32_t q_tile = q_addr + i * NA * kAtom;
    const int first_row = 32 * (warp & 3), words = 2 * ksteps;  // of this warp; 16-byte words of a row
    const bool flat = p.scale_log2 == 0.f;
    // queries of the next segment on their way into the swizzled tile: a warp its 32 rows, neighbouring lanes the words
    // of a row
    auto fetch_q = [&]() {
      if (cp.q_tma) {
        if (row == 0) {
          uint64_t* bar = as_is ? &b.q_full[i] : &b.q_raw[i];
          mbar_expect_tx(bar, NA * kAtom);
          const int t = u.first + p.by_g(u.rt * kUnitRows + i * kTileRows);
          for (int a = 0; a < NA; ++a) tma_load_3d(q_tile + a * kAtom, &cp.q, bar, 64 * a, u.h * p.G, t);
        }
        return;
      }
      constexpr int kRowLanes = 8 * NA, kRowStep = 32 / kRowLanes;
      const int word = lane % kRowLanes, sub_row = lane / kRowLanes;
      if (word < words) {
#pragma unroll 4
        for (int c = 0; c < 32 / kRowStep; ++c) {
          const int x = first_row + kRowStep * c + sub_row, ru = i * kTileRows + x;
          const int r = u.rt * kUnitRows + ru, t = p.by_g(r);
          const bool on = ru < u.rows && !flat;
          const __nv_bfloat16* src =
              on ? p.q + static_cast<long long>(u.first + t) * p.q_st + static_cast<long long>(u.h * p.G + r - t * p.G) * p.q_sh : p.q;
          copy16(swz(q_tile, x, word), src + (on ? 8 * word : 0), on);
        }
      }
    };
    constexpr int kParts = TP / 32;                // of a row of S
    // until the x-th tile's product with V is in O.  With two places the barrier's phase before it, of tile x - 2, is past:
    // S of tile x has been seen, which was made behind that product.
    auto o_wait = [&](uint32_t x) { return wait_hot(&b.o_done[i][kAlias ? x & 1u : 0u], (kAlias ? x >> 1 : x) & 1, abort_flag); };
    uint32_t nk = 0, ns = 0, nq = 0;               // tiles loaded, S of this tile, its segments with work so far
    bool ok = true, have = plans.next(u, lane);
    if (have && (i == 0 ? u.n0 : u.n1) > 0) fetch_q();
    while (ok && have) {
      const int n = max(u.n0, u.n1), mine = i == 0 ? u.n0 : u.n1;
      const int ru = i * kTileRows + row;          // row of the unit
      const bool real = ru < u.rows;
      const int r = u.rt * kUnitRows + ru;         // row of the sequence's head
      const int pos = real ? u.len - u.n + p.by_g(r) : -1;
      const int w0 = u.rt * kUnitRows + i * kTileRows + first_row;             // positions of this warp's rows
      const int pos_lo = u.len - u.n + p.by_g(min(w0, u.n * p.G - 1)), pos_hi = u.len - u.n + p.by_g(min(w0 + 31, u.n * p.G - 1));
      float f = flat ? 1.f : fabsf(p.scale_log2);
      if (mine > 0 && !(as_is && cp.q_tma)) {
        if (cp.q_tma) {
          ok = __all_sync(0xffffffffu, mbar_wait(&b.q_raw[i], nq & 1, abort_flag));
          if (!ok) break;
        } else {
          copies_wait_all();
        }
        __syncwarp();
        const bool flip = p.scale_log2 < 0.f;
        if (!as_is) {
          uint4 v[8 * NA];
          uint32_t top = 0;
#pragma unroll
          for (int c = 0; c < 8 * NA; ++c) {
            v[c] = c < words ? ld_shared_v4(swz(q_tile, row, c)) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
          }
          float up = flat ? 0.f : flip ? -1.f : 1.f;
          const uint32_t e = top >> 7;             // fp16 queries, scaled by a power of two (see the few-row kernel)
          if (kF16 && e >= 16u && e != 255u) {
            up *= __uint_as_float((261u - e) << 23);
            f *= __uint_as_float((e - 7u) << 23);
          }
#pragma unroll
          for (int c = 0; c < 8 * NA; ++c) {
            if (c >= words) continue;
            if (kF16) {
              float t[8];
              bf16x8_to_f32(v[c], t);
              st_shared_v4(swz(q_tile, row, c), pack_f16x2(t[0] * up, t[1] * up), pack_f16x2(t[2] * up, t[3] * up),
                           pack_f16x2(t[4] * up, t[5] * up), pack_f16x2(t[6] * up, t[7] * up));
            } else {
              const uint32_t sign = flip ? 0x80008000u : 0u, keep = flat ? 0u : 0xffffffffu;
              st_shared_v4(swz(q_tile, row, c), (v[c].x ^ sign) & keep, (v[c].y ^ sign) & keep, (v[c].z ^ sign) & keep, (v[c].w ^ sign) & keep);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.q_full[i]);
      }
      if (mine > 0) ++nq;
      float m = kFloor, l = 0.f;
      for (int j = 0; j < mine; ++j, ++ns) {
        const uint32_t st = (nk + j) % kMeta;
        const uint32_t at = kAlias ? ns & 1u : 0u;         // which S
        ok = __all_sync(0xffffffffu, wait_hot(&b.s_full[i][at], (kAlias ? ns >> 1 : ns) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_at = s_base + at * TP, p_at = kAlias ? s_at : p_base;
        const uint32_t gone = absent[st];
        float keep[64];
        if (kKeep) tmem_ld64_now(s_at, keep);              // before it is known whether anything is hidden: rarely
        const int x0 = place<TP>(u, j);
        const bool hidden = gone != 0u || x0 + TP > pos_lo + 1 || x0 < pos_hi - p.window + 1;
        // of columns 32 c ..: score (in powers of two) = product * fc + ev
        float fc[kParts], ev[kParts];
#pragma unroll
        for (int c = 0; c < kParts; ++c) {
          const float* e = reinterpret_cast<const float*>(smem + L::kExp) + st * 8 + c;
          fc[c] = kF16 ? f * e[0] : f;
          fc[c] = fc[c] < kLeastScale ? kLeastScale : fc[c];     // 0 would make NaN of a hidden score; NaN stays
          ev[c] = kF16 ? e[4] : 0.f;
        }
        // what a row does not see is -inf and weighs nothing: in TMEM, so that the tiles in between, most of them, have
        // nothing to do with it
        float top = kSeen;
        if (hidden) {
          bool any = false;
#pragma unroll 1
          for (int c = 0; c < TP / 16; ++c) {
            const int x = x0 + 16 * c;                 // sixteen columns: most are seen, or not, by all rows of a warp
            const uint32_t away = gone >> (8 * (c >> 1) + (c & 1)) & 1u;
            if (away == 0u && x + 15 <= pos_lo && (x > pos_hi - p.window || x + 15 < p.sinks)) {
              any = true;
              continue;
            }
            uint32_t w[16];
            if (away != 0u || x > pos_hi || (x + 15 <= pos_lo - p.window && x >= p.sinks)) {
#pragma unroll
              for (int k = 0; k < 16; ++k) w[k] = 0xff800000u;
            } else {
              float y[16];
              tmem_ld16_now(s_at + 16 * c, y);
              const uint32_t seen = seen32(x, pos, p.window, p.sinks);
              any = any || (seen & 0xffffu) != 0u;
#pragma unroll
              for (int k = 0; k < 16; ++k) w[k] = (seen >> k) & 1u ? __float_as_uint(y[k]) : 0xff800000u;
            }
            tmem_st16(s_at + 16 * c, w);
          }
          tmem_st_wait();
          if (kKeep) tmem_ld64_now(s_at, keep);
          top = any ? kSeen : kFloor;
        }
        // a row of 64 stays in registers where they suffice; two passes over S elsewhere
#pragma unroll
        for (int h = 0; h < TP / 64; ++h) {
          if (!kKeep) tmem_ld64_now(s_at + 64 * h, keep);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float* y = keep + 32 * c;
            float t0 = max_nan(y[0], y[1]), t1 = max_nan(y[2], y[3]);
#pragma unroll
            for (int k = 4; k < 32; k += 4) {
              t0 = max_nan(t0, y[k], y[k + 1]);
              t1 = max_nan(t1, y[k + 2], y[k + 3]);
            }
            top = max_nan(top, fmaf(max_nan(t0, t1), fc[2 * h + c], ev[2 * h + c]));   // fc >= 0
          }
        }
        // a score that is NaN, or inf, less itself NaN too: the row's result is. It goes by the maximum, since exp2_poly
        // does not hand on NaN
        top = top < INFINITY ? top : __uint_as_float(0x7fc00000u);
        // O complete up to the tile before, and the columns of a P of its own free
        auto o_ready = [&]() {
          ok = __all_sync(0xffffffffu, o_wait(ns - 1));
          tc_fence_after();
        };
        if (!kAlias && j > 0) {
          o_ready();
          if (!ok) break;
        }
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xffffffffu, !(top <= m + kSlack))) {
          if (kAlias) {
            o_ready();
            if (!ok) break;
          }
          const float m_new = max_nan(m, top), d = exp2_fast(m - m_new);
          for (int c = 0; c < ksteps; ++c) {
            float o[16];
            tmem_ld16_now(o_at + 16 * c, o);
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k] * d);
            tmem_st16(o_at + 16 * c, w);
          }
          tmem_st_wait();
          l *= d;
          m = m_new;
        }
        // fp16 weights: 2^14 at most, so that 2^-24 of one is 2^-30 of the reference
        const float ref = kF16 ? m - 6.f : m;
        float xs[2][32];
        if (kAhead) tmem_ld32(s_at, xs[0]);
#pragma unroll
        for (int c = 0; c < kParts; ++c) {
          float* x = kKeep ? keep + 32 * (c & 1) : xs[kAhead ? c & 1 : 0];
          if (kAhead) {
            tmem_ld_wait_dep32(x);
            if (c < kParts - 1) tmem_ld32(s_at + 32 * (c + 1), xs[(c + 1) & 1]);
          } else if (!kKeep) {
            tmem_ld32_now(s_at + 32 * c, x);
          }
          if (!kAlias && c == kParts - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.s_free[i]);
          }
          const float off = ev[c] - ref;
          float2 sum = make_float2(0.f, 0.f);
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float2 y = fma2(make_float2(x[k], x[k + 1]), make_float2(fc[c], fc[c]), make_float2(off, off));
            y = (k / 2) % 16 < kPoly<KIND, NA> ? exp2_poly(y) : make_float2(exp2_fast(y.x), exp2_fast(y.y));
            sum = add2(sum, y);
            w[k / 2] = kF16 ? pack_f16x2(y.x, y.y) : pack_bf16x2(y.x, y.y);
          }
          tmem_st16(p_at + 16 * c, w);             // where P takes the place of S: columns already read
          const float part = sum.x + sum.y;
          l += kF16 ? part * exp2_fast(-ev[c]) : part;
          if (c & 1) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(c == kParts - 1 ? &b.p_full[i][at] : &b.p_half[i]);
          }
        }
        if (!ok) break;
      }
      nk += n;
      if (!ok) break;
      // every S of the unit is done: its queries make room for the next ones
      const bool whole = u.whole != 0;
      const float inv = over_sum(l, m);
      float* piece = p.part + (2 * static_cast<size_t>(blockIdx.x) + u.slot) * piece_floats<kUnitRows>(dh);
      __nv_bfloat16* dst = real ? out_row(p, u.first, u.h, r) : nullptr;
      have = plans.next(u, lane);
      if (have && (i == 0 ? u.n0 : u.n1) > 0) fetch_q();
      if (mine > 0) {
        ok = __all_sync(0xffffffffu, o_wait(ns - 1));
        if (!ok) break;
        tc_fence_after();
      }
      if (real && !whole) reinterpret_cast<float2*>(piece)[ru] = make_float2(m, l);
      float4* to = reinterpret_cast<float4*>(piece + 2 * kUnitRows) + ru;
      float odd = 0.f;
      for (int c = 0; c < ksteps; ++c) {
        float o[16];
        if (mine > 0) {
          tmem_ld16_now(o_at + 16 * c, o);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0.f;
        }
        if (!real) continue;
        if (KIND != kInt8) {
#pragma unroll
          for (int k = 0; k < 16; ++k) odd = track_odd(odd, o[k]);
        }
        if (whole) {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = pack_bf16x2(o[2 * k] * inv, o[2 * k + 1] * inv);
          st_global_v8(dst + 16 * c, w);
        } else {                                   // four columns of all rows after four columns of all rows
#pragma unroll
          for (int k = 0; k < 4; ++k)
            to[(4 * c + k) * kUnitRows] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        }
      }
      if (odd != odd && l < INFINITY) *static_cast<volatile int*>(&b.again) = 1;
      tc_fence_before();                           // O has been read: the next unit's P may follow
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(p.w.c.status, kStatusWaitTimeout);
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) { }         // copies and MMAs in flight end before the memory goes
    __syncthreads();
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  const bool redo = (KIND != kInt8 && *static_cast<volatile int*>(&b.again)) || (kF16 && *static_cast<volatile int*>(&b.apart));
  if (redo && *abort_flag == 0) segments_again<KIND, TP>(p);
}

// What several blocks left of a unit, in order: a block takes 32 rows, a lane per row, a warp per sixteen columns.
__global__ void __launch_bounds__(256) paged_merge_chunk_kernel(const AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = blockIdx.x, dh = p.w.c.dh, lane = threadIdx.x & 31, col = 16 * (threadIdx.x >> 5);
  const int r = blockIdx.y * 32 + lane;
  Unit u;
  int last;
  if (!shared_unit<kUnitRows>(p, i, lane, u, last)) return;
  if (r >= u.rows) return;
  float top = kFloor, sum = 0.f, a[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) a[k] = 0.f;
#pragma unroll 2
  for (int j = i; j <= last; ++j) {
    const float* from = p.part + (2 * static_cast<size_t>(j) + (j == i ? 1 : 0)) * piece_floats<kUnitRows>(dh);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(from) + r);
    const float4* o4 = reinterpret_cast<const float4*>(from + 2 * kUnitRows) + (col / 4) * kUnitRows + r;
    float4 o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = __ldcg(o4 + k * kUnitRows);
    const float most = fmaxf(top, ml.x), x = exp2_fast(top - most), w = exp2_fast(ml.x - most);
    top = most;
    sum = fmaf(sum, x, w * ml.y);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[4 * k] = fmaf(a[4 * k], x, w * o[k].x);
      a[4 * k + 1] = fmaf(a[4 * k + 1], x, w * o[k].y);
      a[4 * k + 2] = fmaf(a[4 * k + 2], x, w * o[k].z);
      a[4 * k + 3] = fmaf(a[4 * k + 3], x, w * o[k].w);
    }
  }
  const float inv = over_sum(sum, top);
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = pack_bf16x2(a[2 * k] * inv, a[2 * k + 1] * inv);
  __nv_bfloat16* dst = out_row(p, u, u.rt * kUnitRows + r) + col;
  st_global_v8(dst, w);
}

// Pages as [n_pages * H][page][dh], boxes of 64 columns by one page (a tile's positions at most).
int page_map(CUtensorMap* map, const void* pool, const AttnParams& a) {
  const DsbPaged& c = a.w.c;
  const int most = c.dh <= 64 ? kTP<1> : kTP<2>;
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return 1;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.dh), static_cast<cuuint64_t>(c.page),
                        static_cast<cuuint64_t>(c.n_pages) * static_cast<cuuint64_t>(c.H)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.dh) * 2, static_cast<cuuint64_t>(c.dh) * 2 * c.page};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(c.page < most ? c.page : most), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  if (dims[2] == 0) {                         // no page: nothing is fetched, but a map wants an address
    dims[2] = 1;
    pool = a.q;
  }
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(pool), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : 2;
}

// Queries as [N][Hq][dh], boxes of 64 columns, a group of heads and as many tokens as 128 rows hold.
int query_map(CUtensorMap* map, const AttnParams& a) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return 1;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.w.c.dh), static_cast<cuuint64_t>(a.Hq), static_cast<cuuint64_t>(a.w.c.N)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.q_sh) * 2, static_cast<cuuint64_t>(a.q_st) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.G), static_cast<cuuint32_t>(kTileRows / a.G)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(a.q), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : 2;
}

template <int KIND, int NA>
int launch(const ChunkParams& p, cudaStream_t stream) {
  static std::atomic<int> most[kDevices];
  if (allow_smem(paged_chunk_kernel<KIND, NA>, Smem<NA>::kTotal, most)) return 950;
  return launch_early(paged_chunk_kernel<KIND, NA>, dim3(p.a.workers), kThreadsOf<KIND>, Smem<NA>::kTotal, p, stream) ? 951 : 0;
}

template <int KIND>
int launch_dim(const ChunkParams& p, cudaStream_t stream) {
  return p.a.w.c.dh <= 64 ? launch<KIND, 1>(p, stream) : launch<KIND, 2>(p, stream);
}

}  // namespace

long long chunk_workspace(const DsbPaged* c) { return workspace_bytes(device_sms(), kUnitRows, c->dh); }

int launch_chunk(AttnParams& a, void* workspace, cudaStream_t stream) {
  ChunkParams p;
  a.workers = device_sms();
  a.meta = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(a.meta + a.workers);
  p.a = a;
  // strides that a tensor map takes (positive, below 2^40), a group that divides the rows of a tile: copies row by row
  // otherwise
  p.q_tma = a.G <= kTileRows && kTileRows % a.G == 0 && a.q_sh > 0 && a.q_st > 0 && a.q_sh < (1LL << 38) && a.q_st < (1LL << 38) &&
            query_map(&p.q, a) == 0;
  int rc;
  if (a.w.c.kind == kBf16) {
    if (page_map(&p.k, a.w.c.k, a) || page_map(&p.v, a.w.c.v, a)) return 952;
    rc = launch_dim<kBf16>(p, stream);
  } else if (a.w.c.kind == kE4m3) {
    rc = launch_dim<kE4m3>(p, stream);
  } else {
    rc = launch_dim<kInt8>(p, stream);
  }
  return rc ? rc : launch_early(paged_merge_chunk_kernel, dim3(a.workers, kUnitRows / 32), 2 * a.w.c.dh, 0, a, stream);
}

}  // namespace paged
}  // namespace dsb
