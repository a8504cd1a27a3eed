// Attention of a few query rows per key/value head (single tokens, drafted ones) over a paged cache.
//
// A warp streams tiles of positions straight from global memory into matrix-instruction fragments:
//   S^T [positions, rows] = K Q^T        m16n8k16, K the M side: eight rows fill the N side, so that one row costs
//                                        the same as eight and a tile's scores need no shared memory;
//   O^T [dh, rows]       += V^T P^T      V^T the M side; the transposed P comes from movmatrix, the transposed V
//                                        from pairs of rows interleaved with byte permutes.
// Any order of the contraction will do as long as both operands have it, so a lane takes eight neighbouring
// elements of a row (16 bytes of bf16, 8 of codes) where the fragment wants pairs 2t, 2t+1, 2t+8, 2t+9; 8-bit codes
// become bf16 in registers, exactly, their scales go to the scores and the weights in fp32.  The running maximum and
// sum of the softmax stay in registers.
//
// Two ways to share the work (kSplit): short caches take one block per unit, its warps interleaved over the tiles
// and merged in shared memory: one launch.  Long ones take as many warps as the GPU holds, each with an equal run of
// consecutive tiles of all units; a unit that several warps share is left in pieces, which a second kernel adds up in
// order.  The lengths are read on the device, so a captured call follows them.
#include "common/paged_units.cuh"
#include "common/ptx.cuh"

namespace dsb {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr float kFloor = -3.0e38f;     // below every score

__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight elements of a row as they lie in memory.
template <int KIND> struct Raw { uint2 v; };
template <> struct Raw<kBf16> { uint4 v; };

template <int KIND>
__device__ __forceinline__ void clear(Raw<KIND>& r) { r.v = make_uint2(0u, 0u); }
template <>
__device__ __forceinline__ void clear<kBf16>(Raw<kBf16>& r) { r.v = make_uint4(0u, 0u, 0u, 0u); }

__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ldg8(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
template <int KIND>
__device__ __forceinline__ Raw<KIND> load_raw(const void* pool, size_t elem) {
  Raw<KIND> r;
  r.v = ldg8(static_cast<const uint8_t*>(pool) + elem);
  return r;
}
template <>
__device__ __forceinline__ Raw<kBf16> load_raw<kBf16>(const void* pool, size_t elem) {
  Raw<kBf16> r;
  r.v = ldg16(static_cast<const __nv_bfloat16*>(pool) + elem);
  return r;
}
template <int KIND>
__device__ __forceinline__ void words(const Raw<KIND>& r, uint32_t* o) {
  const uint2 a = codes_to_bf16<KIND>(r.v.x), b = codes_to_bf16<KIND>(r.v.y);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}
template <>
__device__ __forceinline__ void words<kBf16>(const Raw<kBf16>& r, uint32_t* o) {
  o[0] = r.v.x; o[1] = r.v.y; o[2] = r.v.z; o[3] = r.v.w;
}

// One warp's state for a unit: NT tiles of eight rows.  Lane (g, t) = (lane / 4, lane % 4) holds rows 2t and 2t+1 of
// a tile and, of O^T, the eight elements 64 jj + 8 g ..; its queries are row g's.
template <int KIND, int DC, int NT, int MT>
struct Warp {
  static constexpr int kRows = 8 * NT, kTP = 16 * MT, kJ = (DC + 1) / 2;
  uint32_t q[NT][DC][4];
  float o[NT][kJ][4][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void begin(const AttnParams& p, const Unit& u, int g, int t) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = u.rt * kRows + 8 * nt + g;
      const bool live = 8 * nt + g < u.rows;
      const __nv_bfloat16* row = p.q;
      if (live) row += static_cast<long long>(u.first + r / p.G) * p.q_st + static_cast<long long>(u.h * p.G + r % p.G) * p.q_sh;
#pragma unroll
      for (int j = 0; j < DC; ++j) {
        const int col = 32 * j + 8 * t;
        const uint4 v = live && col < p.w.c.dh ? __ldg(reinterpret_cast<const uint4*>(row + col)) : make_uint4(0u, 0u, 0u, 0u);
        q[nt][j][0] = v.x; q[nt][j][1] = v.y; q[nt][j][2] = v.z; q[nt][j][3] = v.w;
      }
      m[nt][0] = m[nt][1] = kFloor;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int jj = 0; jj < kJ; ++jj)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][jj][c][e] = 0.f;
    }
  }

  // Tiles t0, t0 + step, .. below t1 of the unit.
  __device__ void run(const AttnParams& p, const Unit& u, int t0, int t1, int step, int lane) {
    const int g = lane >> 2, t = lane & 3, dh = p.w.c.dh, shift = p.w.shift;
    int pos_of[NT][2];                                   // positions of this lane's rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
        pos_of[nt][e] = r < u.rows ? u.len - u.n + (u.rt * kRows + r) / p.G : -1;
      }
    const int* table = p.w.c.table + static_cast<size_t>(u.b) * p.w.c.width;
    // lane i < MT: the page of the tile's i-th sixteen positions, -1 where no row sees any of them
    auto page_ids = [&](int tile) {
      int id = -1;
      const int x = (tile < u.st ? tile : tile + u.skip) * kTP + 16 * lane;
      if (lane < MT && tile < t1 && x < u.hi && (x + 16 > u.lo || x < u.s_end)) {
        id = __ldg(table + (x >> shift));
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.w.c.n_pages)) {
          atomicExch(p.w.c.status, kStatusBadPage);
          id = -1;
        }
      }
      return id;
    };
    int ids = page_ids(t0);
    for (int tile = t0; tile < t1; tile += step) {
      const int x0 = (tile < u.st ? tile : tile + u.skip) * kTP;
      Raw<KIND> kr[MT][2][DC], vr[MT][4][kJ];
      float ks[MT][2], vs[MT][2];
      uint32_t live = 0;                                 // bit 2 mt + e: position x0 + 16 mt + 8 e + g may be seen
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int id = __shfl_sync(0xffffffffu, ids, mt), x = x0 + 16 * mt;
        const size_t base = ((static_cast<size_t>(max(id, 0)) * p.w.c.H + u.h) << shift) + (x & (p.w.c.page - 1));
        auto seen = [&](int i) { return id >= 0 && x + i < u.hi && (x + i >= u.lo || x + i < u.s_end); };
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool on = seen(g + 8 * e);
          live |= static_cast<uint32_t>(on) << (2 * mt + e);
#pragma unroll
          for (int j = 0; j < DC; ++j) {
            clear(kr[mt][e][j]);
            if (on && 32 * j + 8 * t < dh) kr[mt][e][j] = load_raw<KIND>(p.w.c.k, (base + g + 8 * e) * dh + 32 * j + 8 * t);
          }
          ks[mt][e] = vs[mt][e] = 1.f;
          if (KIND != kBf16 && on) {
            ks[mt][e] = __ldg(p.w.c.k_scale + base + g + 8 * e);
            vs[mt][e] = __ldg(p.w.c.v_scale + base + g + 8 * e);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {                    // positions 2t, 2t+1, 2t+8, 2t+9: the fragment's own order
          const int row = 2 * t + (i & 1) + 8 * (i >> 1);
          const bool on = seen(row);
#pragma unroll
          for (int jj = 0; jj < kJ; ++jj) {
            clear(vr[mt][i][jj]);
            if (on && 64 * jj + 8 * g < dh) vr[mt][i][jj] = load_raw<KIND>(p.w.c.v, (base + row) * dh + 64 * jj + 8 * g);
          }
        }
      }
      ids = page_ids(tile + step);                       // one tile ahead of the loads that need them
      // ---- scores
      float s[NT][MT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < DC; ++j) {
          uint32_t a[4], b[4];
          words<KIND>(kr[mt][0][j], a);
          words<KIND>(kr[mt][1][j], b);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(s[nt][mt], a[0], b[0], a[1], b[1], q[nt][j][0], q[nt][j][1]);
            mma16816(s[nt][mt], a[2], b[2], a[3], b[3], q[nt][j][2], q[nt][j][3]);
          }
        }
      // ---- weights: s[.][.][c] is position g + 8 (c / 2), row 2t + c % 2
      uint32_t pt[NT][MT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2] = {kFloor, kFloor};
        uint32_t vis = 0;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int x = x0 + 16 * mt + g + 8 * (c >> 1), pr = pos_of[nt][c & 1];
            const bool on = ((live >> (2 * mt + (c >> 1))) & 1u) && x <= pr && (x > pr - p.window || x < p.sinks);
            vis |= static_cast<uint32_t>(on) << (4 * mt + c);
            s[nt][mt][c] *= p.scale_log2 * ks[mt][c >> 1];
            if (on) top[c & 1] = fmaxf(top[c & 1], s[nt][mt][c]);
          }
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
          top[e] = fmaxf(top[e], m[nt][e]);
          f[e] = exp2_fast(m[nt][e] - top[e]);
          m[nt][e] = top[e];
          l[nt][e] *= f[e];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
          for (int jj = 0; jj < kJ; ++jj)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][jj][c][e] *= f[e & 1];
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            w[c] = (vis >> (4 * mt + c)) & 1u ? exp2_fast(s[nt][mt][c] - m[nt][c & 1]) : 0.f;
            l[nt][c & 1] += w[c];
            if (KIND != kBf16) w[c] = w[c] > 0.f ? w[c] * vs[mt][c >> 1] : w[c];
          }
          // the one rounding of a weight (to bf16, with its position's scale): 2^-8 at most
          pt[nt][mt][0] = transpose8x8(pack_bf16x2(w[0], w[1]));
          pt[nt][mt][1] = transpose8x8(pack_bf16x2(w[2], w[3]));
        }
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int jj = 0; jj < kJ; ++jj) {
          uint32_t r[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) words<KIND>(vr[mt][i][jj], r[i]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t a0 = __byte_perm(r[0][c], r[1][c], 0x5410), a1 = __byte_perm(r[0][c], r[1][c], 0x7632);
            const uint32_t a2 = __byte_perm(r[2][c], r[3][c], 0x5410), a3 = __byte_perm(r[2][c], r[3][c], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][jj][c], a0, a1, a2, a3, pt[nt][mt][0], pt[nt][mt][1]);
          }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
  }

  // This lane's eight elements (from column 64 jj + 8 g) of row 8 nt + 2 t + e.
  __device__ __forceinline__ void eight(int nt, int jj, int e, float* f) const {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      f[2 * c] = o[nt][jj][c][e];
      f[2 * c + 1] = o[nt][jj][c][2 + e];
    }
  }
};

__device__ __forceinline__ __nv_bfloat16* out_row(const AttnParams& p, const Unit& u, int row) {
  return p.out + (static_cast<size_t>(u.first + row / p.G) * p.Hq + u.h * p.G + row % p.G) * p.w.c.dh;
}

__device__ __forceinline__ uint4 pack8(const float* f, float s) {
  return make_uint4(pack_bf16x2(f[0] * s, f[1] * s), pack_bf16x2(f[2] * s, f[3] * s), pack_bf16x2(f[4] * s, f[5] * s),
                    pack_bf16x2(f[6] * s, f[7] * s));
}

// One block per unit: grid (row tiles, heads, sequences); more row tiles than the grid has are taken in turn.
template <int KIND, int DC, int NT, int MT>
__global__ void __launch_bounds__(32 * kWarps) paged_few_block_kernel(const AttnParams p) {
  using W = Warp<KIND, DC, NT, MT>;
  __shared__ float s_o[kWarps][W::kRows][16 * 8 + 4];
  __shared__ float s_ml[kWarps][W::kRows][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, dh = p.w.c.dh;
  if (blockIdx.x == 0 && blockIdx.y == 0) zero_other_rows(p, blockIdx.z * blockDim.x + threadIdx.x, gridDim.z * blockDim.x);
  Unit u;
  unit_sequence(p, u, blockIdx.z);
  u.h = blockIdx.y;
  const int nrt = row_tiles<W::kRows>(u.n, p.G);
  for (u.rt = blockIdx.x; u.rt < nrt; u.rt += gridDim.x) {
    unit_range<W::kRows, W::kTP>(p, u);
    W s;
    s.begin(p, u, g, t);
    s.run(p, u, warp, u.tiles, kWarps, lane);
    __syncthreads();                                   // the last unit's readers are done
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
#pragma unroll
        for (int jj = 0; jj < W::kJ; ++jj) {
          float f[8];
          s.eight(nt, jj, e, f);
          float4* d = reinterpret_cast<float4*>(&s_o[warp][r][64 * jj + 8 * g]);
          d[0] = make_float4(f[0], f[1], f[2], f[3]);
          d[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
        if (g == 0) {
          s_ml[warp][r][0] = s.m[nt][e];
          s_ml[warp][r][1] = s.l[nt][e];
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < u.rows * (dh / 8); i += blockDim.x) {
      const int r = i / (dh / 8), c = 8 * (i - r * (dh / 8));
      float top = kFloor, sum = 0.f, f[8];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w][r][0]);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float x = exp2_fast(s_ml[w][r][0] - top);
        sum = fmaf(x, s_ml[w][r][1], sum);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = fmaf(x, s_o[w][r][c + k], f[k]);
      }
      *reinterpret_cast<uint4*>(out_row(p, u, u.rt * W::kRows + r) + c) = pack8(f, sum > 0.f ? 1.f / sum : 0.f);
    }
  }
}

// Where a worker's run of tiles begins, among all tiles of all units in order (sequence, head, row tile).
struct Run { long long begin, end, total; };

// Equal runs of the warps: worker i of n takes tiles [i T / n, (i + 1) T / n).
template <int ROWS, int TP>
__device__ __forceinline__ Run share(const AttnParams& p, int lane, long long worker, int least, int& b, long long& before) {
  const int B = p.w.c.B;
  long long total = 0;
  for (int i = 0; i < B; i += 32) {
    long long x = i + lane < B ? sequence_tiles<ROWS, TP>(p, i + lane) : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    total += x;
  }
  const long long most = total / least;
  const long long n = most < 1 ? 1 : most < p.workers ? most : p.workers;
  Run r = {0, 0, total};
  if (worker >= n) return r;
  r.begin = worker * total / n;
  r.end = (worker + 1) * total / n;
  b = 0;
  before = 0;
  for (int i = 0; i < B; i += 32) {                    // the sequence that holds tile r.begin
    const long long x = i + lane < B ? sequence_tiles<ROWS, TP>(p, i + lane) : 0;
    long long c = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, c, d);
      if (lane >= d) c += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + c > r.begin);
    if (past != 0u) {
      const int k = __ffs(past) - 1;
      b = i + k;
      before += __shfl_sync(0xffffffffu, c - x, k);
      return r;
    }
    before += __shfl_sync(0xffffffffu, c, 31);
  }
  return r;
}

// A piece of a unit in the workspace: per row maximum and sum, then O.
template <int ROWS>
__host__ __device__ constexpr int piece_floats(int dh) { return ROWS * (dh + 2); }

constexpr int kLeastTiles = 2;

// Equal runs of tiles for every warp.  Piece 2 i + 1 of worker i: a unit that begins in its run and ends in a later
// one; piece 2 i: a unit that began in an earlier run.  meta[i] = {unit of piece 2 i + 1 or -1 .., rows | 1 << 16 if
// piece 2 i ends its unit}.
template <int KIND, int DC, int NT, int MT>
__global__ void __launch_bounds__(32 * kWarps) paged_few_run_kernel(const AttnParams p) {
  using W = Warp<KIND, DC, NT, MT>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, dh = p.w.c.dh;
  const int worker = blockIdx.x * kWarps + (threadIdx.x >> 5);
  zero_other_rows(p, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
  int b = 0;
  long long before = 0;
  const Run run = share<W::kRows, W::kTP>(p, lane, worker, kLeastTiles, b, before);
  int4 meta = make_int4(-1, 0, 0, 0);
  long long at = run.begin;
  if (at < run.end) {
    Unit u;
    unit_sequence(p, u, b);
    int nrt = row_tiles<W::kRows>(u.n, p.G);
    // head and row tile of the first unit
    long long per_head = 0, off = at - before;
    for (u.rt = 0; u.rt < nrt; ++u.rt) {
      unit_range<W::kRows, W::kTP>(p, u);
      per_head += u.tiles;
    }
    u.h = static_cast<int>(off / per_head);
    off -= u.h * per_head;
    for (u.rt = 0;; ++u.rt) {
      unit_range<W::kRows, W::kTP>(p, u);
      if (off < u.tiles) break;
      off -= u.tiles;
    }
    int t0 = static_cast<int>(off);
    while (true) {
      const long long left = run.end - at;
      const int t1 = static_cast<int>(min(static_cast<long long>(u.tiles), t0 + left));
      W s;
      s.begin(p, u, g, t);
      s.run(p, u, t0, t1, 1, lane);
      const bool whole = t0 == 0 && t1 == u.tiles;
      float* piece = p.part + (2 * static_cast<size_t>(worker) + (t0 == 0 ? 1 : 0)) * piece_floats<W::kRows>(dh);
      if (!whole) {
        if (t0 == 0) {
          meta.x = u.b;
          meta.y = u.h;
          meta.z = u.rt;
        } else if (t1 == u.tiles) {
          meta.w = 1;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * nt + 2 * t + e;
          if (r >= u.rows) continue;
          const float inv = s.l[nt][e] > 0.f ? 1.f / s.l[nt][e] : 0.f;
          if (!whole && g == 0) *reinterpret_cast<float2*>(piece + 2 * r) = make_float2(s.m[nt][e], s.l[nt][e]);
#pragma unroll
          for (int jj = 0; jj < W::kJ; ++jj) {
            const int c = 64 * jj + 8 * g;
            if (c >= dh) continue;
            float f[8];
            s.eight(nt, jj, e, f);
            if (whole) {
              *reinterpret_cast<uint4*>(out_row(p, u, u.rt * W::kRows + r) + c) = pack8(f, inv);
            } else {
              float4* d = reinterpret_cast<float4*>(piece + 2 * W::kRows + r * dh + c);
              d[0] = make_float4(f[0], f[1], f[2], f[3]);
              d[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
          }
        }
      at += t1 - t0;
      if (at >= run.end) break;
      // the next unit
      t0 = 0;
      if (++u.rt >= nrt) {
        u.rt = 0;
        if (++u.h >= p.w.c.H) {
          u.h = 0;
          do {
            unit_sequence(p, u, u.b + 1);
            nrt = row_tiles<W::kRows>(u.n, p.G);
          } while (nrt == 0);
        }
      }
      unit_range<W::kRows, W::kTP>(p, u);
    }
  }
  if (lane == 0) p.meta[worker] = meta;
}

constexpr int kMergeThreads = 128;

// One block per worker whose last unit goes on in later runs: its piece and theirs, in order.
template <int ROWS>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s_w[ROWS];
  __shared__ int s_last;
  const int i = blockIdx.x, dh = p.w.c.dh;
  const int4 meta = p.meta[i];
  if (meta.x < 0) return;
  Unit u;
  unit_sequence(p, u, meta.x);
  u.h = meta.y;
  u.rt = meta.z;
  unit_range<ROWS, 16>(p, u);
  if (threadIdx.x < 32) {                              // the worker that ends the unit
    int j = i + 1;
    for (;; j += 32) {
      const int k = j + static_cast<int>(threadIdx.x);
      const unsigned end = __ballot_sync(0xffffffffu, k >= p.workers || p.meta[k].w != 0);
      if (end != 0u) {
        j += __ffs(end) - 1;
        break;
      }
    }
    if (threadIdx.x == 0) s_last = min(j, p.workers - 1);
  }
  __syncthreads();
  const int last = s_last, stride = piece_floats<ROWS>(dh);
  auto piece = [&](int j) { return p.part + (2 * static_cast<size_t>(j) + (j == i ? 1 : 0)) * stride; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float s_top[ROWS];
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
      s_w[r] = sum > 0.f ? 1.f / sum : 0.f;
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k < u.rows * (dh / 4); k += kMergeThreads) {
    const int r = k / (dh / 4), c = 4 * (k - r * (dh / 4));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = i; j <= last; ++j) {
      const float* d = piece(j);
      const float x = exp2_fast(d[2 * r] - s_top[r]);
      const float4 o = *reinterpret_cast<const float4*>(d + 2 * ROWS + r * dh + c);
      a.x = fmaf(x, o.x, a.x);
      a.y = fmaf(x, o.y, a.y);
      a.z = fmaf(x, o.z, a.z);
      a.w = fmaf(x, o.w, a.w);
    }
    *reinterpret_cast<uint2*>(out_row(p, u, u.rt * ROWS + r) + c) =
        make_uint2(pack_bf16x2(a.x * s_w[r], a.y * s_w[r]), pack_bf16x2(a.z * s_w[r], a.w * s_w[r]));
  }
}

int device_sms() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

constexpr int kBlocksPerSm = 2;

int few_workers() { return device_sms() * kBlocksPerSm * kWarps; }

// Short caches: a block per unit.
bool by_blocks(const DsbPaged* c) { return static_cast<long long>(c->width) * c->page <= 1024; }

template <int KIND, int DC, int NT>
int launch(AttnParams& p, int max_rt, cudaStream_t stream) {
  // positions of a tile: what 128 registers of keys and values hold
  constexpr int MT = NT == 2 ? (KIND == kBf16 ? 1 : 2) : (DC > 2 ? (KIND == kBf16 ? 2 : 4) : 4);
  if (by_blocks(&p.w.c)) {
    const dim3 grid(max_rt, p.w.c.H, p.w.c.B);
    paged_few_block_kernel<KIND, DC, NT, MT><<<grid, 32 * kWarps, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : 944;
  }
  paged_few_run_kernel<KIND, DC, NT, MT><<<p.workers / kWarps, 32 * kWarps, 0, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return 945;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.workers);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_merge_kernel<8 * NT>, p) == cudaSuccess ? 0 : 946;
}

template <int KIND, int NT>
int launch_dim(AttnParams& p, int max_rt, cudaStream_t stream) {
  const int dc = (p.w.c.dh + 31) / 32;
  if (dc == 1) return launch<KIND, 1, NT>(p, max_rt, stream);
  if (dc == 2) return launch<KIND, 2, NT>(p, max_rt, stream);
  if (dc == 3) return launch<KIND, 3, NT>(p, max_rt, stream);
  return launch<KIND, 4, NT>(p, max_rt, stream);
}

template <int KIND>
int launch_rows(AttnParams& p, int max_new, cudaStream_t stream) {
  const long long rows = static_cast<long long>(max_new) * p.G;
  if (rows <= 8) return launch_dim<KIND, 1>(p, 1, stream);
  const long long rt = (rows + 15) / 16;
  return launch_dim<KIND, 2>(p, static_cast<int>(rt > 65535 ? 65535 : rt), stream);
}

}  // namespace
}  // namespace paged
}  // namespace dsb

using namespace dsb::paged;

extern "C" long long dsb_paged_attention_workspace(const DsbPaged* c, int Hq, int max_new) {
  if (c->N == 0 || c->B == 0 || c->H <= 0 || by_blocks(c)) return 0;
  const int rows = static_cast<long long>(max_new) * (Hq / c->H) <= 8 ? 8 : 16;
  const long long w = few_workers();
  return w * static_cast<long long>(sizeof(int4)) + 2 * w * rows * (c->dh + 2) * static_cast<long long>(sizeof(float));
}

extern "C" int dsb_paged_attention(const DsbPaged* c, const void* q, long long q_st, long long q_sh, void* out, int Hq,
                                   int max_new, int window, int sinks, float scale, void* workspace, cudaStream_t stream) {
  if (bad_cache(c) || Hq <= 0 || Hq % c->H != 0 || window < 0 || sinks < 0 || max_new < 0) return 940;
  if ((reinterpret_cast<uintptr_t>(q) & 15) != 0 || q_st % 8 || q_sh % 8 || c->H > 65535 || c->B > 65535) return 941;
  if (c->N == 0) return 0;
  if (c->B == 0) {
    const size_t bytes = static_cast<size_t>(c->N) * Hq * c->dh * sizeof(__nv_bfloat16);
    return cudaMemsetAsync(out, 0, bytes, stream) == cudaSuccess ? 0 : 942;
  }
  if (!by_blocks(c) && workspace == nullptr) return 943;
  AttnParams p;
  p.w = make_view(c);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.Hq = Hq;
  p.G = Hq / c->H;
  p.window = window > 0 && window < kMostPositions ? window : kMostPositions;
  p.sinks = sinks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.workers = few_workers();
  p.meta = static_cast<int4*>(workspace);
  p.part = reinterpret_cast<float*>(p.meta + p.workers);
  if (max_new < 1) max_new = 1;
  if (max_new > c->N) max_new = c->N;
  if (c->kind == kBf16) return launch_rows<kBf16>(p, max_new, stream);
  if (c->kind == kE4m3) return launch_rows<kE4m3>(p, max_new, stream);
  return launch_rows<kInt8>(p, max_new, stream);
}
