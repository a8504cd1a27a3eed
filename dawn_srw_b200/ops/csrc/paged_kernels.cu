// Paged key/value cache: rows into pages (rounded to the pages' type on the way), pages back to dense
// tensors, attention of new tokens over pages.  Types, layouts and bounds: dsb_api_paged.h.
#include <cuda_fp8.h>

#include "common/paged_launch.h"

namespace dsb {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr float kLeast = 7.888609e-31f;      // 2^-100: a row without a larger value is stored as zeros

// Lanes that share a row: eight elements each, a power of two of them.
__host__ __device__ constexpr int lanes_per_row(int dh) {
  return dh <= 16 ? 2 : dh <= 32 ? 4 : dh <= 64 ? 8 : 16;
}

struct Eight { float f[8]; };

template <bool SRC_BF16>
__device__ __forceinline__ Eight load_src(const void* p, size_t at) {
  Eight e;
  if (SRC_BF16) {
    bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at)), e.f);
  } else {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    *reinterpret_cast<float4*>(e.f) = __ldg(q);
    *reinterpret_cast<float4*>(e.f + 4) = __ldg(q + 1);
  }
  return e;
}

// One row's share of eight elements into a pool.  8-bit kinds take the row's largest magnitude as bits, so that
// NaN and infinity, which sort above every number, are seen: such a row is stored as zeros with a NaN scale.
//   e4m3: scale = the smallest power of two with largest / scale <= 448: x / scale is exact and the code is the
//         only rounding.  int8: scale = largest / 127, code = rint(x * (127 / largest)).
template <int KIND, int LPR>
__device__ __forceinline__ void store_row(void* pool, float* scales, size_t row, int dh, int lane, const Eight& e) {
  const int col = 8 * lane;
  const bool on = col < dh;
  if (KIND == kBf16) {
    if (on)
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(pool) + row * dh + col) =
          make_uint4(pack_bf16x2(e.f[0], e.f[1]), pack_bf16x2(e.f[2], e.f[3]), pack_bf16x2(e.f[4], e.f[5]),
                     pack_bf16x2(e.f[6], e.f[7]));
    return;
  }
  uint32_t top = 0;
  if (on) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(e.f[i]) & 0x7fffffffu);
  }
#pragma unroll
  for (int x = 1; x < LPR; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float amax = __uint_as_float(top);
  const bool odd = top >= 0x7f800000u, some = !odd && amax >= kLeast;
  float scale = 1.f, inv = 1.f;
  if (some) {
    if (KIND == kE4m3) {
      const uint32_t s = (top >> 23) - ((top & 0x7fffffu) <= 0x600000u ? 8u : 7u);   // biased exponent
      scale = __uint_as_float(s << 23);
      inv = __uint_as_float((254u - s) << 23);
    } else {
      scale = __fdiv_rn(amax, 127.f);
      inv = __fdiv_rn(127.f, amax);
    }
  }
  uint32_t w[2] = {0u, 0u};
  if (!odd) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = e.f[i] * inv, b = e.f[i + 1] * inv;
      uint32_t c;
      if (KIND == kE4m3)
        c = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
      else
        c = (static_cast<uint32_t>(__float2int_rn(a)) & 0xffu) | ((static_cast<uint32_t>(__float2int_rn(b)) & 0xffu) << 8);
      w[i >> 2] |= c << (8 * (i & 2));
    }
  }
  if (on) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + row * dh + col) = make_uint2(w[0], w[1]);
  if (lane == 0) scales[row] = odd ? __uint_as_float(0x7fc00000u) : scale;
}

// A group of LPR lanes per (new token, head): its key and its value.  Issue slots bound it more than bytes do: 24 prompts of
// 37 to 512 tokens, 16 heads of 128, fp32 to e4m3 (101 MB) take 23 us, 4.4 TB/s of 6.5, with DRAM at 50 % and 68 % of the
// slots taken, by the codes and by finding each row's sequence, length and page, loads that stand one behind the other.
// Two heads to a group were slower.  One token of 6 heads: 4 us, a launch.
template <int KIND, bool SRC_BF16, int LPR>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(const View w, const void* __restrict__ k,
                                                               const void* __restrict__ v, long long k_st, long long k_sh,
                                                               long long v_st, long long v_sh) {
  const long long g = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) / LPR;
  const int lane = threadIdx.x % LPR, col = 8 * lane;
  const long long rows = static_cast<long long>(w.c.N) * w.c.H;
  int t = -1, h = 0, page = -1, pos = -1;
  if (g < rows) {
    t = static_cast<int>(rows >> 31 == 0 ? static_cast<uint32_t>(g) / static_cast<uint32_t>(w.c.H) : g / w.c.H);
    h = static_cast<int>(g - static_cast<long long>(t) * w.c.H);
  }
  // the rows are on their way while their places are looked up, in three loads that depend on one another
  Eight ek, ev;
#pragma unroll
  for (int i = 0; i < 8; ++i) ek.f[i] = ev.f[i] = 0.f;
  if (t >= 0 && col < w.c.dh) {
    ek = load_src<SRC_BF16>(k, static_cast<size_t>(t) * k_st + static_cast<size_t>(h) * k_sh + col);
    ev = load_src<SRC_BF16>(v, static_cast<size_t>(t) * v_st + static_cast<size_t>(h) * v_sh + col);
  }
  int b = -1;
  for (unsigned todo = __ballot_sync(0xffffffffu, t >= 0); todo != 0u;) {      // a token, or two, of a warp's rows
    const int one = __shfl_sync(0xffffffffu, t, __ffs(todo) - 1);
    const int x = seq_of_row_warp(w, one, threadIdx.x & 31);
    if (t == one) b = x;
    todo &= ~__ballot_sync(0xffffffffu, t == one);
  }
  if (b >= 0) {
    const Rows r = seq_rows(w, b);
    const int len = seq_length(w, b);
    pos = len - r.count + (t - r.first);
    if (pos >= 0 && pos < len) page = page_of(w, b, pos);
  }
  // every lane takes part in the shuffles; a group without a page stores nothing
  const size_t row = page >= 0 ? slot_row(w, page, h, pos) : 0;
  const int dh = page >= 0 ? w.c.dh : 0;
  if (KIND == kBf16) {
    store_row<KIND, LPR>(w.c.k, nullptr, row, dh, lane, ek);
    store_row<KIND, LPR>(w.c.v, nullptr, row, dh, lane, ev);
  } else {
    store_row<KIND, LPR>(w.c.k, w.c.k_scale, row, dh, page >= 0 ? lane : 99, ek);
    store_row<KIND, LPR>(w.c.v, w.c.v_scale, row, dh, page >= 0 ? lane : 99, ev);
  }
}

template <int KIND>
__device__ __forceinline__ Eight read8(const void* pool, const float* scales, size_t row, int dh, int col) {
  Eight e;
  if (KIND == kBf16) {
    bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(pool) + row * dh + col)), e.f);
    return e;
  }
  const uint2 c = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + row * dh + col));
  const float s = __ldg(scales + row);
  bf16x8_to_f32(make_uint4(codes_to_bf16<KIND>(c.x).x, codes_to_bf16<KIND>(c.x).y, codes_to_bf16<KIND>(c.y).x,
                           codes_to_bf16<KIND>(c.y).y), e.f);
  if (KIND == kE4m3 && (odd_codes<kE4m3>(c.x) || odd_codes<kE4m3>(c.y))) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0x7fu) == 0x7fu) e.f[i] = __uint_as_float(0x7fc00000u);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) e.f[i] *= s;
  return e;
}

template <bool DST_BF16>
__device__ __forceinline__ void write8(void* p, size_t at, const Eight& e) {
  if (DST_BF16) {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at) =
        make_uint4(pack_bf16x2(e.f[0], e.f[1]), pack_bf16x2(e.f[2], e.f[3]), pack_bf16x2(e.f[4], e.f[5]),
                   pack_bf16x2(e.f[6], e.f[7]));
  } else {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    q[0] = *reinterpret_cast<const float4*>(e.f);
    q[1] = *reinterpret_cast<const float4*>(e.f + 4);
  }
}

// A group of LPR lanes per (sequence, head, position): blockIdx.x = sequence and head, blockIdx.y = positions.  The dense
// result's bytes bound it: 40 int8 sequences of 100 to 2000, 16 heads of 128, to bf16 (777 MB) take 131 us, 5.9 TB/s of
// 6.5 (four positions a group at once: slower); 5 of 60 to 512 in bf16 to fp32, 16 heads of 80 (33 MB), 8 us, 4.0 TB/s.
template <int KIND, bool DST_BF16, int LPR>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const View w, void* __restrict__ k, void* __restrict__ v,
                                                              int max_len) {
  const int b = blockIdx.x / w.c.H, h = blockIdx.x - b * w.c.H;
  const int col = 8 * (threadIdx.x % LPR), len = min(seq_length(w, b), max_len);
  if (col >= w.c.dh) return;
  for (long long p = blockIdx.y * (kThreads / LPR) + threadIdx.x / LPR; p < max_len;
       p += static_cast<long long>(gridDim.y) * (kThreads / LPR)) {
    const int pos = static_cast<int>(p);
    Eight ek, ev;
#pragma unroll
    for (int i = 0; i < 8; ++i) ek.f[i] = ev.f[i] = 0.f;
    const int page = pos < len ? page_of(w, b, pos) : -1;
    if (page >= 0) {
      const size_t row = slot_row(w, page, h, pos);
      ek = read8<KIND>(w.c.k, w.c.k_scale, row, w.c.dh, col);
      ev = read8<KIND>(w.c.v, w.c.v_scale, row, w.c.dh, col);
    }
    const size_t at = (static_cast<size_t>(blockIdx.x) * max_len + pos) * w.c.dh + col;
    write8<DST_BF16>(k, at, ek);
    write8<DST_BF16>(v, at, ev);
  }
}

template <int KIND, bool SRC_BF16>
int launch_write(const View& w, const void* k, const void* v, long long k_st, long long k_sh, long long v_st,
                 long long v_sh, cudaStream_t stream) {
  const int lpr = lanes_per_row(w.c.dh);
  const long long groups = static_cast<long long>(w.c.N) * w.c.H;
  const long long blocks = (groups * lpr + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return 932;
  const unsigned n = static_cast<unsigned>(blocks);
#define DSB_WRITE(L) paged_write_kernel<KIND, SRC_BF16, L><<<n, kThreads, 0, stream>>>(w, k, v, k_st, k_sh, v_st, v_sh)
  if (lpr == 2) DSB_WRITE(2);
  else if (lpr == 4) DSB_WRITE(4);
  else if (lpr == 8) DSB_WRITE(8);
  else DSB_WRITE(16);
#undef DSB_WRITE
  return cudaGetLastError() == cudaSuccess ? 0 : 933;
}

template <int KIND, bool DST_BF16>
int launch_read(const View& w, void* k, void* v, int max_len, cudaStream_t stream) {
  const int lpr = lanes_per_row(w.c.dh), per = kThreads / lpr;
  const long long bh = static_cast<long long>(w.c.B) * w.c.H;
  if (bh > 0x7fffffffLL) return 935;
  long long y = (static_cast<long long>(max_len) + per - 1) / per;
  if (y > 65535) y = 65535;
  const dim3 grid(static_cast<unsigned>(bh), static_cast<unsigned>(y));
#define DSB_READ(L) paged_read_kernel<KIND, DST_BF16, L><<<grid, kThreads, 0, stream>>>(w, k, v, max_len)
  if (lpr == 2) DSB_READ(2);
  else if (lpr == 4) DSB_READ(4);
  else if (lpr == 8) DSB_READ(8);
  else DSB_READ(16);
#undef DSB_READ
  return cudaGetLastError() == cudaSuccess ? 0 : 936;
}

}  // namespace
}  // namespace paged
}  // namespace dsb

using namespace dsb::paged;

extern "C" int dsb_paged_write(const DsbPaged* c, const void* k, const void* v, int src_bf16, long long k_st,
                               long long k_sh, long long v_st, long long v_sh, cudaStream_t stream) {
  if (bad_cache(c)) return 930;
  const int step = src_bf16 ? 8 : 4;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0 || k_st % step || k_sh % step ||
      v_st % step || v_sh % step)
    return 931;
  if (c->N == 0 || c->B == 0) return 0;
  const View w = make_view(c);
#define DSB_KIND(K)                                                                     \
  (src_bf16 ? launch_write<K, true>(w, k, v, k_st, k_sh, v_st, v_sh, stream)            \
            : launch_write<K, false>(w, k, v, k_st, k_sh, v_st, v_sh, stream))
  if (c->kind == kBf16) return DSB_KIND(kBf16);
  if (c->kind == kE4m3) return DSB_KIND(kE4m3);
  return DSB_KIND(kInt8);
#undef DSB_KIND
}

extern "C" int dsb_paged_read(const DsbPaged* c, void* k, void* v, int dst_bf16, int max_len, cudaStream_t stream) {
  if (bad_cache(c) || max_len < 0 || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0) return 934;
  if (c->B == 0 || max_len == 0) return 0;
  const View w = make_view(c);
#define DSB_KIND(K) (dst_bf16 ? launch_read<K, true>(w, k, v, max_len, stream) : launch_read<K, false>(w, k, v, max_len, stream))
  if (c->kind == kBf16) return DSB_KIND(kBf16);
  if (c->kind == kE4m3) return DSB_KIND(kE4m3);
  return DSB_KIND(kInt8);
#undef DSB_KIND
}

namespace {

// Query rows of a head above which the tensor cores take over (units of 256 rows).  Microseconds, few / many rows:
// 8 sequences of 200 to 6000, 8 heads of 64: 16 rows 17 / 27, 24 rows 31 / 28; one of 4000, 16 heads of 128: 16 rows
// 27 / 24, 24 rows 49 / 24; 4 of 1000 to 3000 in int8, 16 heads of 128: 16 rows 21 / 46, 24 rows 35 / 41.
constexpr long long kFewRows = 16;

int new_of(const DsbPaged* c, int max_new) { return max_new < 1 ? 1 : max_new > c->N ? c->N : max_new; }

}  // namespace

extern "C" long long dsb_paged_attention_workspace(const DsbPaged* c, int Hq, int max_new, int window, int sinks) {
  if (bad_cache(c) || c->N == 0 || c->B == 0) return 0;
  max_new = new_of(c, max_new);
  const long long rows = static_cast<long long>(max_new) * (Hq / c->H);
  return rows <= kFewRows ? few_workspace(c, window, sinks, max_new, static_cast<int>(rows)) : chunk_workspace(c);
}

extern "C" int dsb_paged_attention(const DsbPaged* c, const void* q, long long q_st, long long q_sh, void* out, int Hq,
                                   int max_new, int window, int sinks, float scale, void* workspace, cudaStream_t stream) {
  if (bad_cache(c) || Hq <= 0 || Hq % c->H != 0 || window < 0 || sinks < 0 || max_new < 0) return 940;
  if ((reinterpret_cast<uintptr_t>(q) & 15) != 0 || q_st % 8 || q_sh % 8 || c->H > 65535 || c->B > 65535 ||
      static_cast<long long>(c->N) * (Hq / c->H) > kMostPositions)
    return 941;
  // results leave in words of 32 bytes, pieces come and go in words of 16
  if ((reinterpret_cast<uintptr_t>(out) & 31) != 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return 941;
  if (c->N == 0) return 0;
  if (c->B == 0) {
    const size_t bytes = static_cast<size_t>(c->N) * Hq * c->dh * sizeof(__nv_bfloat16);
    return cudaMemsetAsync(out, 0, bytes, stream) == cudaSuccess ? 0 : 942;
  }
  if (workspace == nullptr && dsb_paged_attention_workspace(c, Hq, max_new, window, sinks) > 0) return 943;
  AttnParams p;
  p.w = make_view(c);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.Hq = Hq;
  p.G = Hq / c->H;
  p.by_g = make_divisor(p.G);
  p.window = window > 0 && window < kMostPositions ? window : kMostPositions;
  p.sinks = sinks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = nullptr;
  p.meta = nullptr;
  p.workers = 0;
  max_new = new_of(c, max_new);
  const long long rows = static_cast<long long>(max_new) * p.G;
  return rows <= kFewRows ? launch_few(p, window, sinks, max_new, rows, workspace, stream) : launch_chunk(p, workspace, stream);
}
