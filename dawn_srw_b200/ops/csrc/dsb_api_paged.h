// C ABI of the paged key/value cache (paged_kernels.cu): writing, reading back, attention over pages.
// Device pointers; asynchronous on `stream`; return 0 on a successful launch.
#pragma once
#include <cuda_runtime.h>

#ifdef __cplusplus
extern "C" {
#endif

// Pages of keys and values [n_pages, H, page, dh] and the sequences that own them.
//   kind 0: bf16;  1: e4m3 codes;  2: int8 codes (8-bit kinds with fp32 scales [n_pages, H, page])
//   table [B, width] int32: page of positions [i * page, (i + 1) * page) of a sequence;
//   lengths [B]: positions of a sequence, its new tokens included;
//   starts [B + 1] or null: rows starts[b] .. starts[b + 1] of the N packed rows are the last tokens of
//   sequence b (null: row b is the last token of sequence b, N == B).  starts ascends; no two rows that are written
//   in one call may have one place (not checked: their words, codes and scales would mix).
// Page size: a power of two, 16 .. 256; dh a multiple of 16, at most 128; everything 16-byte aligned, the
// attention's result 32-byte.
// A length above width * page or a page outside the pool sets *status to 4; what it names counts as absent.
struct DsbPaged {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int* table;
  const int* lengths;
  const int* starts;
  int* status;
  int kind, n_pages, H, page, dh, B, width, N;
};

// Rows k, v [N, H, dh] (fp32 or bf16, strides in elements, unit inner stride) into their pages.
int dsb_paged_write(const struct DsbPaged* c, const void* k, const void* v, int src_bf16, long long k_st,
                    long long k_sh, long long v_st, long long v_sh, cudaStream_t stream);
// Pages to dense k, v [B, H, max_len, dh] (fp32 or bf16): zeros at and behind a length.
int dsb_paged_read(const struct DsbPaged* c, void* k, void* v, int dst_bf16, int max_len, cudaStream_t stream);
// out [N, Hq, dh] bf16 = softmax(scale * q k^T) v over the keys at or before a row's position; with window > 0 only
// the last `window` of them and the first `sinks` positions.  q bf16 [N, Hq, dh] (strides in elements), Hq a multiple
// of H; B and H at most 65535.  A row without a key, or of no sequence, is zero; what a row does not see never reaches it,
// NaN and infinities included.  max_new: the most new tokens a
// sequence has, as far as the caller knows (it chooses the kernel; a wrong one costs time only).  workspace:
// dsb_paged_attention_workspace bytes of scratch, 16-byte aligned, this call's alone while it runs.
long long dsb_paged_attention_workspace(const struct DsbPaged* c, int Hq, int max_new, int window, int sinks);
int dsb_paged_attention(const struct DsbPaged* c, const void* q, long long q_st, long long q_sh, void* out, int Hq,
                        int max_new, int window, int sinks, float scale, void* workspace, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
