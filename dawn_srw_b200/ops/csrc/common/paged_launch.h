// Host side of the attention over pages, between its launchers.
#pragma once
#include "paged_units.cuh"

namespace dsb {
namespace paged {

// Few query rows per head (paged_few_kernels.cu): units of 8 or 16 rows.
long long few_workspace(const DsbPaged* c, int window, int sinks, int max_new, int rows);
int launch_few(AttnParams& p, int window, int sinks, int max_new, long long rows, void* workspace, cudaStream_t stream);
// Many (paged_chunk_kernels.cu): units of 256 rows on the tensor cores.
long long chunk_workspace(const DsbPaged* c);
int launch_chunk(AttnParams& p, void* workspace, cudaStream_t stream);

}  // namespace paged
}  // namespace dsb
