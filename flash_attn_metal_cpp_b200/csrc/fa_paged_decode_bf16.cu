// Instantiations of the few-rows paged attention kernel for bf16.
#include "fa_paged_decode.cuh"

namespace fa {

cudaError_t launch_paged_decode_bf16(const PagedArgs& a, cudaStream_t st) { return decode::launch_t<__nv_bfloat16>(a, st); }

}  // namespace fa
