// Instantiations of the many-rows paged attention kernel: head_dim up to 64, f16.
#include "fa_paged_sm100.cuh"

namespace fa {

cudaError_t launch_paged_tc_d64_f16(const PagedArgs& a, const PagedTc& tc, const CUtensorMap& tk, const CUtensorMap& tv,
                                   cudaStream_t st) {
  return paged_tc::launch_dt<64, __half>(a, tc, tk, tv, st);
}

}  // namespace fa
