// Instantiations of the few-rows paged attention kernel for fp16, and its launch rules.
#include "fa_paged_decode.cuh"

namespace fa {

cudaError_t launch_paged_decode_bf16(const PagedArgs& a, cudaStream_t st);

// Rows of a unit: one MMA tile of 16 query rows, or two when a request has
// more on a KV head (not above 128 columns: O of 32 rows would not fit the
// registers).
int decode_rows_per_unit(int D, long long rows) { return rows > 16 && D <= 128 ? 32 : 16; }

// One wave of blocks: two an SM, one where the ring of a block fills it. More
// and shorter runs measured slower (64 requests of up to 32769 tokens: 262 us
// with one wave, 271 with two, 280 with three).
int decode_ctas(int D, int rows_per_unit) {
  return 148 * ((D > 128 || (D > 64 && rows_per_unit == 32)) ? 1 : 2);
}

cudaError_t launch_paged_decode(const PagedArgs& a, int dtype, cudaStream_t st) {
  return dtype == kBF16 ? launch_paged_decode_bf16(a, st) : decode::launch_t<__half>(a, st);
}

}  // namespace fa
