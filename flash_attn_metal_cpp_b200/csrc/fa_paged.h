// fa_paged.h - declarations shared by the paged-cache operators: the page
// planner, the cache append, the attention over a paged cache and their host
// side (fa_paged_api.cu).
#pragma once

#include <atomic>
#include <cstdint>
#include <string>

#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/fa_b200.h"
#include "fa_internal.h"

namespace fa {

// ------------------------------------------------ host state kept in fa_api.cu
fa_status paged_fail(fa_status st, const std::string& msg);
// The current device's status words: [0] timeouts, [1] bad page, slot or length.
fa_status paged_status_words(unsigned** words);
// Cached RoPE tables of `theta` with at least `rows` rows. Refused while
// `stream` is being captured unless they are there already (building them
// allocates and synchronises).
fa_status paged_rope(float theta, int D, int rows, cudaStream_t stream, const float** cs, const float** sn);
// Tensor map of a [pages, slots, heads, D] cache of 16-bit values: boxes of
// `box_rows` slots by 64 columns of one head, 128-byte swizzle.
fa_status paged_encode(CUtensorMap* m, const void* base, bool bf16, int D, int H, int slots, int pages, int64_t sp,
                       int64_t ss, int64_t sh, int box_rows);
unsigned long long paged_wait_limit_ns();

// ------------------------------------------------------------- page planning
struct PlanArgs {
  int B, max_pages, page_size, n_free, rows;
  const int* cached;
  const int* fresh;
  const int* free_pages;
  const int* free_begin;   // NULL = 0
  int* table;
  int64_t table_stride;
  int* seq_lens;           // [B]
  int* cu;                 // [B + 1]
  int64_t* slots;          // [rows]
  int* positions;          // [rows]
  int* free_end;           // [1]
  unsigned* status;        // bad-index word
};
constexpr int kPlanMaxRequests = 8192;
cudaError_t launch_plan_pages(const PlanArgs& a, cudaStream_t stream);

// -------------------------------------------------------------- cache append
struct StoreArgs {
  int T, Hq, Hk, D, page_size;
  long long n_slots;       // num_pages * page_size
  const int64_t* slots;
  const int* positions;    // NULL: no rotation
  int table_rows;
  const float* cs;
  const float* sn;
  const void* k;
  const void* v;
  const void* q;           // NULL: none
  int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh;
  void* kc;
  void* vc;
  int64_t kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh;
  void* qo;                // contiguous [T, Hq, D]
  unsigned* status;
};
cudaError_t launch_store_kv(const StoreArgs& a, int dtype, bool vec, cudaStream_t stream);

// Lets a kernel use `bytes` of dynamic shared memory on the current device:
// asked of the driver once a device (`done`: one bit each).
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Division by a number known on the host, for numerators below 2^31:
// n / d = (umulhi(n, m) + n) >> s with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1 (Granlund and Montgomery 1994). A block of
// the attention kernels lives for a few microseconds and runs its index
// arithmetic once: what counts there is the number of instructions.
struct Div {
  unsigned m, s;
  int d;
  Div() = default;
  explicit Div(int div) : d(div) {
    s = 0;
    while ((1ull << s) < (unsigned long long)div) ++s;
    m = (unsigned)((1ull << 32) * ((1ull << s) - (unsigned long long)div) / (unsigned long long)div + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((unsigned)n, m) + (unsigned)n) >> s); }
#endif
};

// ----------------------------------------------------- attention over pages
// One call's description for every paged attention kernel. The query tokens
// of request i are rows [cu_q[i], cu_q[i + 1]) of q (row i alone when cu_q is
// NULL). Its keys are, in order, the first `pre` slots of the pages in
// pre_table and then the first seq_lens[i] slots of the pages in table row i;
// query token j of n sits at key position pre + seq_lens[i] - n + j.
struct PagedArgs {
  int B, total_q, Hq, Hk, D, group;
  int page_size, num_pages, max_pages;
  int max_len;             // most keys a table row holds (below 2^29)
  Div by_group, by_page, by_hk;
  const int* table;
  int64_t table_stride;
  const int* seq_lens;
  const int* cu_q;
  int pre;
  const int* pre_table;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_st, q_sh;
  int64_t k_sp, k_ss, k_sh;
  int64_t v_sp, v_ss, v_sh;
  void* o;
  int64_t o_st, o_sh;
  int out_dtype;
  float* lse;              // [Hq, total_q] natural log (NULL = not written)
  float scale, scale_log2;
  float softcap;           // > 0: x = softcap * tanh(scale * q.k / softcap)
  float cap_in;            // scale / softcap
  int causal, win_left, win_right;
  const float* alibi;      // [Hq] (NULL = none)
  // Partial results of whole rows, joined by a last kernel: normalised o
  // [n_parts, total_q, Hq, D] and natural-log lse [n_parts, total_q, Hq].
  int n_parts;
  int own_part;            // part that the few-rows and CUDA-core kernels write (-1: the output)
  float* parts_o;
  float* parts_lse;
  int late_wait;           // few-rows kernel: wait for the kernel in front only before ending
  // Work that the kernels cut in n_ctas equal runs (split = 1, fa_paged.cuh):
  // per run two partial units of rows_per_unit rows, and where they belong.
  int split;
  int n_ctas;
  Div by_min_run;          // least length of a run
  int units_per_req;       // uncut work, one block a unit (0: the kernel sums up the requests)
  Div by_units;
  int cluster_shift;       // > 0: a cluster of 1 << cluster_shift blocks shares an uncut unit's tiles
  int rows_per_unit;
  int join_rows;           // most rows a unit can have here (for the join's grid)
  float* slot_o;           // [n_ctas, 2, rows_per_unit, D] unnormalised
  float2* slot_ml;         // [n_ctas, 2, rows_per_unit] running max (log2 units) and sum
  struct RunMeta* meta;    // [n_ctas]
  unsigned* status;        // [0] timeouts, [1] bad index
  unsigned long long wait_limit_ns;
};

// launch_pdl with the grid in clusters of `cluster` blocks.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl_cluster(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                               unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// Where one run of the cut work begins (written by the attention kernel, read
// by the join).
struct RunMeta {
  int begin;               // of the run, in the call's line of work
  int unit_begin;          // of the unit it begins in
  int unit_end;
  int total;               // length of the line
  int n_runs;              // runs in use (0: run not in use)
  int q0;                  // first query row of the unit's request
  int row0;                // first packed row of the unit (row = token * group + head of the group)
  int rows;                // packed rows of the unit
  int hk;
};

// CUDA-core kernel: fp32 inputs, and 16-bit inputs the tensor cores' copies
// cannot take (any head_dim <= 256, any strides and alignment).
int simt_rows_per_unit(int dtype, bool vec, int D, long long rows);
int simt_ctas(int D, int rows_per_unit);
cudaError_t launch_paged_simt(const PagedArgs& a, int dtype, bool vec, cudaStream_t stream);
// Tensor-core kernel for few rows (16-bit, rows of 16-byte pieces).
int decode_rows_per_unit(int D, long long rows);
int decode_ctas(int D, int rows_per_unit);
cudaError_t launch_paged_decode(const PagedArgs& a, int dtype, cudaStream_t stream);
// Tensor-core kernel for many rows (16-bit, head_dim <= 128, pages of 8 slots
// or more): what it needs besides PagedArgs.
struct PagedTc {
  int shared;        // 1: the rows of all requests against the prefix
  int n_blocks;      // blocks of 256 packed rows (an upper bound)
  int n_split;       // parts the keys of a block are cut in
  Div by_split;
  int box_rows;      // slots of one TMA box
  int partial;       // 1: normalised partial results to part0 + split
  int part0;
  int out_vec;       // output rows start at 16-byte boundaries
};
cudaError_t launch_paged_tc_d64_f16(const PagedArgs&, const PagedTc&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);
cudaError_t launch_paged_tc_d64_bf16(const PagedArgs&, const PagedTc&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);
cudaError_t launch_paged_tc_d128_f16(const PagedArgs&, const PagedTc&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);
cudaError_t launch_paged_tc_d128_bf16(const PagedArgs&, const PagedTc&, const CUtensorMap&, const CUtensorMap&, cudaStream_t);
// Join of whole-row partial results (PagedArgs::parts_*) into o and lse.
cudaError_t launch_paged_merge(const PagedArgs& a, cudaStream_t stream);
// Join of the runs' partial units.
cudaError_t launch_paged_join(const PagedArgs& a, cudaStream_t stream);

}  // namespace fa
