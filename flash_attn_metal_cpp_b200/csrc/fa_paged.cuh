// fa_paged.cuh - device side shared by the paged attention kernels: the view
// of one request, the cut of a call's key tiles into equal runs, and the end
// of a finished row (join with partial results, division, store).
//
// Lengths live on the device, so the host cannot balance a batch of requests
// of very different lengths. Instead every block sums up the tiles of the
// call itself: a unit is (request, KV head, chunk of packed query rows), its
// key range is cut in tiles, all tiles of the call stand in one line, and
// block c of n takes tiles [c * T / n, (c + 1) * T / n). A block so holds the
// end of one unit, whole units, and the beginning of another; the two open
// ends go to the block's two partial slots and a second kernel joins them in
// the order of the blocks, so results do not depend on timing. Calls whose
// keys are few by the table's width are not cut (PagedArgs::split): the line
// then counts units and nothing is joined, or a cluster of blocks takes each
// unit and joins it in shared memory (join_cluster).
#pragma once

#include "fa_paged.h"
#include "fa_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace fa {

// Bit of the bad-index status word.
enum : unsigned { FA_DEV_BAD_INDEX = 1u };

__device__ __forceinline__ void note_bad_index(unsigned* status) { atomicOr(status + 1, FA_DEV_BAD_INDEX); }

template <typename T>
__device__ __forceinline__ float cvt_in(T x);
template <>
__device__ __forceinline__ float cvt_in<float>(float x) { return x; }
template <>
__device__ __forceinline__ float cvt_in<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float cvt_in<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// A unit costs about as much as this many tiles besides its own: Q in, rows
// joined over the warps, out. It stands in the line in front of the unit's
// tiles, so a run of many short units is not longer than one of a few long
// ones (33 requests of 1 to 8193 tokens: 33 us, 44 us without; 64 requests of
// 64 to 32769 tokens: 262 us, 297 us without).
constexpr int kUnitCost = 2;

// One request: its query rows, its keys, and the key tiles any of its rows sees.
struct ReqView {
  int q0, qlen;      // query tokens
  int klen;          // keys: shared ones in front, own ones behind
  int key_lo;        // first key the sliding window leaves visible to any row
  int tile_lo, tiles;
  int units;         // chunks * Hk
  // What a unit and the request add to the line (uncut work counts units).
  __device__ __forceinline__ int per_unit(const PagedArgs& a) const { return a.split ? tiles + kUnitCost : 1; }
  __device__ __forceinline__ int work(const PagedArgs& a) const { return units * per_unit(a); }
};

// Lengths and tables. Read past L1 by a kernel that has not waited for the one
// in front of it (PagedArgs::late_wait); else through L1, which holds the next
// tiles' entries (from L2 a ragged batch took 290 us instead of 262).
__device__ __forceinline__ int ld_index(const PagedArgs& a, const int* p) { return a.late_wait ? __ldcg(p) : *p; }

// Lengths outside the table and query ranges outside q are clipped (and noted
// in the status word): a wrong length gives a wrong row, never a wrong access.
template <int TN>
__device__ __forceinline__ ReqView view_request(const PagedArgs& a, int i, int rows_per_unit) {
  ReqView r;
  bool bad = false;
  if (a.cu_q != nullptr) {
    const int b = ld_index(a, a.cu_q + i), e = ld_index(a, a.cu_q + i + 1);
    const int b0 = min(max(b, 0), a.total_q), e0 = min(max(e, b0), a.total_q);
    bad = b0 != b || e0 != e;
    r.q0 = b0;
    r.qlen = e0 - b0;
  } else {
    r.q0 = i;
    r.qlen = i < a.total_q ? 1 : 0;
  }
  const int len = ld_index(a, a.seq_lens + i);
  const int own = min(max(len, 0), a.max_len);
  bad |= own != len;
  if (bad) note_bad_index(a.status);
  r.klen = a.pre + own;
  r.key_lo = a.win_left >= 0 ? min(max(0, r.klen - r.qlen - a.win_left), r.klen) : 0;
  r.tile_lo = (unsigned)r.key_lo / TN;
  r.tiles = max(1, (int)((unsigned)(r.klen + TN - 1) / TN) - r.tile_lo);  // a row without keys is still written
  const int chunks = (int)(((unsigned)r.qlen * (unsigned)a.group + rows_per_unit - 1u) / (unsigned)rows_per_unit);
  r.units = chunks * a.Hk;
  return r;
}

// Equal runs of a line of `total`: the first total % n are one longer. (The
// host cuts work only while the line is shorter than 2^31.)
struct Cuts {
  int quot, rest, n;
  __device__ __forceinline__ Cuts(int total, int runs) : n(runs) {
    quot = (unsigned)total / (unsigned)runs;
    rest = total - quot * runs;
  }
  __device__ __forceinline__ int begin(int run) const { return quot * run + min(run, rest); }
  // First run that begins at or behind `at`.
  __device__ __forceinline__ int first_from(int at) const {
    const int longer = rest * (quot + 1);
    if (at <= longer) return (unsigned)(at + quot) / (unsigned)(quot + 1);
    return rest + (unsigned)(at - longer + quot - 1) / (unsigned)quot;
  }
};

// The run of one block: [begin, end) of the line. A cut that falls on a unit's
// own cost, not on its tiles, is moved to the unit's beginning.
struct Run {
  int begin, end, total;
  int n_runs;
  int req;                 // request the run begins in
  int req_begin;           // where that request begins
  ReqView view;            // of that request
};

// Sums up the line and finds the block's run. Every thread of the block calls
// it; `sh` is shared scratch. A run has at least PagedArgs::min_run of the
// line: shorter runs cost more in joining than they save.
struct RunScratch {
  int part[8];
  int req_begin[2], cut[2], req[2];
  ReqView view;
};
template <int TN, int NTHREADS>
__device__ __forceinline__ Run find_run(const PagedArgs& a, int rows_per_unit, RunScratch* sh) {
  constexpr int NW = NTHREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, block = blockIdx.x;
  Run r;
  if (a.units_per_req > 0) {
    // Uncut units, as many in every request: no sum is needed.
    const int unit = block >> a.cluster_shift;
    r.n_runs = gridDim.x;
    r.total = r.n_runs;
    r.req = a.by_units(unit);
    r.req_begin = r.req * a.units_per_req;
    r.view = view_request<TN>(a, r.req, rows_per_unit);
    r.begin = unit;
    r.end = r.view.units > 0 ? unit + 1 : unit;  // (q may have fewer rows than requests)
    return r;
  }
  const int seg = a.B <= NTHREADS ? 1 : (unsigned)(a.B + NTHREADS - 1) / NTHREADS;
  const int i0 = min(tid * seg, a.B), i1 = min(i0 + seg, a.B);
  ReqView mine;  // the first of this thread's requests (mostly its only one)
  int sum = 0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    const ReqView v = view_request<TN>(a, i, rows_per_unit);
    if (i == i0) mine = v;
    sum += v.work(a);
  }
  int inc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += v;
  }
  if (lane == 31) sh->part[warp] = inc;
  if (tid < 2) sh->req[tid] = -1;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += sh->part[w];
    total += sh->part[w];
  }
  r.total = total;
  r.n_runs = min((int)gridDim.x, max(1, a.split ? a.by_min_run(total) : total));
  r.begin = r.end = 0;
  if (total == 0 || block >= r.n_runs) return r;
  const int at = before + inc - sum;
  const Cuts cuts(total, r.n_runs);
#pragma unroll 1
  for (int e = 0; e < 2; ++e) {
    const int cut = cuts.begin(block + e);
    if (cut >= at && cut < at + sum) {
      int b = at;
      ReqView v = mine;
#pragma unroll 1
      for (int i = i0; i < i1; ++i) {
        if (i > i0) v = view_request<TN>(a, i, rows_per_unit);
        const int w = v.work(a);
        if (cut < b + w) {
          if (e == 0) sh->view = v;
          const int per = v.per_unit(a);
          const int unit_begin = b + (int)((unsigned)(cut - b) / (unsigned)per) * per;
          sh->req[e] = i;
          sh->req_begin[e] = b;
          sh->cut[e] = cut - unit_begin <= kUnitCost ? unit_begin : cut;
          break;
        }
        b += w;
      }
    }
  }
  __syncthreads();
  r.req = sh->req[0];
  if (r.req < 0) return r;  // (offsets that overlap can make a sum no request holds)
  r.req_begin = sh->req_begin[0];
  r.view = sh->view;
  r.begin = sh->cut[0];
  r.end = sh->req[1] >= 0 ? sh->cut[1] : total;
  return r;
}

// First tile (counted from the unit's first) at `off` of a unit's stretch.
__device__ __forceinline__ int tile_at(int off) { return off <= kUnitCost ? 0 : off - kUnitCost; }

// Table entry of key `key` of a request and its slot in the page. The entry
// is not checked here, so that the load can stay in flight: valid_page does.
__device__ __forceinline__ int2 find_key(const PagedArgs& a, int req, int key) {
  const bool shared = key < a.pre;
  const int own = shared ? key : key - a.pre;
  const int p = a.by_page(own);
  const int slot = own - p * a.page_size;
  const int* entry = shared ? a.pre_table + p : a.table + (int64_t)req * a.table_stride + p;
  return make_int2(ld_index(a, entry), slot);
}

// The page, or -1 (and a note) when the table names none of the cache's.
__device__ __forceinline__ int valid_page(const PagedArgs& a, int page) {
  if ((unsigned)page < (unsigned)a.num_pages) return page;
  note_bad_index(a.status);
  return -1;
}

// Keys [lo, hi) visible to the query at key position `pos` of a request with
// `klen` keys.
__device__ __forceinline__ int2 visible_keys(const PagedArgs& a, int klen, int pos) {
  // (klen < 2^30 and windows <= 2^30: no sum passes 31 bits)
  int hi = klen, lo = 0;
  if (a.causal) hi = min(hi, pos + 1);
  if (a.win_right >= 0) hi = min(hi, pos + a.win_right + 1);
  if (a.win_left >= 0) lo = min(max(0, pos - a.win_left), klen);
  return make_int2(lo, max(hi, 0));
}

__device__ __forceinline__ void store_out4(void* base, int64_t idx, int out_dtype, const float (&x)[4], int n) {
  if (out_dtype == kF32) {
    float* p = reinterpret_cast<float*>(base) + idx;
    if (n == 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0)
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else
      for (int i = 0; i < n; ++i) p[i] = x[i];
  } else if (out_dtype == kF16) {
    __half* p = reinterpret_cast<__half*>(base) + idx;
    if (n == 4 && (reinterpret_cast<uintptr_t>(p) & 7) == 0)
      *reinterpret_cast<uint2*>(p) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    else
      for (int i = 0; i < n; ++i) p[i] = __float2half_rn(x[i]);
  } else {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(base) + idx;
    if (n == 4 && (reinterpret_cast<uintptr_t>(p) & 7) == 0)
      *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf162(x[0], x[1]), pack_bf162(x[2], x[3]));
    else
      for (int i = 0; i < n; ++i) p[i] = __float2bfloat16_rn(x[i]);
  }
}

// 16 bytes global -> shared (zeros, and no read, when `on` is false).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

// The running maximum of the tensor-core kernels is held this much (log2 units)
// below the true one, so weights reach 2^7 (2^15 where the many-rows kernel lets
// its maximum lag by 2^8) and fp16 holds them with full precision down to 2^-21
// of the largest, instead of 2^-14: thousands of small weights beside a large
// one would otherwise be rounded off, or away. bf16 has the range anyway.
template <typename T>
__device__ constexpr float weight_bias() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

// tanh for the score cap of the tensor-core kernels: the odd series up to y^9
// below 1/4 (its next term is under 2^-26 of the value there), else
// 1 - 2 / (1 + e^(2y)) with hardware exponential and division. Relative error
// below 2^-19, so the cap may be of any size.
__device__ __forceinline__ float cap_tanh(float y) {
  const float y2 = y * y;
  const float series =
      y * fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  const float quot = 1.f - __fdividef(2.f, 1.f + ex2_approx(y * (2.f * kLog2e)));
  return fabsf(y) < 0.25f ? series : quot;
}

// Natural-log LSE of a row with maximum m (log2 units) and sum l, and what its
// O is multiplied by. The sum is 0 only for a row without visible keys (else its
// largest weight is 1 or more, up to rounding); a NaN sum stays NaN in both.
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l)); }
__device__ __forceinline__ float row_inv(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Columns [col, col + 4) of a finished row (token, head): x holds
// sum exp2(s - m) v and l the sum of exp2(s - m), both over the row's keys
// (m in log2 units, -inf for no key). Writes the quotient and the row's lse,
// to the output or, when more partial results of the row are to be joined,
// to the call's own part of them.
__device__ __forceinline__ void finish_row4(const PagedArgs& a, int token, int head, int col, float (&x)[4], float m,
                                            float l) {
  const float inv = row_inv(l), lse = row_lse(m, l);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] *= inv;
  if (a.own_part >= 0) {
    const int64_t row = ((int64_t)a.own_part * a.total_q + token) * a.Hq + head;
    store_out4(a.parts_o, row * a.D + col, kF32, x, min(4, a.D - col));
    if (col == 0) a.parts_lse[row] = lse;
  } else {
    store_out4(a.o, (int64_t)token * a.o_st + (int64_t)head * a.o_sh + col, a.out_dtype, x, min(4, a.D - col));
    if (col == 0 && a.lse != nullptr) a.lse[(int64_t)head * a.total_q + token] = lse;
  }
}

// Units of a few tiles are cut between the blocks of a cluster, one unit a
// cluster, and joined through its shared memory instead of by a second kernel:
// a launch and its wait less. (On 8 KV heads, D = 128, one request of 500 keys
// 12.3 -> 7.0 us, 16 requests 16.4 -> 11.0 us.)

// First of a unit's tiles that block `rank` of its cluster takes.
__device__ __forceinline__ int share_begin(const PagedArgs& a, int tiles, int rank) {
  return (int)(((long long)tiles * rank) >> a.cluster_shift);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Address of a shared variable of this block in block `rank` of its cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// The end of a cluster's unit: block `rank` left its partial rows (o to `m`,
// as in finish_row4) at part_at(number of its tiles) of its own shared memory,
// [MR][DM] values and then [MR] pairs (m, l). Each block joins a part of the
// rows, in the order of the shares.
template <int MR, int DM, int NTHREADS, typename PartAt>
__device__ __forceinline__ void join_cluster(const PagedArgs& a, const ReqView& v, int row0, int rows, int hk,
                                             PartAt part_at) {
  const int n = 1 << a.cluster_shift, rank = blockIdx.x & (n - 1);
  cluster_sync();
#pragma unroll 1
  for (int e = rank * NTHREADS + threadIdx.x; e < rows * (DM / 4); e += n * NTHREADS) {
    const int r = e / (DM / 4), col = e % (DM / 4) * 4;
    if (col >= a.D) continue;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f, top = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const int tiles = share_begin(a, v.tiles, k + 1) - share_begin(a, v.tiles, k);
      if (tiles == 0) continue;
      const uint32_t part = cluster_addr(part_at(tiles), k);
      const float2 ml = ld_cluster2(part + MR * DM * 4 + r * 8);
      const float4 y = ld_cluster4(part + (r * DM + col) * 4);
      const float m_new = fmaxf(top, ml.x);
      const float f0 = top == -INFINITY ? 0.f : exp2f(top - m_new);
      const float f1 = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m_new);
      x[0] = fmaf(x[0], f0, y.x * f1);
      x[1] = fmaf(x[1], f0, y.y * f1);
      x[2] = fmaf(x[2], f0, y.z * f1);
      x[3] = fmaf(x[3], f0, y.w * f1);
      ls = fmaf(ls, f0, ml.y * f1);
      top = m_new;
    }
    const int row = row0 + r, j = a.by_group(row);
    finish_row4(a, v.q0 + j, hk * a.group + row - j * a.group, col, x, top, ls);
  }
  cluster_sync();  // the others have read this block's part
}

}  // namespace fa
