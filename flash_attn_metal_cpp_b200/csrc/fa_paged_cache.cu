// fa_paged_cache.cu - the paged cache's own kernels: page planning (block
// tables, slot map, positions and offsets of a step, from request lengths
// that live on the device) and the cache append (rotate-half RoPE of K and Q,
// scatter of K and V to their slots).
#include "fa_paged.cuh"

#include <algorithm>

namespace fa {
namespace {

// ------------------------------------------------------------------ planning
// With c_i tokens cached, n_i new and P slots a page:
//   held_i  = ceil(c_i / P),  need_i = ceil((c_i + n_i) / P) - held_i
//   first_i = free_begin + sum of need before i,  cu_i = sum of n before i
//   table[i, held_i + j] = free_pages[first_i + j]            j < need_i
//   token cu_i + j: position c_i + j, slot table[i, pos / P] * P + pos % P
// A few bytes a token: bound by launch and by the latency of one scan over
// the requests (256 requests of one token 3.8 us, 48 prompts of 41447 tokens
// 5.7 us). Every block does that scan itself (8192 requests at most, in
// shared memory) and takes a share of the tokens and of the new pages; a new
// page's id is taken from the free list, not from the table another block is
// writing, so one launch does it all.
constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 1024;  // tokens a block

__device__ __forceinline__ int pages_of(int n, int page) { return (n + page - 1) / page; }

struct PlanReq {
  int c, n, held, need;
  bool bad;
};
__device__ __forceinline__ PlanReq plan_request(const PlanArgs& a, int i) {
  constexpr int kMax = 1 << 29;
  PlanReq r;
  const int c = a.cached[i], n = a.fresh[i];
  r.c = min(max(c, 0), kMax);
  r.n = min(max(n, 0), kMax);
  // Tokens behind the table's last column get no page.
  const int held = pages_of(r.c, a.page_size), after = pages_of(r.c + r.n, a.page_size);
  r.bad = r.c != c || r.n != n || after > a.max_pages;
  r.held = min(held, a.max_pages);
  r.need = min(after, a.max_pages) - r.held;
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const PlanArgs a) {
  extern __shared__ int plan_sm[];
  int* cu = plan_sm;                 // [B + 1] first token of each request
  int* first = plan_sm + a.B + 1;    // [B + 1] first entry of the free list, from free_begin
  __shared__ long long part_n[kPlanThreads / 32], part_p[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch_dependents();

  const int seg = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(tid * seg, a.B), i1 = min(i0 + seg, a.B);
  long long n_sum = 0, p_sum = 0;
  bool bad = false;
  for (int i = i0; i < i1; ++i) {
    const PlanReq r = plan_request(a, i);
    n_sum += r.n;
    p_sum += r.need;
    bad |= r.bad;
  }
  long long n_inc = n_sum, p_inc = p_sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, n_inc, off), y = __shfl_up_sync(0xffffffffu, p_inc, off);
    if (lane >= off) {
      n_inc += x;
      p_inc += y;
    }
  }
  if (lane == 31) {
    part_n[warp] = n_inc;
    part_p[warp] = p_inc;
  }
  __syncthreads();
  long long n_at = n_inc - n_sum, p_at = p_inc - p_sum, n_all = 0, p_all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) {
      n_at += part_n[w];
      p_at += part_p[w];
    }
    n_all += part_n[w];
    p_all += part_p[w];
  }
  constexpr long long kTop = 0x7fffffff;
  const bool lead = blockIdx.x == 0;
  for (int i = i0; i < i1; ++i) {
    const PlanReq r = plan_request(a, i);
    cu[i] = (int)min(n_at, kTop);
    first[i] = (int)min(p_at, kTop);
    if (lead) {
      a.cu[i] = cu[i];
      a.seq_lens[i] = r.c + r.n;
    }
    n_at += r.n;
    p_at += r.need;
  }
  int begin = a.free_begin ? *a.free_begin : 0;
  const int begin_ok = min(max(begin, 0), a.n_free);
  bad |= begin_ok != begin;
  begin = begin_ok;
  if (tid == 0) {
    cu[a.B] = (int)min(n_all, kTop);
    first[a.B] = (int)min(p_all, kTop);
    if (lead) {
      a.cu[a.B] = cu[a.B];
      *a.free_end = (int)min((long long)a.n_free, begin + p_all);
      bad |= begin + p_all > a.n_free || n_all > a.rows;
    }
  }
  if (lead && bad) note_bad_index(a.status);
  __syncthreads();

  // Largest i with at[i] <= x.
  auto find = [&](const int* at, int x) {
    int lo = 0, hi = a.B;  // at[lo] <= x < at[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  // Page `p` new pages from free_begin on; -1 behind the end of the list.
  auto free_page = [&](int p) { return p < a.n_free - begin ? a.free_pages[begin + p] : -1; };

  const int new_pages = first[a.B];
  for (long long pl = blockIdx.x * kPlanThreads + tid; pl < new_pages; pl += (long long)gridDim.x * kPlanThreads) {
    const int p = (int)pl;
    const int i = find(first, p);
    const int held = min(pages_of(min(max(a.cached[i], 0), 1 << 29), a.page_size), a.max_pages);
    a.table[(int64_t)i * a.table_stride + held + (p - first[i])] = free_page(p);
  }
  const int tokens = cu[a.B];
  const int t_end = min(a.rows, (int)(blockIdx.x + 1) * kPlanTokens);
  for (int t = blockIdx.x * kPlanTokens + tid; t < t_end; t += kPlanThreads) {
    int64_t slot = -1;
    int pos = 0;
    if (t < tokens) {
      const int i = find(cu, t);
      const PlanReq r = plan_request(a, i);
      pos = r.c + (t - cu[i]);
      const int p = pos / a.page_size;
      if (p < a.max_pages) {
        const int page = p < r.held ? a.table[(int64_t)i * a.table_stride + p] : free_page(first[i] + (p - r.held));
        if (page >= 0) slot = (int64_t)page * a.page_size + (pos - p * a.page_size);
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

// -------------------------------------------------------------- cache append
// A thread takes 8 columns of each half of a row (the pairs (i, i + D/2) of
// the rotation) for up to kHeads heads of one token, so the angles are read
// once for them; neighbouring threads hold neighbouring columns. Copy bound:
// every row is read and written once (30001 tokens, 32 query and 8 KV heads of
// 128, bf16: 738 MB in 116 us, 6.4 TB/s).
constexpr int kHeads = 4;
constexpr int kStoreThreads = 256;

template <typename T>
struct Vec8 {
  static constexpr int N = sizeof(T) * 8 / 16;  // 16-byte words
  uint4 w[N];
};
template <typename T>
__device__ __forceinline__ Vec8<T> ld8(const T* p) {
  Vec8<T> v;
#pragma unroll
  for (int i = 0; i < Vec8<T>::N; ++i) v.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return v;
}
template <typename T>
__device__ __forceinline__ void st8(T* p, const Vec8<T>& v) {
#pragma unroll
  for (int i = 0; i < Vec8<T>::N; ++i) reinterpret_cast<uint4*>(p)[i] = v.w[i];
}
template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T>& v, float (&x)[8]);
template <>
__device__ __forceinline__ void unpack8<float>(const Vec8<float>& v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __uint_as_float(v.w[i].x);
    x[4 * i + 1] = __uint_as_float(v.w[i].y);
    x[4 * i + 2] = __uint_as_float(v.w[i].z);
    x[4 * i + 3] = __uint_as_float(v.w[i].w);
  }
}
template <>
__device__ __forceinline__ void unpack8<__half>(const Vec8<__half>& v, float (&x)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const Vec8<__nv_bfloat16>& v, float (&x)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ Vec8<T> pack8(const float (&x)[8]) {
  Vec8<T> v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v.w[i] = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]),
                          __float_as_uint(x[4 * i + 3]));
  } else if constexpr (std::is_same<T, __half>::value) {
    v.w[0] = make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
  } else {
    v.w[0] = make_uint4(pack_bf162(x[0], x[1]), pack_bf162(x[2], x[3]), pack_bf162(x[4], x[5]), pack_bf162(x[6], x[7]));
  }
  return v;
}

// Cache page and slot of token t; false when it is not stored (a negative
// slot: padding; a slot behind the cache: noted).
__device__ __forceinline__ bool find_slot(const StoreArgs& a, int t, int64_t* page, int* off) {
  const int64_t slot = a.slots[t];
  if (slot < 0) return false;
  if (slot >= a.n_slots) {
    note_bad_index(a.status);
    return false;
  }
  if (a.n_slots < (1ll << 31)) {  // the usual case: a 32-bit division
    *page = (unsigned)slot / (unsigned)a.page_size;
  } else {
    *page = slot / a.page_size;
  }
  *off = (int)(slot - *page * a.page_size);
  return true;
}

// Row of the angle tables of token t, -1 for no rotation.
__device__ __forceinline__ int find_angle(const StoreArgs& a, int t) {
  if (a.positions == nullptr) return -1;
  const int p = a.positions[t];
  if ((unsigned)p >= (unsigned)a.table_rows) {
    note_bad_index(a.status);
    return -1;
  }
  return p;
}

template <typename T>
__global__ void __launch_bounds__(kStoreThreads) store_kv_vec_kernel(const StoreArgs a) {
  const int half = a.D / 2, chunks = half / 8;
  const int gq = (a.Hq + kHeads - 1) / kHeads, gk = (a.Hk + kHeads - 1) / kHeads;
  const int per_token = (gq + 2 * gk) * chunks;
  const long long total = (long long)a.T * per_token;
  grid_dep_wait();
  grid_dep_launch_dependents();
  for (long long e = blockIdx.x * (long long)kStoreThreads + threadIdx.x; e < total;
       e += (long long)gridDim.x * kStoreThreads) {
    const int t = (int)(e / per_token);
    const int rest = (int)(e - (long long)t * per_token);
    const int grp = rest / chunks, col = (rest - grp * chunks) * 8;
    const bool is_q = grp < gq, is_k = !is_q && grp < gq + gk;
    const int h0 = (is_q ? grp : is_k ? grp - gq : grp - gq - gk) * kHeads;
    const int n = min(kHeads, (is_q ? a.Hq : a.Hk) - h0);
    const T* src;
    T* dst;
    int64_t sh, dh;
    if (is_q) {
      src = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.q_st + (int64_t)h0 * a.q_sh;
      dst = reinterpret_cast<T*>(a.qo) + ((int64_t)t * a.Hq + h0) * a.D;
      sh = a.q_sh;
      dh = a.D;
    } else {
      int64_t page;
      int off;
      if (!find_slot(a, t, &page, &off)) continue;
      if (is_k) {
        src = reinterpret_cast<const T*>(a.k) + (int64_t)t * a.k_st + (int64_t)h0 * a.k_sh;
        dst = reinterpret_cast<T*>(a.kc) + page * a.kc_sp + (int64_t)off * a.kc_ss + (int64_t)h0 * a.kc_sh;
        sh = a.k_sh;
        dh = a.kc_sh;
      } else {
        src = reinterpret_cast<const T*>(a.v) + (int64_t)t * a.v_st + (int64_t)h0 * a.v_sh;
        dst = reinterpret_cast<T*>(a.vc) + page * a.vc_sp + (int64_t)off * a.vc_ss + (int64_t)h0 * a.vc_sh;
        sh = a.v_sh;
        dh = a.vc_sh;
      }
    }
    src += col;
    dst += col;
    Vec8<T> x[kHeads], y[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
      if (h < n) {
        x[h] = ld8<T>(src + h * sh);
        y[h] = ld8<T>(src + h * sh + half);
      }
    const int pos = (is_q || is_k) ? find_angle(a, t) : -1;
    if (pos >= 0) {
      float c[8], s[8];
      unpack8<float>(ld8<float>(a.cs + (int64_t)pos * half + col), c);
      unpack8<float>(ld8<float>(a.sn + (int64_t)pos * half + col), s);
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        if (h < n) {
          float xa[8], xb[8], ra[8], rb[8];
          unpack8<T>(x[h], xa);
          unpack8<T>(y[h], xb);
          rope_rotate8(xa, xb, c, s, ra, rb);
          x[h] = pack8<T>(ra);
          y[h] = pack8<T>(rb);
        }
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
      if (h < n) {
        st8<T>(dst + h * dh, x[h]);
        st8<T>(dst + h * dh + half, y[h]);
      }
  }
}

template <typename T>
__device__ __forceinline__ T cvt_to(float x);
template <>
__device__ __forceinline__ float cvt_to<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half cvt_to<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 cvt_to<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Any head_dim, stride and alignment: one pair of columns (or the last
// column of an odd row, which has no partner and is kept) a step.
template <typename T>
__global__ void __launch_bounds__(kStoreThreads) store_kv_elem_kernel(const StoreArgs a) {
  const int half = a.D / 2, pairs = a.D - half;
  const int per_token = (a.Hq + 2 * a.Hk) * pairs;
  const long long total = (long long)a.T * per_token;
  grid_dep_wait();
  grid_dep_launch_dependents();
  for (long long e = blockIdx.x * (long long)kStoreThreads + threadIdx.x; e < total;
       e += (long long)gridDim.x * kStoreThreads) {
    const int t = (int)(e / per_token);
    const int rest = (int)(e - (long long)t * per_token);
    int h = rest / pairs;
    const int i = rest - h * pairs;
    const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hk;
    const T* src;
    T* dst;
    if (is_q) {
      src = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
      dst = reinterpret_cast<T*>(a.qo) + ((int64_t)t * a.Hq + h) * a.D;
    } else {
      int64_t page;
      int off;
      if (!find_slot(a, t, &page, &off)) continue;
      h -= is_k ? a.Hq : a.Hq + a.Hk;
      if (is_k) {
        src = reinterpret_cast<const T*>(a.k) + (int64_t)t * a.k_st + (int64_t)h * a.k_sh;
        dst = reinterpret_cast<T*>(a.kc) + page * a.kc_sp + (int64_t)off * a.kc_ss + (int64_t)h * a.kc_sh;
      } else {
        src = reinterpret_cast<const T*>(a.v) + (int64_t)t * a.v_st + (int64_t)h * a.v_sh;
        dst = reinterpret_cast<T*>(a.vc) + page * a.vc_sp + (int64_t)off * a.vc_ss + (int64_t)h * a.vc_sh;
      }
    }
    if (i >= half) {  // last column of an odd head_dim
      dst[a.D - 1] = src[a.D - 1];
      continue;
    }
    const int pos = (is_q || is_k) ? find_angle(a, t) : -1;
    if (pos < 0) {
      dst[i] = src[i];
      dst[i + half] = src[i + half];
    } else {
      const float c = a.cs[(int64_t)pos * half + i], s = a.sn[(int64_t)pos * half + i];
      const float xa = cvt_in<T>(src[i]), xb = cvt_in<T>(src[i + half]);
      dst[i] = cvt_to<T>(__fmaf_rn(xa, c, -__fmul_rn(xb, s)));
      dst[i + half] = cvt_to<T>(__fmaf_rn(xa, s, __fmul_rn(xb, c)));
    }
  }
}

template <typename T>
cudaError_t launch_store_t(const StoreArgs& a, bool vec, cudaStream_t st) {
  long long items;
  if (vec) items = (long long)a.T * ((a.Hq + kHeads - 1) / kHeads + 2 * ((a.Hk + kHeads - 1) / kHeads)) * (a.D / 16);
  else items = (long long)a.T * (a.Hq + 2 * a.Hk) * (a.D - a.D / 2);
  const long long blocks = std::min<long long>((items + kStoreThreads - 1) / kStoreThreads, 148 * 16);
  auto kern = vec ? store_kv_vec_kernel<T> : store_kv_elem_kernel<T>;
  cudaError_t e = launch_pdl(kern, dim3((unsigned)blocks), dim3(kStoreThreads), 0, st, a);
  note_launch();
  return e;
}

}  // namespace

cudaError_t launch_plan_pages(const PlanArgs& a, cudaStream_t st) {
  // Asked for once, for the largest plan: what a call may use depends neither on
  // the calls before it nor on another thread's (the kernel's static shared
  // memory counts against the 48 KB that need no asking).
  constexpr int most = 2 * (kPlanMaxRequests + 1) * (int)sizeof(int);
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(plan_pages_kernel), most, done);
  if (e != cudaSuccess) return e;
  const size_t smem = 2 * (size_t)(a.B + 1) * sizeof(int);
  const int blocks = std::max(1, (a.rows + kPlanTokens - 1) / kPlanTokens);
  e = launch_pdl(plan_pages_kernel, dim3((unsigned)blocks), dim3(kPlanThreads), smem, st, a);
  note_launch();
  return e;
}

cudaError_t launch_store_kv(const StoreArgs& a, int dtype, bool vec, cudaStream_t st) {
  if (a.T == 0 || a.Hq + a.Hk == 0) return cudaSuccess;
  switch (dtype) {
    case kF16: return launch_store_t<__half>(a, vec, st);
    case kBF16: return launch_store_t<__nv_bfloat16>(a, vec, st);
    default: return launch_store_t<float>(a, vec, st);
  }
}

}  // namespace fa
