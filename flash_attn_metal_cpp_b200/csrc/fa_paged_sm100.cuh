// fa_paged_sm100.cuh - attention of many query rows over a paged cache
// (fp16 / bf16) on the 5th-generation tensor cores: prompt chunks, runs of
// tokens to verify, and the shared prefix of a batch, whose keys meet the
// query rows of all requests at once.
//
// The rows that read the same keys are packed: row r = token * group + head
// of the group, so a KV head's whole group (and, for a shared prefix, the
// whole batch) fills the 128 rows of an MMA. One block takes 256 packed rows
// (two tiles) of one KV head and a range of the keys. The mapping on the SM
// is that of the contiguous kernel (fa_fwd_sm100.cuh): two softmax
// warpgroups, one per tile, that ping-pong with one MMA thread; S and P in
// TMEM, O in TMEM, lazily rescaled. What differs:
//   * K and V come page by page: a tile of 128 keys is up to 16 TMA boxes of
//     gcd(page_size, 128) slots by 64 columns, each sent by its own lane of
//     the producer warp, which looked its page up one tile earlier.
//   * Slots outside the visible range hold anything, NaN included. Scores of
//     such keys are masked by selection; their V rows (0 * NaN is NaN) are
//     zeroed by the V producer after its copies landed and before the MMA
//     thread is told: only edge tiles pay for that.
//   * Q rows are gathered by the softmax warps (whole rows, cp.async) into the
//     swizzled layout the MMA reads, so any packing and stride is fine.
//   * P has V's type (one MMA takes one type): rounded to bf16 or fp16, half
//     a step of 2^-8 or 2^-11 of each weight; everything else is fp32.
//   * Columns beyond head_dim (below 64 or 128) are zero-filled by the TMA.
// What bounds it: the chain of a step (S = Q K^T, load, maximum, exponentials,
// P, O += P V, and only then the tile's next S, whose columns P takes), which
// two row tiles do not hide. No pipe is full: in prompt chunks and in a prefix
// of 32768 keys the tensor pipe is busy 48 and 64 % of the time, the
// exponentials' 42 and 56 %, 33 % of the issue slots are taken. K and V come
// from L2 for all blocks of one KV head but the first. A step of 256 rows by
// 128 keys takes 2.2 us at D = 128 (1120 TFLOP/s with all SMs at it; its MMAs
// alone would take 1.5, its exponentials 1.1), a block's start and end 6 to 9
// us: a prefix of 32768 keys under 2048 rows on 8 KV heads takes 290 us in 128
// blocks of 128 steps, 4 prompt chunks of 335 to 840 tokens over 1165 to 3932
// cached ones 126 us.
#pragma once

#include "fa_paged.cuh"

#include <type_traits>

namespace fa {
namespace paged_tc {

constexpr int BM = 128, NT = 2, BN = 128;
constexpr int kThreads = 384;
constexpr int kKWarp = 8, kMmaWarp = 9, kVWarp = 10;
// As in fa_fwd_sm100.cuh: 384 x 168 registers at launch = 2 x 128 x 216 + 128 x 72.
constexpr uint32_t kRegsLaunch = 168, kRegsSoftmax = 216, kRegsOther = 72;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsOther <= kThreads * kRegsLaunch, "register split exceeds launch");
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;
constexpr float kRescaleThreshold = 8.0f;
constexpr float kFastCap = 256.f;

template <int D>
struct Cfg {
  static constexpr int NBOX = D / 64;
  static constexpr int BOX_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = NBOX * BOX_BYTES;
  static constexpr int NS = (D == 128) ? 2 : 4;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = NT * TILE_BYTES;
  static constexpr int OFF_V = OFF_K + NS * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_V + NS * TILE_BYTES;
  static constexpr int SMEM_BYTES = OFF_BAR + 1024 + 1024;  // barriers and scratch, alignment slack
};

// Which rows and keys the block works on.
struct Block {
  int q0, qlen, klen;   // query tokens and keys of its request (shared prefix: all tokens, the prefix)
  int req;
  int row0, rows;       // packed rows [row0, min(row0 + 256, rows))
};

struct Bars {
  uint64_t q_full[NT], s_full[NT], p_full[NT][2], o_full[NT];
  uint64_t mma_final, v_raw;
  uint64_t k_full[4], v_full[4], k_empty[4], v_empty[4];
  uint32_t tmem_base;
  int abort_flag;
  // block search
  int part[kThreads / 32];
  int min_ahead;
  Block work;
};
static_assert(sizeof(Bars) <= 1024, "barrier space");

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The smaller of both, NaN when one of them is (fminf drops a NaN, and a NaN
// score would become the full cap).
__device__ __forceinline__ float min_nan(float x, float y) {
  float z;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
template <typename T>
__device__ __forceinline__ uint32_t pack_p(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) return pack_half2(lo, hi);
  else return pack_bf162(lo, hi);
}

// Sum of one int per thread before the calling thread (and the total); only
// the first `warps` warps have any.
__device__ __forceinline__ int scan_block(int x, int warps, int* part, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += y;
  }
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll 1
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += part[w];
    all += part[w];
  }
  *total = all;
  return before + inc - x;
}

// XF: what a score goes through before the softmax. 0: scale alone (positive);
// 1: any scale, ALiBi; 2: the tanh cap with a positive scale, caps up to
// kFastCap; 3: the tanh cap, any size and scale, ALiBi.
//
// XF 2 uses cap tanh(y) = cap (1 - 2 r), r = 1 / (1 + e^(2y)), which is
// monotone in the score: the row maximum is taken of the raw scores, and the
// weight is exp2(cap' - m - 2 cap' r) with cap' = cap log2(e). Two scores share
// one reciprocal (r1 = d2 R, r2 = d1 R, R = 1 / (d1 d2); e^(2y) is held below
// 2^40, where r is below 2^-40 anyway, so the product stays finite): 2.5
// special-function operations a score instead of 3, and 5 others (prefix of
// 32768 keys, 2048 rows on 8 KV heads: 528 us; 860 us through XF 3). A quarter
// of the weights through a polynomial on the FMA pipe measured 515 where this
// measured 538, half of them 553: left out, 4 % of one kind of call for a second
// exponential with an error of its own. r is off by at most 2^-22.5, the score
// by 2^-21 cap; caps beyond kFastCap take XF 3, whose tanh is exact in the
// relative sense. A NaN score stays NaN (min_nan).
template <int D, typename T, int XF>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_sm100(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const PagedArgs a, const PagedTc tc) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  const uint32_t sQ = smem_addr(smem + C::OFF_Q), sK = smem_addr(smem + C::OFF_K), sV = smem_addr(smem + C::OFF_V);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned long long wlim = a.wait_limit_ns ? a.wait_limit_ns : kWaitLimitNs;

  // Set-up that touches no global memory overlaps the end of the kernel in front.
  if (threadIdx.x == kKWarp * 32) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      mbar_init(smem_addr(&bars->q_full[t]), 4);
      mbar_init(smem_addr(&bars->s_full[t]), 1);
      mbar_init(smem_addr(&bars->p_full[t][0]), 4);
      mbar_init(smem_addr(&bars->p_full[t][1]), 4);
      mbar_init(smem_addr(&bars->o_full[t]), 1);
    }
    mbar_init(smem_addr(&bars->mma_final), 1);
    mbar_init(smem_addr(&bars->v_raw), 1);
    for (int s = 0; s < C::NS; ++s) {
      mbar_init(smem_addr(&bars->k_full[s]), 1);
      mbar_init(smem_addr(&bars->v_full[s]), 1);
      mbar_init(smem_addr(&bars->k_empty[s]), 1);
      mbar_init(smem_addr(&bars->v_empty[s]), 1);
    }
    bars->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_addr(&bars->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  volatile int* abort_flag = &bars->abort_flag;
  auto leave = [&]() {  // a block without work
    if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
  };
  grid_dep_wait();
  grid_dep_launch_dependents();

  // ------------------------------------------------------------ work item
  // Blocks of a request's rows stand in one line over the requests, the last
  // ones first (under a causal mask they have the most keys); within a block
  // the KV heads, within a head the parts of the keys.
  const int per_split = tc.by_split(blockIdx.x);
  const int split = blockIdx.x - per_split * tc.n_split;
  const int bi = a.by_hk(per_split);
  const int hk = per_split - bi * a.Hk;
  Block b;
  if (tc.shared) {
    const int last = a.cu_q ? min(max(a.cu_q[a.B], 0), a.total_q) : min(a.B, a.total_q);
    b.req = -1;
    b.q0 = 0;
    b.qlen = last;
    b.klen = a.pre;
    b.rows = last * a.group;
    b.row0 = bi * NT * BM;
    if (b.row0 >= b.rows) {
      leave();
      return;
    }
    if (a.win_left >= 0) {
      // The window may leave most of the prefix unseen: the earliest query of
      // the batch says how much.
      int ahead = 1 << 30;
      for (int i = threadIdx.x; i < a.B; i += kThreads) {
        const ReqView v = view_request<BN>(a, i, BM);
        if (v.qlen > 0) ahead = min(ahead, v.klen - v.qlen);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) ahead = min(ahead, __shfl_xor_sync(0xffffffffu, ahead, off));
      if (lane == 0) bars->part[warp] = ahead;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; ++w) ahead = min(ahead, bars->part[w]);
        bars->min_ahead = ahead;
      }
    }
  } else {
    const int seg = (a.B + kThreads - 1) / kThreads;
    const int i0 = min((int)threadIdx.x * seg, a.B), i1 = min(i0 + seg, a.B);
    auto blocks_of = [&](const ReqView& v) { return (v.qlen * a.group + NT * BM - 1) / (NT * BM); };
    ReqView mine;  // the first of this thread's requests (mostly its only one)
    int n = 0;
    for (int i = i0; i < i1; ++i) {
      const ReqView v = view_request<BN>(a, i, BM);
      if (i == i0) mine = v;
      n += blocks_of(v);
    }
    if (threadIdx.x == 0) bars->work.req = -1;
    int total;
    int at = scan_block(n, a.B >= kThreads ? kThreads / 32 : (a.B + 31) / 32, bars->part, &total);
    const int want = total - 1 - bi;
    if (want < 0) {
      leave();
      return;
    }
    if (want >= at && want < at + n) {
      for (int i = i0; i < i1; ++i) {
        const ReqView v = i == i0 ? mine : view_request<BN>(a, i, BM);
        const int nb = blocks_of(v);
        if (want < at + nb) {
          bars->work = Block{v.q0, v.qlen, v.klen, i, (want - at) * NT * BM, v.qlen * a.group};
          break;
        }
        at += nb;
      }
    }
    __syncthreads();
    b = bars->work;
    if (b.req < 0) {  // (offsets that overlap can make a sum no request holds)
      leave();
      return;
    }
  }

  if (tc.shared && a.win_left >= 0) __syncthreads();  // min_ahead

  // Key tiles of each row tile (absolute, in tiles of 128 keys), then the
  // part of them that this split takes. All threads compute the same.
  int lo_t[NT], hi_t[NT];
  int k_lo = 0x7fffffff, k_hi = 0;   // keys any row of the block sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r0 = b.row0 + t * BM;
    int lo = 0, hi = 0;
    if (r0 < b.rows) {
      hi = b.klen;
      if (tc.shared) {
        if (a.win_left >= 0) lo = max(0, bars->min_ahead - a.win_left);
      } else {
        const int r1 = min(r0 + BM, b.rows) - 1;
        const int p0 = b.klen - b.qlen + a.by_group(r0);
        const int p1 = b.klen - b.qlen + a.by_group(r1);
        lo = visible_keys(a, b.klen, p0).x;
        hi = visible_keys(a, b.klen, p1).y;
      }
      if (lo >= hi) lo = hi = 0;
      else {
        k_lo = min(k_lo, lo);
        k_hi = max(k_hi, hi);
      }
    }
    lo_t[t] = lo / BN;
    hi_t[t] = (hi + BN - 1) / BN;
  }
  int j_min = 0, n_kv = 0, s_lo[NT], n_kv_t[NT];
  {
    int first = 0, last = 0;
    if (k_hi > k_lo) {
      const int t0 = k_lo / BN, n = (k_hi + BN - 1) / BN - t0;
      // (n < 2^23 tiles, at most 64 parts)
      first = t0 + tc.by_split(n * split);
      last = t0 + tc.by_split(n * (split + 1));
    }
    j_min = first;
    n_kv = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int lo = max(lo_t[t], first), hi = min(hi_t[t], last);
      s_lo[t] = lo - first;
      n_kv_t[t] = max(0, hi - lo);
      if (n_kv_t[t] > 0) n_kv = max(n_kv, hi - first);
    }
  }

  if (warp >= 8) {
    reg_alloc_dec<kRegsOther>();
    if ((warp == kKWarp || warp == kVWarp) && n_kv > 0) {
      // ------------------------------------------------------ producers
      const bool is_k = warp == kKWarp;
      const CUtensorMap* tm = is_k ? &tm_k : &tm_v;
      const uint32_t ring = is_k ? sK : sV;
      uint64_t* full = is_k ? bars->k_full : bars->v_full;
      uint64_t* empty = is_k ? bars->k_empty : bars->v_empty;
      const uint32_t raw = smem_addr(&bars->v_raw);
      const int box = tc.box_rows, box_log = 31 - __clz(box), boxes = BN >> box_log;  // (a power of two)
      const int* table = tc.shared ? a.pre_table : a.table + (int64_t)b.req * a.table_stride;
      // Table entry and first slot of this lane's box in tile j (slot -1:
      // nothing to load); the entry is checked when it is used.
      auto look_up = [&](int j) {
        const int key = (j_min + j) * BN + lane * box;
        if (lane >= boxes || j >= n_kv || key >= k_hi || key + box <= k_lo) return make_int2(-1, -1);
        const int p = a.by_page(key);
        return make_int2(table[p], key - p * a.page_size);
      };
      int2 next = look_up(0);
      int raw_phase = 0, issued = 0;
      for (int j = 0; j < n_kv; ++j) {
        const int st = j % C::NS;
        bool ok = true;
        if (lane == 0) {
          ok = !*abort_flag && fa_wait(smem_addr(&empty[st]), ((j / C::NS) + 1) & 1, a.status, wlim);
          if (!ok) *abort_flag = 1;
        }
        if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
        const int kv0 = (j_min + j) * BN;
        const int page = next.y < 0 ? -1 : valid_page(a, next.x), slot = next.y;
        const unsigned on = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t bytes = (uint32_t)__popc(on) * box * 128 * C::NBOX;
        // Edge tile: some of its rows are not of visible keys.
        const bool edge = __popc(on) != boxes || kv0 < k_lo || kv0 + BN > k_hi;
        const bool clean = !is_k && edge;
        const uint32_t bfull = smem_addr(&full[st]);
        const uint32_t bar = clean ? raw : bfull;
        if (lane == 0) {
          if (bytes) mbar_arrive_expect_tx(bar, bytes);
          else mbar_arrive(bar);
        }
        __syncwarp();
        if (page >= 0) {
          const uint32_t dst = ring + st * C::TILE_BYTES + lane * box * 128;
#pragma unroll
          for (int bx = 0; bx < C::NBOX; ++bx)
            tma_load_4d(dst + bx * C::BOX_BYTES, tm, bar, bx * 64, hk, slot, page);
        }
        __syncwarp();
        next = look_up(j + 1);
        if (clean) {
          if (lane == 0) ok = fa_wait(raw, raw_phase, a.status, wlim);
          if (!__shfl_sync(0xffffffffu, (int)ok, 0)) {
            if (lane == 0) {
              *abort_flag = 1;
              fa_wait(raw, raw_phase, a.status, wlim);  // its copies are still on their way
            }
            break;
          }
          raw_phase ^= 1;
          uint8_t* tile = smem + C::OFF_V + st * C::TILE_BYTES;
          for (int e = lane; e < BN * 8; e += 32) {
            const int row = e >> 3, key = kv0 + row;
            if (key >= k_lo && key < k_hi && ((on >> (row >> box_log)) & 1)) continue;
#pragma unroll
            for (int bx = 0; bx < C::NBOX; ++bx)
              *reinterpret_cast<uint4*>(tile + bx * C::BOX_BYTES + e * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bfull);
        }
        issued = j + 1;
      }
      // Never leave the CTA with bulk copies still writing shared memory.
      if (lane == 0)
        for (int j = max(0, issued - C::NS); j < issued; ++j)
          fa_wait(smem_addr(&full[j % C::NS]), (j / C::NS) & 1, a.status, wlim);
    } else if (warp == kMmaWarp && lane == 0 && n_kv > 0) {
      // ------------------------------------------------------ MMA issuer
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_s = make_idesc(BM, BN, fmt, 0, 0);
      constexpr uint32_t idesc_o = make_idesc(BM, D, fmt, 0, 1 /*V is MN-major*/);
      const uint64_t qk_desc0 = smem_desc(smem_addr(smem), 16, 1024);
      const uint64_t v_desc0 = smem_desc(sV, C::BOX_BYTES, 1024);
      const uint32_t qk_lo0 = (uint32_t)qk_desc0, qk_hi = (uint32_t)(qk_desc0 >> 32);
      const uint32_t v_lo0 = (uint32_t)v_desc0, v_hi = (uint32_t)(v_desc0 >> 32);
      bool ok = true;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (ok && n_kv_t[t] > 0) ok = fa_wait(smem_addr(&bars->q_full[t]), 0, a.status, wlim);
      for (int j = 0; ok && j <= n_kv; ++j) {
        if (*abort_flag) { ok = false; break; }
        bool k_ready = false, v_ready = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t tS = tmem + kColS + t * 128, tO = tmem + kColO + t * 128;
          if (j >= 1 && j - 1 >= s_lo[t] && j - 1 < s_lo[t] + n_kv_t[t]) {
            const int i = j - 1, it = i - s_lo[t];
            if (!v_ready) {
              if (!fa_wait(smem_addr(&bars->v_full[i % C::NS]), (i / C::NS) & 1, a.status, wlim)) { ok = false; break; }
              v_ready = true;
            }
            const uint32_t v_lo = v_lo0 + (uint32_t)((i % C::NS) * C::TILE_BYTES >> 4);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (!fa_wait(smem_addr(&bars->p_full[t][half]), it & 1, a.status, wlim)) { ok = false; break; }
              tc_fence_after();
#pragma unroll
              for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                mma_ts_lohi(tO, tS + kk * 8, v_lo + kk * (16 * 128 >> 4), v_hi, idesc_o, (it > 0 || kk > 0) ? 1u : 0u);
            }
            if (!ok) break;
            if (it == n_kv_t[t] - 1) mma_commit(smem_addr(&bars->o_full[t]));
          }
          if (j >= s_lo[t] && j < s_lo[t] + n_kv_t[t]) {
            if (!k_ready) {
              if (!fa_wait(smem_addr(&bars->k_full[j % C::NS]), (j / C::NS) & 1, a.status, wlim)) { ok = false; break; }
              k_ready = true;
            }
            tc_fence_after();
            const uint32_t q_lo = qk_lo0 + (uint32_t)((C::OFF_Q + t * C::TILE_BYTES) >> 4);
            const uint32_t k_lo_d = qk_lo0 + (uint32_t)((C::OFF_K + (j % C::NS) * C::TILE_BYTES) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * C::BOX_BYTES + (kk & 3) * 32) >> 4;
              mma_ss_lohi(tS, q_lo + off, qk_hi, k_lo_d + off, qk_hi, idesc_s, kk > 0 ? 1u : 0u);
            }
            mma_commit(smem_addr(&bars->s_full[t]));
          }
        }
        if (!ok) break;
        // A stage that neither row tile used is released as well, once its
        // copies have landed.
        if (j < n_kv) {
          if (!k_ready && !fa_wait(smem_addr(&bars->k_full[j % C::NS]), (j / C::NS) & 1, a.status, wlim)) { ok = false; break; }
          mma_commit(smem_addr(&bars->k_empty[j % C::NS]));
        }
        if (j >= 1) {
          const int i = j - 1;
          if (!v_ready && !fa_wait(smem_addr(&bars->v_full[i % C::NS]), (i / C::NS) & 1, a.status, wlim)) { ok = false; break; }
          mma_commit(smem_addr(&bars->v_empty[i % C::NS]));
        }
      }
      if (!ok) *abort_flag = 1;
      mma_commit(smem_addr(&bars->mma_final));
      fa_wait(smem_addr(&bars->mma_final), 0, a.status, wlim);
    }
  } else {
    // ---------------------------------------------------------- softmax
    reg_alloc_inc<kRegsSoftmax>();
    const int t = warp >> 2;
    const int row = threadIdx.x & 127;
    const int pr = b.row0 + t * BM + row;      // packed row
    const bool row_ok = pr < b.rows;
    const int my_kv = (t == 0) ? n_kv_t[0] : n_kv_t[1];
    const int my_lo = j_min + ((t == 0) ? s_lo[0] : s_lo[1]);
    const int pj = a.by_group(pr);
    const int tok = row_ok ? b.q0 + pj : 0;
    const int head = hk * a.group + (pr - pj * a.group);
    constexpr int CH = D / 8;          // 16-byte pieces of a 16-bit row
    constexpr int RPI = 32 / CH;       // rows a warp moves with one instruction
    // Element offset of row `i` of the warp's 32 (a lane's own is `mine`), -1
    // for a row that does not exist.
    auto row_at = [&](int64_t mine, int i) {
      const unsigned lo = __shfl_sync(0xffffffffu, (unsigned)mine, i);
      const int hi = __shfl_sync(0xffffffffu, (int)(mine >> 32), i);
      return (int64_t)hi << 32 | lo;
    };
    if (my_kv > 0) {
      // Whole rows at a time: a lane per row would touch 32 lines with every
      // load (16 such loads took 2.5 us of a block's 12 us start-up and end).
      const T* Q = reinterpret_cast<const T*>(a.q);
      const int64_t q_at = row_ok ? (int64_t)tok * a.q_st + (int64_t)head * a.q_sh : -1;
      const int c = lane % CH;
      const uint32_t dst = sQ + t * C::TILE_BYTES + (warp & 3) * 32 * 128 + (c >> 3) * C::BOX_BYTES;
      // Hardly unrolled, here and where the output leaves: this code runs once
      // a block, and fetching its instructions takes longer than the copies.
#pragma unroll 4
      for (int i = 0; i < CH; ++i) {
        const int r = i * RPI + lane / CH;
        const int64_t at = row_at(q_at, r);
        const bool on = at >= 0 && c * 8 < a.D;
        cp_async16(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), on ? Q + at + c * 8 : Q, on);
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&bars->q_full[t]));
    }
    // Key position of the row's query, and the keys [row_lo, row_hi) it sees.
    int qpos = 0, row_lo = 0, row_hi = 0x7fffffff;
    if (row_ok) {
      if (tc.shared) {
        row_hi = b.klen;
        if (a.causal || a.win_left >= 0 || a.win_right >= 0 || (XF & 1) != 0) {
          int i = tok;
          if (a.cu_q != nullptr) {
            int lo = 0, hi = a.B;  // the last request that begins at or before the token
            while (hi - lo > 1) {
              const int mid = (lo + hi) >> 1;
              if (a.cu_q[mid] <= tok) lo = mid;
              else hi = mid;
            }
            i = lo;
          }
          const ReqView v = view_request<BN>(a, i, BM);
          qpos = v.klen - v.qlen + (tok - v.q0);
          const int2 see = visible_keys(a, v.klen, qpos);
          row_lo = see.x;
          row_hi = min(see.y, b.klen);
        }
      } else {
        qpos = b.klen - b.qlen + pj;
        const int2 see = visible_keys(a, b.klen, qpos);
        row_lo = see.x;
        row_hi = see.y;
      }
    }
    const float slope = ((XF & 1) != 0 && a.alibi != nullptr) ? a.alibi[head] * kLog2e : 0.f;
    const float cap_in = a.cap_in, cap_log2 = a.softcap * kLog2e;
    const float sl2 = XF == 0 ? a.scale_log2 : 1.f;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = lane_base + kColS + t * 128;
    const uint32_t tO = lane_base + kColO + t * 128;
    const uint32_t b_s_full = smem_addr(&bars->s_full[t]);
    const uint32_t b_p_full = smem_addr(&bars->p_full[t][0]);
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;

    for (int j = 0; j < my_kv; ++j) {
      if (*abort_flag) { ok = false; break; }
      const bool got = fa_wait(b_s_full, j & 1, a.status, wlim);
      if (!__all_sync(0xffffffffu, got)) { ok = false; *abort_flag = 1; break; }
      tc_fence_after();
      float s[BN];
      tmem_ld128(tS, s);
      const int kv0 = (my_lo + j) * BN;
      const int key_beg = row_lo - kv0, key_lim = row_hi - kv0;
      const bool need_mask = __any_sync(0xffffffffu, key_beg > 0 || key_lim < BN);
      if constexpr (XF == 1) {
        const float base = (float)(kv0 - qpos);
#pragma unroll
        for (int c = 0; c < BN; ++c) s[c] = fmaf(s[c], a.scale_log2, slope * (base + (float)c));
      }
      if constexpr (XF == 3) {
        const float base = (float)(kv0 - qpos);
#pragma unroll
        for (int c = 0; c < BN; ++c) s[c] = fmaf(cap_log2, cap_tanh(s[c] * cap_in), slope * (base + (float)c));
      }
      float ext;
      if (!need_mask) {
        ext = row_max128(s);
      } else {
        ext = -INFINITY;
#pragma unroll
        for (int c = 0; c < BN; ++c) ext = fmaxf(ext, (c < key_lim && c >= key_beg) ? s[c] : -INFINITY);
      }
      // (XF 2: e^(2y) and the score of the row maximum)
      const float cap_k = cap_in * (2.f * kLog2e);
      float m_cand = ext * sl2;
      if constexpr (XF == 2)
        m_cand = ext == -INFINITY ? -INFINITY
                                  : cap_log2 * (1.f - __fdividef(2.f, 1.f + ex2_approx(min_nan(ext * cap_k, 40.f))));
      const float m_new = fmaxf(m_run, m_cand - weight_bias<T>());
      const bool grow = m_new > m_run + kRescaleThreshold;
      const bool any_grow = __any_sync(0xffffffffu, grow);
      const float m_use = any_grow ? m_new : m_run;
      const float m_sub = (m_use == -INFINITY) ? 0.f : m_use;
      const float alpha = (m_use == m_run || m_use == -INFINITY) ? 1.f : ex2_approx(m_run - m_use);
      if (any_grow && j > 0) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(tO + c * 32, r);
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
          tmem_st32(tO + c * 32, r);
        }
      }
      float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
      // The exponent of a weight is u * sc2 + nm2: u the score, XF 2: r.
      const float sc = XF == 2 ? -2.f * cap_log2 : sl2, nm = XF == 2 ? cap_log2 - m_sub : -m_sub;
      const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
      const float2 ck2 = make_float2(cap_k, cap_k);
      auto exponents = [&](float s0, float s1) {
        float2 u = make_float2(s0, s1);
        if constexpr (XF == 2) {
          u = __fmul2_rn(u, ck2);
          u = make_float2(min_nan(u.x, 40.f), min_nan(u.y, 40.f));
          const float2 d = __fadd2_rn(make_float2(ex2_approx(u.x), ex2_approx(u.y)), make_float2(1.f, 1.f));
          const float inv = rcp_approx(d.x * d.y);
          u = __fmul2_rn(make_float2(d.y, d.x), make_float2(inv, inv));
        }
        return __ffma2_rn(u, sc2, nm2);
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[32];
        if (need_mask) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c = h * 64 + 2 * i;
            // (a masked score may be NaN and shares its reciprocal: it goes first)
            const bool on0 = c < key_lim && c >= key_beg, on1 = c + 1 < key_lim && c + 1 >= key_beg;
            const float2 x = exponents(on0 ? s[c] : 0.f, on1 ? s[c + 1] : 0.f);
            const float p0 = on0 ? ex2_approx(x.x) : 0.f, p1 = on1 ? ex2_approx(x.y) : 0.f;
            acc0 = __fadd2_rn(acc0, make_float2(p0, p1));
            p[i] = pack_p<T>(p0, p1);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c = h * 64 + 2 * i;
            const float2 x = exponents(s[c], s[c + 1]);
            const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            if (i & 1) acc1 = __fadd2_rn(acc1, e);
            else acc0 = __fadd2_rn(acc0, e);
            p[i] = pack_p<T>(e.x, e.y);
          }
        }
        tmem_st32(tS + h * 32, p);
        if (h == 0) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(b_p_full);
        }
      }
      l_run = l_run * alpha + (acc0.x + acc0.y) + (acc1.x + acc1.y);
      m_run = m_use;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_p_full + 8);
    }

    // -------------------------------------------------------- epilogue
    if (ok && my_kv > 0) {
      const bool got = fa_wait(smem_addr(&bars->o_full[t]), 0, a.status, wlim);
      if (!__all_sync(0xffffffffu, got)) { ok = false; *abort_flag = 1; }
      tc_fence_after();
    }
    if (ok && b.row0 + t * BM < b.rows) {
      const float inv_l = row_inv(l_run);
      const float lse = l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * kLn2;
      // 32 columns of the row's O, divided by the sum.
      auto take32 = [&](int col, float (&x)[32]) {
        uint32_t u[32];
        if (my_kv > 0) tmem_ld32(tO + col, u);
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = my_kv > 0 ? __uint_as_float(u[i]) * inv_l : 0.f;
      };
      const int part = tc.part0 + split;
      const int64_t prow = ((int64_t)part * a.total_q + tok) * a.Hq + head;
      if (row_ok) {
        if (tc.partial) a.parts_lse[prow] = lse;
        else if (a.lse != nullptr) a.lse[(int64_t)head * a.total_q + tok] = lse;
      }
      const int64_t o_at = (int64_t)tok * a.o_st + (int64_t)head * a.o_sh;
      if (tc.partial || tc.out_vec) {
        // Whole rows at a time here too: each warp turns its 32 rows around in
        // its part of the row tile's Q space (free: o_full came after the last
        // S MMA), 16-byte pieces XOR-swizzled by row. A 16-bit row fills its
        // 2 D bytes at once, a float32 row takes two passes.
        uint8_t* buf = smem + C::OFF_Q + t * C::TILE_BYTES + (warp & 3) * 32 * (D * 2);
        const int dt = tc.partial ? (int)kF32 : a.out_dtype;
        const int elem = dt == kF32 ? 4 : 2;
        uint8_t* base = tc.partial ? reinterpret_cast<uint8_t*>(a.parts_o) : reinterpret_cast<uint8_t*>(a.o);
        const int64_t mine = row_ok ? (tc.partial ? prow * a.D : o_at) * elem : -1;
        const int r = lane, c = lane % CH;
        const int passes = dt == kF32 ? 2 : 1, cols = D / passes;
        const int col = c * (16 / elem);  // of this lane's piece, in a pass
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass) {
#pragma unroll 1
          for (int k = 0; k < cols; k += 32) {
            float x[32];
            take32(pass * cols + k, x);
            uint8_t* to = buf + r * (D * 2);
            const int sw = r & 7;
            if (dt == kF32) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4*>(to + (((k / 4 + i) ^ sw) << 4)) =
                    make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float* y = x + 8 * i;
                *reinterpret_cast<uint4*>(to + (((k / 8 + i) ^ sw) << 4)) =
                    dt == kF16 ? make_uint4(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]), pack_half2(y[4], y[5]), pack_half2(y[6], y[7]))
                               : make_uint4(pack_bf162(y[0], y[1]), pack_bf162(y[2], y[3]), pack_bf162(y[4], y[5]), pack_bf162(y[6], y[7]));
              }
            }
          }
          __syncwarp();
          const bool col_on = pass * cols + col < a.D;
          uint8_t* dst = base + (int64_t)(pass * cols + col) * elem;
#pragma unroll 4
          for (int i = 0; i < CH; ++i) {
            const int rr = i * RPI + lane / CH;
            const int64_t at = row_at(mine, rr);
            if (at >= 0 && col_on)
              *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(buf + rr * (D * 2) + ((c ^ (rr & 7)) << 4));
          }
          __syncwarp();
        }
      } else {
        // Rows that start anywhere: element by element.
#pragma unroll 1
        for (int k = 0; k < D; k += 32) {
          float x[32];
          take32(k, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float y[4] = {x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
            if (row_ok && k + 4 * i < a.D) store_out4(a.o, o_at + k + 4 * i, a.out_dtype, y, 4);
          }
        }
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int D, typename T, int XF>
cudaError_t launch_xf(const PagedArgs& a, const PagedTc& tc, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  auto kern = paged_attn_sm100<D, T, XF>;
  constexpr int smem = Cfg<D>::SMEM_BYTES;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  const long long blocks = (long long)tc.n_blocks * a.Hk * tc.n_split;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  e = launch_pdl(kern, dim3((unsigned)blocks), dim3(kThreads), smem, st, tk, tv, a, tc);
  note_launch();
  return e;
}

template <int D, typename T>
cudaError_t launch_dt(const PagedArgs& a, const PagedTc& tc, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  if (a.softcap > 0.f && a.softcap <= kFastCap && a.scale > 0.f && a.alibi == nullptr)
    return launch_xf<D, T, 2>(a, tc, tk, tv, st);
  if (a.softcap > 0.f) return launch_xf<D, T, 3>(a, tc, tk, tv, st);
  if (a.alibi != nullptr || !(a.scale > 0.f)) return launch_xf<D, T, 1>(a, tc, tk, tv, st);
  return launch_xf<D, T, 0>(a, tc, tk, tv, st);
}

}  // namespace paged_tc
}  // namespace fa
