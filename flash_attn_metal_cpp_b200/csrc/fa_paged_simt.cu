// fa_paged_simt.cu - CUDA-core attention over a paged cache, and the join of
// partial units that it shares with the tensor-core decoding kernel.
//
// Right for every case: fp32 (kept in fp32 end to end), any head_dim up to
// 256, any strides and alignment, any number of query rows. Online softmax in
// log2 units as in the other kernels: x = scale q.k (capped, biased), running
// m and l, o = sum exp2(x - m) v.
//
// One block of 4 warps works through its run of tiles (fa_paged.cuh). In a
// warp 8 lanes share one key (each holds every 8th 16-byte piece of its row),
// so 4 keys are in work at once and a dot product needs 3 shuffles; every group
// of 8 lanes keeps its own m, l and o until the unit ends. A unit has 1 row (one
// query head on a KV head) or 4 rows (2 for head_dim above 128) that use each
// key row loaded.
//
// Bound by memory latency: with one row the warps an SM holds cover it better
// than a second key a lane group has in flight (D = 64, 64 requests of 8000
// tokens on 8 heads: 363 us, 5.8 TB/s, with 24 warps, 457 with 16 warps and two
// keys); with 4 rows the registers decide the warps, and two keys give the
// scheduler 8 independent dot products (32 heads on 8 KV heads: 739 and 770 us).
// 16 or 32 lanes a key, for fewer registers at D = 128 and 256, double the
// shuffles and the softmax work: 1525 us instead of 1190. Clusters (narrow
// tables) leave warps over, so there 4 keys in flight pay (16 requests of 250
// tokens, 16 heads of 64: 9.4 us, with one key 10.2; not above 64 columns: 8
// requests of 250, 4 KV heads of 256, 9.8 us with two keys, 9.1 with one). 8
// requests of 200 to 1025 tokens, 8 heads of 64, take 9.2 us, of 8000 tokens
// 55 us (4.8 TB/s).
//
// More than 4 rows a unit share nothing: a prompt chunk reads its keys again
// for every 4 rows (2 above 128 columns), from L2, and a shared prefix is read
// by every request. 8 requests of 4 tokens over 2000, 32 heads on 8 KV heads of
// 128, take 162 us, 4 chunks of 512 tokens over 2000 10.2 ms (7 TFLOP/s), 64
// single tokens behind a prefix of 4096 keys 436 us.
#include "fa_paged.cuh"

#include <algorithm>

namespace fa {
namespace {

constexpr int kTile = 32;
constexpr int kThreads = 128;

// DPL elements of a row: lane `sub` of 8 holds vectors sub, sub + 8, ...
template <typename T, int DPL, bool VEC>
__device__ __forceinline__ void load_slice(const T* row, int sub, int D, float (&x)[DPL]) {
  if constexpr (VEC) {
    static_assert(sizeof(T) == 4, "vector slices are used for fp32 only");
#pragma unroll
    for (int i = 0; i < DPL / 4; ++i) {
      const int col = (i * 8 + sub) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < D) v = *reinterpret_cast<const float4*>(row + col);
      x[4 * i] = v.x;
      x[4 * i + 1] = v.y;
      x[4 * i + 2] = v.z;
      x[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      const int col = i * 8 + sub;
      x[i] = col < D ? cvt_in<T>(row[col]) : 0.f;
    }
  }
}

template <int DPL, bool VEC>
__device__ __forceinline__ int slice_col(int sub, int i) {
  return VEC ? ((i / 4) * 8 + sub) * 4 + (i & 3) : i * 8 + sub;
}

// CL: clusters of blocks share uncut units (PagedArgs::cluster_shift).
template <typename T, int DM, int R, bool VEC, bool CL>
__global__ void __launch_bounds__(kThreads) paged_simt_kernel(const PagedArgs a) {
  constexpr int DPL = DM / 8;
  // Keys a lane group has in flight.
  constexpr int U = CL && R == 1 && DM <= 64 ? 4 : R > 1 && DM <= 128 ? 2 : 1;
  __shared__ RunScratch scratch;
  __shared__ float sm_o[4][R][DM];
  __shared__ float sm_m[4][R], sm_l[4][R];
  __shared__ __align__(16) float sm_part[CL ? R * DM + 2 * R : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int sub = lane & 7, kg = lane >> 3;
  const int sd = (a.D + 3) & ~3;

  grid_dep_wait();
  grid_dep_launch_dependents();
  const Run run = find_run<kTile, kThreads>(a, R, &scratch);
  if (run.end <= run.begin) {
    if (!CL && a.split && tid == 0) a.meta[blockIdx.x].n_runs = 0;
    return;
  }
  const T* Q = reinterpret_cast<const T*>(a.q);
  const T* K = reinterpret_cast<const T*>(a.k);
  const T* V = reinterpret_cast<const T*>(a.v);

  int req = run.req;
  int req_begin = run.req_begin;
  ReqView v = run.view;
  int at = run.begin;
  while (at < run.end) {
    const int per = v.per_unit(a);
    const int off = at - req_begin;
    if (off >= v.units * per) {
      req_begin += v.units * per;
      if (++req >= a.B) break;
      v = view_request<kTile>(a, req, R);
      continue;
    }
    const int unit = (unsigned)off / (unsigned)per;
    const int unit_begin = req_begin + unit * per;
    const int t_end = v.tile_lo + v.tiles;
    int t0 = v.tile_lo, t1 = t_end;
    if constexpr (CL) {
      const int rank = blockIdx.x & ((1 << a.cluster_shift) - 1);
      t1 = t0 + share_begin(a, v.tiles, rank + 1);
      t0 += share_begin(a, v.tiles, rank);
    } else if (a.split) {
      t0 += tile_at(at - unit_begin);
      if (run.end < unit_begin + per) t1 = v.tile_lo + tile_at(run.end - unit_begin);
    }
    const int chunk = a.by_hk(unit);
    const int hk = unit - chunk * a.Hk;
    const int row0 = chunk * R;
    const int rows = min(R, v.qlen * a.group - row0);
    if (!CL && a.split && at == run.begin && tid == 0) {
      RunMeta& mt = a.meta[blockIdx.x];
      mt.begin = run.begin;
      mt.unit_begin = unit_begin;
      mt.unit_end = unit_begin + per;
      mt.total = run.total;
      mt.n_runs = run.n_runs;
      mt.q0 = v.q0;
      mt.row0 = row0;
      mt.rows = rows;
      mt.hk = hk;
    }

    float q[R][DPL], o[R][DPL], m[R], l[R];
    int2 vis[R];
    float slope[R];
    int qpos[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + min(r, rows - 1);
      const int j = a.by_group(row), head = hk * a.group + row - j * a.group;
      load_slice<T, DPL, VEC>(Q + (int64_t)(v.q0 + j) * a.q_st + (int64_t)head * a.q_sh, sub, a.D, q[r]);
      qpos[r] = v.klen - v.qlen + j;
      vis[r] = visible_keys(a, v.klen, qpos[r]);
      slope[r] = a.alibi ? a.alibi[head] : 0.f;
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) o[r][i] = 0.f;
    }
    const int key_begin = max(v.key_lo, t0 * kTile), key_end = min(v.klen, t1 * kTile);
    // Table entries one step ahead of the rows they lead to.
    int2 next[U];
    auto fetch = [&](int base) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = base + u * 16 + kg;
        next[u] = key >= key_begin && key < key_end ? find_key(a, req, key) : make_int2(-1, -1);
      }
    };
    const int base0 = t0 * kTile + warp * 4;
    fetch(base0);
    for (int base = base0; base < key_end; base += 16 * U) {
      float kx[U][DPL], vx[U][DPL];
      bool on[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        on[u] = next[u].y >= 0 && valid_page(a, next[u].x) >= 0;
        if (on[u]) {
          const int64_t page = next[u].x, slot = next[u].y;
          load_slice<T, DPL, VEC>(K + page * a.k_sp + slot * a.k_ss + (int64_t)hk * a.k_sh, sub, a.D, kx[u]);
          load_slice<T, DPL, VEC>(V + page * a.v_sp + slot * a.v_ss + (int64_t)hk * a.v_sh, sub, a.D, vx[u]);
        } else {
#pragma unroll
          for (int i = 0; i < DPL; ++i) kx[u][i] = vx[u][i] = 0.f;
        }
      }
      fetch(base + 16 * U);
      // Every score of the step before any of its branches, so that the dot
      // products and their shuffles overlap.
      float x[U][R];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[u][r] = 0.f;
#pragma unroll
          for (int i = 0; i < DPL; ++i) x[u][r] = fmaf(q[r][i], kx[u][i], x[u][r]);
        }
      }
#pragma unroll
      for (int d = 1; d < 8; d *= 2) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) x[u][r] += __shfl_xor_sync(0xffffffffu, x[u][r], d);
      }
      if (a.softcap > 0.f) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) x[u][r] = a.softcap * tanhf(x[u][r] * a.cap_in);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) x[u][r] *= a.scale;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int key = base + u * 16 + kg;
          x[u][r] = fmaf(slope[r], (float)(key - qpos[r]), x[u][r]) * kLog2e;
          if (!on[u] || key < vis[r].x || key >= vis[r].y) x[u][r] = -INFINITY;
          top = fmaxf(top, x[u][r]);
        }
        if (top > m[r]) {
          const float f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top);
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < DPL; ++i) o[r][i] *= f;
          m[r] = top;
        }
        // (a score of -inf, hidden or an overflow, leaves the row as it is)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (x[u][r] != -INFINITY) {
            const float p = exp2f(x[u][r] - m[r]);
            l[r] += p;
#pragma unroll
            for (int i = 0; i < DPL; ++i) o[r][i] = fmaf(p, vx[u][i], o[r][i]);
          }
        }
      }
    }
    // The warp's four key groups, then the block's four warps.
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top);
      float ls = l[r] * f;
      ls += __shfl_xor_sync(0xffffffffu, ls, 8);
      ls += __shfl_xor_sync(0xffffffffu, ls, 16);
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        float x = o[r][i] * f;
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (kg == 0) sm_o[warp][r][slice_col<DPL, VEC>(sub, i)] = x;
      }
      if (lane == 0) {
        sm_m[warp][r] = top;
        sm_l[warp][r] = ls;
      }
    }
    __syncthreads();
    const bool whole = t0 == v.tile_lo && t1 == t_end;
    const int slot = blockIdx.x * 2 + (at == run.begin ? 0 : 1);
    for (int e = tid; e < rows * (DM / 4); e += kThreads) {
      const int r = e / (DM / 4), col = e % (DM / 4) * 4;
      if (col >= a.D) continue;
      float top = sm_m[0][r];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, sm_m[w][r]);
      float x[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = sm_m[w][r] == -INFINITY ? 0.f : exp2f(sm_m[w][r] - top);
        ls = fmaf(f, sm_l[w][r], ls);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fmaf(f, sm_o[w][r][col + i], x[i]);
      }
      if constexpr (CL) {
        *reinterpret_cast<float4*>(sm_part + r * DM + col) = make_float4(x[0], x[1], x[2], x[3]);
        if (col == 0) *reinterpret_cast<float2*>(sm_part + R * DM + 2 * r) = make_float2(top, ls);
      } else if (whole) {
        const int row = row0 + r, j = a.by_group(row);
        finish_row4(a, v.q0 + j, hk * a.group + row - j * a.group, col, x, top, ls);
      } else {
        const int64_t sr = (int64_t)slot * a.rows_per_unit + r;
        *reinterpret_cast<float4*>(a.slot_o + sr * sd + col) = make_float4(x[0], x[1], x[2], x[3]);
        if (col == 0) a.slot_ml[sr] = make_float2(top, ls);
      }
    }
    if constexpr (CL) {
      const uint32_t part = smem_addr(sm_part);
      join_cluster<R, DM, kThreads>(a, v, row0, rows, hk, [part](int) { return part; });
      return;
    }
    __syncthreads();
    at = unit_begin + per;
  }
}

// One block joins one row of one unit that was cut between runs: the block of
// the unit's first cut does it, the others return. A single long request on
// one KV head leaves as many partial rows as there are runs, so eight warps
// share them; the order is fixed.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedArgs a) {
  __shared__ float sm_o[kJoinWarps][256];
  __shared__ float sm_m[kJoinWarps], sm_l[kJoinWarps];
  grid_dep_wait();
  grid_dep_launch_dependents();
  const int b = blockIdx.x + 1, r = blockIdx.y;
  const RunMeta mt = a.meta[b];
  if (mt.n_runs == 0 || r >= mt.rows || mt.begin == mt.unit_begin) return;
  // Run b - 1 begins in the unit's tiles too: its block joins the unit.
  const Cuts cuts(mt.total, mt.n_runs);
  const int prev = cuts.begin(b - 1);
  if (prev - mt.unit_begin > kUnitCost) return;
  const int first = b - 1, last = min(mt.n_runs, cuts.first_from(mt.unit_end));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sd = (a.D + 3) & ~3;
  auto row_of = [&](int run) {
    const int slot = run * 2 + ((run == first && prev < mt.unit_begin) ? 1 : 0);
    return (int64_t)slot * a.rows_per_unit + r;
  };
  // Each warp joins every eighth run, four of them in flight.
  float top = -INFINITY, acc[2][4] = {}, l = 0.f;
  for (int j0 = first + warp; j0 < last; j0 += 4 * kJoinWarps) {
    float2 ml[4];
    float4 x[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * kJoinWarps;
      ml[i] = make_float2(-INFINITY, 0.f);
      if (j < last) {
        const int64_t sr = row_of(j);
        ml[i] = a.slot_ml[sr];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (c * 128 + lane * 4 < a.D) x[i][c] = *reinterpret_cast<const float4*>(a.slot_o + sr * sd + c * 128 + lane * 4);
      }
    }
    float nt = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) nt = fmaxf(nt, ml[i].x);
    const float g = top == -INFINITY ? 0.f : exp2f(top - nt);
    top = nt;
    l *= g;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[c][k] *= g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (a part without visible keys has the sum 0; a row of NaN scores has no
      // maximum either, but a NaN sum, and is joined)
      if (ml[i].y == 0.f) continue;
      const float f = exp2f(ml[i].x - top);
      l = fmaf(f, ml[i].y, l);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (c * 128 + lane * 4 < a.D) {
          acc[c][0] = fmaf(f, x[i][c].x, acc[c][0]);
          acc[c][1] = fmaf(f, x[i][c].y, acc[c][1]);
          acc[c][2] = fmaf(f, x[i][c].z, acc[c][2]);
          acc[c][3] = fmaf(f, x[i][c].w, acc[c][3]);
        }
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) sm_o[warp][c * 128 + lane * 4 + i] = acc[c][i];
  if (lane == 0) {
    sm_m[warp] = top;
    sm_l[warp] = l;
  }
  __syncthreads();
  const int col = threadIdx.x * 4;
  if (col >= a.D) return;
  top = sm_m[0];
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) top = fmaxf(top, sm_m[w]);
  float x[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float f = sm_m[w] == -INFINITY ? 0.f : exp2f(sm_m[w] - top);
    ls = fmaf(f, sm_l[w], ls);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(f, sm_o[w][col + i], x[i]);
  }
  const int row = mt.row0 + r, j = a.by_group(row);
  finish_row4(a, mt.q0 + j, mt.hk * a.group + row - j * a.group, col, x, top, ls);
}

// Join of whole-row partial results: LSE = log sum_p exp(lse_p),
// o = sum_p exp(lse_p - LSE) o_p. W warps of the block's eight share a row's
// parts, so that the loads of a row are all in flight however many they are;
// a lane takes 4 columns (the kernels that write parts have head_dim <= 128).
template <int W>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedArgs a) {
  constexpr int R = 8 / W;  // rows a block
  __shared__ __align__(16) float sm_o[8][128];
  __shared__ float sm_m[8], sm_l[8];
  grid_dep_wait();
  grid_dep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = (int64_t)a.total_q * a.Hq;
  const int64_t row = blockIdx.x * (int64_t)R + warp / W;  // token * Hq + head
  const int tok = (int)(row / a.Hq), head = (int)(row - (int64_t)tok * a.Hq);
  const int first = a.cu_q ? min(max(a.cu_q[0], 0), a.total_q) : 0;
  const int last = a.cu_q ? min(max(a.cu_q[a.B], 0), a.total_q) : min(a.B, a.total_q);
  const bool on = row < rows && tok >= first && tok < last;  // else the row is of no sequence
  const int col = lane * 4;
  float x[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f, top = -INFINITY;
  if (on) {
    for (int p0 = warp % W; p0 < a.n_parts; p0 += 4 * W) {
      float lse[4];
      float4 y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + i * W;
        lse[i] = -INFINITY;
        y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < a.n_parts) {
          lse[i] = a.parts_lse[p * rows + row] * kLog2e;
          if (col < a.D) y[i] = *reinterpret_cast<const float4*>(a.parts_o + (p * rows + row) * a.D + col);
        }
      }
      const float nt = fmaxf(top, fmaxf(fmaxf(lse[0], lse[1]), fmaxf(lse[2], lse[3])));
      const float sub = nt == -INFINITY ? 0.f : nt;
      const float g = exp2f(top - sub);
      top = nt;
      l *= g;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] *= g;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = exp2f(lse[i] - sub);
        l += f;
        x[0] = fmaf(f, y[i].x, x[0]);
        x[1] = fmaf(f, y[i].y, x[1]);
        x[2] = fmaf(f, y[i].z, x[2]);
        x[3] = fmaf(f, y[i].w, x[3]);
      }
    }
  }
  if constexpr (W > 1) {
    *reinterpret_cast<float4*>(&sm_o[warp][col]) = make_float4(x[0], x[1], x[2], x[3]);
    if (lane == 0) {
      sm_m[warp] = top;
      sm_l[warp] = l;
    }
    __syncthreads();
    if (warp % W != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float mw = sm_m[warp + w];
      const float nt = fmaxf(top, mw);
      const float sub = nt == -INFINITY ? 0.f : nt;
      const float g = exp2f(top - sub), f = exp2f(mw - sub);
      top = nt;
      l = l * g + f * sm_l[warp + w];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = x[k] * g + f * sm_o[warp + w][col + k];
    }
  }
  if (!on) return;
  const float inv = row_inv(l);
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] *= inv;
  if (col < a.D) store_out4(a.o, (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + col, a.out_dtype, x, 4);
  if (lane == 0 && a.lse != nullptr)
    a.lse[(int64_t)head * a.total_q + tok] = row_lse(top, l);
}

template <typename T, int DM, int R, bool VEC>
cudaError_t launch_one(const PagedArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.n_ctas), block(kThreads);
  cudaError_t e;
  if (VEC && a.cluster_shift > 0)
    e = launch_pdl_cluster(paged_simt_kernel<T, DM, R, VEC, VEC>, grid, block, 0, st, 1u << a.cluster_shift, a);
  else
    e = launch_pdl(paged_simt_kernel<T, DM, R, VEC, false>, grid, block, 0, st, a);
  note_launch();
  return e;
}

template <typename T, bool VEC>
cudaError_t launch_dm(const PagedArgs& a, cudaStream_t st) {
  const bool one = a.rows_per_unit == 1;
  if constexpr (VEC) {
    if (a.D <= 64) return one ? launch_one<T, 64, 1, true>(a, st) : launch_one<T, 64, 4, true>(a, st);
    if (a.D <= 128) return one ? launch_one<T, 128, 1, true>(a, st) : launch_one<T, 128, 4, true>(a, st);
    return one ? launch_one<T, 256, 1, true>(a, st) : launch_one<T, 256, 2, true>(a, st);
  } else {
    if (a.D <= 64) return launch_one<T, 64, 1, false>(a, st);
    if (a.D <= 128) return launch_one<T, 128, 1, false>(a, st);
    return launch_one<T, 256, 1, false>(a, st);
  }
}

}  // namespace

// Rows a unit: the 16-byte path of fp32 takes 4 (2 above 128 columns, where
// q and o of 4 rows would not fit the registers) as soon as a request has
// more than one row on a KV head.
int simt_rows_per_unit(int dtype, bool vec, int D, long long rows) {
  if (dtype != kF32 || !vec || rows <= 1) return 1;
  return D <= 128 ? 4 : 2;
}

// One wave: what the registers let an SM hold. (D = 64, one row, 8000 tokens: 6
// blocks an SM 363 us, 8 blocks 500, 5 blocks 414.)
int simt_ctas(int D, int rows_per_unit) {
  return 148 * (rows_per_unit == 1 ? (D <= 64 ? 6 : D <= 128 ? 4 : 2) : (D <= 64 ? 3 : 2));
}

cudaError_t launch_paged_simt(const PagedArgs& a, int dtype, bool vec, cudaStream_t st) {
  switch (dtype) {
    case kF16: return launch_dm<__half, false>(a, st);
    case kBF16: return launch_dm<__nv_bfloat16, false>(a, st);
    default: return vec ? launch_dm<float, true>(a, st) : launch_dm<float, false>(a, st);
  }
}

cudaError_t launch_paged_merge(const PagedArgs& a, cudaStream_t st) {
  const bool wide = a.n_parts > 4;
  const long long rows = (long long)a.total_q * a.Hq, blocks = wide ? rows : (rows + 7) / 8;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  cudaError_t e = launch_pdl(wide ? paged_merge_kernel<8> : paged_merge_kernel<1>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  note_launch();
  return e;
}

cudaError_t launch_paged_join(const PagedArgs& a, cudaStream_t st) {
  if (a.n_ctas < 2) return cudaSuccess;
  cudaError_t e = launch_pdl(paged_join_kernel, dim3((unsigned)(a.n_ctas - 1), (unsigned)a.join_rows),
                             dim3(kJoinWarps * 32), 0, st, a);
  note_launch();
  return e;
}

}  // namespace fa
