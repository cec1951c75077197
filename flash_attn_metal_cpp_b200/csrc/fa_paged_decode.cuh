// fa_paged_decode.cuh - attention of few query rows over a paged cache
// (fp16 / bf16): single tokens and short runs of tokens.
//
// What bounds it: the bytes of K and V. With g query heads on a KV head a key
// row of 4 D bytes (K and V) feeds 4 D g operations, so up to some hundred
// rows the tensor cores have idle time and the kernel's task is to keep
// enough loads in flight. What it does with each tile of 64 keys:
//   * 4 warps of 16 keys each. The unit's query rows (heads of the group times
//     tokens, 16 or 32 of them) are the M side of mma.sync m16n8k16, the
//     warp's keys the N side of S = Q K^T and the K side of O += P V, so the
//     score registers become the P operand without leaving the warp. A
//     tcgen05 tile has 128 rows and would leave 7/8 of them empty here, and
//     its softmax would cross TMEM for 16 rows. At the copy rate of the memory
//     (64 requests of 64 to 32769 tokens, 32 heads on 8 KV heads, D = 128:
//     1.68 GB in 262 us, 6.4 TB/s) mma.sync keeps the tensor pipe 19 % and the
//     issue slots 37 % busy.
//   * each warp keeps its own running max, sum and O; they meet only at the
//     end of a unit.
//   * K and V rows arrive by 16-byte cp.async in a ring of NS tiles, so any
//     page size and any row stride works (a TMA box would need pages of 8
//     rows); the page numbers of a tile are looked up one step before its
//     copies are issued, and the Q rows of a unit travel with its first tile.
//     Keys outside [first visible, end) are filled with zeros, never read.
//   * two blocks an SM (one where registers or the ring do not allow two).
// P is rounded to the input type for the PV product (half a step: 2^-8 bf16,
// 2^-11 fp16, of each weight); scores, running max, sum and O stay in fp32,
// and the sum adds the unrounded weights.
#pragma once

#include "fa_paged.cuh"

#include <type_traits>

namespace fa {
namespace decode {

constexpr int kTile = 64;
constexpr int kThreads = 128;

template <int DM, int MT>
struct Cfg {
  static constexpr int KV_BYTES = kTile * DM * 2;          // one K or V tile
  static constexpr int Q_BYTES = MT * 16 * DM * 2;
  static constexpr int STAGE = 2 * KV_BYTES + Q_BYTES;
  static constexpr int BLOCKS = (DM == 256 || (DM == 128 && MT == 2)) ? 1 : 2;  // blocks an SM
  static constexpr int NS = DM == 64 ? 5 : DM == 128 ? (MT == 1 ? 3 : 5) : 3;
};

// One tile of the block's run, as its consumers see it.
struct TileDesc {
  int rows;       // packed rows of the unit; 0 = no tile
  int row0;
  int q0, qlen, klen, key_lo;
  int req, hk, tile;
  int first, last, whole, slot;
};

template <int NS, int MT>
struct Shared {
  RunScratch scratch;
  TileDesc desc[NS + 1];
  longlong2 at[NS + 1][kTile];   // element offsets of each key's K and V row (negative: no row)
  float red_m[4][MT * 16], red_l[4][MT * 16];
};

template <int DM, int MT>
constexpr int smem_bytes() {
  return Cfg<DM, MT>::NS * Cfg<DM, MT>::STAGE + (int)sizeof(Shared<Cfg<DM, MT>::NS, MT>);
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) return pack_half2(lo, hi);
  else return pack_bf162(lo, hi);
}

// Steps through the tiles of a run: request, unit (chunk of rows, KV head), tile.
template <int MR, bool CL>
struct Cursor {
  int left;              // of the line, from the unit's beginning on
  int req, unit, per;    // per: a unit's stretch of the line
  int hk, row0;          // of the unit
  int tile, tile_end;    // of the current piece, from the unit's first tile
  bool run_first;        // the current piece is the run's first
  bool new_piece, whole;
  ReqView v;

  __device__ __forceinline__ void begin_piece(const PagedArgs& a, int first) {
    tile = first;
    tile_end = !CL && a.split && left < per ? tile_at(left) : v.tiles;
    whole = first == 0 && tile_end == v.tiles;
    new_piece = true;
  }
  __device__ __forceinline__ void start(const PagedArgs& a, const Run& run) {
    left = 0;
    run_first = true;
    if (run.end <= run.begin) return;
    req = run.req;
    v = run.view;
    per = v.per_unit(a);
    const int off = run.begin - run.req_begin;
    unit = (unsigned)off / (unsigned)per;
    const int in_unit = off - unit * per;
    left = run.end - run.begin + in_unit;
    const int chunk = a.by_hk(unit);
    hk = unit - chunk * a.Hk;
    row0 = chunk * MR;
    begin_piece(a, !CL && a.split ? tile_at(in_unit) : 0);
    if constexpr (CL) {
      const int rank = blockIdx.x & ((1 << a.cluster_shift) - 1);
      tile = share_begin(a, v.tiles, rank);
      tile_end = share_begin(a, v.tiles, rank + 1);
      whole = false;
      if (tile == tile_end) left = 0;
    }
  }

  // Describes the current tile and moves on.
  __device__ __forceinline__ void next(const PagedArgs& a, TileDesc& d) {
    d.rows = 0;
    if (left <= 0) return;
    d.req = req;
    d.hk = hk;
    d.row0 = row0;
    d.rows = min(MR, v.qlen * a.group - row0);
    d.q0 = v.q0;
    d.qlen = v.qlen;
    d.klen = v.klen;
    d.key_lo = v.key_lo;
    d.tile = v.tile_lo + tile;
    d.first = new_piece;
    d.whole = whole;
    d.slot = run_first ? 0 : 1;
    new_piece = false;
    d.last = ++tile == tile_end;
    if (d.last) {
      run_first = false;
      left -= per;
      if (!CL && left > 0) {
        if (++hk == a.Hk) {
          hk = 0;
          row0 += MR;
        }
        if (++unit == v.units) {
          unit = hk = row0 = 0;
          do {
            if (++req >= a.B) {
              left = 0;
              return;
            }
            v = view_request<kTile>(a, req, MR);
          } while (v.units == 0);
          per = v.per_unit(a);
        }
        begin_piece(a, 0);
      }
    }
  }
};

// CL: clusters of blocks share uncut units (PagedArgs::cluster_shift).
template <typename T, int DM, int MT, bool CL>
__global__ void __launch_bounds__(kThreads, (Cfg<DM, MT>::BLOCKS)) paged_decode_kernel(const PagedArgs a) {
  using C = Cfg<DM, MT>;
  constexpr int NS = C::NS, MR = MT * 16, CPR = DM / 8, NB = DM / 8, KK = DM / 16;
  extern __shared__ __align__(128) uint8_t ring[];
  Shared<NS, MT>& sh = *reinterpret_cast<Shared<NS, MT>*>(ring + NS * C::STAGE);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring_addr = smem_addr(ring);
  const T* Q = reinterpret_cast<const T*>(a.q);
  const T* K = reinterpret_cast<const T*>(a.k);
  const T* V = reinterpret_cast<const T*>(a.v);

  // With late_wait the kernel in front is the shared prefix's: this one needs
  // nothing of it and may run beside it, on the SMs it leaves free. All blocks
  // of that kernel have waited for everything before it by the time they let
  // this one start, so lengths, tables and caches are complete (and read from
  // L2). One block waits at its end instead, so that "this kernel is done"
  // still means "that one is done too" for the join that follows; the others
  // make room for the next block when their run is finished.
  if (CL || !a.late_wait) grid_dep_wait();
  grid_dep_launch_dependents();
  const Run run = find_run<kTile, kThreads>(a, MR, &sh.scratch);
  if (run.end <= run.begin) {
    if (!CL && a.split && tid == 0) a.meta[blockIdx.x].n_runs = 0;
    if (!CL && a.late_wait && blockIdx.x == 0) grid_dep_wait();
    return;
  }
  Cursor<MR, CL> cur;
  cur.start(a, run);
  if (!CL && a.split && tid == 0) {
    RunMeta& mt = a.meta[blockIdx.x];
    mt.begin = run.begin;
    mt.unit_begin = run.req_begin + cur.unit * cur.per;
    mt.unit_end = mt.unit_begin + cur.per;
    mt.total = run.total;
    mt.n_runs = run.n_runs;
    mt.q0 = cur.v.q0;
    mt.row0 = cur.row0;
    mt.rows = min(MR, cur.v.qlen * a.group - mt.row0);
    mt.hk = cur.hk;
  }

  // Table entry and slot of key `tid` of a tile (slot -1: no key).
  // put_rows() checks the entry and turns it into row offsets a tile later:
  // the load is in flight until then, and the copies need one addition each.
  auto look_up = [&](const TileDesc& d) {
    int2 ps = make_int2(-1, -1);
    if (tid < kTile && d.rows > 0) {
      const int key = d.tile * kTile + tid;
      if (key >= d.key_lo && key < d.klen) ps = find_key(a, d.req, key);
    }
    return ps;
  };
  auto put_rows = [&](int i, int2 ps, int hk) {
    if (tid >= kTile) return;
    longlong2 at = make_longlong2(-1, -1);
    if (ps.y >= 0 && valid_page(a, ps.x) >= 0) {
      at.x = (int64_t)ps.x * a.k_sp + (int64_t)ps.y * a.k_ss + (int64_t)hk * a.k_sh;
      at.y = (int64_t)ps.x * a.v_sp + (int64_t)ps.y * a.v_ss + (int64_t)hk * a.v_sh;
    }
    sh.at[i][tid] = at;
  };
  // Copies of tile `i` (slot i of desc and page) into stage `st`.
  auto issue = [&](int i, int st) {
    const TileDesc& d = sh.desc[i];
    if (d.rows > 0) {
      const uint32_t sk = ring_addr + st * C::STAGE, sv = sk + C::KV_BYTES;
      // A thread copies the same 16-byte column of every row it takes.
      const int c = tid % CPR, row0 = tid / CPR;
      const bool col_on = c * 8 < a.D;
      const T* kc = K + c * 8;
      const T* vc = V + c * 8;
#pragma unroll
      for (int n = 0; n < kTile * CPR / kThreads; ++n) {
        const int row = row0 + n * (kThreads / CPR);
        const longlong2 at = sh.at[i][row];
        const bool on = at.x >= 0 && col_on;
        const uint32_t off = row * (DM * 2) + ((c ^ (row & 7)) << 4);
        cp_async16(sk + off, on ? kc + at.x : K, on);
        cp_async16(sv + off, on ? vc + at.y : V, on);
      }
      if (d.first) {
        const uint32_t sq = sk + 2 * C::KV_BYTES;
#pragma unroll
        for (int n = 0; n < MR * CPR / kThreads; ++n) {
          const int e = n * kThreads + tid, r = e / CPR, c = e % CPR;
          const bool on = r < d.rows && c * 8 < a.D;
          const int row = d.row0 + (on ? r : 0);
          const int j = a.by_group(row), head = d.hk * a.group + row - j * a.group;
          const T* qs = on ? Q + (int64_t)(d.q0 + j) * a.q_st + (int64_t)head * a.q_sh + c * 8 : Q;
          cp_async16(sq + r * (DM * 2) + ((c ^ (r & 7)) << 4), qs, on);
        }
      }
    }
    cp_async_commit();
  };

  {
    // The first NS tiles' page numbers together. Loops stay rolled here, and
    // the first copies are issued by the main loop's code: what runs once a
    // block waits for its instructions from L2 longer than for anything else.
#pragma unroll 1
    for (int i = 0; i < NS; ++i) {
      TileDesc d;
      cur.next(a, d);
      if (tid == 0) sh.desc[i] = d;
    }
    __syncthreads();
    int2 ps[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) ps[i] = look_up(sh.desc[i]);
#pragma unroll
    for (int i = 0; i < NS; ++i) put_rows(i, ps[i], sh.desc[i].hk);
    __syncthreads();
  }

  uint32_t qf[MT][KK][4];
  float o[MT][NB][4];
  float m[MT][2], l[MT][2], slope[MT][2];
  int lo[MT][2], hi[MT][2], qpos[MT][2];
  int full_lo = 0, full_hi = 0;  // keys that every row of the unit sees
  const bool plain = a.softcap == 0.f && a.alibi == nullptr && a.scale > 0.f;
  const float cap_in = a.cap_in;
  const float cap_log2 = a.softcap * kLog2e;

  int di = 0, st = 0;          // slot and stage of the current tile
  int di_in = 0, st_in = 0;    // of the next tile to be copied
  int ahead = NS - 1;          // copies to issue before the first tile is awaited
  while (true) {
    if (ahead == 0) {
      cp_async_wait<NS - 2>();
      __syncthreads();
      if (sh.desc[di].rows == 0) break;
    }
    issue(di_in, st_in);
    di_in = di_in == NS ? 0 : di_in + 1;
    st_in = st_in == NS - 1 ? 0 : st_in + 1;
    if (ahead > 0) {
      --ahead;
      continue;
    }
    const TileDesc& d = sh.desc[di];
    TileDesc dn;
    cur.next(a, dn);
    const int2 pn = look_up(dn);

    const uint32_t sk = ring_addr + st * C::STAGE, sv = sk + C::KV_BYTES;
    if (d.first) {
      const int p0 = d.klen - d.qlen + a.by_group(d.row0), p1 = d.klen - d.qlen + a.by_group(d.row0 + d.rows - 1);
      full_hi = plain ? visible_keys(a, d.klen, p0).y : 0;
      full_lo = max(visible_keys(a, d.klen, p1).x, d.key_lo);
      const uint32_t sq = sk + 2 * C::KV_BYTES;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16 + (lane & 15);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          ldm_x4(qf[mt][kk], sq + r * (DM * 2) + (((kk * 2 + (lane >> 4)) ^ (r & 7)) << 4));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = d.row0 + min(mt * 16 + e * 8 + (lane >> 2), d.rows - 1);
          const int j = a.by_group(row);
          qpos[mt][e] = d.klen - d.qlen + j;
          const int2 see = visible_keys(a, d.klen, qpos[mt][e]);
          lo[mt][e] = see.x;
          hi[mt][e] = see.y;
          slope[mt][e] = a.alibi ? __ldcg(a.alibi + d.hk * a.group + row - j * a.group) * kLog2e : 0.f;
          m[mt][e] = -INFINITY;
          l[mt][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.f;
      }
    }

    // S = Q K^T of the warp's 16 keys (two blocks of 8).
    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.f;
    {
      const int kr = warp * 16 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t b[4];
        ldm_x4(b, sk + kr * (DM * 2) + (((kk * 2 + ((lane >> 3) & 1)) ^ (kr & 7)) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<T>(s[mt][0], qf[mt][kk], b[0], b[1]);
          mma16816<T>(s[mt][1], qf[mt][kk], b[2], b[3]);
        }
      }
    }
    // Online softmax of the warp's rows (log2 units). A tile that every row
    // sees whole, with nothing but a positive scale on the scores, needs no
    // masks and folds the scale into the exponent.
    const bool fast = d.tile * kTile >= full_lo && (d.tile + 1) * kTile <= full_hi;
    uint32_t p[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top[2];
      if (fast) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          top[e] = fmaxf(fmaxf(s[mt][0][2 * e], s[mt][0][2 * e + 1]), fmaxf(s[mt][1][2 * e], s[mt][1][2 * e + 1]));
      } else {
        const int key0 = d.tile * kTile + warp * 16 + (lane & 3) * 2;
        top[0] = top[1] = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = i >> 1, key = key0 + n * 8 + (i & 1);
            float x;
            if (a.softcap > 0.f) x = cap_log2 * cap_tanh(s[mt][n][i] * cap_in);
            else x = s[mt][n][i] * a.scale_log2;
            x = fmaf(slope[mt][e], (float)(key - qpos[mt][e]), x);
            x = (key >= lo[mt][e] && key < hi[mt][e]) ? x : -INFINITY;
            s[mt][n][i] = x;
            top[e] = fmaxf(top[e], x);
          }
      }
      const float mul = fast ? a.scale_log2 : 1.f;
      float f[2], sub[2];
      bool grow = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
        const float nm = fmaxf(m[mt][e], top[e] * mul - weight_bias<T>());
        grow |= nm > m[mt][e];
        sub[e] = nm == -INFINITY ? 0.f : nm;
        f[e] = ex2_approx(m[mt][e] - sub[e]);  // 0 for the first keys of a row
        m[mt][e] = nm;
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[mt][n][0] *= f[0];
          o[mt][n][1] *= f[0];
          o[mt][n][2] *= f[1];
          o[mt][n][3] *= f[1];
        }
        l[mt][0] *= f[0];
        l[mt][1] *= f[1];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ex2_approx(fmaf(s[mt][n][i], mul, -sub[i >> 1]));
        l[mt][0] += x[0] + x[1];
        l[mt][1] += x[2] + x[3];
        p[mt][2 * n] = pack2<T>(x[0], x[1]);
        p[mt][2 * n + 1] = pack2<T>(x[2], x[3]);
      }
    }
    // O += P V.
    {
      const int vr = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
      for (int n = 0; n < NB; n += 2) {
        uint32_t b[4];
        ldm_x4_t(b, sv + vr * (DM * 2) + (((n + (lane >> 4)) ^ (vr & 7)) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<T>(o[mt][n], p[mt], b[0], b[1]);
          mma16816<T>(o[mt][n + 1], p[mt], b[2], b[3]);
        }
      }
    }

    if (d.last) {
      // The four warps' rows meet in the stage just consumed (the copies in
      // flight go to the other stages).
      float* buf = reinterpret_cast<float*>(ring + st * C::STAGE);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 1);
          l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 2);
          if ((lane & 3) == 0) {
            sh.red_m[warp][mt * 16 + e * 8 + (lane >> 2)] = m[mt][e];
            sh.red_l[warp][mt * 16 + e * 8 + (lane >> 2)] = l[mt][e];
          }
        }
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (mt * 16 >= d.rows) break;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = e * 8 + (lane >> 2);
          float top = sh.red_m[0][mt * 16 + r];
#pragma unroll
          for (int w = 1; w < 4; ++w) top = fmaxf(top, sh.red_m[w][mt * 16 + r]);
          const float f = m[mt][e] == -INFINITY ? 0.f : ex2_approx(m[mt][e] - top);
          float* row = buf + (warp * 16 + r) * DM;
          if (mt * 16 + r >= d.rows) continue;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const int c4 = n * 2 + ((lane & 3) >> 1);
            *reinterpret_cast<float2*>(row + (((c4 ^ (r & 7)) << 2) | ((lane & 1) << 1))) =
                make_float2(o[mt][n][2 * e] * f, o[mt][n][2 * e + 1] * f);
          }
        }
        __syncthreads();
        const int rows = min(16, d.rows - mt * 16);
        for (int e = tid; e < rows * (DM / 4); e += kThreads) {
          const int r = e / (DM / 4), c4 = e % (DM / 4), col = c4 * 4;
          if (col >= a.D) continue;
          const int rr = mt * 16 + r;
          float top = sh.red_m[0][rr];
#pragma unroll
          for (int w = 1; w < 4; ++w) top = fmaxf(top, sh.red_m[w][rr]);
          float x[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float mw = sh.red_m[w][rr];
            ls = fmaf(mw == -INFINITY ? 0.f : ex2_approx(mw - top), sh.red_l[w][rr], ls);
            const float4 y = *reinterpret_cast<const float4*>(buf + (w * 16 + r) * DM + ((c4 ^ (r & 7)) << 2));
            x[0] += y.x;
            x[1] += y.y;
            x[2] += y.z;
            x[3] += y.w;
          }
          if (!CL && d.whole) {
            const int row = d.row0 + rr, j = a.by_group(row);
            finish_row4(a, d.q0 + j, d.hk * a.group + row - j * a.group, col, x, top, ls);
          } else if (CL) {
            float* part = reinterpret_cast<float*>(ring + (st == 0 ? 1 : 0) * C::STAGE);
            *reinterpret_cast<float4*>(part + rr * DM + col) = make_float4(x[0], x[1], x[2], x[3]);
            if (col == 0) reinterpret_cast<float2*>(part + MR * DM)[rr] = make_float2(top, ls);
          } else {
            const int64_t sr = ((int64_t)blockIdx.x * 2 + d.slot) * MR + rr;
            *reinterpret_cast<float4*>(a.slot_o + sr * a.D + col) = make_float4(x[0], x[1], x[2], x[3]);
            if (col == 0) a.slot_ml[sr] = make_float2(top, ls);
          }
        }
        if (mt + 1 < MT) __syncthreads();
      }
    }
    // Slot (di + NS) mod (NS + 1) was the tile before this one: free again.
    const int dp = di == 0 ? NS : di - 1;
    put_rows(dp, pn, dn.hk);
    if (tid == 0) sh.desc[dp] = dn;
    di = di == NS ? 0 : di + 1;
    st = st == NS - 1 ? 0 : st + 1;
  }
  cp_async_wait<0>();
  if constexpr (CL) {
    // A block's part is in stage 1 if its last tile was in stage 0, else in
    // stage 0 (and nowhere when it had no tile).
    const int rows = min(MR, cur.v.qlen * a.group - cur.row0);
    join_cluster<MR, DM, kThreads>(a, cur.v, cur.row0, rows, cur.hk, [&](int tiles) {
      return ring_addr + ((unsigned)(tiles - 1) % NS == 0 ? C::STAGE : 0);
    });
  }
  if (!CL && a.late_wait && blockIdx.x == 0) grid_dep_wait();
}

template <typename T, int DM, int MT, bool CL = false>
cudaError_t launch(const PagedArgs& a, cudaStream_t st) {
  constexpr int smem = smem_bytes<DM, MT>();
  static_assert(smem <= 227 * 1024 && Cfg<DM, MT>::BLOCKS * (smem + 1024) <= 228 * 1024, "shared memory");
  auto kern = paged_decode_kernel<T, DM, MT, CL>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)a.n_ctas), block(kThreads);
  e = CL ? launch_pdl_cluster(kern, grid, block, smem, st, 1u << a.cluster_shift, a)
         : launch_pdl(kern, grid, block, smem, st, a);
  note_launch();
  return e;
}

template <typename T>
cudaError_t launch_t(const PagedArgs& a, cudaStream_t st) {
  const bool two = a.rows_per_unit == 32;
  if (a.cluster_shift > 0) {  // (one MMA tile of rows only)
    if (a.D <= 64) return launch<T, 64, 1, true>(a, st);
    return a.D <= 128 ? launch<T, 128, 1, true>(a, st) : launch<T, 256, 1, true>(a, st);
  }
  if (a.D <= 64) return two ? launch<T, 64, 2>(a, st) : launch<T, 64, 1>(a, st);
  if (a.D <= 128) return two ? launch<T, 128, 2>(a, st) : launch<T, 128, 1>(a, st);
  return launch<T, 256, 1>(a, st);
}

}  // namespace decode
}  // namespace fa
