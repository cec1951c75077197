// fa_paged_api.cu - host side of the paged-cache operators: argument checks,
// choice of kernel, scratch layout, launches (include/fa_b200.h).
//
// Nothing here reads device memory, allocates or synchronises (the RoPE
// tables of a new theta excepted), so every call can be captured in a graph
// and replayed while the lengths, pages and slots on the device change.
#include "fa_paged.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <iterator>

namespace fa {
namespace {

size_t elem_size(int dt) { return dt == kF32 ? 4 : 2; }
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

fa_status cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return FA_OK;
  cudaGetLastError();  // reported here, not by the next call
  return paged_fail(FA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

struct Checked {
  PagedArgs a;
  int dtype;
  bool vec;              // strides are multiples of 16 bytes
  int64_t nk[2], nv[2];  // strides of the new rows (append)
};

// `grouped`: query heads share the KV heads (the append takes any number).
fa_status check(const fa_paged_params* p, Checked* c, bool grouped = true) {
  if (!p) return paged_fail(FA_ERR_INVALID_ARG, "params is NULL");
  if (p->dtype < 0 || p->dtype > 2) return paged_fail(FA_ERR_INVALID_ARG, "dtype must be 0 (f16), 1 (bf16) or 2 (f32)");
  if (p->out_dtype > 2) return paged_fail(FA_ERR_INVALID_ARG, "out_dtype must be -1, 0, 1 or 2");
  if (p->head_dim == 0 || p->head_dim > 256) return paged_fail(FA_ERR_UNSUPPORTED, "head_dim must be in [1, 256]");
  if (p->num_heads_k == 0 || p->num_heads_q > 65535 || p->num_heads_k > 65535 ||
      (grouped && p->num_heads_q % p->num_heads_k != 0))
    return paged_fail(FA_ERR_INVALID_ARG, "num_heads_q must be a positive multiple of num_heads_k");
  const uint64_t lim = 1ull << 30;
  if (p->page_size == 0) return paged_fail(FA_ERR_INVALID_ARG, "page_size must be positive");
  if (p->batch_size > lim || p->total_q > lim || p->page_size > lim || p->num_pages > lim || p->max_pages > lim ||
      p->prefix_pages > lim)
    return paged_fail(FA_ERR_INVALID_ARG, "tensor dimensions out of range");
  if (grouped && (uint64_t)p->total_q * p->num_heads_q > lim)
    return paged_fail(FA_ERR_INVALID_ARG, "total_q * num_heads_q must not exceed 2^30");
  if (grouped && (uint64_t)p->batch_size * p->num_heads_q > lim)
    return paged_fail(FA_ERR_INVALID_ARG, "batch_size * num_heads_q must not exceed 2^30");
  if (p->prefix_len > lim / 2 || (uint64_t)p->prefix_len > (uint64_t)p->prefix_pages * p->page_size)
    return paged_fail(FA_ERR_INVALID_ARG, "prefix_len is beyond the pages of the prefix table");
  if (!std::isfinite(p->softmax_scale)) return paged_fail(FA_ERR_INVALID_ARG, "softmax_scale must be finite");
  if (!std::isfinite(p->softcap) || p->softcap < 0.f)
    return paged_fail(FA_ERR_INVALID_ARG, "softcap must be 0 (off) or positive and finite");

  PagedArgs& a = c->a;
  std::memset(&a, 0, sizeof(a));
  a.B = (int)p->batch_size;
  a.total_q = (int)p->total_q;
  a.Hq = (int)p->num_heads_q;
  a.Hk = (int)p->num_heads_k;
  a.D = (int)p->head_dim;
  a.group = a.Hq / a.Hk;
  a.page_size = (int)p->page_size;
  a.num_pages = (int)p->num_pages;
  a.max_pages = (int)p->max_pages;
  a.table_stride = p->table_stride ? p->table_stride : (int64_t)p->max_pages;
  a.pre = (int)p->prefix_len;
  a.max_len = (int)std::min<uint64_t>((uint64_t)p->max_pages * p->page_size, (1u << 29) - 1);
  a.by_group = Div(std::max(1, a.group));
  a.by_page = Div(a.page_size);
  a.by_hk = Div(a.Hk);
  const int64_t row_q = (int64_t)a.Hq * a.D, row_k = (int64_t)a.Hk * a.D;
  auto two = [&](const int64_t in[2], int64_t row, int64_t* s0, int64_t* s1) {
    const bool none = in[0] == 0 && in[1] == 0;
    *s0 = none ? row : in[0];
    *s1 = none ? a.D : in[1];
    return *s0 >= 0 && *s1 >= 0;
  };
  auto three = [&](const int64_t in[3], int64_t* s0, int64_t* s1, int64_t* s2) {
    const bool none = in[0] == 0 && in[1] == 0 && in[2] == 0;
    *s0 = none ? row_k * a.page_size : in[0];
    *s1 = none ? row_k : in[1];
    *s2 = none ? a.D : in[2];
    return *s0 >= 0 && *s1 >= 0 && *s2 >= 0;
  };
  bool ok = a.table_stride >= 0;
  ok &= two(p->q_stride, row_q, &a.q_st, &a.q_sh);
  ok &= two(p->o_stride, row_q, &a.o_st, &a.o_sh);
  ok &= two(p->new_k_stride, row_k, &c->nk[0], &c->nk[1]);
  ok &= two(p->new_v_stride, row_k, &c->nv[0], &c->nv[1]);
  ok &= three(p->k_stride, &a.k_sp, &a.k_ss, &a.k_sh);
  ok &= three(p->v_stride, &a.v_sp, &a.v_ss, &a.v_sh);
  if (!ok) return paged_fail(FA_ERR_INVALID_ARG, "strides must be non-negative");
  a.out_dtype = p->out_dtype < 0 ? p->dtype : p->out_dtype;
  a.scale = p->softmax_scale;
  a.scale_log2 = (float)((double)p->softmax_scale * 1.4426950408889634);
  a.softcap = p->softcap;
  // (finite for the smallest caps: 0 * cap_in stays 0)
  if (a.softcap > 0.f) a.cap_in = std::max(-1e37f, std::min(1e37f, a.scale / a.softcap));
  a.causal = p->is_causal ? 1 : 0;
  a.win_left = p->window_left < 0 ? -1 : std::min(p->window_left, 1 << 30);
  a.win_right = p->window_right < 0 ? -1 : std::min(p->window_right, 1 << 30);
  a.alibi = p->alibi_slopes;
  c->dtype = p->dtype;
  const int64_t m = 16 / (int64_t)elem_size(p->dtype);
  auto al = [&](int64_t s) { return s % m == 0; };
  c->vec = a.D % m == 0 && al(a.q_st) && al(a.q_sh) && al(a.k_sp) && al(a.k_ss) && al(a.k_sh) && al(a.v_sp) &&
           al(a.v_ss) && al(a.v_sh);
  return FA_OK;
}

// Most packed rows (query tokens times heads of a group) of one request.
long long max_rows(const fa_paged_params* p, const PagedArgs& a, bool one_token) {
  if (one_token) return a.group;
  const long long q = p->max_seqlen_q ? std::min(p->max_seqlen_q, p->total_q) : p->total_q;
  return std::max(1ll, q) * a.group;
}

// Scratch of the cut work: run records, running max and sum, partial rows.
struct CutLayout {
  size_t ml, o, bytes;
};
CutLayout cut_layout(int n_ctas, int rows, int D) {
  CutLayout l;
  l.ml = up256((size_t)n_ctas * sizeof(RunMeta));
  l.o = l.ml + up256((size_t)n_ctas * 2 * rows * sizeof(float2));
  l.bytes = l.o + up256((size_t)n_ctas * 2 * rows * ((D + 3) & ~3) * sizeof(float));
  return l;
}

void place_cut(PagedArgs& a, const CutLayout& l, void* ws) {
  uint8_t* w = static_cast<uint8_t*>(ws);
  a.meta = reinterpret_cast<RunMeta*>(w);
  a.slot_ml = reinterpret_cast<float2*>(w + l.ml);
  a.slot_o = reinterpret_cast<float*>(w + l.o);
}

// Which kernels a call takes, and its scratch.
struct Choice {
  bool tensor;     // few-rows tensor-core kernel, else CUDA cores
  bool many;       // the requests' own keys go to the many-rows kernel
  bool shared;     // the prefix is computed once for all rows (many-rows kernel)
  int box;         // slots of a TMA box
  int own_split, pre_split;        // parts the keys are cut in
  int own_blocks, pre_blocks;      // blocks of 256 packed rows
  int rows_per_unit, n_ctas, join_rows, split;
  int units_per_req, cluster_shift;
  int n_parts;                     // whole-row partial results to join (0: none)
  CutLayout cut;
  size_t parts_lse, parts_o, bytes;  // offsets of the partial results
};

// Parts that the keys of `blocks` blocks (256 rows, up to `tiles` tiles of
// 128 keys) are cut in. A wave of 148 blocks takes one tile in 2.15 us (D =
// 128; 1.8 at 64) and about 14 us more to begin and end (64 blocks of 256
// tiles: 568 us in 1 part, 315 in 2 = one wave, 368 in 4 = two waves, 375 in 9
// = four); every part writes and reads its partial rows once (about 5 TB/s).
// One part needs no join. With the few-rows kernel running `beside`, a single
// wave leaves it a quarter of the SMs, or costs its time (some 10 us, from one
// size only) on top. (24 requests of 4 tokens, 8 heads on one KV head, a prefix
// of 50001 keys: 74 us with 16 parts, 52 with 31, 56 with 49.)
//
// For a request's own keys `tiles` is what its table has room for, as the host
// does not know the lengths; parts behind a request's end cost their start and
// their empty rows. (4 prompt chunks of 335 to 840 tokens over 1165 to 3932: 126
// us with a table of 4272 tokens, 187 with 8192 and 32768, 573 with 2^20.)
int choose_parts(long long blocks, long long tiles, int D, double row_bytes, bool join_anyway, bool beside) {
  const double tile = D <= 64 ? 1.8e-6 : 2.15e-6;
  const int top = (int)std::max(1ll, std::min(64ll, tiles / 2));
  int best = 1;
  double best_cost = 0;
  for (int n = 1; n <= top; ++n) {
    const double waves = (double)((blocks * n + 147) / 148);
    double cost = waves * ((double)((tiles + n - 1) / n) * tile + 14e-6);
    if (n > 1 || join_anyway) cost += 2.0 * n * row_bytes / 5e12;
    if (n > 1 && !join_anyway) cost += 3e-6;  // the join's own launch
    if (beside && blocks * n > 112 && blocks * n <= 148) cost += 10e-6;
    if (n == 1 || cost < best_cost) {
      best = n;
      best_cost = cost;
    }
  }
  return best;
}

int gcd(int a, int b) {
  while (b) {
    const int t = a % b;
    a = b;
    b = t;
  }
  return a;
}

// `one`: one query token a request (no cu_seqlens_q).
Choice choose(const fa_paged_params* p, const Checked& c, bool vec, bool one) {
  const PagedArgs& a = c.a;
  Choice h{};
  const long long rows = max_rows(p, a, one);
  const long long all_rows = (long long)a.total_q * a.group;
  const long long own_keys = a.max_len;
  // 16-bit rows of whole 16-byte pieces go to the tensor cores; fp32 and
  // everything that cannot be copied in such pieces to the CUDA cores.
  h.tensor = c.dtype != kF32 && vec && a.num_pages > 0;
  h.box = gcd(a.page_size, 128);
  const bool tma = h.tensor && a.D <= 128 && h.box >= 8 && a.k_sp > 0 && a.k_ss > 0 && a.k_sh > 0 && a.v_sp > 0 &&
                   a.v_ss > 0 && a.v_sh > 0;
  // Above 32 rows the few-rows kernel reads the keys more than once. (16
  // requests of 8000 keys, 32 heads on 8 KV heads: 16 rows 97 us and 119 in the
  // many-rows kernel, 32 rows 103 and 119, 48 rows 245 and 119.)
  h.many = tma && rows > 32;
  // A prefix is computed apart when each request's reading it (from L2) would
  // cost more than a kernel and a join. (In this place and apart, D = 128, 8 KV
  // heads: 8 requests of 500 keys, 16 MB, 13.6 and 16.2 us; of 1000 keys 16.3
  // and 16.5; of 2000 keys 20.8 and 17.1; 64 requests of 600 keys 41 and 21.)
  h.shared = tma && a.pre > 0 &&
             (h.many || (a.B > 1 && a.pre >= 128 && (double)a.B * a.pre * a.Hk * a.D * 4 >= 32e6));
  const double row_bytes = (double)a.total_q * a.Hq * a.D * 4;
  if (h.shared) {
    h.pre_blocks = (int)((all_rows + 255) / 256);
    h.pre_split = choose_parts((long long)h.pre_blocks * a.Hk, (a.pre + 127) / 128, a.D, row_bytes, true, !h.many);
  }
  if (h.many) {
    h.own_blocks = (int)(one ? (long long)a.B * ((a.group + 255) / 256) : (all_rows + 255) / 256 + a.B);
    h.own_split = choose_parts((long long)h.own_blocks * a.Hk, (own_keys + 127) / 128, a.D, row_bytes, h.shared, false);
  }
  if (!h.many) {
    if (h.tensor) {
      h.rows_per_unit = decode_rows_per_unit(a.D, rows);
      h.n_ctas = decode_ctas(a.D, h.rows_per_unit);
    } else {
      h.rows_per_unit = simt_rows_per_unit(c.dtype, vec, a.D, rows);
      h.n_ctas = simt_ctas(a.D, h.rows_per_unit);
    }
    const int wave = h.n_ctas;
    h.join_rows = (int)std::min<long long>(h.rows_per_unit, one ? (long long)a.group : all_rows);
    const long long keys = own_keys + (h.shared ? 0 : a.pre);
    // A unit of few keys is not worth cutting: its block takes 0.6 to 1.2 us a
    // tile of 64 keys, the join 4 us. One request on 8 KV heads, D = 128, uncut
    // and cut: 250 keys 8.6 and 11.4 us, 380 keys 11.1 and 11.4, 500 keys 13.4
    // and 12.5; 4 requests on 16 heads, D = 64: 250 keys 8.2 and 11.0, 500 keys
    // 12.0 and 11.3; 40 requests on 8 heads, D = 128: 250 keys 18.2 and 17.4, 500
    // keys 29 and 24. CUDA cores, 8 requests on 8 heads, D = 64: 160 keys 8.9 and
    // 10.1, 200 keys 10.5 and 10.2, 250 keys 12.3 and 10.4.
    const long long per_req = (a.group + h.rows_per_unit - 1) / h.rows_per_unit * a.Hk;
    const long long units = one ? a.B * per_req : (all_rows / h.rows_per_unit + a.B) * a.Hk;
    h.split = keys > (h.tensor ? 384 : 192);
    // The line the kernels cut is counted in 32 bits.
    if (units * (keys / 32 + 4) >= (1ll << 31)) h.split = 0;
    if (!h.split) {
      h.n_ctas = (int)std::min<long long>(units, one ? 1 << 30 : 148 * 16);
      h.units_per_req = one && units <= (1 << 30) ? (int)per_req : 0;
    }
    // Units of few tiles are cut between the blocks of a cluster instead, which
    // saves the join's launch but balances nothing, so a block's share by the
    // table's width is at most 128 KB of K and V. (Times of graphs of five calls,
    // some 0.8 us above those of longer graphs. One request on 8 KV heads, D =
    // 128, cut in runs and in clusters: 500 keys 13.1 and 7.9 us, 2000 keys, 4
    // tiles a share, 13.6 and 11.4, 4000 keys 13.3 and 15.9; 16 requests of 1 to
    // 1000 keys, 8 tiles a share, 13.0 and 15.8. Uncut and in clusters: 200 keys
    // 9.3 and 7.0, 160 keys 8.2 and 8.1, D = 64 200 keys 8.7 and 7.5, 160 keys 7.7
    // and 8.0; fp32, 90 keys 9.4 and 8.3, 250 keys 14.9 and 7.9.) Blocks that fill an SM go in fours: eights
    // took 17.9 us where fours take 15.9. Beside the prefix's kernel more
    // blocks find no SM free (16 requests of up to 200 keys 19.1 us, uncut 17.8).
    const bool can = h.tensor ? h.rows_per_unit == 16 : vec && c.dtype == kF32;  // (the kernels with cluster variants)
    if (one && can && !h.shared && keys > (h.tensor ? 192 : 64)) {
      const int tile = h.tensor ? 64 : 32, most = h.tensor && a.D > 128 ? 2 : 3;
      const long long tiles = (keys + tile - 1) / tile;
      int shift = 0;
      while (shift < most && (units << (shift + 1)) <= wave && (2ll << shift) <= tiles) ++shift;
      if (shift > 0 && (tiles >> shift) * a.D <= 512) {
        h.cluster_shift = shift;
        h.split = 0;
        h.n_ctas = (int)units << shift;
        h.units_per_req = (int)per_req;
      }
    }
    h.cut = cut_layout(h.split ? h.n_ctas : 0, h.rows_per_unit, a.D);
    h.bytes = h.cut.bytes;
  }
  // Whole-row partial results: the prefix's, then the own keys' (the few-rows
  // kernel makes one part of them).
  h.n_parts = h.pre_split + (h.many ? (h.shared || h.own_split > 1 ? h.own_split : 0) : (h.shared ? 1 : 0));
  const size_t parts = (size_t)h.n_parts;
  h.parts_lse = h.bytes;
  h.parts_o = h.parts_lse + up256(parts * a.Hq * a.total_q * sizeof(float));
  h.bytes = h.parts_o + up256(parts * (size_t)a.total_q * a.Hq * a.D * sizeof(float));
  return h;
}

// Every choice the tensors' base addresses (bit 0: 16-byte aligned) and
// cu_seqlens_q (bit 1: none) can lead to; returns the scratch of the largest.
size_t choose_all(const fa_paged_params* p, const Checked& c, Choice (&all)[4]) {
  size_t bytes = 256;  // (0 means invalid parameters)
  for (int i = 0; i < 4; ++i) {
    if ((i & 1) && !c.vec) continue;
    all[i] = choose(p, c, (i & 1) != 0, (i & 2) != 0);
    bytes = std::max(bytes, all[i].bytes);
  }
  return bytes;
}

cudaError_t launch_tc(const PagedArgs& a, const PagedTc& t, int dtype, const CUtensorMap& tk, const CUtensorMap& tv,
                      cudaStream_t s) {
  if (a.D <= 64)
    return dtype == kF16 ? launch_paged_tc_d64_f16(a, t, tk, tv, s) : launch_paged_tc_d64_bf16(a, t, tk, tv, s);
  return dtype == kF16 ? launch_paged_tc_d128_f16(a, t, tk, tv, s) : launch_paged_tc_d128_bf16(a, t, tk, tv, s);
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

void fa_paged_params_init(fa_paged_params* p) {
  if (!p) return;
  std::memset(p, 0, sizeof(*p));
  p->window_left = -1;
  p->window_right = -1;
  p->dtype = FA_F16;
  p->out_dtype = -1;
}

fa_status fa_plan_pages(uint32_t batch, uint32_t page_size, uint32_t max_pages, uint32_t n_free, uint32_t rows,
                        const int32_t* cached, const int32_t* fresh, const int32_t* free_pages,
                        const int32_t* free_begin, int32_t* table, int64_t table_stride, int32_t* seq_lens,
                        int32_t* cu, int64_t* slots, int32_t* positions, int32_t* free_end, void* stream) {
  if (batch > (uint32_t)kPlanMaxRequests)
    return paged_fail(FA_ERR_UNSUPPORTED, "at most " + std::to_string(kPlanMaxRequests) + " requests a plan");
  const uint32_t lim = 1u << 30;
  if (page_size == 0 || page_size > lim || max_pages > lim || n_free > lim || rows > lim || table_stride < 0)
    return paged_fail(FA_ERR_INVALID_ARG, "plan dimensions out of range");
  if ((batch && (!cached || !fresh || !seq_lens || (max_pages && !table))) || !cu || !free_end ||
      (rows && (!slots || !positions)) || (n_free && !free_pages))
    return paged_fail(FA_ERR_INVALID_ARG, "NULL plan pointer");
  // Every block reads the lengths again while the first one writes its results.
  // (The table has rows apart from one another, so what lies between them is
  // the caller's.)
  struct Span {
    const char* name;
    const void* p;
    size_t bytes;
  };
  const size_t n = batch;
  const Span out[] = {{"seq_lens", seq_lens, n * 4}, {"cu", cu, (n + 1) * 4}, {"slots", slots, (size_t)rows * 8},
                      {"positions", positions, (size_t)rows * 4}, {"free_end", free_end, 4}};
  const Span in[] = {{"cached", cached, n * 4}, {"fresh", fresh, n * 4}, {"free_pages", free_pages, (size_t)n_free * 4},
                     {"free_begin", free_begin, free_begin ? 4u : 0u}};
  auto meet = [](const Span& x, const Span& y) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x.p), b = reinterpret_cast<uintptr_t>(y.p);
    return x.bytes && y.bytes && a < b + y.bytes && b < a + x.bytes;
  };
  auto refuse = [](const Span& x, const Span& y) {
    return paged_fail(FA_ERR_INVALID_ARG, std::string(x.name) + " and " + y.name + " must not overlap");
  };
  for (size_t i = 0; i < std::size(out); ++i) {
    for (const Span& x : in)
      if (meet(out[i], x)) return refuse(x, out[i]);
    for (size_t j = 0; j < i; ++j)
      if (meet(out[i], out[j])) return refuse(out[j], out[i]);
  }
  unsigned* words = nullptr;
  fa_status st = paged_status_words(&words);
  if (st != FA_OK) return st;
  PlanArgs a{};
  a.B = (int)batch;
  a.max_pages = (int)max_pages;
  a.page_size = (int)page_size;
  a.n_free = (int)n_free;
  a.rows = (int)rows;
  a.cached = cached;
  a.fresh = fresh;
  a.free_pages = free_pages;
  a.free_begin = free_begin;
  a.table = table;
  a.table_stride = table_stride ? table_stride : (int64_t)max_pages;
  a.seq_lens = seq_lens;
  a.cu = cu;
  a.slots = slots;
  a.positions = positions;
  a.free_end = free_end;
  a.status = words;
  return cuda_status(launch_plan_pages(a, static_cast<cudaStream_t>(stream)), "page planning");
}

fa_status fa_store_kv(const fa_paged_params* p, const void* k, const void* v, void* k_cache, void* v_cache,
                      const int64_t* slots, const int32_t* positions, const float* cos, const float* sin,
                      uint32_t table_rows, float rope_theta, const void* q, void* q_out, void* stream) {
  Checked c;
  fa_status st = check(p, &c, false);
  if (st != FA_OK) return st;
  const PagedArgs& g = c.a;
  if (g.total_q == 0) return FA_OK;
  if (!k || !v || !slots || (g.num_pages && (!k_cache || !v_cache)))
    return paged_fail(FA_ERR_INVALID_ARG, "NULL tensor pointer");
  if ((q == nullptr) != (q_out == nullptr)) return paged_fail(FA_ERR_INVALID_ARG, "q and q_out go together");
  if ((cos == nullptr) != (sin == nullptr)) return paged_fail(FA_ERR_INVALID_ARG, "cos and sin tables go together");
  if (table_rows > (1u << 30)) return paged_fail(FA_ERR_INVALID_ARG, "table_rows out of range");
  const bool rotate = positions != nullptr;
  if (rotate && !cos && (!(rope_theta > 0.f) || !std::isfinite(rope_theta)))
    return paged_fail(FA_ERR_INVALID_ARG, "positions need cos/sin tables or rope_theta > 0");
  if (rotate && !cos && g.D % 2 != 0)
    return paged_fail(FA_ERR_UNSUPPORTED, "RoPE from rope_theta needs an even head_dim");
  if (!rotate && (cos || rope_theta != 0.f))
    return paged_fail(FA_ERR_INVALID_ARG, "cos/sin tables and rope_theta need positions");
  StoreArgs a{};
  st = paged_status_words(&a.status);
  if (st != FA_OK) return st;
  const float *cs = cos, *sn = sin;
  if (rotate && !cos && table_rows > 0) {
    st = paged_rope(rope_theta, g.D, (int)table_rows, static_cast<cudaStream_t>(stream), &cs, &sn);
    if (st != FA_OK) return st;
  }
  a.T = g.total_q;
  a.Hq = q ? g.Hq : 0;
  a.Hk = g.Hk;
  a.D = g.D;
  a.page_size = g.page_size;
  a.n_slots = (long long)g.num_pages * g.page_size;
  a.slots = slots;
  a.positions = positions;
  a.table_rows = rotate ? (int)table_rows : 0;
  a.cs = cs;
  a.sn = sn;
  a.k = k;
  a.v = v;
  a.q = q;
  a.k_st = c.nk[0];
  a.k_sh = c.nk[1];
  a.v_st = c.nv[0];
  a.v_sh = c.nv[1];
  a.q_st = g.q_st;
  a.q_sh = g.q_sh;
  a.kc = k_cache;
  a.vc = v_cache;
  a.kc_sp = g.k_sp;
  a.kc_ss = g.k_ss;
  a.kc_sh = g.k_sh;
  a.vc_sp = g.v_sp;
  a.vc_ss = g.v_ss;
  a.vc_sh = g.v_sh;
  a.qo = q_out;
  // 16-byte pieces of 8 columns in both halves of a row, from every tensor.
  const int64_t m = 16 / (int64_t)elem_size(c.dtype);
  auto al = [&](int64_t s) { return s % m == 0; };
  bool vec = g.D % 16 == 0 && al(a.k_st) && al(a.k_sh) && al(a.v_st) && al(a.v_sh) && al(a.kc_sp) && al(a.kc_ss) &&
             al(a.kc_sh) && al(a.vc_sp) && al(a.vc_ss) && al(a.vc_sh) && aligned(k, 16) && aligned(v, 16) &&
             aligned(k_cache, 16) && aligned(v_cache, 16);
  if (q) vec &= al(a.q_st) && al(a.q_sh) && aligned(q, 16) && aligned(q_out, 16);
  if (rotate) vec &= aligned(cs, 16) && aligned(sn, 16);
  return cuda_status(launch_store_kv(a, c.dtype, vec, static_cast<cudaStream_t>(stream)), "cache append");
}

size_t fa_paged_workspace_size(const fa_paged_params* p) {
  Checked c;
  if (check(p, &c) != FA_OK) return 0;
  Choice all[4];
  return choose_all(p, c, all);
}

fa_status fa_paged_forward(const fa_paged_params* p, const void* q, const void* k_cache, const void* v_cache,
                           const int32_t* block_table, const int32_t* seq_lens, const int32_t* cu_seqlens_q,
                           const int32_t* prefix_table, void* o, float* lse, void* workspace,
                           size_t workspace_bytes, void* stream) {
  Checked c;
  fa_status st = check(p, &c);
  if (st != FA_OK) return st;
  PagedArgs& a = c.a;
  if (a.total_q == 0 || a.B == 0 || a.Hq == 0) return FA_OK;
  if (!q || !o || !seq_lens || (a.max_pages && !block_table) || (a.pre && !prefix_table) ||
      (a.num_pages && (!k_cache || !v_cache)))
    return paged_fail(FA_ERR_INVALID_ARG, "NULL tensor pointer");
  Choice all[4];
  const size_t need = choose_all(p, c, all);
  if (!workspace || workspace_bytes < need)
    return paged_fail(FA_ERR_INVALID_ARG, "workspace smaller than fa_paged_workspace_size()");
  if (!aligned(workspace, 256)) return paged_fail(FA_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
  st = paged_status_words(&a.status);
  if (st != FA_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  a.table = block_table;
  a.seq_lens = seq_lens;
  a.cu_q = cu_seqlens_q;
  a.pre_table = prefix_table;
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.o = o;
  a.lse = lse;
  a.wait_limit_ns = paged_wait_limit_ns();
  const bool vec = c.vec && aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16);
  const Choice& h = all[(vec ? 1 : 0) + (cu_seqlens_q == nullptr ? 2 : 0)];
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.n_parts = h.n_parts;
  a.own_part = h.n_parts > 0 && !h.many ? h.pre_split : -1;
  a.parts_lse = reinterpret_cast<float*>(ws + h.parts_lse);
  a.parts_o = reinterpret_cast<float*>(ws + h.parts_o);
  CUtensorMap tk, tv;
  PagedTc t{};
  t.box_rows = h.box;
  const int64_t om = 16 / (int64_t)elem_size(a.out_dtype);
  t.out_vec = aligned(o, 16) && a.o_st % om == 0 && a.o_sh % om == 0;
  if (h.shared || h.many) {
    const bool bf = c.dtype == kBF16;
    st = paged_encode(&tk, k_cache, bf, a.D, a.Hk, a.page_size, a.num_pages, a.k_sp, a.k_ss, a.k_sh, h.box);
    if (st == FA_OK)
      st = paged_encode(&tv, v_cache, bf, a.D, a.Hk, a.page_size, a.num_pages, a.v_sp, a.v_ss, a.v_sh, h.box);
    if (st != FA_OK) return st;
  }
  if (h.shared) {
    t.shared = 1;
    t.n_blocks = h.pre_blocks;
    t.n_split = h.pre_split;
    t.by_split = Div(t.n_split);
    t.partial = 1;
    st = cuda_status(launch_tc(a, t, c.dtype, tk, tv, s), "shared prefix attention");
    if (st != FA_OK) return st;
    a.pre = 0;  // what follows sees each request's own keys
    a.pre_table = nullptr;
  }
  if (h.many) {
    t.shared = 0;
    t.n_blocks = h.own_blocks;
    t.n_split = h.own_split;
    t.by_split = Div(t.n_split);
    t.partial = h.n_parts > 0;
    t.part0 = h.pre_split;
    st = cuda_status(launch_tc(a, t, c.dtype, tk, tv, s), "paged attention (many rows)");
  } else {
    a.rows_per_unit = h.rows_per_unit;
    a.n_ctas = h.n_ctas;
    a.join_rows = h.join_rows;
    // Shortest run, kUnitCost + 1 (one request of 1000 keys, 8 KV heads, D =
    // 128: 11.6 us, with 4 instead of 3 12.7 us).
    a.by_min_run = Div(3);
    a.units_per_req = h.units_per_req;
    a.by_units = Div(std::max(1, h.units_per_req));
    a.split = h.split;
    a.cluster_shift = h.cluster_shift;
    place_cut(a, h.cut, workspace);
    a.late_wait = h.shared;
    st = h.tensor ? cuda_status(launch_paged_decode(a, c.dtype, s), "paged attention (few rows)")
                  : cuda_status(launch_paged_simt(a, c.dtype, vec, s), "paged attention (CUDA cores)");
    if (st == FA_OK && a.split) st = cuda_status(launch_paged_join(a, s), "paged attention (join)");
  }
  if (st == FA_OK && h.n_parts > 0) st = cuda_status(launch_paged_merge(a, s), "paged attention (merge)");
  return st;
}

}  // extern "C"
