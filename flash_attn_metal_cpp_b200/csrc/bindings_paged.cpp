// bindings_paged.cpp - the `_flash_attn_paged` extension: plan_pages,
// store_kv, paged_forward and shared_prefix_forward over the C ABI in
// fa_b200.h. CUDA torch tensors only; every call runs on the tensors' device
// and its current stream and returns without synchronising.
//
// A decoding step makes these calls for every layer, each a few microseconds
// of GPU time, so tensors are read and results allocated through torch's C++
// interface (reading eight tensors and allocating five through Python took
// 14 us). That is why they live in an extension of their own, which
// `_flash_attn_metal` loads when one of them is first used: the rest of the
// module works without torch.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <pybind11/pybind11.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/fa_b200.h"

namespace py = pybind11;

namespace {

[[noreturn]] void paged_error(const std::string& what) { throw std::runtime_error("Paged cache error: " + what); }

void check_status(fa_status st) {
  if (st == FA_OK) return;
  std::string s = fa_last_error();
  paged_error(s.empty() ? "status " + std::to_string((int)st) : s);
}

// Device of the call: the first tensor sets it, the others must be there too.
struct Device {
  int index = -1;
};

constexpr int kMaxDims = 4;
struct View {
  void* ptr = nullptr;
  int nd = 0;
  int64_t size[kMaxDims] = {}, stride[kMaxDims] = {};
  at::ScalarType dtype = at::kFloat;
  bool contiguous() const {
    int64_t run = 1;
    for (int i = nd; i-- > 0;) {
      if (size[i] != 1 && stride[i] != run) return false;
      run *= size[i];
    }
    return true;
  }
};

View view(py::handle o, const char* what, int nd, Device& dev) {
  if (!THPVariable_Check(o.ptr())) paged_error(std::string(what) + " must be a CUDA torch tensor");
  const at::Tensor& t = THPVariable_Unpack(o.ptr());
  if (!t.is_cuda()) paged_error(std::string(what) + " must be a CUDA torch tensor");
  const int index = t.get_device();
  if (dev.index < 0) dev.index = index;
  else if (dev.index != index) paged_error(std::string(what) + " is on another device than the other tensors");
  if (t.dim() != nd) paged_error(std::string(what) + " must have " + std::to_string(nd) + " dimensions");
  View v;
  v.nd = nd;
  for (int i = 0; i < nd; ++i) {
    v.size[i] = t.size(i);
    v.stride[i] = t.stride(i);
  }
  v.ptr = t.data_ptr();
  v.dtype = t.scalar_type();
  return v;
}

int float_code(const View& v, const char* what) {
  switch (v.dtype) {
    case at::kHalf: return FA_F16;
    case at::kBFloat16: return FA_BF16;
    case at::kFloat: return FA_F32;
    default: paged_error(std::string(what) + " must be float16, bfloat16 or float32");
  }
}
at::ScalarType type_of(int code) { return code == FA_F16 ? at::kHalf : code == FA_BF16 ? at::kBFloat16 : at::kFloat; }

// int32 vector of n values (any n when n < 0), contiguous.
View int_vector(py::handle o, const char* what, int64_t n, Device& dev) {
  View v = view(o, what, 1, dev);
  if (v.dtype != at::kInt) paged_error(std::string(what) + " must be int32");
  if (!v.contiguous()) paged_error(std::string(what) + " must be contiguous");
  if (n >= 0 && v.size[0] != n) paged_error(std::string(what) + " must have " + std::to_string(n) + " entries");
  return v;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const Device& dev) {
  // (what at::empty ends in, without the dispatcher on the way)
  return at::detail::empty_cuda(shape, dtype, at::Device(at::kCUDA, (c10::DeviceIndex)dev.index), std::nullopt);
}

py::object wrap(const at::Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

void* stream_of(const Device& dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev.index).stream(); }

// Makes the tensors' device current for the call and puts the caller's back.
using OnDevice = c10::cuda::CUDAGuard;
OnDevice on_device(const Device& dev) { return OnDevice((c10::DeviceIndex)dev.index); }

// Strides (in elements) of the `n` leading dimensions. Dimensions of one entry
// get their row's length, so that the C ABI's "all zero = contiguous" is never
// met by accident; a broadcast tensor that would mean it is refused.
void copy_strides(const View& v, int n, int64_t* out, const char* what) {
  bool any = false;
  for (int i = 0; i < n; ++i) {
    out[i] = v.size[i] > 1 ? v.stride[i] : v.size[v.nd - 1];
    any |= out[i] != 0;
  }
  if (!any) paged_error(std::string(what) + " is one row broadcast: make it contiguous");
}

// True when no two indices of a tensor that is written share memory.
void no_overlap(const View& v, const char* what) {
  bool used[kMaxDims] = {};
  int64_t reach = 1;  // elements the dimensions so far span
  for (int n = 0; n < v.nd; ++n) {
    int best = -1;
    for (int i = 0; i < v.nd; ++i)
      if (!used[i] && (best < 0 || v.stride[i] < v.stride[best])) best = i;
    used[best] = true;
    if (v.size[best] <= 1) continue;
    if (v.stride[best] < reach) paged_error(std::string(what) + " overlaps itself");
    reach = v.stride[best] * (v.size[best] - 1) + reach;
  }
}

uint32_t u32(int64_t x, const char* what) {
  if (x < 0 || x > 0xffffffffll) paged_error(std::string(what) + " out of range");
  return (uint32_t)x;
}

// K and V cache: [num_pages, page_size, Hk, D], one type, one shape.
void fill_cache(fa_paged_params& p, const View& k, const View& v) {
  for (int i = 0; i < 4; ++i)
    if (k.size[i] != v.size[i]) paged_error("k_cache and v_cache must have one shape");
  if (k.dtype != v.dtype) paged_error("k_cache and v_cache must have one dtype");
  if ((k.size[3] > 1 && k.stride[3] != 1) || (v.size[3] > 1 && v.stride[3] != 1))
    paged_error("k_cache and v_cache need a unit innermost stride");
  p.num_pages = u32(k.size[0], "num_pages");
  p.page_size = u32(k.size[1], "page_size");
  p.num_heads_k = u32(k.size[2], "num_heads_k");
  p.head_dim = u32(k.size[3], "head_dim");
  copy_strides(k, 3, p.k_stride, "k_cache");
  copy_strides(v, 3, p.v_stride, "v_cache");
}

void unit_inner(const View& v, const char* what) {
  if (v.size[v.nd - 1] > 1 && v.stride[v.nd - 1] != 1)
    paged_error(std::string(what) + " needs a unit innermost stride");
}

// ------------------------------------------------------------------ planning
py::tuple plan_pages(py::object cached_lens, py::object new_lens, py::object block_table, py::object free_pages,
                     int64_t page_size, int64_t total_new, py::object free_begin) {
  Device dev;
  const View c = int_vector(cached_lens, "cached_lens", -1, dev);
  const View n = int_vector(new_lens, "new_lens", c.size[0], dev);
  const View tb = view(block_table, "block_table", 2, dev);
  if (tb.dtype != at::kInt) paged_error("block_table must be int32");
  if (tb.size[0] != c.size[0]) paged_error("block_table must have one row per request");
  if (tb.size[1] > 1 && tb.stride[1] != 1) paged_error("block_table needs a unit innermost stride");
  if (tb.size[0] > 1 && tb.stride[0] < tb.size[1]) paged_error("block_table rows must not overlap");
  const View f = int_vector(free_pages, "free_pages", -1, dev);
  if (page_size <= 0) paged_error("page_size must be positive");
  if (total_new < 0) paged_error("total_new must not be negative");
  const int32_t* begin = nullptr;
  if (!free_begin.is_none()) begin = static_cast<const int32_t*>(int_vector(free_begin, "free_begin", 1, dev).ptr);
  const OnDevice guard = on_device(dev);
  const int64_t b = c.size[0];
  const at::Tensor lens = empty({b}, at::kInt, dev), cu = empty({b + 1}, at::kInt, dev),
                   slots = empty({total_new}, at::kLong, dev), pos = empty({total_new}, at::kInt, dev),
                   end = empty({1}, at::kInt, dev);
  check_status(fa_plan_pages(u32(b, "batch"), u32(page_size, "page_size"), u32(tb.size[1], "max_pages"),
                             u32(f.size[0], "free_pages"), u32(total_new, "total_new"),
                             static_cast<const int32_t*>(c.ptr), static_cast<const int32_t*>(n.ptr),
                             static_cast<const int32_t*>(f.ptr), begin, static_cast<int32_t*>(tb.ptr),
                             tb.size[0] > 1 ? tb.stride[0] : tb.size[1], static_cast<int32_t*>(lens.data_ptr()),
                             static_cast<int32_t*>(cu.data_ptr()), static_cast<int64_t*>(slots.data_ptr()),
                             static_cast<int32_t*>(pos.data_ptr()), static_cast<int32_t*>(end.data_ptr()), stream_of(dev)));
  return py::make_tuple(wrap(lens), wrap(cu), wrap(slots), wrap(pos), wrap(end));
}

// -------------------------------------------------------------- cache append
py::object store_kv(py::object k, py::object v, py::object k_cache, py::object v_cache, py::object slots, py::object q,
                    py::object positions, py::object cos, py::object sin, py::object rope_theta,
                    py::object max_position) {
  Device dev;
  const View kn = view(k, "k", 3, dev), vn = view(v, "v", 3, dev);
  const View kc = view(k_cache, "k_cache", 4, dev), vc = view(v_cache, "v_cache", 4, dev);
  fa_paged_params p;
  fa_paged_params_init(&p);
  fill_cache(p, kc, vc);
  p.dtype = float_code(kc, "k_cache");
  if (kn.dtype != kc.dtype || vn.dtype != kc.dtype) paged_error("k, v and the cache must have one dtype");
  for (const View* x : {&kn, &vn})
    if (x->size[0] != kn.size[0] || x->size[1] != kc.size[2] || x->size[2] != kc.size[3])
      paged_error("k and v must be [tokens, num_heads_k, head_dim] of the cache's heads");
  unit_inner(kn, "k");
  unit_inner(vn, "v");
  const int64_t tokens = kn.size[0];
  p.total_q = u32(tokens, "tokens");
  p.num_heads_q = p.num_heads_k;
  copy_strides(kn, 2, p.new_k_stride, "k");
  copy_strides(vn, 2, p.new_v_stride, "v");
  no_overlap(kc, "k_cache");
  no_overlap(vc, "v_cache");
  const View sl = view(slots, "slots", 1, dev);
  if (sl.dtype != at::kLong || !sl.contiguous() || sl.size[0] != tokens)
    paged_error("slots must be a contiguous int64 vector with one entry per token");
  const int32_t* pos = nullptr;
  if (!positions.is_none()) pos = static_cast<const int32_t*>(int_vector(positions, "positions", tokens, dev).ptr);
  View qv;
  const bool has_q = !q.is_none();
  if (has_q) {
    qv = view(q, "q", 3, dev);
    if (qv.dtype != kc.dtype) paged_error("q and the cache must have one dtype");
    if (qv.size[0] != tokens || qv.size[2] != kc.size[3])
      paged_error("q must be [tokens, num_heads_q, head_dim]");
    unit_inner(qv, "q");
    p.num_heads_q = u32(qv.size[1], "num_heads_q");
    copy_strides(qv, 2, p.q_stride, "q");
  }
  const float *cp = nullptr, *sp = nullptr;
  int64_t rows = 0;
  if (cos.is_none() != sin.is_none()) paged_error("cos and sin go together");
  if (!cos.is_none()) {
    const View cv = view(cos, "cos", 2, dev), sv = view(sin, "sin", 2, dev);
    const int64_t half = kc.size[3] / 2;
    for (const View* x : {&cv, &sv})
      if (x->dtype != at::kFloat || !x->contiguous() || x->size[1] != half || x->size[0] != cv.size[0])
        paged_error("cos and sin must be contiguous float32 [positions, head_dim / 2] tensors");
    if (!rope_theta.is_none()) paged_error("give cos and sin or rope_theta, not both");
    cp = static_cast<const float*>(cv.ptr);
    sp = static_cast<const float*>(sv.ptr);
    rows = cv.size[0];
  }
  float theta = 0.f;
  if (!rope_theta.is_none()) {
    theta = rope_theta.cast<float>();
    if (max_position.is_none()) paged_error("rope_theta needs max_position, one past the largest position");
    rows = max_position.cast<int64_t>();
  }
  const OnDevice guard = on_device(dev);
  at::Tensor out;
  void *qp = nullptr, *qo = nullptr;
  if (has_q) {
    out = empty({tokens, qv.size[1], qv.size[2]}, kc.dtype, dev);
    if (tokens > 0 && qv.size[1] > 0) {
      qp = qv.ptr;
      qo = out.data_ptr();
    }
  }
  check_status(fa_store_kv(&p, kn.ptr, vn.ptr, kc.ptr, vc.ptr, static_cast<const int64_t*>(sl.ptr), pos, cp, sp,
                           u32(rows, "max_position"), theta, qp, qo, stream_of(dev)));
  return has_q ? wrap(out) : py::none();
}

// ----------------------------------------------------- attention over pages
py::object attention(py::object q, py::object k_cache, py::object v_cache, const py::object* prefix_table,
                     int64_t prefix_len, py::object block_table, py::object seq_lens, float softmax_scale,
                     bool is_causal, py::object cu_seqlens_q, py::object max_seqlen_q, float softcap,
                     py::object window_size, py::object alibi_slopes, py::object out_dtype, bool return_lse,
                     py::object out) {
  Device dev;
  const View qv = view(q, "q", 3, dev);
  const View kc = view(k_cache, "k_cache", 4, dev), vc = view(v_cache, "v_cache", 4, dev);
  fa_paged_params p;
  fa_paged_params_init(&p);
  fill_cache(p, kc, vc);
  p.dtype = float_code(kc, "k_cache");
  if (qv.dtype != kc.dtype) paged_error("q and the cache must have one dtype");
  if (qv.size[2] != kc.size[3]) paged_error("q must be [tokens, num_heads_q, head_dim] of the cache's head_dim");
  unit_inner(qv, "q");
  const View lens = int_vector(seq_lens, "seq_lens", -1, dev);
  const int64_t b = lens.size[0];
  const View tb = view(block_table, "block_table", 2, dev);
  if (tb.dtype != at::kInt) paged_error("block_table must be int32");
  if (tb.size[0] != b) paged_error("block_table must have one row per request");
  if (tb.size[1] > 1 && tb.stride[1] != 1) paged_error("block_table needs a unit innermost stride");
  p.batch_size = u32(b, "batch");
  p.total_q = u32(qv.size[0], "tokens");
  p.num_heads_q = u32(qv.size[1], "num_heads_q");
  p.max_pages = u32(tb.size[1], "max_pages");
  p.table_stride = tb.size[0] > 1 ? tb.stride[0] : tb.size[1];
  copy_strides(qv, 2, p.q_stride, "q");
  p.softmax_scale = softmax_scale;
  p.softcap = softcap;
  p.is_causal = is_causal ? 1 : 0;
  if (!window_size.is_none()) {
    py::tuple ws = window_size.cast<py::tuple>();
    if (py::len(ws) != 2) paged_error("window_size must be (left, right)");
    p.window_left = ws[0].cast<int>();
    p.window_right = ws[1].cast<int>();
  }
  if (!alibi_slopes.is_none()) {
    const View al = view(alibi_slopes, "alibi_slopes", 1, dev);
    if (al.dtype != at::kFloat || !al.contiguous() || al.size[0] != qv.size[1])
      paged_error("alibi_slopes must hold one float32 slope per query head");
    p.alibi_slopes = static_cast<const float*>(al.ptr);
  }
  const int32_t* cu = nullptr;
  if (!cu_seqlens_q.is_none()) {
    cu = static_cast<const int32_t*>(int_vector(cu_seqlens_q, "cu_seqlens_q", b + 1, dev).ptr);
    if (!max_seqlen_q.is_none()) {
      const int64_t m = max_seqlen_q.cast<int64_t>();
      if (m < 0) paged_error("max_seqlen_q must not be negative");
      p.max_seqlen_q = u32(m, "max_seqlen_q");
    }
  } else {
    if (qv.size[0] < b) paged_error("without cu_seqlens_q, q needs one row per request");
    p.max_seqlen_q = 1;  // (no scratch for the routes of several tokens)
  }
  const int32_t* pre = nullptr;
  if (prefix_table) {
    const View pt = int_vector(*prefix_table, "prefix_table", -1, dev);
    if (prefix_len < 0) paged_error("prefix_len must not be negative");
    p.prefix_len = u32(prefix_len, "prefix_len");
    p.prefix_pages = u32(pt.size[0], "prefix_table");
    pre = static_cast<const int32_t*>(pt.ptr);
  }
  int oc = p.dtype;
  if (!out_dtype.is_none()) {
    const std::string n = py::str(out_dtype);
    oc = n == "float16" || n == "torch.float16"     ? FA_F16
         : n == "bfloat16" || n == "torch.bfloat16" ? FA_BF16
         : n == "float32" || n == "torch.float32"   ? FA_F32
                                                    : -1;
    if (oc < 0) paged_error("out_dtype must be float16, bfloat16 or float32");
  }
  p.out_dtype = oc;
  const OnDevice guard = on_device(dev);
  void* op;
  if (out.is_none()) {
    out = wrap(empty({qv.size[0], qv.size[1], qv.size[2]}, type_of(oc), dev));
    op = THPVariable_Unpack(out.ptr()).data_ptr();
  } else {
    const View ov = view(out, "out", 3, dev);
    if (ov.size[0] != qv.size[0] || ov.size[1] != qv.size[1] || ov.size[2] != qv.size[2])
      paged_error("out has the wrong shape");
    if (ov.dtype != type_of(oc)) paged_error("out has the wrong dtype");
    unit_inner(ov, "out");
    no_overlap(ov, "out");
    copy_strides(ov, 2, p.o_stride, "out");
    op = ov.ptr;
  }
  at::Tensor lse;
  float* lp = nullptr;
  if (return_lse) {
    lse = empty({qv.size[1], qv.size[0]}, at::kFloat, dev);
    lp = static_cast<float*>(lse.data_ptr());
  }
  // The scratch is the call's own: torch hands it out on the current stream
  // (and, while a graph is captured, from that graph's memory).
  const size_t bytes = fa_paged_workspace_size(&p);
  const at::Tensor ws = empty({(int64_t)bytes}, at::kByte, dev);
  check_status(fa_paged_forward(&p, qv.ptr, kc.ptr, vc.ptr, static_cast<const int32_t*>(tb.ptr),
                                static_cast<const int32_t*>(lens.ptr), cu, pre, op, lp, ws.data_ptr(), bytes,
                                stream_of(dev)));
  if (return_lse) return py::make_tuple(out, wrap(lse));
  return out;
}

py::object paged_forward(py::object q, py::object k_cache, py::object v_cache, py::object block_table,
                         py::object seq_lens, float softmax_scale, bool is_causal, py::object cu_seqlens_q,
                         py::object max_seqlen_q, float softcap, py::object window_size, py::object alibi_slopes,
                         py::object out_dtype, bool return_lse, py::object out) {
  return attention(q, k_cache, v_cache, nullptr, 0, block_table, seq_lens, softmax_scale, is_causal, cu_seqlens_q,
                   max_seqlen_q, softcap, window_size, alibi_slopes, out_dtype, return_lse, out);
}

py::object shared_prefix_forward(py::object q, py::object k_cache, py::object v_cache, py::object prefix_table,
                                 int64_t prefix_len, py::object block_table, py::object seq_lens, float softmax_scale,
                                 bool is_causal, py::object cu_seqlens_q, py::object max_seqlen_q, float softcap,
                                 py::object window_size, py::object alibi_slopes, py::object out_dtype,
                                 bool return_lse, py::object out) {
  return attention(q, k_cache, v_cache, &prefix_table, prefix_len, block_table, seq_lens, softmax_scale, is_causal,
                   cu_seqlens_q, max_seqlen_q, softcap, window_size, alibi_slopes, out_dtype, return_lse, out);
}

}  // namespace

PYBIND11_MODULE(_flash_attn_paged, m) {
  m.doc() = "Paged KV cache: planning, append, attention over pages (CUDA torch tensors)";
  m.def("plan_pages", &plan_pages, py::arg("cached_lens"), py::arg("new_lens"), py::arg("block_table"),
        py::arg("free_pages"), py::arg("page_size"), py::arg("total_new"), py::kw_only(),
        py::arg("free_begin") = py::none(),
        "Plan one step of a paged cache on the GPU: takes the pages that the new tokens need from free_pages "
        "(from entry free_begin on), writes them into block_table, and returns (seq_lens, cu_seqlens, slots, "
        "positions, free_end); slots and positions have total_new rows, slot -1 behind the last token");
  m.def("store_kv", &store_kv, py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"),
        py::kw_only(), py::arg("q") = py::none(), py::arg("positions") = py::none(), py::arg("cos") = py::none(),
        py::arg("sin") = py::none(), py::arg("rope_theta") = py::none(), py::arg("max_position") = py::none(),
        "Write the K and V rows of new tokens to their cache slots (distinct; negative = skip). With positions, "
        "K and q are rotated by rotate-half RoPE (cos/sin tables, or rope_theta and max_position); returns the "
        "rotated q, or None without q");
  m.def("paged_forward", &paged_forward, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"),
        py::arg("seq_lens"), py::arg("softmax_scale") = 0.0f, py::arg("is_causal") = false, py::kw_only(),
        py::arg("cu_seqlens_q") = py::none(), py::arg("max_seqlen_q") = py::none(), py::arg("softcap") = 0.0f,
        py::arg("window_size") = py::none(), py::arg("alibi_slopes") = py::none(), py::arg("out_dtype") = py::none(),
        py::arg("return_lse") = false, py::arg("out") = py::none(),
        "Attention of packed query tokens [tokens, Hq, D] over a paged cache [pages, page_size, Hk, D]; the query "
        "tokens of a request are the last of its seq_lens[i] keys");
  m.def("shared_prefix_forward", &shared_prefix_forward, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("prefix_table"), py::arg("prefix_len"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("softmax_scale") = 0.0f, py::arg("is_causal") = false, py::kw_only(),
        py::arg("cu_seqlens_q") = py::none(), py::arg("max_seqlen_q") = py::none(), py::arg("softcap") = 0.0f,
        py::arg("window_size") = py::none(), py::arg("alibi_slopes") = py::none(), py::arg("out_dtype") = py::none(),
        py::arg("return_lse") = false, py::arg("out") = py::none(),
        "paged_forward for a batch whose requests all begin with the same prefix_len keys (the pages of "
        "prefix_table): block_table and seq_lens describe what each request has behind them");
}
