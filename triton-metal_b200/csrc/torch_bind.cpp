// Python binding of the entry points of a serving step, for callers that issue
// one call per layer per token: the kernels take a few microseconds, so the
// host cost of reaching them (argument checks, pointers, the caller's current
// stream) decides whether a step is host-bound.
// This module does those checks in C++ on the at::Tensor arguments and calls
// the C-ABI entry points (include/b2.h) of libb2.so; it holds no kernels of its
// own.
//
// Every function here answers its operator's common case only.  It returns None
// when the arguments are not that case (the Python operator then takes its
// general path, with its own checks and messages), the operator's result on
// success, and the nonzero b2 status as an int when the call failed (the Python
// operator raises the matching B2Error).
//
// int4_matmul(input, weight, scales, group_size, out) mirrors the fast path of
// b200kern.quant.int4_matmul (the reference operator int4_matmul,
// triton_metal/codegen/_msl_templates.py:2682-2745, GPTQ layout, symmetric).
//
// The others take tensors of one CUDA device, the current one, with the types,
// shapes and strides that their kernels read as they are; see attention.py and
// paged.py for what they compute.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAFunctions.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>

#include "b2.h"

namespace {

py::object int4_matmul(const at::Tensor& x, const at::Tensor& w, const at::Tensor& s, int64_t group_size,
                       const c10::optional<at::Tensor>& out) {
  const auto st = x.scalar_type();
  int dt;
  if (st == at::kHalf)
    dt = B2_F16;
  else if (st == at::kBFloat16)
    dt = B2_BF16;
  else
    return py::none();
  if (w.scalar_type() != at::kInt || s.scalar_type() != st || !x.is_cuda() || !w.is_cuda() || !s.is_cuda())
    return py::none();
  if (x.dim() != 2 || w.dim() != 2 || s.dim() != 2 || !x.is_contiguous() || !w.is_contiguous() ||
      !s.is_contiguous())
    return py::none();
  const int64_t M = x.size(0), K = x.size(1), N = w.size(1);
  if (group_size <= 0 || w.size(0) * 8 != K || K % group_size || s.size(0) != K / group_size || s.size(1) != N)
    return py::none();
  at::Tensor res;
  bool into_out = false;
  if (out.has_value()) {
    const at::Tensor& o = *out;
    into_out = o.scalar_type() == st && o.is_cuda() && o.is_contiguous() && o.dim() == 2 && o.size(0) == M &&
               o.size(1) == N;
    if (into_out) res = o;
  }
  if (!into_out) res = at::empty({M, N}, x.options());
  if (M) {
    cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
    const int rc = b2_int4_matmul(x.data_ptr(), w.data_ptr(), res.data_ptr(), s.data_ptr(), nullptr, M, N, K,
                                  group_size, dt, (void*)stream);
    if (rc != 0) return py::int_(rc);
  }
  if (out.has_value() && !into_out) {
    // a caller-given output of another layout: filled by a copy, as the
    // Python path does
    out->copy_(res);
    return py::cast(*out);
  }
  return py::cast(res);
}

using OptT = c10::optional<at::Tensor>;

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return B2_F16;
    case at::kBFloat16: return B2_BF16;
    case at::kFloat: return B2_F32;
    default: return -1;
  }
}
// the device of a call: its first tensor's, which has to be the current one
bool device_of(const at::Tensor& t, c10::DeviceIndex& dev) {
  if (!t.is_cuda()) return false;
  dev = t.get_device();
  return dev == c10::cuda::current_device();
}
bool here(const at::Tensor& t, c10::DeviceIndex dev) { return t.is_cuda() && t.get_device() == dev; }
bool here(const OptT& t, c10::DeviceIndex dev) { return !t.has_value() || here(*t, dev); }
bool is_i32(const at::Tensor& t, std::initializer_list<int64_t> shape) {
  return t.scalar_type() == at::kInt && t.is_contiguous() && t.sizes() == at::IntArrayRef(shape);
}
// a cap as the kernels' fp32 argument: beyond these bounds the weights are the same
// in fp32, but a float could round to 0 (no cap) or to infinity
float cap_arg(double cap) { return cap > 0 ? (float)std::min(std::max(cap, 1e-30), 1e30) : 0.f; }
const void* ptr(const OptT& t) { return t.has_value() ? t->data_ptr() : nullptr; }
void* current_stream() { return (void*)at::cuda::getCurrentCUDAStream().stream(); }
// the output to write: the caller's, when it is what the operator would make
bool output(const OptT& out, const at::Tensor& like, at::IntArrayRef shape, at::Tensor& res) {
  if (!out.has_value()) {
    res = at::empty(shape, like.options());
    return true;
  }
  res = *out;
  return res.is_cuda() && res.get_device() == like.get_device() && res.scalar_type() == like.scalar_type() &&
         res.sizes() == shape && res.is_contiguous();
}

py::object build_page_table(const at::Tensor& ctx, const at::Tensor& fresh, int64_t page_size, const at::Tensor& free,
                            const at::Tensor& table, int64_t max_tokens) {
  c10::DeviceIndex dev;
  if (!device_of(ctx, dev) || !here(fresh, dev) || !here(free, dev) || !here(table, dev) || ctx.dim() != 1 ||
      free.dim() != 1 || table.dim() != 2)
    return py::none();
  const int64_t B = ctx.size(0);
  if (!is_i32(ctx, {B}) || !is_i32(fresh, {B}) || !is_i32(free, {free.size(0)}) ||
      !is_i32(table, {B, table.size(1)}) || page_size <= 0 || max_tokens < 0)
    return py::none();
  const auto i32 = ctx.options();
  at::Tensor slots = at::empty({max_tokens}, i32.dtype(at::kLong)), offsets = at::empty({B + 1}, i32),
             used = at::empty({1}, i32);
  const int64_t width = table.size(1);
  const int rc = b2_build_page_table(ctx.data_ptr<int>(), fresh.data_ptr<int>(), free.data_ptr<int>(),
                                     table.data_ptr<int>(), slots.data_ptr<int64_t>(), offsets.data_ptr<int>(),
                                     used.data_ptr<int>(), B, page_size, free.size(0), width, width, max_tokens,
                                     current_stream());
  if (rc != 0) return py::int_(rc);
  return py::make_tuple(table, slots, offsets, used);
}

py::object store_kv(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kp, const at::Tensor& vp,
                    const at::Tensor& slots) {
  c10::DeviceIndex dev;
  const int src = dtype_code(k), dst = dtype_code(kp);
  if (!device_of(k, dev) || !here(v, dev) || !here(kp, dev) || !here(vp, dev) || !here(slots, dev) || k.dim() != 3 ||
      kp.dim() != 4 || v.sizes() != k.sizes() || vp.sizes() != kp.sizes() || src < 0 || dst < 0 ||
      (src != dst && src != B2_F32) || v.scalar_type() != k.scalar_type() || vp.scalar_type() != kp.scalar_type())
    return py::none();
  const int64_t N = k.size(0), H = k.size(1), D = k.size(2);
  if (kp.size(2) != H || kp.size(3) != D || kp.size(1) == 0 || H == 0 || D == 0 || k.stride(2) != 1 ||
      v.stride(2) != 1 || !kp.is_contiguous() || !vp.is_contiguous() || slots.scalar_type() != at::kLong ||
      slots.dim() != 1 || slots.size(0) != N || !slots.is_contiguous())
    return py::none();
  const int rc = b2_store_kv(k.data_ptr(), v.data_ptr(), kp.data_ptr(), vp.data_ptr(), slots.data_ptr<int64_t>(), N, H,
                             D, kp.size(0), kp.size(1), k.strides().data(), v.strides().data(), kp.strides().data(),
                             vp.strides().data(), src, dst, current_stream());
  if (rc != 0) return py::int_(rc);
  return py::make_tuple(kp, vp);
}

// K/V of a cache and its page table: [B, Hkv, S, D] or [n_pages, page_size, Hkv, D]
struct Cache {
  int64_t Hkv, keys, page_size, max_pages, n_pages;
  bool take(const at::Tensor& k, const at::Tensor& v, const OptT& table, int64_t B, int64_t D,
            c10::DeviceIndex dev) {
    if (!here(k, dev) || !here(v, dev) || !here(table, dev) || k.dim() != 4 || v.sizes() != k.sizes() ||
        v.scalar_type() != k.scalar_type() || k.size(3) != D || k.stride(3) != 1 || v.stride(3) != 1 || dtype_code(k) < 0)
      return false;
    n_pages = k.size(0);
    if (!table.has_value()) {
      Hkv = k.size(1);
      keys = k.size(2);
      page_size = max_pages = 0;
      return n_pages == B && keys > 0 && Hkv > 0;
    }
    if (table->dim() != 2 || !is_i32(*table, {B, table->size(1)})) return false;
    page_size = k.size(1);
    Hkv = k.size(2);
    max_pages = table->size(1);
    keys = page_size * max_pages;
    return keys > 0 && Hkv > 0 && n_pages > 0;
  }
};

py::object tree_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& ctx,
                          const at::Tensor& mask, const OptT& draft, const OptT& table, double scale, double softcap,
                          const OptT& out) {
  c10::DeviceIndex dev;
  const int qd = dtype_code(q);
  if (!device_of(q, dev) || q.dim() != 4 || q.stride(3) != 1 || q.numel() == 0 || qd < 0) return py::none();
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3);
  Cache c;
  if (!c.take(k, v, table, B, D, dev) || Hq % c.Hkv || !here(ctx, dev) || !here(mask, dev) || !here(draft, dev) ||
      !is_i32(ctx, {B}) || (draft.has_value() && !is_i32(*draft, {B})) || !mask.is_contiguous() ||
      (mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) || !(softcap >= 0 && std::isfinite(softcap)))
    return py::none();
  const bool each = mask.dim() == 3;
  if (mask.sizes() != (each ? at::IntArrayRef({B, T, T}) : at::IntArrayRef({T, T}))) return py::none();
  at::Tensor o;
  if (!output(out, q, q.sizes(), o)) return py::none();
  const int kd = dtype_code(k);
  const size_t need = b2_tree_attn_workspace_size(B, T, Hq, c.Hkv, D, c.keys, qd, kd);
  at::Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  const int rc = b2_tree_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), (const int32_t*)ptr(table),
                              ctx.data_ptr<int>(), (const int32_t*)ptr(draft), (const uint8_t*)mask.data_ptr(),
                              each ? T * T : 0, need ? ws.data_ptr() : nullptr, B, T, Hq, c.Hkv, D, c.keys, c.page_size,
                              c.max_pages, c.n_pages, q.strides().data(), k.strides().data(), v.strides().data(),
                              o.strides().data(), (float)scale, cap_arg(softcap), qd, kd, current_stream());
  if (rc != 0) return py::int_(rc);
  return py::cast(o);
}

bool slopes_ok(const OptT& s, int64_t Hq, c10::DeviceIndex dev) {
  return !s.has_value() ||
         (here(*s, dev) && s->scalar_type() == at::kFloat && s->dim() == 1 && s->size(0) == Hq && s->is_contiguous());
}

py::object decode_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& lens,
                            const OptT& table, double scale, double softcap, const OptT& slopes, const OptT& out) {
  c10::DeviceIndex dev;
  const int qd = dtype_code(q);
  if (!device_of(q, dev) || q.dim() != 3 || !q.is_contiguous() || q.numel() == 0 || qd < 0) return py::none();
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  Cache c;
  if (!c.take(k, v, table, B, D, dev) || Hq % c.Hkv || !here(lens, dev) || !is_i32(lens, {B}) || !(softcap >= 0 && std::isfinite(softcap)) ||
      !slopes_ok(slopes, Hq, dev))
    return py::none();
  at::Tensor o;
  if (!output(out, q, q.sizes(), o)) return py::none();
  const size_t need = softcap > 0 || slopes.has_value()
                          ? b2_decode_attn_scored_workspace_size(B, Hq, c.Hkv, D, c.keys)
                          : b2_decode_attn_workspace_size(B, Hq, c.Hkv, D, c.keys);
  at::Tensor ws = at::empty({(int64_t)(need ? need : 1)}, q.options().dtype(at::kByte));
  const int rc = b2_decode_attn_scored(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                       (const int32_t*)ptr(table), lens.data_ptr<int>(), ws.data_ptr(), B, Hq, c.Hkv, D,
                                       c.keys, c.page_size, c.max_pages, c.n_pages, k.strides().data(),
                                       v.strides().data(), nullptr, 0, nullptr, (float)scale, cap_arg(softcap),
                                       (const float*)ptr(slopes), qd, dtype_code(k), current_stream());
  if (rc != 0) return py::int_(rc);
  return py::cast(o);
}

py::object flash_scored(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal, double scale,
                        int64_t window, double softcap, const OptT& slopes, const OptT& docs, const OptT& prefix,
                        const OptT& out) {
  c10::DeviceIndex dev;
  const int dt = dtype_code(q);
  if (!device_of(q, dev) || !here(k, dev) || !here(v, dev) || q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() ||
      q.numel() == 0 || k.numel() == 0 || dt < 0 || k.scalar_type() != q.scalar_type() ||
      v.scalar_type() != q.scalar_type() || q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1)
    return py::none();
  const int64_t B = q.size(0), Hq = q.size(1), S = q.size(2), D = q.size(3), Hkv = k.size(1), Skv = k.size(2);
  if (k.size(0) != B || k.size(3) != D || Hq % Hkv || ((causal || docs.has_value()) && S != Skv) || window < 0 ||
      (window && !causal) || !(softcap >= 0 && std::isfinite(softcap)) || !slopes_ok(slopes, Hq, dev) || !here(docs, dev) || !here(prefix, dev))
    return py::none();
  int64_t n_docs = 0;
  if (docs.has_value()) {
    if (docs->dim() != 2 || docs->size(1) < 2 || !is_i32(*docs, {B, docs->size(1)})) return py::none();
    n_docs = docs->size(1) - 1;
  }
  if (prefix.has_value() &&
      (!causal || window || !(n_docs ? is_i32(*prefix, {B, n_docs}) : is_i32(*prefix, {B}))))
    return py::none();
  at::Tensor o;
  if (!output(out, q, q.sizes(), o)) return py::none();
  const int rc = b2_flash_attn_fwd_scored(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), B, Hq, Hkv, S, Skv, D,
                                          q.strides().data(), k.strides().data(), v.strides().data(),
                                          o.strides().data(), (float)scale, causal, window, cap_arg(softcap),
                                          (const float*)ptr(slopes), (const int32_t*)ptr(docs), n_docs,
                                          (const int32_t*)ptr(prefix), dt, current_stream());
  if (rc != 0) return py::int_(rc);
  return py::cast(o);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "C++ argument handling for the calls of a serving step";
  m.def("int4_matmul", &int4_matmul, py::arg("input"), py::arg("weight"), py::arg("scales"),
        py::arg("group_size"), py::arg("out") = py::none());
  m.def("build_page_table", &build_page_table);
  m.def("store_kv", &store_kv);
  m.def("tree_attention", &tree_attention);
  m.def("decode_attention", &decode_attention);
  m.def("flash_scored", &flash_scored);
}
