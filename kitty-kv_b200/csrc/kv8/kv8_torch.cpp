// Torch side of the 8-bit cache operators: checks the tensors, fills the argument
// structs of include/kitty_kv8.h and calls the entry points on the tensors' current
// stream.  The calls of a decode step take a few microseconds on the GPU, so the checks
// are made here and not in Python, where they would take longer than the kernels.
// Everything that is refused raises RuntimeError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <limits>

#include "../../../include/kitty_kv8.h"

namespace {

using at::Tensor;

// A tensor argument; undefined for None.
Tensor tensor(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return Tensor();
  TORCH_CHECK(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}

struct Call {
  c10::Device device{c10::kCPU};
  // A tensor of the call: all on one CUDA device.
  const Tensor& on(const Tensor& t) {
    if (!t.defined()) return t;
    TORCH_CHECK(t.is_cuda(), "Kitty B200 kernels need CUDA tensors (there is no CPU path); got a tensor on ", t.device());
    if (device.is_cpu()) device = t.device();
    TORCH_CHECK(t.device() == device, "tensors on different devices: ", device, " and ", t.device());
    return t;
  }
  Tensor arg(PyObject* o, const char* name, bool optional = false) {
    Tensor t = tensor(o, name, optional);
    on(t);
    return t;
  }
};

// These operators have no backward pass and no forward derivative: a tensor that asks for one is
// refused, what is written included.
void no_grad(std::initializer_list<const Tensor*> tensors) {
  const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    TORCH_CHECK(!backward || !t->requires_grad(), "this operator has no backward pass: call it under "
                "torch.no_grad() or on detached tensors");
    TORCH_CHECK(!forward || !t->_fw_grad(0).defined(), "this operator has no forward derivative: call it on the "
                "primal of a dual tensor");
  }
}

// What autograd has saved of a tensor that was written is no longer what it was.
void written(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

int dtype_code(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kHalf) return KITTY_KV8_F16;
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, what, " must be float16 or bfloat16, got ", t.scalar_type());
  return KITTY_KV8_BF16;
}

int32_t i32(int64_t v, const char* what) {
  TORCH_CHECK(v <= std::numeric_limits<int32_t>::max(), what, " does not fit 32 bits");
  return int32_t(v);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Row and head strides of a (rows, heads, D) tensor; true if its rows are 16-byte aligned.
bool row_strides(const Tensor& t, int64_t& s0, int64_t& s1) {
  s0 = t.size(0) > 1 ? t.stride(0) : 0;
  s1 = t.size(1) > 1 ? t.stride(1) : 0;
  return (t.stride(2) == 1 || t.size(2) <= 1) && s0 % 8 == 0 && s1 % 8 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// A contiguous tensor on the device of `like` (without the way through the dispatcher).
Tensor make(at::IntArrayRef shape, const Tensor& like) {
  return at::detail::empty_cuda(shape, like.scalar_type(), like.device(), std::nullopt);
}

// An input of aligned rows, copied if it has none.
const void* input_rows(Tensor& t, int64_t& s0, int64_t& s1) {
  if (!row_strides(t, s0, s1)) {
    t = t.clone(at::MemoryFormat::Contiguous);
    s0 = t.size(1) * t.size(2);
    s1 = t.size(2);
  }
  return t.data_ptr();
}

// A caller's output: refused if its rows are not aligned or overlap.  Undefined: made here.
void* output_rows(Tensor& t, const Tensor& like, const char* name, int64_t& s0, int64_t& s1) {
  if (!t.defined()) {
    t = make(like.sizes(), like);
    s0 = like.size(1) * like.size(2);
    s1 = like.size(2);
    return t.data_ptr();
  }
  TORCH_CHECK(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type(), name, " must be ", like.sizes(), " ",
              like.scalar_type());
  const bool ok = row_strides(t, s0, s1);
  TORCH_CHECK(ok, name, " needs unit channel stride and 16-byte aligned rows");
  // rows that follow one another in either order, heads inside tokens or tokens inside heads
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2);
  TORCH_CHECK(n * h <= 1 || (n <= 1 ? s1 >= d : h <= 1 ? s0 >= d : (s1 >= d && s0 >= (h - 1) * s1 + d) ||
                                                                     (s0 >= d && s1 >= (n - 1) * s0 + d)),
              name, " has rows that overlap");
  return t.data_ptr();
}

// The places of (rows, heads, D) 16-bit values, strides in elements (0 where there is one).
struct Places {
  const void* p;
  int64_t n, h, d, s0, s1;
  bool operator==(const Places& o) const { return p == o.p && n == o.n && h == o.h && s0 == o.s0 && s1 == o.s1; }
};

Places places(const Tensor& t, const void* p, int64_t s0, int64_t s1) {
  return Places{p, t.size(0), t.size(1), t.size(2), t.size(0) > 1 ? s0 : 0, t.size(1) > 1 ? s1 : 0};
}

// Whether two of them, of equally many rows, share a value.  Exact where their row strides are
// the same (the parts of fused rows lie between one another); otherwise whether their ranges meet.
bool meet(const Places& a, const Places& b) {
  if (a.n == 0 || a.h == 0 || b.h == 0) return false;
  const int64_t off = (reinterpret_cast<intptr_t>(b.p) - reinterpret_cast<intptr_t>(a.p)) / 2;
  const int64_t wide_a = (a.h - 1) * a.s1 + a.d, wide_b = (b.h - 1) * b.s1 + b.d, s = a.s0;
  if (off >= (a.n - 1) * a.s0 + wide_a || -off >= (b.n - 1) * b.s0 + wide_b) return false;
  if (a.s0 != b.s0) return true;
  if (s > 0) {     // the rows of one between those of the other
    const int64_t in = (off % s + s) % s;
    if (in >= wide_a && in + wide_b <= s) return false;
  }
  for (int64_t i = 0; i < a.h; ++i)
    for (int64_t j = 0; j < b.h; ++j) {
      // head j of b against head i of a, k rows away: | e + k s | < d for a k of -(n - 1) .. n - 1
      const int64_t e = off + j * b.s1 - i * a.s1;
      const int64_t k = s > 0 ? std::max(-(a.n - 1), std::min(a.n - 1, -e / s)) : 0;
      for (int64_t x = std::max(k - 1, -(a.n - 1)); x <= std::min(k + 1, a.n - 1); ++x)
        if (std::abs(e + x * s) < a.d) return true;
    }
  return false;
}

const int32_t* index(Tensor& t, const char* name, int64_t n) {
  if (!t.defined()) return nullptr;
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n, name, " must be (", n, ",) int32");
  if (!t.is_contiguous()) t = t.contiguous();
  return static_cast<const int32_t*>(t.data_ptr());
}

void check(int rc, const char* what) {
  static const char* const kind[] = {"", "invalid argument", "unsupported", "CUDA error", "workspace"};
  TORCH_CHECK(rc == 0, what, " failed (", rc > 0 && rc < 5 ? kind[rc] : "?", "): ", kitty_kv8_last_error());
}

template <typename Fn, typename Args>
void launch(const Call& call, Fn fn, const Args& args, const char* what) {
  const c10::cuda::CUDAGuard guard(call.device);
  check(fn(&args, c10::cuda::getCurrentCUDAStream(call.device.index()).stream()), what);
}

// The arrays of a cache, in the order of the Python functions: lengths, block_table,
// key_codes, value_codes, key_scale, value_scale, tail_k, tail_v.
struct CacheArrays {
  Tensor lengths, table, key_codes, value_codes, key_scale, value_scale, tail_k, tail_v;
};

CacheArrays fill_cache(Call& call, PyObject* const* o, KittyKv8Cache& c) {
  CacheArrays r{call.arg(o[0], "lengths"), call.arg(o[1], "block_table"), call.arg(o[2], "key_codes"),
                call.arg(o[3], "value_codes"), call.arg(o[4], "key_scale"), call.arg(o[5], "value_scale"),
                call.arg(o[6], "tail_k"), call.arg(o[7], "tail_v")};
  TORCH_CHECK(r.key_codes.dim() == 4 && r.value_codes.sizes() == r.key_codes.sizes(),
              "key_codes and value_codes must both be (P, H, G, D)");
  const auto code = r.key_codes.scalar_type();
  TORCH_CHECK((code == at::kFloat8_e4m3fn || code == at::kChar) && r.value_codes.scalar_type() == code,
              "key_codes and value_codes must both be float8_e4m3fn or both int8");
  const int64_t pages = r.key_codes.size(0), h = r.key_codes.size(1), g = r.key_codes.size(2), d = r.key_codes.size(3);
  TORCH_CHECK(r.lengths.dim() == 1 && r.lengths.scalar_type() == at::kInt, "lengths must be (slots,) int32");
  const int64_t slots = r.lengths.size(0);
  TORCH_CHECK(r.table.dim() == 2 && r.table.scalar_type() == at::kInt && r.table.size(0) == slots,
              "block_table must be (slots, M) int32 with a row for each entry of lengths");
  TORCH_CHECK(r.table.size(1) <= 1 || r.table.stride(1) == 1, "block_table rows need unit stride");
  c.dtype = dtype_code(r.tail_k, "tail_k and tail_v");
  TORCH_CHECK(r.tail_v.scalar_type() == r.tail_k.scalar_type(), "tail_k and tail_v must have one dtype");
  TORCH_CHECK(r.tail_k.dim() == 4 && r.tail_k.size(0) == slots && r.tail_k.size(1) == h && r.tail_k.size(2) == g &&
              r.tail_k.size(3) == d && r.tail_v.sizes() == r.tail_k.sizes(),
              "tail_k and tail_v must be (", slots, ", ", h, ", ", g, ", ", d, ")");
  for (const Tensor* t : {&r.key_scale, &r.value_scale})
    TORCH_CHECK(t->dim() == 2 && t->scalar_type() == at::kFloat && t->size(0) == pages && t->size(1) == h,
                "key_scale and value_scale must be (", pages, ", ", h, ") float32");
  TORCH_CHECK(r.key_codes.is_contiguous() && r.value_codes.is_contiguous() && r.key_scale.is_contiguous() &&
              r.value_scale.is_contiguous() && r.tail_k.is_contiguous() && r.tail_v.is_contiguous() &&
              r.lengths.is_contiguous(), "pools, scales, tails and lengths must be contiguous");
  no_grad({&r.key_codes, &r.value_codes, &r.key_scale, &r.value_scale, &r.tail_k, &r.tail_v});
  c.key_codes = ptr(r.key_codes);
  c.value_codes = ptr(r.value_codes);
  c.key_scale = static_cast<float*>(ptr(r.key_scale));
  c.value_scale = static_cast<float*>(ptr(r.value_scale));
  c.tail_k = ptr(r.tail_k);
  c.tail_v = ptr(r.tail_v);
  c.block_table = static_cast<const int32_t*>(ptr(r.table));
  c.lengths = static_cast<const int32_t*>(ptr(r.lengths));
  c.bt_s_slot = r.table.stride(0);
  c.pages = pages;
  c.slots = i32(slots, "slots");
  c.max_pages = i32(r.table.size(1), "block_table");
  c.num_heads = i32(h, "heads");
  c.head_dim = i32(d, "head_dim");
  c.page_size = i32(g, "page_size");
  c.code = code == at::kChar ? KITTY_KV8_INT8 : KITTY_KV8_E4M3;
  return r;
}

constexpr int kCache = 8;     // tensors of a cache

// qk_norm_rope(q, k, positions, table, q_weight, k_weight, eps, interleaved, q_out, k_out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 10, "qk_norm_rope takes 10 arguments");
  Call call;
  Tensor q = call.arg(o[0], "q"), k = call.arg(o[1], "k"), pos = call.arg(o[2], "positions"),
         table = call.arg(o[3], "table"), wq = call.arg(o[4], "q_weight", true), wk = call.arg(o[5], "k_weight", true),
         q_out = call.arg(o[8], "q_out", true), k_out = call.arg(o[9], "k_out", true);
  no_grad({&q, &k, &wq, &wk, &table, &q_out, &k_out});
  KittyQkNormRopeArgs a{};
  a.eps = float(PyFloat_AsDouble(o[6]));
  a.interleaved = PyObject_IsTrue(o[7]);
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2),
              "q must be (N, Hq, D) and k (N, H, D)");
  a.dtype = dtype_code(q, "q and k");
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have one dtype, got ", q.scalar_type(), " and ",
              k.scalar_type());
  const int64_t n = q.size(0), d = q.size(2);
  TORCH_CHECK((pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong) && pos.dim() == 1 && pos.size(0) == n,
              "positions must be (", n, ",) int32 or int64");
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kFloat && table.is_contiguous(),
              "table must be (max_positions, R) float32, contiguous");
  TORCH_CHECK(wq.defined() == wk.defined(), "q_weight and k_weight must be given together");
  if (wq.defined()) {
    TORCH_CHECK(wq.dim() == 1 && wk.dim() == 1 && wq.size(0) == d && wk.size(0) == d,
                "q_weight and k_weight must be (", d, ",)");
    a.weight_f32 = wq.scalar_type() == at::kFloat;
    TORCH_CHECK(wk.scalar_type() == wq.scalar_type() && (a.weight_f32 || wq.scalar_type() == q.scalar_type()),
                "q_weight and k_weight must both be ", q.scalar_type(), " or both float32");
    wq = wq.contiguous();
    wk = wk.contiguous();
  }
  pos = pos.contiguous();
  const bool given = q_out.defined() || k_out.defined();
  a.q_out = output_rows(q_out, q, "q_out", a.qo_s_row, a.qo_s_head);
  a.k_out = output_rows(k_out, k, "k_out", a.ko_s_row, a.ko_s_head);
  a.q = input_rows(q, a.q_s_row, a.q_s_head);
  a.k = input_rows(k, a.k_s_row, a.k_s_head);
  if (given) {     // warps take the heads of a token apart, and read ahead of what they store
    const Places in[2] = {places(q, a.q, a.q_s_row, a.q_s_head), places(k, a.k, a.k_s_row, a.k_s_head)},
                 out[2] = {places(q_out, a.q_out, a.qo_s_row, a.qo_s_head), places(k_out, a.k_out, a.ko_s_row, a.ko_s_head)};
    for (int i = 0; i < 2; ++i)
      TORCH_CHECK((out[i] == in[i] || !meet(out[i], in[i])) && !meet(out[i], in[1 - i]), i ? "k_out" : "q_out",
                  " overlaps an input (it may be ", i ? "k" : "q", " itself, with the same strides)");
    TORCH_CHECK(!meet(out[0], out[1]), "q_out and k_out overlap");
  }
  a.q_weight = ptr(wq);
  a.k_weight = ptr(wk);
  a.positions = ptr(pos);
  a.positions64 = pos.scalar_type() == at::kLong;
  a.table = static_cast<const float*>(ptr(table));
  a.table_rows = table.size(0);
  a.rows = i32(n, "N");
  a.num_q_heads = i32(q.size(1), "Hq");
  a.num_k_heads = i32(k.size(1), "H");
  a.head_dim = i32(d, "D");
  a.rot = i32(table.size(1), "R");
  launch(call, kitty_qk_norm_rope, a, "kitty_qk_norm_rope");
  written({&q_out, &k_out});
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(q_out));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(k_out));
  return r;
  END_HANDLE_TH_ERRORS
}

// write(key, value, <cache>, row_offsets, seq_map)
PyObject* write(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 4 + kCache, "write takes 12 arguments");
  Call call;
  KittyKv8WriteArgs a{};
  Tensor key = call.arg(o[0], "key"), value = call.arg(o[1], "value");
  no_grad({&key, &value});
  const CacheArrays c = fill_cache(call, o + 2, a.cache);
  Tensor offsets = call.arg(o[10], "row_offsets", true), map = call.arg(o[11], "seq_map", true);
  TORCH_CHECK(key.dim() == 3 && key.sizes() == value.sizes() && key.size(1) == a.cache.num_heads &&
              key.size(2) == a.cache.head_dim && key.scalar_type() == c.tail_k.scalar_type() &&
              value.scalar_type() == c.tail_k.scalar_type(),
              "key and value must be (N, ", a.cache.num_heads, ", ", a.cache.head_dim, ") ", c.tail_k.scalar_type());
  const int64_t rows = key.size(0);
  const int64_t n = map.defined() ? map.numel() : offsets.defined() ? offsets.numel() - 1 : rows;
  TORCH_CHECK(n >= 0, "row_offsets must have n + 1 entries");
  TORCH_CHECK(offsets.defined() || n == rows, "without row_offsets key and value must have one row for each slot");
  a.seq_map = index(map, "seq_map", n);
  a.row_offsets = index(offsets, "row_offsets", n + 1);
  a.key = input_rows(key, a.k_s_row, a.k_s_head);
  a.value = input_rows(value, a.v_s_row, a.v_s_head);
  a.n = i32(n, "entries");
  a.rows = i32(rows, "N");
  launch(call, kitty_kv8_write, a, "kitty_kv8_write");
  written({&c.key_codes, &c.value_codes, &c.key_scale, &c.value_scale, &c.tail_k, &c.tail_v});
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// read(<cache>, row_offsets, rows, first, seq_map, key_out, value_out)
PyObject* read(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 6 + kCache, "read takes 14 arguments");
  Call call;
  KittyKv8ReadArgs a{};
  const CacheArrays c = fill_cache(call, o, a.cache);
  Tensor offsets = call.arg(o[8], "row_offsets"), first = call.arg(o[10], "first", true),
         map = call.arg(o[11], "seq_map", true);
  Tensor out[2] = {call.arg(o[12], "key_out", true), call.arg(o[13], "value_out", true)};
  no_grad({&out[0], &out[1]});
  const int64_t rows = PyLong_AsLongLong(o[9]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t n = offsets.numel() - 1;
  TORCH_CHECK(n >= 0 && rows >= 0, "row_offsets must have n + 1 entries and rows must not be negative");
  a.row_offsets = index(offsets, "row_offsets", n + 1);
  a.first = index(first, "first", n);
  a.seq_map = index(map, "seq_map", n);
  const int64_t shape[3] = {rows, a.cache.num_heads, a.cache.head_dim};
  for (Tensor& t : out) {
    if (!t.defined()) t = make(shape, c.tail_k);
    TORCH_CHECK(t.sizes() == at::IntArrayRef(shape) && t.scalar_type() == c.tail_k.scalar_type() && t.is_contiguous(),
                "key_out and value_out must be (", rows, ", ", shape[1], ", ", shape[2], ") ", c.tail_k.scalar_type(),
                ", contiguous");
  }
  const int64_t row = shape[1] * shape[2];
  TORCH_CHECK(!meet(Places{ptr(out[0]), rows, 1, row, row, 0}, Places{ptr(out[1]), rows, 1, row, row, 0}),
              "key_out and value_out overlap");
  a.key = ptr(out[0]);
  a.value = ptr(out[1]);
  a.n = i32(n, "entries");
  a.rows = i32(rows, "rows");
  launch(call, kitty_kv8_read, a, "kitty_kv8_read");
  written({&out[0], &out[1]});
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out[0]));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(out[1]));
  return r;
  END_HANDLE_TH_ERRORS
}

// attention(q, <cache>, sm_scale, seq_map, out)
PyObject* attention(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n_args == 4 + kCache, "attention takes 12 arguments");
  Call call;
  KittyKv8AttentionArgs a{};
  Tensor q = call.arg(o[0], "q");
  const CacheArrays c = fill_cache(call, o + 1, a.cache);
  Tensor map = call.arg(o[10], "seq_map", true), out = call.arg(o[11], "out", true);
  no_grad({&q, &out});
  TORCH_CHECK(q.dim() == 3 && q.size(2) == a.cache.head_dim && q.scalar_type() == c.tail_k.scalar_type(),
              "q must be (B, Hq, ", a.cache.head_dim, ") ", c.tail_k.scalar_type());
  const int64_t b = q.size(0), hq = q.size(1);
  TORCH_CHECK(hq > 0 && a.cache.num_heads > 0 && hq % a.cache.num_heads == 0,
              "num_q_heads must be a multiple of num_kv_heads");
  a.sm_scale = o[9] == Py_None ? float(1.0 / std::sqrt(double(a.cache.head_dim))) : float(PyFloat_AsDouble(o[9]));
  if (PyErr_Occurred()) return nullptr;
  a.seq_map = index(map, "seq_map", b);
  a.out = output_rows(out, q, "out", a.out_s_seq, a.out_s_head);
  a.q = input_rows(q, a.q_s_seq, a.q_s_head);
  const Places from = places(q, a.q, a.q_s_seq, a.q_s_head), to = places(out, a.out, a.out_s_seq, a.out_s_head);
  TORCH_CHECK(from == to || !meet(from, to), "out overlaps q (it may be q itself, with the same strides)");
  a.batch = i32(b, "B");
  a.num_q_heads = i32(hq, "Hq");
  const c10::cuda::CUDAGuard guard(call.device);
  check(kitty_kv8_attention_workspace_size(&a, &a.workspace_bytes), "kitty_kv8_attention_workspace_size");
  // from the allocator of this stream (and of this graph, in a capture), and back to it on return
  const c10::DataPtr scratch = c10::cuda::CUDACachingAllocator::get()->allocate(a.workspace_bytes);
  a.workspace = scratch.get();
  launch(call, kitty_kv8_attention, a, "kitty_kv8_attention");
  written({&out});
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

#define KITTY_FN(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {KITTY_FN(qk_norm_rope), KITTY_FN(write), KITTY_FN(read), KITTY_FN(attention),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kv8_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8_torch() { return PyModule_Create(&kModule); }
