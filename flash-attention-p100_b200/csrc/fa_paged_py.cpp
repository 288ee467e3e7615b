// fa_paged_py.cpp -- the torch side of the paged cache's operators: checks of
// arguments, outputs and workspaces, and the calls of the C ABI
// (include/fa_b200.h), as a CPython module (_fa_paged) that fa_p100_paged.py
// wraps. The same work in Python cost 7 to 14 us of host time a call, more than
// most of these kernels take; here it is under 2. The C ABI is called
// through addresses that bind() gets from the library _lib.py has loaded, so the
// release and the checked library serve alike and nothing links against either.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/fa_b200.h"

namespace {

struct Abi {
  decltype(&fa_b200_paged_extend) extend = nullptr;
  decltype(&fa_b200_paged_release) release = nullptr;
  decltype(&fa_b200_paged_append) append = nullptr;
  decltype(&fa_b200_paged_attn) attn = nullptr;
  decltype(&fa_b200_paged_attn_workspace_bytes) attn_workspace_bytes = nullptr;
  decltype(&fa_b200_paged_table_workspace_bytes) table_workspace_bytes = nullptr;
  decltype(&fa_b200_status_string) status_string = nullptr;
  decltype(&fa_b200_last_error) last_error = nullptr;
} abi;

template <typename F>
void take(F& f, const pybind11::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const pybind11::dict& addresses) {
  take(abi.extend, addresses, "fa_b200_paged_extend");
  take(abi.release, addresses, "fa_b200_paged_release");
  take(abi.append, addresses, "fa_b200_paged_append");
  take(abi.attn, addresses, "fa_b200_paged_attn");
  take(abi.attn_workspace_bytes, addresses, "fa_b200_paged_attn_workspace_bytes");
  take(abi.table_workspace_bytes, addresses, "fa_b200_paged_table_workspace_bytes");
  take(abi.status_string, addresses, "fa_b200_status_string");
  take(abi.last_error, addresses, "fa_b200_last_error");
}

// A refusal: RuntimeError in Python.
std::string text(const char* x) { return x; }
std::string text(const std::string& x) { return x; }
std::string text(int64_t x) { return std::to_string(x); }
std::string text(at::Device x) { return x.str(); }
std::string text(at::ScalarType x) { return c10::toString(x); }

template <typename... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  std::string all;
  (void)std::initializer_list<int>{(all += text(parts), 0)...};
  throw std::runtime_error(all);
}

void check_status(int status, const char* name) {
  if (status == FA_B200_OK) return;
  const std::string detail = abi.last_error();
  refuse(name, ": ", abi.status_string(status), " (status ", static_cast<int64_t>(status), ")",
         detail.empty() ? "" : ": ", detail);
}

const at::Tensor& tensor(pybind11::handle h, const char* name) {
  if (!THPVariable_Check(h.ptr())) refuse(name, " must be a tensor");
  return THPVariable_Unpack(h.ptr());
}

// A contiguous 1-D tensor of n whole numbers (n < 0: any number).
const at::Tensor& ints(pybind11::handle h, const char* name, int64_t n, at::ScalarType dtype = at::kInt) {
  const at::Tensor& t = tensor(h, name);
  if (t.scalar_type() != dtype || t.dim() != 1 || (n >= 0 && t.numel() != n))
    refuse(name, " must be a ", dtype == at::kInt ? "torch.int32" : "torch.bool", " tensor of shape (",
           n >= 0 ? std::to_string(n) : std::string("P"), ",)");
  if (!t.is_contiguous()) refuse(name, " must be contiguous");
  return t;
}

struct Table {
  const at::Tensor& t;
  int64_t W, stride;
};

Table table(pybind11::handle h, int64_t B) {
  const at::Tensor& t = tensor(h, "block_table");
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != B || t.size(1) < 1)
    refuse("block_table must be an int32 tensor of shape (", B, ", W), W >= 1");
  const int64_t W = t.size(1);
  if ((W > 1 && t.stride(1) != 1) || (B > 1 && t.stride(0) < W))
    refuse("block_table: the columns must be contiguous and the rows apart");
  return {t, W, B > 1 ? t.stride(0) : W};
}

void check_page_size(int64_t page, int64_t P, int64_t W) {
  if (page < 16 || page > 4096 || page % 16)
    refuse("page_size must be a multiple of 16 up to 4096, got ", page);
  if (P < 1) refuse("the cache needs at least one page");
  if (std::max(P, W) * page > (int64_t{1} << 30))
    refuse("a cache, or a row of the block table, may hold up to 2**30 tokens");
}

void fits_int(int64_t n, const char* name) {
  if (n > 0x7fffffff) refuse(name, " must be below 2**31, got ", n);
}

// Strides (batch, head, row) of a 16-bit tensor; those of a size-1 axis are never
// used and taken as 8. False where 16-byte accesses cannot address it.
bool strides(const at::Tensor& t, int64_t batch, int64_t head, int64_t row, fa_b200_strides* s) {
  const auto at_axis = [&](int64_t axis) { return axis < 0 || t.size(axis) == 1 ? int64_t{8} : t.stride(axis); };
  *s = {at_axis(batch), at_axis(head), at_axis(row)};
  return t.stride(t.dim() - 1) == 1 && ((s->batch | s->head | s->row) & 7) == 0 && s->batch >= 0 && s->head >= 0 &&
         s->row >= 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

struct Caches {
  const at::Tensor &k, &v;
  int64_t P, Hkv, page, D;
  fa_b200_strides sk, sv;
  int dtype;
};

Caches caches(pybind11::handle hk, pybind11::handle hv) {
  const at::Tensor &k = tensor(hk, "k_cache"), &v = tensor(hv, "v_cache");
  if (k.dim() != 4) refuse("k_cache must be (P, Hkv, page_size, D)");
  if (v.dim() != 4) refuse("v_cache must be (P, Hkv, page_size, D)");
  if (k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16) refuse("k_cache must be fp16 or bf16");
  if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
    refuse("k_cache and v_cache must have one shape and one dtype");
  Caches c{k, v, k.size(0), k.size(1), k.size(2), k.size(3), {}, {},
           k.scalar_type() == at::kHalf ? FA_B200_DTYPE_FP16 : FA_B200_DTYPE_BF16};
  if (c.D != 64 && c.D != 128) refuse("head dim must be 64 or 128, got ", c.D);
  if (c.Hkv < 1) refuse("the cache needs at least one head");
  fits_int(c.Hkv, "the number of heads");
  check_page_size(c.page, c.P, 1);
  if (!strides(k, 0, 1, 2, &c.sk) || !strides(v, 0, 1, 2, &c.sv))
    refuse("the caches' D axis must be contiguous, and their bases and strides multiples of 16 bytes");
  return c;
}

// Whether two tensors share a byte. Their elements are sums of index times stride, so
// they do if some difference of indices makes up the distance of their bases: looked
// for axis by axis, the largest stride first, with what the smaller ones can still make
// up as the bound. Caches, rows and slices of one buffer have strides that nest, and
// leave at most two choices an axis. Layouts that leave many more count as shared.
struct Axis {
  int64_t stride, lo, hi;   // bytes; differences of indices
};
bool makes_up(const Axis* axis, const Axis* end, int64_t distance, int& budget) {
  if (axis == end) return distance == 0;
  int64_t lo = 0, hi = 0;   // of the smaller strides
  for (const Axis* x = axis + 1; x != end; ++x) {
    lo += x->lo * x->stride;
    hi += x->hi * x->stride;
  }
  const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t first = std::max(axis->lo, -floor_div(hi - distance, axis->stride));
  const int64_t last = std::min(axis->hi, floor_div(distance - lo, axis->stride));
  for (int64_t i = first; i <= last; ++i)
    if (--budget < 0 || makes_up(axis + 1, end, distance - i * axis->stride, budget)) return true;
  return false;
}

// The bytes from a tensor's first element to behind its last: most tensors are told
// apart by these alone.
struct Span {
  const at::Tensor& t;
  uintptr_t first;
  int64_t bytes;   // 0 without an element
  explicit Span(const at::Tensor& x) : t(x), first(reinterpret_cast<uintptr_t>(x.const_data_ptr())) {
    const auto sizes = x.sizes(), strides = x.strides();
    int64_t last = 0;
    for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
    bytes = x.numel() == 0 ? 0 : (last + 1) * static_cast<int64_t>(x.itemsize());
  }
};
bool share_memory(const Span& sa, const Span& sb) {
  const auto distance = static_cast<int64_t>(sb.first - sa.first);
  if (sa.bytes == 0 || sb.bytes == 0 || distance >= sa.bytes || -distance >= sb.bytes) return false;
  const at::Tensor &a = sa.t, &b = sb.t;
  Axis axes[16];   // the tensors have up to 4 axes each
  int n = 0;
  const auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
    if (stride == 0 || lo == hi) return;
    int i = 0;
    while (i < n && axes[i].stride > stride) ++i;
    if (i < n && axes[i].stride == stride) {
      axes[i].lo += lo;
      axes[i].hi += hi;
      return;
    }
    std::copy_backward(axes + i, axes + n, axes + n + 1);
    axes[i] = {stride, lo, hi};
    ++n;
  };
  for (int64_t i = 0; i < a.dim(); ++i) add(a.stride(i) * a.element_size(), 0, a.size(i) - 1);
  for (int64_t i = 0; i < b.dim(); ++i) add(b.stride(i) * b.element_size(), 1 - b.size(i), 0);
  add(1, 0, a.element_size() - 1);   // an element's bytes
  add(1, 1 - b.element_size(), 0);
  int budget = 10000;
  return makes_up(axes, axes + n, distance, budget);
}

struct Named {
  const char* name;
  const at::Tensor& t;
};

// The one GPU that holds all tensors.
at::Device one_device(std::initializer_list<Named> all) {
  const at::Device device = all.begin()->t.device();
  for (const Named& x : all) {
    if (!x.t.is_cuda()) refuse(x.name, " must be a CUDA tensor");
    if (x.t.device() != device) refuse(x.name, " must be on ", device, ", got ", x.t.device());
  }
  return device;
}

// Forward-mode tangents are refused under torch.no_grad() too, which does not turn
// that mode off.
void no_grad(std::initializer_list<Named> all) {
  const bool records = c10::GradMode::is_enabled();
  for (const Named& x : all) {
    if (records && x.t.requires_grad())
      refuse("the paged cache has no backward: call it under torch.no_grad() or detach ", x.name);
    if (x.t._fw_grad(0).defined())
      refuse("the paged cache has no forward-mode derivative: ", x.name, " carries a tangent");
  }
}

// A caller's tensor that a call has written changes as under torch's own in-place
// operations: a backward that saved it (or a view) raises. Inference tensors have no
// version.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// On the device of the call from here on; outputs are plain allocations there.
struct Call {
  c10::cuda::CUDAGuard device;
  at::AutoDispatchBelowADInplaceOrView plain;
  void* stream;
  explicit Call(at::Device d) : device(d), stream(c10::cuda::getCurrentCUDAStream(d.index()).stream()) {}
};

at::Tensor empty(at::IntArrayRef shape, const at::Tensor& like, at::ScalarType dtype) {
  return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt);
}

at::Tensor bytes_of(int64_t n, const at::Tensor& like) { return empty({n}, like, at::kByte); }

// A contiguous tensor over the bytes of `all` from `at` on, a multiple of its item
// size: a view without the dispatcher (0.2 us of host time; an allocation is 1.3).
at::Tensor piece(const at::Tensor& all, int64_t at, at::IntArrayRef shape, at::ScalarType dtype) {
  const auto type = c10::scalarTypeToTypeMeta(dtype);
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(all.storage()),
                                                          all.key_set(), type);
  t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(type.itemsize()));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  return t;
}

int* data(const at::Tensor& t) { return static_cast<int*>(t.data_ptr()); }

struct Requests {
  const at::Tensor &lens, &free_pages, &free_count;
  Table table;
  int64_t B, P;
};

Requests requests(pybind11::handle lens, pybind11::handle block_table, pybind11::handle free_pages,
                  pybind11::handle free_count, int64_t page) {
  const at::Tensor& l = tensor(lens, "lens");
  if (l.dim() != 1 || l.numel() < 1) refuse("lens must be an int32 tensor of shape (B,), B >= 1");
  const int64_t B = l.numel();
  fits_int(B, "the number of requests");
  ints(lens, "lens", B);
  const Table t = table(block_table, B);
  const at::Tensor& p = ints(free_pages, "free_pages", -1);
  const Requests r{l, p, ints(free_count, "free_count", 1), t, B, p.numel()};
  check_page_size(page, r.P, t.W);
  return r;
}

// The workspace of a table call, its further outputs `granted` and `slots` if it has
// them, and the caller's lens_out and free_count_out or new ones: pieces of one
// allocation, 24 bytes a request and more that live as long as any of them. Many slots
// are an allocation of their own, which a length that is kept does not hold (extend for
// 64 tokens 7.3 us of host time so, 6.8 with its slots among the pieces).
struct TableOutputs {
  static constexpr int64_t kFewSlots = 16384;
  at::Tensor all, granted, slots, lens, free_count;
  size_t ws_bytes;
  bool own_lens, own_free_count;   // no caller's
  TableOutputs(const Requests& r, bool extends, int64_t total, pybind11::handle lens_out,
               pybind11::handle free_count_out)
      : ws_bytes(abi.table_workspace_bytes(static_cast<int>(r.B))),
        own_lens(lens_out.is_none()),
        own_free_count(free_count_out.is_none()) {
    const int64_t few = total <= kFewSlots ? total : 0, more = extends ? r.B + few : 0;
    const int64_t ws = (static_cast<int64_t>(ws_bytes) + 3) / 4 * 4;
    all = bytes_of(ws + 4 * (more + r.B + 1), r.lens);
    const auto ints_at = [&](int64_t i, int64_t n) { return piece(all, ws + 4 * i, {n}, at::kInt); };
    if (extends) {
      granted = ints_at(0, r.B);
      slots = few == total ? ints_at(r.B, total) : empty({total}, r.lens, at::kInt);
    }
    lens = own_lens ? ints_at(more, r.B) : given(lens_out, "lens_out", r.lens);
    free_count = own_free_count ? ints_at(more + r.B, 1) : given(free_count_out, "free_count_out", r.free_count);
  }
  void mark_written() const {
    if (!own_lens) written(lens);
    if (!own_free_count) written(free_count);
  }
  static at::Tensor given(pybind11::handle h, const char* name, const at::Tensor& like) {
    const at::Tensor& t = ints(h, name, like.numel());
    if (t.device() != like.device()) refuse(name, " must be on ", like.device(), ", got ", t.device());
    return t;
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> extend(
    pybind11::handle new_lens, pybind11::handle lens, pybind11::handle block_table, pybind11::handle free_pages,
    pybind11::handle free_count, int64_t page, int64_t total, pybind11::handle lens_out,
    pybind11::handle free_count_out) {
  const Requests r = requests(lens, block_table, free_pages, free_count, page);
  const at::Tensor& n = ints(new_lens, "new_lens", r.B);
  if (total < 0 || total > 0x7fffffff) refuse("total_tokens must be in [0, 2**31), got ", total);
  Call call(one_device({{"lens", r.lens}, {"new_lens", n}, {"block_table", r.table.t}, {"free_pages", r.free_pages},
                        {"free_count", r.free_count}}));
  const TableOutputs out(r, true, total, lens_out, free_count_out);
  check_status(abi.extend(data(n), data(r.lens), data(r.table.t), r.table.stride, data(r.free_pages),
                          data(r.free_count), data(out.slots), data(out.granted), data(out.lens), data(out.free_count),
                          out.all.data_ptr(), out.ws_bytes, static_cast<int>(r.B), static_cast<int>(r.table.W), static_cast<int>(r.P),
                          static_cast<int>(page), static_cast<int>(total), call.stream),
               "fa_b200_paged_extend");
  written(r.table.t);
  out.mark_written();
  return {out.slots, out.granted, out.lens, out.free_count};
}

std::tuple<at::Tensor, at::Tensor> release(pybind11::handle finished, pybind11::handle lens,
                                           pybind11::handle block_table, pybind11::handle free_pages,
                                           pybind11::handle free_count, int64_t page, pybind11::handle lens_out,
                                           pybind11::handle free_count_out) {
  const Requests r = requests(lens, block_table, free_pages, free_count, page);
  const at::Tensor& f = ints(finished, "finished", r.B, at::kBool);
  Call call(one_device({{"lens", r.lens}, {"finished", f}, {"block_table", r.table.t}, {"free_pages", r.free_pages},
                        {"free_count", r.free_count}}));
  const TableOutputs out(r, false, 0, lens_out, free_count_out);
  check_status(abi.release(static_cast<const unsigned char*>(f.data_ptr()), data(r.lens), data(r.table.t),
                           r.table.stride, data(r.free_pages), data(r.free_count), data(out.lens),
                           data(out.free_count), out.all.data_ptr(), out.ws_bytes, static_cast<int>(r.B), static_cast<int>(r.table.W), static_cast<int>(r.P),
                           static_cast<int>(page), call.stream),
               "fa_b200_paged_release");
  written(r.free_pages);
  out.mark_written();
  return {out.lens, out.free_count};
}

void append(pybind11::handle k_new, pybind11::handle v_new, pybind11::handle slots, pybind11::handle k_cache,
            pybind11::handle v_cache) {
  const Caches c = caches(k_cache, v_cache);
  at::Tensor k = tensor(k_new, "k"), v = tensor(v_new, "v");
  for (const Named& x : {Named{"k", k}, Named{"v", v}}) {
    if (x.t.dim() != 3 || x.t.size(1) != c.Hkv || x.t.size(2) != c.D)
      refuse(x.name, " must be (T, ", c.Hkv, ", ", c.D, ")");
    if (x.t.scalar_type() != c.k.scalar_type())
      refuse(x.name, " must have the caches' dtype ", c.k.scalar_type(), ", got ", x.t.scalar_type());
  }
  const int64_t T = k.size(0);
  if (T != v.size(0)) refuse("k and v must match");
  fits_int(T, "the number of tokens");
  const at::Tensor& s = ints(slots, "slots", T);
  for (const fa_b200_strides& st : {c.sk, c.sv})
    if (st.batch == 0 || st.head == 0 || st.row == 0)
      refuse("k_cache and v_cache are written and must not be expanded views");
  const Span in_k(c.k), in_v(c.v);
  if (share_memory(in_k, in_v)) refuse("k_cache and v_cache must be different memory");
  for (const Named& x : {Named{"k", k}, Named{"v", v}, Named{"slots", s}})
    if (const Span span(x.t); share_memory(span, in_k) || share_memory(span, in_v))
      refuse(x.name, " must not overlap the caches");
  no_grad({{"k", k}, {"v", v}, {"k_cache", c.k}, {"v_cache", c.v}});
  Call call(one_device({{"k_cache", c.k}, {"v_cache", c.v}, {"k", k}, {"v", v}, {"slots", s}}));
  if (T == 0) return;
  // rows that 16-byte accesses cannot address are copied first
  fa_b200_strides sk, sv;
  if (!strides(k, -1, 1, 0, &sk)) strides(k = k.clone(at::MemoryFormat::Contiguous), -1, 1, 0, &sk);
  if (!strides(v, -1, 1, 0, &sv)) strides(v = v.clone(at::MemoryFormat::Contiguous), -1, 1, 0, &sv);
  check_status(abi.append(k.data_ptr(), sk, v.data_ptr(), sv, data(s), c.k.data_ptr(), c.sk, c.v.data_ptr(), c.sv,
                          static_cast<int>(T), static_cast<int>(c.Hkv), static_cast<int>(c.D),
                          static_cast<int>(c.P), static_cast<int>(c.page), c.dtype, call.stream),
               "fa_b200_paged_append");
  written(c.k);
  written(c.v);
}

std::tuple<at::Tensor, at::Tensor> attn(pybind11::handle query, pybind11::handle k_cache, pybind11::handle v_cache,
                                        pybind11::handle block_table, pybind11::handle lens) {
  const Caches c = caches(k_cache, v_cache);
  at::Tensor q = tensor(query, "q");
  if (q.dim() != 3 || q.size(2) != c.D || q.size(0) < 1) refuse("q must be (B, Hq, ", c.D, "), B >= 1");
  if (q.scalar_type() != c.k.scalar_type())
    refuse("q must have the caches' dtype ", c.k.scalar_type(), ", got ", q.scalar_type());
  const int64_t B = q.size(0), Hq = q.size(1);
  fits_int(B * std::max<int64_t>(Hq, 1), "requests * heads");
  if (Hq < 1 || Hq % c.Hkv)
    refuse("query heads (", Hq, ") must be a multiple of key/value heads (", c.Hkv, ")");
  const at::Tensor& l = ints(lens, "lens", B);
  const Table t = table(block_table, B);
  check_page_size(c.page, c.P, t.W);
  no_grad({{"q", q}, {"k_cache", c.k}, {"v_cache", c.v}});
  Call call(one_device({{"q", q}, {"k_cache", c.k}, {"v_cache", c.v}, {"block_table", t.t}, {"lens", l}}));
  fa_b200_strides sq;
  if (!strides(q, 0, 1, -1, &sq)) strides(q = q.clone(at::MemoryFormat::Contiguous), 0, 1, -1, &sq);
  const at::Tensor out = bytes_of(B * Hq * (2 * c.D + 4), q);
  at::Tensor o = piece(out, 0, {B, Hq, c.D}, q.scalar_type());
  at::Tensor lse = piece(out, 2 * B * Hq * c.D, {B, Hq}, at::kFloat);
  const fa_b200_strides so{Hq * c.D, c.D, c.D};
  const int ib = static_cast<int>(B), ihq = static_cast<int>(Hq), ihkv = static_cast<int>(c.Hkv);
  const int id = static_cast<int>(c.D), iw = static_cast<int>(t.W), ip = static_cast<int>(c.page);
  const size_t bytes = abi.attn_workspace_bytes(ib, ihq, ihkv, iw, id, ip);
  at::Tensor ws;
  if (bytes) ws = bytes_of(static_cast<int64_t>(bytes), q);
  check_status(abi.attn(q.data_ptr(), sq, c.k.data_ptr(), c.sk, c.v.data_ptr(), c.sv, data(t.t), t.stride, data(l),
                        o.data_ptr(), so, static_cast<float*>(lse.data_ptr()), bytes ? ws.data_ptr() : nullptr, bytes,
                        ib, ihq, ihkv, id, static_cast<int>(c.P), iw, ip, c.dtype, call.stream),
               "fa_b200_paged_attn");
  return {o, lse};
}

}  // namespace

PYBIND11_MODULE(_fa_paged, m) {
  m.attr("build_key") = FA_PAGED_KEY;   // what this was compiled against (_build.binding_key)
  m.def("bind", &bind);
  m.def("extend", &extend);
  m.def("release", &release);
  m.def("append", &append);
  m.def("attn", &attn);
  m.def("check_page_size", &check_page_size);
}
