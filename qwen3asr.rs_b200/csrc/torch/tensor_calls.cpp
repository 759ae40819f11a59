// tensor_calls.cpp — module _vasr_calls: the tensor-level entry points of the
// rotary, scored-attention, eviction and verification operators.
//
// Each takes the tensors of the Python call that documents it (fused.py,
// eviction.py, speculative.py), checks them, allocates the results, finds the
// stream's workspace and forwards raw pointers to the C ABI. These calls are
// made once per layer and decode step on a few microseconds of GPU work, and
// the same checks in Python with a ctypes call of 20 to 30 arguments took 15
// us of host time (8 in Python, 2.5 in the argument conversions); here they
// take 1 to 2. The C functions' addresses come from the loaded library
// (bind), so that this module and the ctypes binding always run the same one.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <map>
#include <string>
#include <utility>
#include <vector>

#include "vasr_pa.h"

namespace {

// ------------------------------------------------------------- the C functions
decltype(&vasr_pa_mrope) c_mrope;
decltype(&vasr_pa_fused_qk_norm_mrope_append) c_mrope_append;
decltype(&vasr_pa_paged_attention_scored) c_scored;
decltype(&vasr_pa_paged_attention_scored_workspace_size) c_scored_size;
decltype(&vasr_pa_evict_kv) c_evict;
decltype(&vasr_pa_verify_draft_tokens) c_verify;
decltype(&vasr_pa_verify_draft_tokens_workspace_size) c_verify_size;
PyObject *error_class;  // VasrPaError(status, what)

// A refusal: VasrPaError(status, what).
struct Refused {
  int status;
  std::string what;
};
void require(bool ok, int status, const char *what) {
  if (!ok) throw Refused{status, what};
}

// ------------------------------------------------------------------- arguments
const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) throw Refused{VASR_PA_EINVAL_POINTER, std::string(name) + " must be a tensor"};
  return THPVariable_Unpack(o);
}
const at::Tensor *maybe(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }
struct PyFailed {};  // a Python exception is set
int64_t whole(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyFailed{};
  return v;
}
int32_t whole32(PyObject *o, const char *name) {
  const int64_t v = whole(o);
  if (v < INT32_MIN || v > INT32_MAX) throw Refused{VASR_PA_EINVAL_SHAPE, std::string(name) + " out of range"};
  return (int32_t)v;
}
double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
  return v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailed{};
  return v != 0;
}

template <typename T = void>
T *ptr(const at::Tensor &t) { return static_cast<T *>(t.data_ptr()); }
template <typename T = void>
T *ptr(const at::Tensor *t) { return t ? ptr<T>(*t) : nullptr; }

int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return VASR_PA_F32;
    case at::kBFloat16: return VASR_PA_BF16;
    case at::kHalf: return VASR_PA_F16;
    default: throw Refused{VASR_PA_EINVAL_DTYPE, std::string("unsupported paged cache dtype ") + toString(t.scalar_type())};
  }
}
bool is_index32(const at::Tensor &t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32; }
bool shape_is(const at::Tensor &t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s); }
bool is_f32(const at::Tensor &t) { return t.scalar_type() == at::kFloat; }

// The device of a call's tensors: one CUDA device.
c10::DeviceIndex common_device(std::initializer_list<const at::Tensor *> ts) {
  const c10::Device d = (*ts.begin())->device();
  for (const at::Tensor *t : ts) {
    require(t->is_cuda(), VASR_PA_EINVAL_POINTER, "paged attention tensors must be on a CUDA device");
    require(t->device() == d, VASR_PA_EINVAL_POINTER, "paged attention tensors on different devices");
  }
  return d.index();
}
bool on(const at::Tensor &t, c10::DeviceIndex d) { return t.is_cuda() && t.device().index() == d; }

vasr_pa_stream_t stream_of(c10::DeviceIndex d) {
  return reinterpret_cast<vasr_pa_stream_t>(c10::cuda::getCurrentCUDAStream(d).stream());
}

struct Cache {
  int64_t blocks;
  int32_t heads, dim, block;
  bool fp8;
  int code;  // of the pages; the query's own type's where they are not fp8
};
Cache cache_of(const at::Tensor &k, const at::Tensor &v) {
  require(k.dim() == 5 && v.dim() == 4, VASR_PA_EINVAL_SHAPE, "key cache must have 5 dims and value cache 4");
  const auto s = k.sizes();
  require(shape_is(v, {s[0], s[1], s[2] * s[4], s[3]}) && s[4] * (int64_t)k.element_size() == 16, VASR_PA_EINVAL_SHAPE,
          "paged cache shape mismatch");
  require(k.scalar_type() == v.scalar_type(), VASR_PA_EINVAL_DTYPE, "key/value cache dtype mismatch");
  require(k.is_contiguous() && v.is_contiguous(), VASR_PA_EINVAL_SHAPE, "paged caches must be contiguous");
  Cache c{s[0], (int32_t)s[1], (int32_t)(s[2] * s[4]), (int32_t)s[3], k.scalar_type() == at::kFloat8_e4m3fn, 0};
  c.code = c.fp8 ? (int)VASR_PA_FP8_E4M3 : dtype_code(k);
  return c;
}
// fp8 pages come with both scales; other pages have the rows' type.
void check_rows(const Cache &c, const at::Tensor &rows, const at::Tensor &k, const at::Tensor *ks, const at::Tensor *vs,
                const char *what) {
  if (!c.fp8) {
    require(rows.scalar_type() == k.scalar_type(), VASR_PA_EINVAL_DTYPE, what);
    return;
  }
  for (const at::Tensor *s : {ks, vs})
    require(s && is_f32(*s) && s->numel() == 1 && s->device() == k.device(), VASR_PA_EINVAL_POINTER,
            "fp8 caches need k_scale / v_scale as f32 scalars on the cache device");
}
void check_scores(const at::Tensor &s, const Cache &c, c10::DeviceIndex d) {
  require(is_f32(s) && shape_is(s, {c.blocks, c.heads, c.block}) && on(s, d) && s.is_contiguous(), VASR_PA_EINVAL_SHAPE,
          "score_cache must be a contiguous f32 [num_blocks, num_kv_heads, block_size] on the cache device");
}

void check(int status, const char *what) {
  if (status != VASR_PA_OK) throw Refused{status, what};
}

bool capturing() {
  return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
}

// The scratch of one kind of call: a growing workspace per (device, stream),
// allocated in that stream's order, whichever is current; outgrown ones stay
// allocated, and doubling bounds them by the one in use. A call that is being
// captured takes its scratch from the graph's own memory instead: graphs that
// were captured on one stream may be replayed on several at once.
class Workspaces {
 public:
  explicit Workspaces(const char *what) : what_(what) {}
  const at::Tensor &reserve(c10::DeviceIndex device, uintptr_t stream, size_t bytes) {
    std::vector<at::Tensor> &all = held_[{device, stream}];
    const size_t have = all.empty() ? 0 : (size_t)all.back().numel();
    if (all.empty() || have < bytes) {
      if (capturing())
        throw Refused{VASR_PA_EINVAL_WORKSPACE, what_ + " workspace cannot be reserved while a CUDA graph is captured"};
      const c10::cuda::CUDAStreamGuard guard(
          c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(stream), device));
      all.push_back(allocate(device, std::max({bytes, 2 * have, (size_t)1 << 20})));
    }
    return all.back();
  }
  at::Tensor scratch(c10::DeviceIndex device, vasr_pa_stream_t stream, size_t bytes) {
    if (capturing()) return allocate(device, std::max(bytes, (size_t)1));
    return reserve(device, reinterpret_cast<uintptr_t>(stream), bytes);
  }

 private:
  static at::Tensor allocate(c10::DeviceIndex device, size_t bytes) {
    return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(c10::Device(c10::kCUDA, device)));
  }
  std::string what_;
  std::map<std::pair<c10::DeviceIndex, uintptr_t>, std::vector<at::Tensor>> held_;
};
Workspaces &scored_workspaces() {
  static auto *w = new Workspaces("paged_attention_scored");  // outlives the interpreter's tensors
  return *w;
}
Workspaces &verify_workspaces() {
  static auto *w = new Workspaces("verify_draft_tokens");
  return *w;
}

// ---------------------------------------------------------------------- rotary
struct Rope {
  int32_t sections[4];
  int32_t axes, half;
  at::Tensor positions;  // unit token stride
  int64_t axis_stride;
};
Rope rope_of(const at::Tensor &cos, const at::Tensor &sin, const at::Tensor &positions, PyObject *sections,
             int64_t tokens) {
  Rope r;
  PyObject *seq = PySequence_Fast(sections, "sections must be a sequence");
  if (!seq) throw PyFailed{};
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  r.axes = (int32_t)n;
  r.half = 0;
  bool ok = n >= 1 && n <= 4;
  try {
    for (Py_ssize_t i = 0; ok && i < n; ++i) {
      const int32_t s = whole32(PySequence_Fast_GET_ITEM(seq, i), "sections");
      ok = s >= 0 && s <= 1 << 20;
      r.sections[i] = s;
      r.half += s;
    }
  } catch (...) {
    Py_DECREF(seq);
    throw;
  }
  Py_DECREF(seq);
  require(ok, VASR_PA_EINVAL_SHAPE, "sections must be 1 to 4 sizes");
  require(is_f32(cos) && is_f32(sin) && cos.dim() == 2 && cos.size(1) == r.half && sin.sizes() == cos.sizes(),
          VASR_PA_EINVAL_SHAPE, "cos/sin tables must be f32 [max_position, sum(sections)]");
  require(cos.is_contiguous() && sin.is_contiguous(), VASR_PA_EINVAL_SHAPE, "cos/sin tables must be contiguous");
  require(positions.scalar_type() == at::kLong && shape_is(positions, {n, tokens}), VASR_PA_EINVAL_SHAPE,
          "positions must be int64 [axes, T]");
  r.positions = positions.stride(1) == 1 || tokens <= 1 ? positions : positions.contiguous();
  r.axis_stride = r.positions.stride(0);
  return r;
}

PyObject *mrope(PyObject *const *a) {
  const at::Tensor &x = tensor(a[0], "x"), &cos = tensor(a[1], "cos_table"), &sin = tensor(a[2], "sin_table"),
                   &pos = tensor(a[3], "positions");
  const bool interleaved = truth(a[5]), inverse = truth(a[6]);
  const at::Tensor *given = maybe(a[7], "out");
  const c10::DeviceIndex dev = common_device({&x, &cos, &sin, &pos});
  const c10::cuda::CUDAGuard on_device(dev);
  require(x.dim() == 3 && x.stride(2) == 1, VASR_PA_EINVAL_SHAPE, "x must be [T, H, D] with unit dim stride");
  const int64_t t = x.size(0), h = x.size(1), d = x.size(2);
  const Rope r = rope_of(cos, sin, pos, a[4], t);
  const int code = dtype_code(x);
  if (given)
    require(given->sizes() == x.sizes() && given->scalar_type() == x.scalar_type() && on(*given, dev) && given->stride(2) == 1,
            VASR_PA_EINVAL_SHAPE, "out must have x's shape and dtype, with unit dim stride");
  const at::Tensor out = given ? *given : at::empty({t, h, d}, x.options());
  check(c_mrope(ptr(out), out.stride(0), out.stride(1), ptr(x), x.stride(0), x.stride(1), ptr<float>(cos), ptr<float>(sin),
                cos.size(0), ptr<int64_t>(r.positions), r.axis_stride, r.sections, r.axes, interleaved, inverse, t,
                (int32_t)h, (int32_t)d, code, stream_of(dev)),
        "mrope");
  return THPVariable_Wrap(out);
}

PyObject *mrope_append(PyObject *const *a) {
  const at::Tensor &qkv = tensor(a[0], "qkv");
  const at::Tensor *qw = maybe(a[1], "q_norm_weight"), *kw = maybe(a[2], "k_norm_weight");
  const double eps = real(a[3]);
  const at::Tensor &cos = tensor(a[4], "cos_table"), &sin = tensor(a[5], "sin_table"), &pos = tensor(a[6], "positions"),
                   &kc = tensor(a[8], "key_cache"), &vc = tensor(a[9], "value_cache"), &slots = tensor(a[10], "slot_mapping");
  const int32_t hq = whole32(a[11], "num_heads");
  const bool interleaved = truth(a[12]);
  const at::Tensor *ks = maybe(a[13], "k_scale"), *vs = maybe(a[14], "v_scale"), *scores = maybe(a[15], "score_cache"),
                   *given = maybe(a[16], "q_out");
  const c10::DeviceIndex dev = common_device({&qkv, &kc, &vc, &pos, &slots, &cos, &sin});
  const c10::cuda::CUDAGuard on_device(dev);
  const Cache c = cache_of(kc, vc);
  require(hq > 0 && qkv.dim() == 2 && qkv.stride(1) == 1 && qkv.size(1) == ((int64_t)hq + 2 * c.heads) * c.dim,
          VASR_PA_EINVAL_SHAPE, "qkv must be [T, (Hq + 2 Hkv) * D] with unit column stride");
  const int64_t t = qkv.size(0);
  const Rope r = rope_of(cos, sin, pos, a[7], t);
  require(slots.scalar_type() == at::kLong && shape_is(slots, {t}), VASR_PA_EINVAL_SHAPE, "slot_mapping must be int64 [T]");
  const at::Tensor slot_mapping = slots.contiguous();
  const int code = dtype_code(qkv);
  check_rows(c, qkv, kc, ks, vs, "qkv dtype must equal the cache dtype");
  require(!qw == !kw, VASR_PA_EINVAL_POINTER, "q and k norm weights go together");
  if (qw)
    for (const at::Tensor *w : {qw, kw})
      require(w->scalar_type() == qkv.scalar_type() && shape_is(*w, {c.dim}) && on(*w, dev) && w->is_contiguous(),
              VASR_PA_EINVAL_SHAPE, "norm weights must be [D] of qkv's dtype on its device");
  if (scores) check_scores(*scores, c, dev);
  if (given)
    require(shape_is(*given, {t, hq, c.dim}) && given->scalar_type() == qkv.scalar_type() && on(*given, dev) &&
                given->is_contiguous(),
            VASR_PA_EINVAL_SHAPE, "q_out must be a contiguous [T, Hq, D] of qkv's dtype");
  const at::Tensor q = given ? *given : at::empty({t, hq, c.dim}, qkv.options());
  check(c_mrope_append(ptr(q), ptr(qkv), t > 1 ? qkv.stride(0) : qkv.size(1), ptr(qw), ptr(kw), (float)eps, ptr<float>(cos),
                       ptr<float>(sin), cos.size(0), ptr<int64_t>(r.positions), r.axis_stride, r.sections, r.axes,
                       interleaved, ptr(kc), ptr(vc), ptr<float>(scores), ptr<int64_t>(slot_mapping), t, hq, c.heads, c.dim,
                       c.block, c.blocks, code, c.code, c.fp8 ? ptr<float>(ks) : nullptr, c.fp8 ? ptr<float>(vs) : nullptr,
                       stream_of(dev)),
        "fused_qk_norm_mrope_append");
  return THPVariable_Wrap(q);
}

// ---------------------------------------------------------------------- scored
void check_tables(const at::Tensor &tables, const at::Tensor &lens, int64_t b) {
  require(is_index32(tables) && tables.dim() == 2 && tables.size(0) == b, VASR_PA_EINVAL_SHAPE,
          "block_tables must be u32/i32 [B, cols]");
  require(is_index32(lens) && shape_is(lens, {b}), VASR_PA_EINVAL_SHAPE, "context_lens must be u32/i32 [B]");
}

PyObject *scored(PyObject *const *a) {
  const at::Tensor &q = tensor(a[0], "q");
  const at::Tensor *ks = maybe(a[1], "k_scale"), *vs = maybe(a[2], "v_scale");
  const at::Tensor &kc = tensor(a[3], "key_cache"), &vc = tensor(a[4], "value_cache"), &scores = tensor(a[5], "score_cache"),
                   &bt = tensor(a[6], "block_tables"), &cl = tensor(a[7], "context_lens");
  const int32_t longest = whole32(a[8], "max_context_len");
  const float scale = (float)real(a[9]), softcap = (float)real(a[10]), decay = (float)real(a[11]);
  const at::Tensor *given = maybe(a[13], "out");
  const c10::DeviceIndex dev = common_device({&q, &kc, &vc, &scores, &bt, &cl});
  const c10::cuda::CUDAGuard on_device(dev);
  const Cache c = cache_of(kc, vc);
  const int64_t dims = q.dim();
  require(dims == 3 || dims == 4, VASR_PA_EINVAL_SHAPE, "q must be [B, Hq, D] or [B, W, Hq, D] with packed heads");
  const int64_t b = q.size(0), window = dims == 4 ? q.size(1) : 1, hq = q.size(dims - 2);
  require(q.size(dims - 1) == c.dim && q.stride(dims - 1) == 1 && (q.stride(dims - 2) == c.dim || hq == 1),
          VASR_PA_EINVAL_SHAPE, "q must be [B, Hq, D] or [B, W, Hq, D] with packed heads");
  int64_t q_stride = dims == 4 && window > 1 ? q.stride(1) : q.stride(0);
  require(dims == 3 || b <= 1 || window <= 1 || q.stride(0) == window * q_stride, VASR_PA_EINVAL_SHAPE,
          "q's rows must follow one another at one token stride");
  if (b * window == 1) q_stride = hq * c.dim;
  const int code = dtype_code(q);
  check_rows(c, q, kc, ks, vs, "q dtype must equal the cache dtype");
  check_scores(scores, c, dev);
  check_tables(bt, cl, b);
  const int32_t rows = a[12] == Py_None ? (int32_t)window : whole32(a[12], "score_rows");
  const at::Tensor tables = bt.contiguous(), lens = cl.contiguous();
  if (given)
    require(given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type() && on(*given, dev) && given->is_contiguous(),
            VASR_PA_EINVAL_SHAPE, "out must be contiguous with q's shape and dtype");
  const at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
  const vasr_pa_stream_t stream = stream_of(dev);
  const size_t need = c_scored_size((int32_t)b, (int32_t)window, rows, (int32_t)hq, c.heads, c.dim, c.block, longest);
  const at::Tensor ws = scored_workspaces().scratch(dev, stream, need);
  check(c_scored(ptr(out), ptr(q), ptr(kc), ptr(vc), ptr<float>(scores), ptr<uint32_t>(tables), ptr<uint32_t>(lens),
                 (int32_t)b, (int32_t)window, rows, (int32_t)hq, c.heads, c.dim, c.block, c.blocks, (int32_t)tables.size(1),
                 longest, scale, softcap, decay, q_stride, code, c.code, c.fp8 ? ptr<float>(ks) : nullptr,
                 c.fp8 ? ptr<float>(vs) : nullptr, ptr(ws), (size_t)ws.numel(), stream),
        "paged_attention_scored");
  return THPVariable_Wrap(out);
}

PyObject *pair_of(const at::Tensor &x, const at::Tensor &y) {
  PyObject *t = PyTuple_New(2);
  if (!t) throw PyFailed{};
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(x));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(y));
  return t;
}

// ------------------------------------------------------------------------ evict
PyObject *evict(PyObject *const *a) {
  const at::Tensor &kc = tensor(a[0], "key_cache"), &vc = tensor(a[1], "value_cache"), &scores = tensor(a[2], "score_cache"),
                   &bt = tensor(a[3], "block_tables"), &cl = tensor(a[4], "context_lens");
  const int32_t longest = whole32(a[5], "max_context_len"), budget = whole32(a[6], "budget"),
                sink = whole32(a[7], "num_sink"), recent = whole32(a[8], "num_recent");
  const at::Tensor *lim = maybe(a[9], "budgets"), *to = maybe(a[10], "out_block_tables");
  const c10::DeviceIndex dev = common_device({&kc, &vc, &scores, &bt, &cl});
  const c10::cuda::CUDAGuard on_device(dev);
  const Cache c = cache_of(kc, vc);
  check_scores(scores, c, dev);
  require(bt.dim() == 2, VASR_PA_EINVAL_SHAPE, "block_tables must be u32/i32 [B, cols]");
  const int64_t b = bt.size(0);
  check_tables(bt, cl, b);
  const at::Tensor tables = bt.contiguous(), lens = cl.contiguous();
  at::Tensor out_tables, limits;
  if (to) {
    require(is_index32(*to) && to->dim() == 2 && to->size(0) == b && on(*to, dev), VASR_PA_EINVAL_SHAPE,
            "out_block_tables must be u32/i32 [B, cols] on the cache device");
    out_tables = to->contiguous();
  }
  if (lim) {
    require(is_index32(*lim) && shape_is(*lim, {b}) && on(*lim, dev), VASR_PA_EINVAL_SHAPE,
            "budgets must be u32/i32 [B] on the cache device");
    limits = lim->contiguous();
  }
  const auto i32 = at::TensorOptions().dtype(at::kInt).device(bt.device());
  const at::Tensor kept = at::empty({b, c.heads, budget > 0 ? budget : 0}, i32), new_lens = at::empty({b}, i32);
  check(c_evict(ptr(kc), ptr(vc), ptr<float>(scores), ptr<uint32_t>(tables), (int32_t)tables.size(1),
                to ? ptr<uint32_t>(out_tables) : nullptr, to ? (int32_t)out_tables.size(1) : 0, ptr<uint32_t>(lens), longest,
                lim ? ptr<uint32_t>(limits) : nullptr, budget, sink, recent, ptr<int32_t>(kept), ptr<uint32_t>(new_lens),
                (int32_t)b, c.heads, c.dim, c.block, c.blocks, c.code, stream_of(dev)),
        "evict_kv");
  return pair_of(kept, new_lens);
}

// ----------------------------------------------------------------------- verify
PyObject *verify(PyObject *const *a) {
  const at::Tensor &logits = tensor(a[0], "target_logits"), &dt = tensor(a[1], "draft_tokens");
  const at::Tensor *probs = maybe(a[2], "draft_probs"), *uni = maybe(a[3], "uniform"), *race = maybe(a[4], "race"),
                   *len = maybe(a[6], "draft_lens");
  const c10::DeviceIndex dev = common_device({&logits, &dt});
  const c10::cuda::CUDAGuard on_device(dev);
  require(logits.dim() == 3 && logits.stride(2) == 1 && logits.size(1) >= 1, VASR_PA_EINVAL_SHAPE,
          "target_logits must be [B, K + 1, V] with unit column stride");
  const int64_t b = logits.size(0), k = logits.size(1) - 1, v = logits.size(2);
  const int code = dtype_code(logits);
  require(dt.scalar_type() == at::kInt && shape_is(dt, {b, k}), VASR_PA_EINVAL_SHAPE, "draft_tokens must be int32 [B, K]");
  if (probs)
    require(shape_is(*probs, {b, k, v}) && probs->stride(2) == 1 && on(*probs, dev), VASR_PA_EINVAL_SHAPE,
            "draft_probs must be [B, K, V] with unit column stride");
  if (uni)
    require(is_f32(*uni) && shape_is(*uni, {b, k}) && on(*uni, dev), VASR_PA_EINVAL_SHAPE, "uniform must be f32 [B, K]");
  if (race)
    require(is_f32(*race) && shape_is(*race, {b, v}) && on(*race, dev) && race->stride(1) == 1, VASR_PA_EINVAL_SHAPE,
            "race must be f32 [B, V] with unit column stride");
  if (len)
    require(len->scalar_type() == at::kInt && shape_is(*len, {b}) && on(*len, dev), VASR_PA_EINVAL_SHAPE,
            "draft_lens must be int32 [B]");
  at::Tensor temps;
  float temperature = 1.f;
  if (THPVariable_Check(a[5])) {
    const at::Tensor &t = THPVariable_Unpack(a[5]);
    require(is_f32(t) && shape_is(t, {b}) && on(t, dev), VASR_PA_EINVAL_SHAPE, "temperature must be a number or f32 [B]");
    temps = t.contiguous();
  } else {
    temperature = (float)real(a[5]);
  }
  const at::Tensor drafts = dt.contiguous();
  const at::Tensor uniform = uni ? uni->contiguous() : at::Tensor(), lens = len ? len->contiguous() : at::Tensor();
  const at::Tensor tokens = at::empty({b, k + 1}, dt.options()), accepted = at::empty({b}, dt.options());
  const vasr_pa_stream_t stream = stream_of(dev);
  const at::Tensor ws = verify_workspaces().scratch(dev, stream, c_verify_size((int32_t)b, (int32_t)k, v));
  check(c_verify(ptr<int32_t>(tokens), ptr<int32_t>(accepted), ptr(logits), logits.stride(0), logits.stride(1), code,
                 ptr<int32_t>(drafts), len ? ptr<int32_t>(lens) : nullptr, ptr(probs), probs ? probs->stride(0) : 0,
                 probs ? probs->stride(1) : 0, probs ? dtype_code(*probs) : 0, uni ? ptr<float>(uniform) : nullptr,
                 ptr<float>(race), race ? race->stride(0) : 0, temps.defined() ? ptr<float>(temps) : nullptr, temperature,
                 (int32_t)b, (int32_t)k, v, ptr(ws), (size_t)ws.numel(), stream),
        "verify_draft_tokens");
  return pair_of(tokens, accepted);
}

// ------------------------------------------------------------------- workspaces
// reserve(kind, device index, stream handle, bytes) -> the stream's workspace
PyObject *reserve(PyObject *const *a) {
  const int64_t kind = whole(a[0]);
  Workspaces &w = kind == 0 ? scored_workspaces() : verify_workspaces();
  return THPVariable_Wrap(w.reserve((c10::DeviceIndex)whole(a[1]), (uintptr_t)whole(a[2]), (size_t)whole(a[3])));
}

// bind(error class, address of each C function in the order below)
PyObject *bind(PyObject *const *a) {
  Py_INCREF(a[0]);
  Py_XSETREF(error_class, a[0]);
  auto at = [&](int i) { return reinterpret_cast<void *>((uintptr_t)whole(a[i])); };
  c_mrope = reinterpret_cast<decltype(c_mrope)>(at(1));
  c_mrope_append = reinterpret_cast<decltype(c_mrope_append)>(at(2));
  c_scored = reinterpret_cast<decltype(c_scored)>(at(3));
  c_scored_size = reinterpret_cast<decltype(c_scored_size)>(at(4));
  c_evict = reinterpret_cast<decltype(c_evict)>(at(5));
  c_verify = reinterpret_cast<decltype(c_verify)>(at(6));
  c_verify_size = reinterpret_cast<decltype(c_verify_size)>(at(7));
  Py_RETURN_NONE;
}

// Positional arguments only, as many as the function takes; refusals become
// VasrPaError, torch's own errors (out of memory) what torch makes of them.
template <PyObject *(*kCall)(PyObject *const *), int kArgs>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
    return nullptr;
  }
  if (!error_class && kCall != bind) {
    PyErr_SetString(PyExc_RuntimeError, "_vasr_calls is not bound to the kernel library");
    return nullptr;
  }
  try {
    return kCall(args);
  } catch (const PyFailed &) {
    return nullptr;
  } catch (const Refused &r) {
    PyObject *e = PyObject_CallFunction(error_class, "is", r.status, r.what.c_str());
    if (e) {
      PyErr_SetObject(error_class, e);
      Py_DECREF(e);
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define ENTRY(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(bind, 8),   ENTRY(reserve, 4), ENTRY(mrope, 8), ENTRY(mrope_append, 17), ENTRY(scored, 14),
                         ENTRY(evict, 11), ENTRY(verify, 7),  {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_vasr_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__vasr_calls() { return PyModule_Create(&module); }
