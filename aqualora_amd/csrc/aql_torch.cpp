// Autograd binding of the training operators (LayerNorm with weight gradients, 8-bit checkpoints, adapters of many requests): argument checks,
// output allocation, the calls of the C ABI, and the backward nodes, in C++.
//
// Why not Python like the other wrappers: these operators are short (8-30 us each way at a few thousand rows), and a Python backward node costs
// more than that on the host -- it runs on the engine's device thread, where it has to take the interpreter lock for every line.  Measured for a
// LayerNorm forward + backward of 64 x 320: 155 us of host time with Python nodes (17 us forward alone).
// No kernel is here: everything below ends in an aql_* entry point of libaqualora_hip.so.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <condition_variable>
#include <cstdlib>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/aqualora_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct AqlErr : std::runtime_error {   // becomes aqualora_amd._lib.AqlError in Python
  using std::runtime_error::runtime_error;
};
py::handle aql_error_class;

bool debug_sync() {
  static const bool on = [] { const char* e = std::getenv("AQL_DEBUG_SYNC"); return e && *e; }();
  return on;
}
void ran(int rc, const char* name, aql_stream_t st) {
  if (rc) throw AqlErr(std::string(name) + " failed with status " + std::to_string(rc) + ": " + aql_last_error());
  if (debug_sync()) {   // the debugging aid of _lib.call: name the entry point that faulted
    std::fprintf(stderr, "[aql] %s\n", name);
    std::fflush(stderr);
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)st, &cs) == hipSuccess && cs == hipStreamCaptureStatusNone) (void)hipDeviceSynchronize();
  }
}
[[noreturn]] void bad_value(const std::string& s) { throw py::value_error(s); }
std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// the kernels run on the current device's current stream: a tensor of another device is refused, not followed
void here(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw AqlErr(std::string(name) + ": the HIP path needs a GPU tensor; there is no CPU fallback");
  if (t.get_device() != c10::hip::current_device())
    throw AqlErr(std::string(name) + ": tensor on device " + std::to_string(t.get_device()) + ", but the current device is " +
                 std::to_string(c10::hip::current_device()) + "; wrap the call in torch.cuda.device(...)");
}
aql_stream_t stream_of(const Tensor& t) { return (aql_stream_t)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void hip_ok(hipError_t e, const char* what) {
  if (e != hipSuccess) throw AqlErr(std::string(what) + ": " + hipGetErrorString(e));
}
bool capturing(const c10::hip::HIPStream& s) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(s.stream(), &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
}
// of the capture that a stream is in, never used again; 0: none
unsigned long long capture_id(const c10::hip::HIPStream& s) {
  if (!capturing(s)) return 0;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  hip_ok(hipStreamGetCaptureInfo(s.stream(), &cs, &id), "hipStreamGetCaptureInfo");
  return cs == hipStreamCaptureStatusActive ? id : 0;
}

// at::empty without the dispatcher's way to it: a backward pass allocates up to seven tensors
Tensor fresh(at::IntArrayRef size, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(size, type, like.device(), std::nullopt); }
// two fp32 tensors in one allocation (a pair of gradients: they live and end together); an unwanted one stays undefined
std::pair<Tensor, Tensor> fresh_pair(bool one, at::IntArrayRef a, bool two, at::IntArrayRef b, const Tensor& like) {
  if (!one || !two) return {one ? fresh(a, at::kFloat, like) : Tensor(), two ? fresh(b, at::kFloat, like) : Tensor()};
  const int64_t na = (c10::multiply_integers(a) + 3) / 4 * 4;   // (both 16-byte aligned)
  const Tensor buf = fresh({na + c10::multiply_integers(b)}, at::kFloat, like);
  const auto view = [&](at::IntArrayRef size, int64_t offset) {
    Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
    return t;
  };
  return {view(a, 0), view(b, na)};
}
// workspace of one call, returned to the caching allocator behind it on the same stream
c10::DataPtr workspace(long floats) { return c10::hip::HIPCachingAllocator::get()->allocate(floats * 4); }

int dt(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : 1; }
bool bf16_or_f32(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
template <class T = void>
T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }

struct Rows {
  Tensor t;
  long ld = 0;
};
// rows with unit column stride that do not overlap
Rows rows2d(const Tensor& t) {
  const long M = t.size(0), C = t.size(1);
  if (M <= 1) return {t.is_contiguous() ? t : t.contiguous(), C};
  if (t.stride(1) != 1 || t.stride(0) < C) return {t.contiguous(), C};
  return {t, t.stride(0)};
}
// rows as the matrix kernels read them: 16-byte aligned, a multiple of 8 elements apart
Rows gemm_rows(const Tensor& t) {
  Rows r = rows2d(t);
  if (r.ld % 8 || r.ld >= (1L << 21) || ((uintptr_t)r.t.data_ptr() & 15)) r = {r.t.clone(at::MemoryFormat::Contiguous), t.size(1)};
  return r;
}

// memory that kernels on stream s use: freed earlier, it is given out again behind them (nothing to do on the stream that it was allocated on)
void used_on(const Tensor& t, const c10::hip::HIPStream& s) {
  if (t.defined()) c10::hip::HIPCachingAllocator::recordStream(t.storage().data_ptr(), s);
}

Tensor leaf(const Tensor& t) { return t.defined() && t.is_leaf() && t.requires_grad() ? t : Tensor(); }

// A leaf's accumulation node runs on the stream on which it was made.  A captured backward pass that reaches one made on another stream (an eager graph of
// the same leaf still lives) would draw that stream into the capture, which ends the process: refused instead.
void leaves_ok(const std::vector<Tensor>& leaves, const Tensor& g, const char* name) {
  const auto here = c10::hip::getCurrentHIPStream(g.get_device());
  if (!capturing(here)) return;
  for (const Tensor& t : leaves) {
    if (!t.defined()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (node && node->stream() && node->stream()->id() != here.id())   // (of one device: here() has seen to that)
      throw AqlErr(std::string(name) + ": this backward pass is being captured, but a graph of the same parameters that was made on another stream still lives; drop it "
                   "(its outputs and losses) before the capture");
  }
}

// A saved tensor as it was saved, whatever hooks of saved tensors made of it meanwhile (moved to the host and back, other strides): the kernels go by its address.
// `rows`: with its row stride, else contiguous
Tensor intact(const Tensor& t, at::IntArrayRef size, at::ScalarType type, const Tensor& like, const char* name, bool rows = false) {
  if (!t.defined()) return t;
  if (t.device() != like.device() || t.scalar_type() != type || t.sizes() != size || t.layout() != at::kStrided)
    throw AqlErr(std::string(name) + ": a tensor saved for the backward pass came back as " + c10::toString(t.scalar_type()) + " " + shape_of(t) + " on " + t.device().str());
  return rows ? t : t.contiguous();
}

// gradients of a backward pass under create_graph: they carry a node that refuses a second backward pass
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  at::AutoGradMode off(false);
  variable_list in;
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
  if (in.empty()) return grads;
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative", (int64_t)in.size());
  auto out = (*err)(std::move(in));
  size_t k = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// ------------------------------------------------------------------------------------------------------------------ 8-bit checkpoint
constexpr long ACT8_COLUMNS = 1 << 24;   // the C entries' limit, checked ahead of their int
std::pair<Tensor, Tensor> act8_alloc(long M, long C, const Tensor& like) {
  const long Cp = (C + 31) / 32 * 32;
  return {fresh({M, Cp}, at::kByte, like), fresh({M, Cp / 32}, at::kByte, like)};
}

std::pair<Tensor, Tensor> act8_pack(const Tensor& x) {
  if (!bf16_or_f32(x)) bad_value(std::string("act8_pack: bfloat16 or float32, not ") + c10::toString(x.scalar_type()));
  if (x.dim() < 1 || x.size(-1) == 0) bad_value("act8_pack: expected [..., columns], got " + shape_of(x));
  if (x.size(-1) > ACT8_COLUMNS) bad_value("act8_pack: at most " + std::to_string(ACT8_COLUMNS) + " columns, got " + shape_of(x));
  here(x, "act8_pack");
  at::AutoGradMode off(false);
  const long C = x.size(-1);
  const Rows r = rows2d(x.numel() ? x.reshape({-1, C}) : x.reshape({0, C}));
  auto [codes, exps] = act8_alloc(r.t.size(0), C, x);
  const auto st = stream_of(x);
  ran(aql_act8_pack(r.t.data_ptr(), dt(x), r.t.size(0), (int)C, r.ld, ptr<uint8_t>(codes), ptr<uint8_t>(exps), st), "aql_act8_pack", st);
  return {codes, exps};
}

Tensor act8_unpack(const Tensor& codes, const Tensor& exps, std::vector<int64_t> shape, bool bf16) {
  const long C = shape.empty() ? 0 : shape.back(), Cp = (C + 31) / 32 * 32;
  int64_t M = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) M *= shape[i];
  const auto fits = [&](const Tensor& t, long w) { return t.scalar_type() == at::kByte && t.dim() == 2 && t.size(0) == M && t.size(1) == w && t.is_contiguous(); };
  if (C < 1 || !fits(codes, Cp) || !fits(exps, Cp / 32) || codes.device() != exps.device())
    bad_value("Act8.unpack: codes uint8 [" + std::to_string(M) + ", " + std::to_string(Cp) + "] and exps uint8 [" + std::to_string(M) + ", " +
              std::to_string(Cp / 32) + "], contiguous on one device, not " + shape_of(codes) + " and " + shape_of(exps));
  if (C > ACT8_COLUMNS) bad_value("Act8.unpack: at most " + std::to_string(ACT8_COLUMNS) + " columns, not " + std::to_string(C));
  here(codes, "Act8.unpack");
  Tensor out = fresh(shape, bf16 ? at::kBFloat16 : at::kFloat, codes);
  const auto st = stream_of(codes);
  ran(aql_act8_unpack(ptr<uint8_t>(codes), ptr<uint8_t>(exps), codes.size(0), (int)C, out.data_ptr(), bf16 ? 0 : 1, C, st), "aql_act8_unpack", st);
  return out;
}

// -------------------------------------------------------------------------------------------------------- LayerNorm with weight gradients
struct NormCall : torch::CustomClassHolder {   // what its backward pass needs besides tensors of the graph
  std::vector<Tensor> leaves;
  bool beta = false;
  long M = 0, C = 0;
  at::ScalarType weights = at::kFloat;
};

struct LayerNormTrain : torch::autograd::Function<LayerNormTrain> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gamma, const std::optional<Tensor>& beta_, double eps, bool ckpt8, bool passthrough) {
    const Tensor beta = beta_ ? *beta_ : Tensor();
    const long M = x.size(0), C = x.size(1);
    const Rows r = rows2d(x);
    Tensor y = fresh({M, C}, x.scalar_type(), x), stats = fresh({M, 2}, at::kFloat, x), codes, exps;
    if (ckpt8) std::tie(codes, exps) = act8_alloc(M, C, x);
    const auto st = stream_of(x);
    ran(aql_layernorm_train_fwd(r.t.data_ptr(), dt(x), M, (int)C, r.ld, gamma.data_ptr(), ptr(beta), dt(gamma), (float)eps, y.data_ptr(), C,
                                ptr<float>(stats), ptr<uint8_t>(codes), ptr<uint8_t>(exps), st), "aql_layernorm_train_fwd", st);
    ctx->save_for_backward({ckpt8 ? Tensor() : r.t, codes, exps, gamma, stats});
    auto c = c10::make_intrusive<NormCall>();
    c->beta = beta.defined(), c->M = M, c->C = C, c->weights = gamma.scalar_type();
    c->leaves = {leaf(x), leaf(gamma), leaf(beta)};
    ctx->set_materialize_grads(false);   // an output that nothing used has no gradient, not one of zeros
    ctx->saved_data["call"] = c10::IValue::make_capsule(std::move(c));
    if (passthrough) return {y, x.view_as(x)};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const auto c = c10::static_intrusive_pointer_cast<NormCall>(ctx->saved_data["call"].toCapsule());
    const long M = c->M, C = c->C;
    const bool want_g = ctx->needs_input_grad(1), want_b = c->beta && ctx->needs_input_grad(2);
    if (!g[0].defined()) {   // only the pass-through output was used: its gradient as it is, and the weights have no part in it
      at::AutoGradMode off(false);
      if (!g.back().defined()) return variable_list(6);
      const auto zeros = [&](bool want) { return want ? at::zeros({C}, g.back().options().dtype(c->weights)) : Tensor(); };
      return {g.size() > 1 ? g[1] : Tensor(), zeros(want_g), zeros(want_b), Tensor(), Tensor(), Tensor()};
    }
    here(g[0], "layernorm_train backward");
    leaves_ok(c->leaves, g[0], "layernorm_train");
    Tensor dx, dg, db;
    {
      at::AutoGradMode off(false);
      dx = fresh({M, C}, g[0].scalar_type(), g[0]);
      if (M == 0) {
        const auto f32 = g[0].options().dtype(at::kFloat);
        if (want_g) dg = at::zeros({C}, f32);
        if (want_b) db = at::zeros({C}, f32);
      } else {
        const char* name = "layernorm_train";
        Rows x;
        if (s[0].defined()) x = rows2d(intact(s[0], {M, C}, dx.scalar_type(), dx, name, true));
        const long nb = (C + 31) / 32;
        const Tensor codes = intact(s[1], {M, nb * 32}, at::kByte, dx, name), exps = intact(s[2], {M, nb}, at::kByte, dx, name);
        const Tensor gamma = intact(s[3], {C}, c->weights, dx, name), stats = intact(s[4], {M, 2}, at::kFloat, dx, name);
        const Rows dy = rows2d(g[0]);
        Rows dres;
        if (g.size() > 1 && g[1].defined()) dres = rows2d(g[1]);
        std::tie(dg, db) = fresh_pair(want_g, {C}, want_b, {C}, dx);
        const long n = aql_layernorm_train_scratch_floats(M, (int)C);
        const c10::DataPtr scratch = workspace(n);
        const auto st = stream_of(dx);
        ran(aql_layernorm_train_bwd(ptr(x.t), ptr<uint8_t>(codes), ptr<uint8_t>(exps), dy.t.data_ptr(), ptr(dres.t), dt(dx), M, (int)C,
                                    x.t.defined() ? x.ld : C, dy.ld, dres.ld, gamma.data_ptr(), dt(gamma), ptr<float>(stats), dx.data_ptr(), C,
                                    ptr<float>(dg), ptr<float>(db), (float*)scratch.get(), n, st), "aql_layernorm_train_bwd", st);
      }
      if (c->weights != at::kFloat) {
        if (dg.defined()) dg = dg.to(c->weights);
        if (db.defined()) db = db.to(c->weights);
      }
    }
    return once({dx, dg, db, Tensor(), Tensor(), Tensor()}, "layernorm_train");
  }
};

py::object layernorm_train(const Tensor& x, const Tensor& gamma, const std::optional<Tensor>& beta_, double eps, bool ckpt8, bool passthrough) {
  if (x.dim() != 2) bad_value("layernorm_train: expected [rows, columns], got " + shape_of(x));
  if (!bf16_or_f32(x)) bad_value(std::string("layernorm_train: bfloat16 or float32 rows, not ") + c10::toString(x.scalar_type()));
  const long C = x.size(1);
  const Tensor beta = beta_ ? *beta_ : Tensor();
  for (const Tensor* p : {&gamma, &beta}) {
    if (!p->defined()) continue;
    if (p->dim() != 1 || p->size(0) != C || !bf16_or_f32(*p) || p->device() != x.device() || (C > 1 && p->stride(0) != 1))
      bad_value("layernorm_train: gamma and beta must be contiguous bfloat16 / float32 [" + std::to_string(C) + "] on " + x.device().str());
    if (p->scalar_type() != gamma.scalar_type()) bad_value("layernorm_train: gamma and beta must have the same type");
  }
  if (C < 1 || C > 8192) bad_value("layernorm_train: 1 to 8192 columns, not " + std::to_string(C));
  here(x, "layernorm_train");
  variable_list out = LayerNormTrain::apply(x, gamma, beta_, eps, ckpt8, passthrough);
  if (passthrough) return py::make_tuple(out[0], out[1]);
  return py::cast(out[0]);
}

// ------------------------------------------------------------------------------------------------------- adapters of many requests
struct Bank {   // the device side of adapters.AdapterBank
  Tensor a, b, at, bt, ranks, scales;
  Tensor down, up;              // what a .. bt are laid out from, and its versions then
  int64_t down_seen = -1, up_seen = -1;
  long G = 0, r = 0, R = 0, K = 0, N = 0;
  bool trainable = false;

  // whether the stacks that a call on the current stream will read are those of the parameters
  bool fresh() const {
    const bool recorded = laid_in && capture_id(current()) == laid_in;   // a layout that the graph being captured holds goes before those outside
    return (int64_t)down._version() == (recorded ? down_rec : down_seen) && (int64_t)up._version() == (recorded ? up_rec : up_seen);
  }

  // The stacks are written in place, by whichever call comes first after a change, and read by all, from any thread and stream.
  //   Threads: `busy` calls are queueing kernels that read the stacks; a layout begins by raising `serial` and making the stacks stale, so that no further call enters,
  //   and then waits for the ones inside.  (A backward pass enters by the serial of its forward pass; the versions are noted ahead of the copies.)
  //   Streams: the first read on a stream behind a layout waits for its event, and a layout waits for every stream that has read since the last one.
  // (What runs inside a graph is ordered by whoever replays it.)
  //   Captures: a layout in a capture changes nothing before a replay.  Only calls in that same capture go by it.
  std::mutex guard;
  std::condition_variable quiet;
  int busy = 0;
  long serial = 0;
  static thread_local const Bank* inside;     // the bank that this thread is queueing reads of
  int64_t down_next = -1, up_next = -1;       // versions that the layout in progress will have seen
  unsigned long long laid_in = 0;             // the capture that holds the last recorded layout, and the versions that it has seen
  int64_t down_rec = -1, up_rec = -1;
  std::optional<c10::hip::HIPStream> home;    // stream of the last layout
  std::vector<c10::hip::HIPStream> readers;   // streams that have read since then
  hipEvent_t laid = nullptr, mark = nullptr;  // behind the last layout; for one wait at a time

  Bank() = default;
  Bank(const Bank&) = delete;
  ~Bank() {
    for (hipEvent_t e : {laid, mark})
      if (e) (void)hipEventDestroy(e);
  }
  c10::hip::HIPStream current() const { return c10::hip::getCurrentHIPStream(a.get_device()); }
  void used_by(const c10::hip::HIPStream& s) const {
    for (const Tensor* t : {&a, &b, &at, &bt, &ranks, &scales}) used_on(*t, s);
  }
  // ahead of kernels on the current stream that read the stacks (guard held)
  void read_on(const c10::hip::HIPStream& s) {
    if (std::find(readers.begin(), readers.end(), s) != readers.end() || capturing(s)) return;
    if (home && *home != s) hip_ok(hipStreamWaitEvent(s.stream(), laid, 0), "AdapterBank");
    used_by(s);
    readers.push_back(s);
  }
  // the transposed stacks, complete
  void publish(const Tensor& at_, const Tensor& bt_) {
    const std::lock_guard<std::mutex> lock(guard);
    at = at_, bt = bt_;
    for (const auto& r : readers) used_by(r);
  }
  void reads() {
    const std::lock_guard<std::mutex> lock(guard);
    read_on(current());
  }
  // around the copies of a layout on the current stream; one at a time (adapters.AdapterBank sees to that)
  void begin_layout() {
    const auto s = current();
    if (inside == this) throw AqlErr("AdapterBank: changed weights cannot be laid out from inside a call that uses the bank (a hook of its saved tensors)");
    std::unique_lock<std::mutex> lock(guard);
    down_next = down._version(), up_next = up._version();
    ++serial;
    if (capturing(s)) return;
    down_seen = up_seen = -1;
    used_by(s);
    quiet.wait(lock, [&] { return busy == 0; });
    const c10::DeviceGuard device(a.device());
    for (hipEvent_t* e : {&laid, &mark})
      if (!*e) hip_ok(hipEventCreateWithFlags(e, hipEventDisableTiming), "AdapterBank");
    if (home && *home != s) hip_ok(hipStreamWaitEvent(s.stream(), laid, 0), "AdapterBank");
    for (const auto& r : readers) {
      if (r == s) continue;
      if (capturing(r)) throw AqlErr("AdapterBank: changed weights cannot be laid out while a stream that has read the old ones is being captured");
      hip_ok(hipEventRecord(mark, r.stream()), "AdapterBank");
      hip_ok(hipStreamWaitEvent(s.stream(), mark, 0), "AdapterBank");
    }
    if (std::find(readers.begin(), readers.end(), s) == readers.end()) readers.push_back(s);   // (for the next layout, if this one ends half way: out of memory)
  }
  void end_layout() {
    const auto s = current();
    const std::lock_guard<std::mutex> lock(guard);
    if ((laid_in = capture_id(s))) {
      down_rec = down_next, up_rec = up_next;
      return;
    }
    hip_ok(hipEventRecord(laid, s.stream()), "AdapterBank");
    home = s;
    readers.clear();
    down_seen = down_next, up_seen = up_next;
  }
};

thread_local const Bank* Bank::inside = nullptr;

// a call that queues kernels which read the stacks on the current stream; `in` is false where they are not what the call needs
struct Reading {
  Bank& bank;
  bool in;
  long serial;
  const Bank* outer = Bank::inside;
  explicit Reading(Bank& b, long want = -1) : bank(b) {   // want: the serial that the stacks must have (-1: that of the parameters' versions)
    const std::lock_guard<std::mutex> lock(b.guard);
    in = want < 0 ? b.fresh() : b.serial == want;
    serial = b.serial;
    if (!in) return;
    b.read_on(b.current());
    ++b.busy;
    Bank::inside = &b;
  }
  Reading(const Reading&) = delete;
  ~Reading() {
    if (!in) return;
    Bank::inside = outer;
    const std::lock_guard<std::mutex> lock(bank.guard);
    if (--bank.busy == 0) bank.quiet.notify_all();
  }
};

struct Plan {   // the device side of adapters.RequestPlan
  Tensor table;
  std::vector<long> start;   // host copy, in units
  long units = 0, requests = 0, live_units = 0, unit_rows = 1;   // unit_rows: rows per unit where the requests have given lengths
  int nseg = 0, nused = 0, nslot = 0, max_id = -1;
  bool equal = false;
  std::vector<long> at;      // offsets of unit_id, perm, used_pos, slot in the table
  std::unordered_map<long, int> slots_by_unit;
  std::vector<c10::hip::HIPStream> readers;
  std::mutex guard;          // of these two: backward passes ask from the engine's threads

  const int* part(int k) const { return (const int*)table.data_ptr() + at[k]; }
  long unit(long rows) const {   // rows per table unit for a call on `rows` rows
    if (!equal) {
      if (rows != units * unit_rows) bad_value("RequestPlan: the requests have " + std::to_string(units * unit_rows) + " rows, the call " + std::to_string(rows));
      return unit_rows;
    }
    if (requests == 0) {
      if (rows) bad_value("RequestPlan: no requests for " + std::to_string(rows) + " rows");
      return 1;
    }
    if (rows % requests) bad_value("RequestPlan: " + std::to_string(rows) + " rows do not divide among " + std::to_string(requests) + " equal requests");
    return std::max(1L, rows / requests);
  }
  void reads() {   // ahead of kernels on the current stream that read the table
    const auto s = c10::hip::getCurrentHIPStream(table.get_device());
    const std::lock_guard<std::mutex> lock(guard);
    if (std::find(readers.begin(), readers.end(), s) != readers.end() || capturing(s)) return;
    used_on(table, s);
    readers.push_back(s);
  }
  int slots(long unit) {   // the most segments, and so adapters, that meet in 16 rows [16 i, 16 i + 16)
    const std::lock_guard<std::mutex> lock(guard);
    auto it = slots_by_unit.find(unit);
    if (it != slots_by_unit.end()) return it->second;
    int most = 0, count = 0;
    long tile = -1;
    for (size_t k = 1; k + 1 < start.size(); ++k) {
      const long row = start[k] * unit;
      if (row % 16 == 0) continue;
      count = row / 16 == tile ? count + 1 : 1;
      tile = row / 16;
      most = std::max(most, count);
    }
    return slots_by_unit[unit] = 1 + most;
  }
};

struct Call : torch::CustomClassHolder {   // what a backward pass of adapter_linear needs besides tensors
  std::shared_ptr<Bank> bank;
  std::shared_ptr<Plan> plan;
  Tensor w, wt, bias;
  std::vector<Tensor> leaves;
  long unit = 1, serial = 0, M = 0, N = 0, K = 0;
  bool train = false, residual = false;
};

// one pass of aql_adapter_linear -> (y [M, N], T [M, parts, R] or undefined)
std::pair<Tensor, Tensor> product(const Rows& x, const Tensor& w, const Tensor& bias, const Rows& res, const Tensor& a, const Tensor& b, const Bank& bank,
                                  Plan& plan, long unit, long N, long K, int parts) {
  const long M = x.t.size(0);
  Tensor y = fresh({M, N}, at::kBFloat16, x.t), T;
  if (plan.nseg) T = fresh({M, parts, bank.R}, at::kBFloat16, y);
  const auto st = stream_of(y);
  ran(aql_adapter_linear(ptr<bf16_t>(x.t), x.ld, ptr<bf16_t>(w), K, ptr<bf16_t>(bias), ptr<bf16_t>(res.t), res.ld, ptr<bf16_t>(y), N, M, (int)N, (int)K,
                         ptr<bf16_t>(a), ptr<bf16_t>(b), ptr<int>(bank.ranks), ptr<float>(bank.scales), (int)bank.R, plan.part(0), (int)unit, plan.nseg,
                         plan.slots(unit), plan.nused, ptr<bf16_t>(T), parts, st), "aql_adapter_linear", st);
  return {y, T};
}

Tensor down(const Rows& x, const Tensor& codes, const Tensor& exps, long M, long K, const Tensor& a, const Bank& bank, Plan& plan, long unit) {
  Tensor T = fresh({M, 3, bank.R}, at::kBFloat16, a);
  const auto st = stream_of(T);
  ran(aql_adapter_down(ptr<bf16_t>(x.t), x.ld, ptr<uint8_t>(codes), ptr<uint8_t>(exps), M, (int)K, ptr<bf16_t>(a), ptr<int>(bank.ranks), ptr<float>(bank.scales),
                       (int)bank.R, plan.part(0), (int)unit, plan.nseg, plan.slots(unit), ptr<bf16_t>(T), 3, st), "aql_adapter_down", st);
  return T;
}

// fp32 gradients of the stacks: dA [G, r, K] where want_a, dB [G, N, r] where want_b
void wgrad(const Tensor& dT, const Rows& x, const Tensor& codes, const Tensor& exps, bool want_a, const Tensor& T, const Rows& dy, bool want_b, long M,
           const Bank& bank, const Plan& plan, long unit, Tensor& dA, Tensor& dB) {
  std::tie(dA, dB) = fresh_pair(want_a, {bank.G, bank.r, bank.K}, want_b, {bank.G, bank.N, bank.r}, bank.scales);
  const long rows = plan.live_units * unit;
  const int n = aql_adapter_wgrad_scratch_floats(rows, plan.nused, want_a ? (int)bank.K : 0, want_b ? (int)bank.N : 0, (int)bank.R);
  if (n < 0) throw AqlErr("adapter_linear: the weight gradients' workspace passes 2^31 elements; train fewer rows or adapters per call");
  const c10::DataPtr scratch = workspace(n);
  const auto st = stream_of(bank.scales);
  ran(aql_adapter_wgrad(ptr<bf16_t>(dT), ptr<bf16_t>(x.t), x.ld, ptr<uint8_t>(codes), ptr<uint8_t>(exps), (int)bank.K, ptr<float>(dA), ptr<bf16_t>(T),
                        ptr<bf16_t>(dy.t), dy.ld, (int)bank.N, ptr<float>(dB), M, (int)bank.G, (int)bank.R, (int)bank.r, ptr<int>(bank.ranks), plan.part(1),
                        plan.part(2), plan.part(3), plan.nused, plan.nslot, (int)unit, rows, (float*)scratch.get(), n, st), "aql_adapter_wgrad", st);
}

struct AdapterLinear : torch::autograd::Function<AdapterLinear> {
  // ckpt8: the backward pass keeps X in 8 bits -- T is computed again from the codes, and dA and dB see their values in the place of X
  static Tensor forward(AutogradContext* ctx, const Tensor& x2d, const Tensor& down, const Tensor& up, const std::optional<Tensor>& residual,
                        c10::intrusive_ptr<Call> c, bool ckpt8, bool train) {
    Rows x = gemm_rows(x2d), res;
    if ((c->residual = residual.has_value())) res = gemm_rows(*residual);
    auto [y, T] = product(x, c->w, c->bias, res, c->bank->a, c->bank->b, *c->bank, *c->plan, c->unit, c->N, c->K, train && !ckpt8 ? 3 : 1);
    Tensor codes, exps, keep = x.t;
    c->train = train;
    c->leaves = {leaf(x2d), leaf(down), leaf(up), residual ? leaf(*residual) : Tensor()};
    if (!train) {
      keep = T = Tensor();
    } else if (ckpt8) {
      std::tie(codes, exps) = act8_alloc(c->M, c->K, y);
      const auto st = stream_of(y);
      ran(aql_act8_pack(x.t.data_ptr(), 0, c->M, (int)c->K, x.ld, ptr<uint8_t>(codes), ptr<uint8_t>(exps), st), "aql_act8_pack", st);
      keep = T = Tensor();
    }
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({keep, T, codes, exps});
    ctx->saved_data["call"] = c10::IValue::make_capsule(c);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto c = c10::static_intrusive_pointer_cast<Call>(ctx->saved_data["call"].toCapsule());
    const Bank& bank = *c->bank;
    const variable_list s = ctx->get_saved_variables();
    const bool want_x = ctx->needs_input_grad(0), want_a = ctx->needs_input_grad(1), want_b = ctx->needs_input_grad(2), want_r = c->residual && ctx->needs_input_grad(3);
    variable_list out(7);
    if (!g[0].defined()) return out;
    here(g[0], "adapter_linear backward");
    leaves_ok(c->leaves, g[0], "adapter_linear");
    const Reading reading(*c->bank, c->serial);
    if (!reading.in) throw AqlErr("adapter_linear: the bank's weights changed between the forward pass and its backward pass");
    {
      at::AutoGradMode off(false);
      if (c->M == 0) {
        if (want_x) out[0] = fresh({0, c->K}, at::kBFloat16, g[0]);
        if (want_a) out[1] = at::zeros({bank.G, bank.r, bank.K}, bank.scales.options());
        if (want_b) out[2] = at::zeros({bank.G, bank.N, bank.r}, bank.scales.options());
      } else {
        const Rows dy = gemm_rows(g[0]);
        const char* name = "adapter_linear";
        const long nb = (c->K + 31) / 32;
        Tensor dT, T = intact(s[1], {c->M, 3, bank.R}, at::kBFloat16, dy.t, name);
        const Tensor codes = intact(s[2], {c->M, nb * 32}, at::kByte, dy.t, name), exps = intact(s[3], {c->M, nb}, at::kByte, dy.t, name);
        Rows x;
        if (s[0].defined()) x = gemm_rows(intact(s[0], {c->M, c->K}, at::kBFloat16, dy.t, name, true));
        if (want_x) std::tie(out[0], dT) = product(dy, c->wt, Tensor(), Rows(), bank.bt, bank.at, bank, *c->plan, c->unit, c->K, c->N, c->train && want_a ? 3 : 1);
        if (c->train && (want_a || want_b)) {
          if (want_a && !dT.defined() && c->plan->nseg) dT = down(dy, Tensor(), Tensor(), c->M, c->N, bank.bt, bank, *c->plan, c->unit);
          if (want_b && !T.defined() && c->plan->nseg) T = down(Rows(), codes, exps, c->M, c->K, bank.a, bank, *c->plan, c->unit);
          wgrad(dT, x, codes, exps, want_a, T, dy, want_b, c->M, bank, *c->plan, c->unit, out[1], out[2]);
        }
      }
      if (want_r) out[3] = g[0];
    }
    return once(std::move(out), "adapter_linear");
  }
};

// -> y, or nothing where the bank has to be laid out first
std::optional<Tensor> adapter_linear(const Tensor& x, const Tensor& w, const Tensor& wt, const std::optional<Tensor>& bias_, const std::shared_ptr<Bank>& bank,
                                     const std::shared_ptr<Plan>& plan, const std::optional<Tensor>& residual_, bool ckpt8) {
  if (!bank->at.defined() && x.requires_grad() && at::GradMode::is_enabled()) return std::nullopt;
  const Tensor &down = bank->down, &up = bank->up;
  if (w.dim() != 2) bad_value("adapter_linear: the projection must be [N, K], not " + shape_of(w));
  const long N = w.size(0), K = w.size(1);
  if (x.dim() != 2 || x.scalar_type() != at::kBFloat16)
    bad_value("adapter_linear: expected bfloat16 [rows, " + std::to_string(K) + "], got " + c10::toString(x.scalar_type()) + " " + shape_of(x));
  const long M = x.size(0);
  if (x.size(1) != K || bank->K != K || bank->N != N)
    bad_value("adapter_linear: input " + shape_of(x) + ", projection [" + std::to_string(N) + ", " + std::to_string(K) + "], adapters on [" +
              std::to_string(bank->N) + ", " + std::to_string(bank->K) + "]");
  if (std::max(N, K) > 0x7fffffffL) bad_value("adapter_linear: projections of less than 2^31 rows and columns");
  if (plan->max_id >= bank->G)
    bad_value("adapter_linear: the plan names adapter " + std::to_string(plan->max_id) + ", the bank has " + std::to_string(bank->G));
  const long unit = plan->unit(M);
  const Tensor res = residual_ ? *residual_ : Tensor(), bias = bias_ ? *bias_ : Tensor();
  if (res.defined() && (res.dim() != 2 || res.size(0) != M || res.size(1) != N || res.scalar_type() != at::kBFloat16))
    bad_value("adapter_linear: residual must be bfloat16 [" + std::to_string(M) + ", " + std::to_string(N) + "], not " + shape_of(res));
  here(x, "adapter_linear");
  const auto operand = [&](const Tensor& t, at::IntArrayRef size) { return t.scalar_type() == at::kBFloat16 && t.sizes() == size && t.is_contiguous() && t.device() == x.device(); };
  if (!operand(w, {N, K}) || !operand(wt, {K, N}) || (bias.defined() && !operand(bias, {N})))
    bad_value("adapter_linear: the projection must be bfloat16 [" + std::to_string(N) + ", " + std::to_string(K) + "], its transpose and a bias of " + std::to_string(N) + ", contiguous on " + x.device().str());
  for (const Tensor* t : {&x, &res, &down, &up})   // (without reverse gradients no node is made that would refuse it)
    if (t->defined() && t->_fw_grad(0).defined()) throw AqlErr("adapter_linear has no forward-mode derivative");
  if (bank->a.device() != x.device() || plan->table.device() != x.device() || w.device() != x.device() || (res.defined() && res.device() != x.device()))
    bad_value("adapter_linear: input, projection, adapters, plan and residual must live on one device");
  const Reading reading(*bank);
  if (!reading.in) return std::nullopt;
  plan->reads();
  const bool train = bank->trainable && at::GradMode::is_enabled() && (down.requires_grad() || up.requires_grad());
  if (at::GradMode::is_enabled() && (train || x.requires_grad() || (res.defined() && res.requires_grad()))) {
    auto c = c10::make_intrusive<Call>();
    c->bank = bank, c->plan = plan, c->w = w, c->wt = wt, c->bias = bias, c->unit = unit, c->serial = reading.serial, c->M = M, c->N = N, c->K = K;
    return AdapterLinear::apply(x, down, up, residual_, c, ckpt8, train);
  }
  Rows r;
  if (res.defined()) r = gemm_rows(res);
  return product(gemm_rows(x), w, bias, r, bank->a, bank->b, *bank, *plan, unit, N, K, 1).first;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("set_error_class", [](py::object cls) { aql_error_class = cls.release(); });
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const AqlErr& e) {
      PyErr_SetString(aql_error_class.ptr() ? aql_error_class.ptr() : PyExc_RuntimeError, e.what());
    }
  });
  m.def("abi_version", [] { return aql_abi_version(); });
  m.def("abi_address", [] { return (uintptr_t)&aql_abi_version; });   // which kernel library this is bound to
  m.def("act8_pack", &act8_pack);
  m.def("act8_unpack", &act8_unpack);
  m.def("layernorm_train", &layernorm_train);
  m.def("adapter_linear", &adapter_linear);
  py::class_<Bank, std::shared_ptr<Bank>>(m, "Bank")
      .def(py::init<>())
      .def_readwrite("a", &Bank::a).def_readwrite("b", &Bank::b).def_readonly("at", &Bank::at).def_readonly("bt", &Bank::bt).def("publish", &Bank::publish)
      .def_readwrite("ranks", &Bank::ranks).def_readwrite("scales", &Bank::scales)
      .def_readwrite("down", &Bank::down).def_readwrite("up", &Bank::up).def("fresh", &Bank::fresh)
      .def("reads", &Bank::reads)
      .def("begin_layout", &Bank::begin_layout, py::call_guard<py::gil_scoped_release>())   // (a call that it waits for may need the interpreter)
      .def("end_layout", &Bank::end_layout)
      .def_readwrite("G", &Bank::G).def_readwrite("r", &Bank::r).def_readwrite("R", &Bank::R).def_readwrite("K", &Bank::K).def_readwrite("N", &Bank::N)
      .def_readonly("serial", &Bank::serial).def_readwrite("trainable", &Bank::trainable);
  py::class_<Plan, std::shared_ptr<Plan>>(m, "Plan")
      .def(py::init<>())
      .def_readwrite("table", &Plan::table).def_readwrite("start", &Plan::start).def_readwrite("at", &Plan::at)
      .def_readwrite("units", &Plan::units).def_readwrite("requests", &Plan::requests).def_readwrite("live_units", &Plan::live_units).def_readwrite("unit_rows", &Plan::unit_rows)
      .def_readwrite("nseg", &Plan::nseg).def_readwrite("nused", &Plan::nused).def_readwrite("nslot", &Plan::nslot)
      .def_readwrite("max_id", &Plan::max_id).def_readwrite("equal", &Plan::equal)
      .def("unit", &Plan::unit).def("slots", &Plan::slots);
}
