// CPython module triton_muon_adamw._objectives: the objectives as torch calls.
//
// What a call does beside its launches (arguments checked, outputs allocated, the node of the autograd graph) is 50 to
// 80 us in Python with ctypes, several times what the kernels of a small batch take, and some 10 us here.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/version.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>

#include <pybind11/pybind11.h>

#include <mutex>
#include <tuple>

#include "muonadamw_amd.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check(int status, const char* what) {
    if (status == MAMW_OK) return;
    if (status < 0) TORCH_CHECK_VALUE(false, what, ": ", mamw_strerror(status), " (status ", status, ")");
    TORCH_CHECK(false, what, ": ", mamw_strerror(status), " (status ", status, ")");
}

mamw_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int float_type(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MAMW_F32;
        case at::kBFloat16: return MAMW_BF16;
        case at::kHalf: return MAMW_F16;
        default: return -1;
    }
}

// ---- arguments

mamw_rows rows_of(const Tensor& x) {
    const int type = float_type(x.scalar_type());
    TORCH_CHECK_TYPE(type >= 0, "logits must be float32, bfloat16 or float16 (got ", x.scalar_type(), ")");
    TORCH_CHECK_VALUE(x.dim() == 2 || x.dim() == 3, "logits must be (rows, vocab) or (batch, length, vocab) (got ",
                      x.sizes(), ")");
    const int64_t vocab = x.size(-1);
    TORCH_CHECK_VALUE(vocab > 0, "logits have an empty vocabulary");
    TORCH_CHECK_VALUE(vocab == 1 || x.stride(-1) == 1 || x.numel() == 0,
                      "logits must be contiguous along the vocabulary");
    mamw_rows r;
    r.data = x.const_data_ptr();
    r.outer = x.dim() == 3 ? x.size(0) : 1;
    r.outer_stride = x.dim() == 3 ? x.stride(0) : 0;
    r.inner = x.size(-2);
    r.inner_stride = x.stride(-2);
    r.vocab = vocab;
    r.type = type;
    r.reserved = 0;
    return r;
}

enum Kind { kF32, kFloats, kInts, kBool };

int type_of(const Tensor& x, const char* name, Kind kind) {
    const at::ScalarType t = x.scalar_type();
    switch (kind) {
        case kF32:
            TORCH_CHECK_TYPE(t == at::kFloat, name, " must be float32 (got ", t, ")");
            return MAMW_F32;
        case kFloats:
            TORCH_CHECK_TYPE(float_type(t) >= 0, name, " must be float32, bfloat16 or float16 (got ", t, ")");
            return float_type(t);
        case kInts:
            TORCH_CHECK_TYPE(t == at::kInt || t == at::kLong, name, " must be int32 or int64 (got ", t, ")");
            return t == at::kInt ? MAMW_I32 : MAMW_I64;
        default:
            TORCH_CHECK_TYPE(t == at::kBool, name, " must be bool (got ", t, ")");
            return MAMW_BOOL;
    }
}

// One value (k > 0: k consecutive ones) for each row of `logits`, broadcast to them.
mamw_per_row per_row(const Tensor& x, const char* name, const Tensor& logits, Kind kind, int64_t k = 0) {
    mamw_per_row p = {};
    if (!x.defined()) return p;
    p.type = type_of(x, name, kind);
    TORCH_CHECK_VALUE(x.device() == logits.device(), name, " is on ", x.device(), ", logits on ", logits.device());
    const int64_t last = k ? 1 : 0, dims = x.dim() - last, want = logits.dim() - 1;
    TORCH_CHECK_VALUE(!k || (x.dim() >= 1 && x.size(-1) == k && (k == 1 || x.stride(-1) == 1)), name, " must have ", k,
                      " values for each row (got ", x.sizes(), ")");
    TORCH_CHECK_VALUE(dims <= want, name, " of shape ", x.sizes(), " does not go with logits of shape ",
                      logits.sizes());
    int64_t strides[2] = {0, 0};  // of the outer and the inner index
    for (int64_t d = 0; d < dims; ++d) {
        const int64_t at = want - dims + d, n = x.size(d);
        TORCH_CHECK_VALUE(n == 1 || n == logits.size(at), name, " of shape ", x.sizes(),
                          " does not go with logits of shape ", logits.sizes());
        strides[2 - want + at] = n == 1 ? 0 : x.stride(d);
    }
    p.data = x.const_data_ptr();
    p.outer_stride = strides[0];
    p.inner_stride = strides[1];
    return p;
}

// (offsets for the device, how many sequences there are)
std::pair<Tensor, int64_t> sequences(const Tensor& offsets, const Tensor& logits, bool needed) {
    if (!offsets.defined()) {
        TORCH_CHECK_VALUE(logits.dim() == 3 || !needed, "logits of shape (rows, vocab) need offsets: where each "
                          "sequence starts, and the end of the last");
        return {Tensor(), logits.dim() == 3 ? logits.size(0) : 1};
    }
    TORCH_CHECK_VALUE(logits.dim() == 2, "offsets go with logits of shape (rows, vocab)");
    type_of(offsets, "offsets", kInts);
    TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 1,
                      "offsets must hold a place for each sequence and the end (got shape ", offsets.sizes(), ")");
    TORCH_CHECK_VALUE(offsets.device() == logits.device(), "offsets are on ", offsets.device(), ", logits on ",
                      logits.device());
    return {offsets.to(at::kLong).contiguous(), offsets.numel() - 1};
}

// Last of the checks: the kernels run on ROCm devices only.
void require_gpu(const Tensor& logits) {
    TORCH_CHECK_NOT_IMPLEMENTED(!logits._fw_grad(/*level=*/0).defined(), "the objectives have no forward-mode derivative");
    TORCH_CHECK(logits.is_cuda(), "logits is on ", logits.device(),
                "; MuonAdamW's HIP kernels need tensors on a ROCm GPU (there is no CPU path)");
}

bool wants_grad(const Tensor& logits) { return at::GradMode::is_enabled() && logits.requires_grad(); }

template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor grad_like(const Tensor& logits) { return at::empty(logits.sizes(), logits.options()); }
Tensor bytes(size_t n, const Tensor& like) {
    return at::empty({int64_t(n < 256 ? 256 : n)}, like.options().dtype(at::kByte));
}

// A tensor that backward reads.  Where saved-tensor hooks are in force (a checkpoint that computes it again, offloading to
// host memory) they have it, nothing of it stays here, and it comes back at another address.  Otherwise its memory stays,
// and who has put other memory under it meanwhile (t.data = ..., which no version counter sees) gets an error.
struct Kept {
    SavedVariable saved;
    Tensor constant;  // of inference mode: without a version, it cannot be saved, nor a change of it be noticed
    c10::Storage storage;
    const void* data = nullptr;
    bool hooked = false;

    Kept() = default;  // of an undefined tensor
    // Of `logits` a gradient is wanted; what is kept of other inputs is their value.
    Kept(const Tensor& t, bool logits = false) {
        if (t.is_inference()) {
            constant = t;
            return;
        }
        saved = SavedVariable(!logits && t.requires_grad() ? t.detach() : t, false);
        hooked = saved.has_hooks();
        if (hooked) return;
        storage = t.storage();
        data = t.const_data_ptr();
    }

    Tensor unpack() const {
        if (constant.defined()) return constant;
        Tensor t = saved.unpack();  // raises where it was released, or changed in place since
        TORCH_CHECK(hooked || !t.defined() || t.const_data_ptr() == data,
                    "a tensor that the gradient needs was given other memory after the forward pass");
        return t;
    }
    // Of logits: `rows` are those of the forward pass, and then of the memory that they are in now.
    Tensor unpack(mamw_rows& rows, const Tensor& like) const {
        Tensor x = unpack();
        TORCH_CHECK(x.device() == like.device() && float_type(x.scalar_type()) == rows.type, "logits of the forward pass on ",
                    like.device(), " came back as ", x.scalar_type(), " on ", x.device());
        const mamw_rows was = rows;
        if (x.dim() == 2 || x.dim() == 3) rows = rows_of(x);
        TORCH_CHECK((x.dim() == 2 || x.dim() == 3) && rows.outer == was.outer && rows.inner == was.inner &&
                        rows.vocab == was.vocab,
                    "logits changed their shape after the forward pass (now ", x.sizes(), ")");
        return x;
    }
    void reset() {
        saved.reset_data();
        constant = Tensor();
        storage = c10::Storage();
    }
};

// ---- the autograd graph

// A gradient that was computed for a graph to be built of it (create_graph) cannot be differentiated again: who tries
// gets an error, not zeros.
Tensor once(const Tensor& grad) {
    if (!at::GradMode::is_enabled()) return grad;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the objectives' gradients cannot be differentiated a second time", 1);
    return (*error)({grad.detach().requires_grad_(true)})[0];
}

// A loss whose forward kernel writes the gradient as well, because a row's gradient needs nothing beyond that row.
// backward hands it out; a gradient of the loss other than 1 has it computed again from the logits with that factor
// (the device decides, so nothing waits), which rounds once and keeps float16 gradients of a scaled loss from
// vanishing first.  Where hooks keep the logits, a gradient of their size is not kept beside them: backward computes it.
struct OnePass : Node {
    std::mutex lock;
    Kept logits;
    std::vector<Kept> inputs;  // what the description points to, in the order of describe()
    mamw_rows rows;
    Tensor grad, workspace;

    // Has the description point to `inputs`, which go with logits x.
    virtual void describe(const Tensor& x, at::ArrayRef<Tensor> inputs) = 0;
    virtual int again(const float* scale, int unless_one, void* out, mamw_stream_t stream) = 0;

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> guard(lock);
        if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
        return {once(gradient(grads[0]))};
    }

    Tensor gradient(const Tensor& grad_output) {
        at::NoGradGuard no_grad;
        const Tensor x = logits.unpack(rows, workspace);
        c10::SmallVector<Tensor, 5> with;
        for (auto& i : inputs) with.push_back(i.unpack());
        describe(x, with);
        const c10::DeviceGuard device(x.device());
        Tensor out = std::move(grad);
        grad = Tensor();
        const bool fresh = !out.defined();  // the graph was retained and the first one is someone else's now, or hooks
        if (fresh) out = grad_like(x);
        const Tensor scale = grad_output.to(at::kFloat);
        check(again(ptr<float>(scale), !fresh, ptr(out), stream_of(x)), name().c_str());
        return out;
    }

    void release_variables() override {
        std::lock_guard<std::mutex> guard(lock);
        logits.reset();
        for (auto& i : inputs) i.reset();
        grad = workspace = Tensor();
    }
};

// tokens, old_logprobs, advantages, ref_logprobs, offsets (int64)
void describe_policy(mamw_policy& p, const Tensor& logits, at::ArrayRef<Tensor> inputs) {
    p.tokens = per_row(inputs[0], "tokens", logits, kInts);
    p.old_logprobs = per_row(inputs[1], "old_logprobs", logits, kF32);
    p.advantages = per_row(inputs[2], "advantages", logits, kF32);
    p.ref_logprobs = per_row(inputs[3], "ref_logprobs", logits, kF32);
    p.offsets = inputs[4].defined() ? inputs[4].const_data_ptr<int64_t>() : nullptr;
}

// teacher_logits, teacher_indices, teacher_lse, mask
void describe_distill(mamw_distill& p, const Tensor& logits, at::ArrayRef<Tensor> inputs) {
    p.teacher_logits = per_row(inputs[0], "teacher_logits", logits, kFloats, p.k);
    p.teacher_indices = per_row(inputs[1], "teacher_indices", logits, kInts, p.k);
    p.teacher_lse = per_row(inputs[2], "teacher_lse", logits, kF32);
    p.mask = per_row(inputs[3], "mask", logits, kBool);
}

struct PolicyLossBackward : OnePass {
    mamw_policy desc;
    std::string name() const override { return "PolicyLossBackward"; }
    void describe(const Tensor& x, at::ArrayRef<Tensor> inputs) override { describe_policy(desc, x, inputs); }
    int again(const float* scale, int unless_one, void* out, mamw_stream_t stream) override {
        return mamw_policy_grad(&rows, &desc, scale, unless_one, out, ptr(workspace), workspace.numel(), stream);
    }
};

struct DistillLossBackward : OnePass {
    mamw_distill desc;
    std::string name() const override { return "DistillLossBackward"; }
    void describe(const Tensor& x, at::ArrayRef<Tensor> inputs) override { describe_distill(desc, x, inputs); }
    int again(const float* scale, int unless_one, void* out, mamw_stream_t stream) override {
        return mamw_distill_grad(&rows, &desc, scale, unless_one, out, ptr(workspace), workspace.numel(), stream);
    }
};

// Gradients from the statistics that the forward pass left: of log-probabilities and entropies, with a gradient for
// each row, and of the preference loss, with one for the loss and the rows' coefficients.
struct FromStats : Node {
    std::mutex lock;
    Kept logits, tokens, entropy;
    mamw_rows rows;
    Tensor stats, coef;  // coef: the preference loss's
    double temperature;
    int64_t ignore_index;

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> guard(lock);
        const bool by_row = !coef.defined();
        const bool second = by_row && grads.size() > 1 && grads[1].defined();
        if (!task_should_compute_output(0) || !(grads[0].defined() || second)) return {Tensor()};
        return {once(gradient(grads, by_row, second))};
    }

    Tensor gradient(const variable_list& grads, bool by_row, bool second) {
        at::NoGradGuard no_grad;
        const Tensor x = logits.unpack(rows, stats), toks = tokens.unpack(), h_out = second ? entropy.unpack() : Tensor();
        const c10::DeviceGuard device(x.device());
        const mamw_per_row at = per_row(toks, "tokens", x, kInts);
        Tensor first = grads[0].defined() ? grads[0].to(at::kFloat) : at::zeros({}, stats.options());
        const Tensor out = grad_like(x);
        mamw_per_row a, h = {};
        Tensor other;
        if (by_row) {
            a = per_row(first, "gradient", x, kF32);
            if (second) {
                other = grads[1].to(at::kFloat);
                h = per_row(other, "gradient", x, kF32);
            }
        } else {
            a = per_row(coef, "coefficients", x, kF32);
        }
        check(mamw_logits_grad(&rows, &at, ignore_index, float(temperature), ptr<float>(stats), &a,
                               second ? &h : nullptr, ptr<float>(h_out), by_row ? nullptr : ptr<float>(first),
                               ptr(out), stream_of(x)),
              name().c_str());
        return out;
    }

    void release_variables() override {
        std::lock_guard<std::mutex> guard(lock);
        logits.reset();
        tokens.reset();
        entropy.reset();
        stats = Tensor();
        if (coef.defined()) coef = floats({0}, coef);
    }
};

struct TokenLogprobsBackward : FromStats {
    std::string name() const override { return "TokenLogprobsBackward"; }
};

struct PreferenceLossBackward : FromStats {
    std::string name() const override { return "PreferenceLossBackward"; }
};

template <typename N>
std::shared_ptr<N> node_of(const Tensor& logits) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    return node;
}

// ---- from Python

struct Args {
    PyObject* const* v;
    Py_ssize_t n;

    Tensor tensor(int i, const char* name) const {
        TORCH_CHECK_TYPE(THPVariable_Check(v[i]), name, " must be a tensor (got ", Py_TYPE(v[i])->tp_name, ")");
        return THPVariable_Unpack(v[i]);
    }
    Tensor maybe_tensor(int i, const char* name) const { return v[i] == Py_None ? Tensor() : tensor(i, name); }
    double real(int i) const {
        const double x = PyFloat_AsDouble(v[i]);
        if (x == -1.0 && PyErr_Occurred()) throw python_error();
        return x;
    }
    int64_t whole(int i) const {
        const int64_t x = PyLong_AsLongLong(v[i]);
        if (x == -1 && PyErr_Occurred()) throw python_error();
        return x;
    }
    bool truth(int i) const {
        const int x = PyObject_IsTrue(v[i]);
        if (x < 0) throw python_error();
        return x != 0;
    }
    void expect(Py_ssize_t count) const { TORCH_CHECK_TYPE(n == count, "expected ", count, " arguments, got ", n); }
};

PyObject* pack(std::initializer_list<Tensor> tensors) {
    THPObjectPtr out(PyTuple_New(Py_ssize_t(tensors.size())));
    if (!out) throw python_error();
    Py_ssize_t i = 0;
    for (const Tensor& t : tensors) {
        PyObject* o = t.defined() ? THPVariable_Wrap(t) : (Py_INCREF(Py_None), Py_None);
        if (!o) throw python_error();
        PyTuple_SET_ITEM(out.get(), i++, o);
    }
    return out.release();
}

// token_logprobs(logits, tokens, temperature, ignore_index, entropy) -> (logprobs, entropies or None)
PyObject* token_logprobs(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Args a{v, n};
    a.expect(5);
    const Tensor logits = a.tensor(0, "logits"), tokens = a.tensor(1, "tokens");
    const double temperature = a.real(2);
    const int64_t ignore_index = a.whole(3);
    const bool with_entropy = a.truth(4);
    const mamw_rows rows = rows_of(logits);
    const mamw_per_row at = per_row(tokens, "tokens", logits, kInts);
    require_gpu(logits);
    const bool grad = wants_grad(logits);
    Tensor logprobs, entropy, stats;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard device(logits.device());
        const auto shape = logits.sizes().slice(0, logits.dim() - 1);
        logprobs = floats(shape, logits);
        if (with_entropy) entropy = floats(shape, logits);
        if (grad) stats = floats({rows.outer, rows.inner, 2}, logits);
        check(mamw_token_logprobs(&rows, &at, ignore_index, float(temperature), ptr<float>(logprobs),
                                  ptr<float>(entropy), ptr<float>(stats), stream_of(logits)),
              "token_logprobs");
    }
    if (grad) {
        auto node = node_of<TokenLogprobsBackward>(logits);
        node->logits = Kept(logits, true);
        node->tokens = Kept(tokens);
        node->rows = rows;
        node->stats = stats;
        if (with_entropy) node->entropy = Kept(entropy.detach());  // an alias: a change in place of the output counts
        node->temperature = temperature;
        node->ignore_index = ignore_index;
        torch::autograd::set_history(logprobs, node);
        if (with_entropy) torch::autograd::set_history(entropy, node);
    }
    return pack({logprobs, entropy});
    END_HANDLE_TH_ERRORS
}

// The forward pass of a loss in one, for `node` (NULL: no gradient).
template <typename N, typename Fn>
Tensor with_node(const Tensor& logits, const std::shared_ptr<N>& node, const mamw_rows& rows, const Tensor& workspace,
                 at::ArrayRef<Tensor> inputs, Fn forward) {
    if (node) node->logits = Kept(logits, true);
    Tensor loss, grad;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        if (node && !node->logits.hooked) grad = grad_like(logits);
        loss = forward(ptr(grad));
    }
    if (node) {
        for (const Tensor& t : inputs) node->inputs.push_back(t.defined() ? Kept(t) : Kept());
        node->rows = rows;
        node->grad = std::move(grad);
        node->workspace = workspace;
        torch::autograd::set_history(loss, node);
    }
    return loss;
}

// policy_loss(logits, tokens, old_logprobs, advantages, ref_logprobs, kl_coef, clip_low, clip_high, by_sequence,
//             offsets, temperature, ignore_index, scale) -> (loss, logprobs, kl, clipped)
PyObject* policy_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Args a{v, n};
    a.expect(13);
    const Tensor logits = a.tensor(0, "logits");
    Tensor inputs[5] = {a.tensor(1, "tokens"), a.tensor(2, "old_logprobs"), a.tensor(3, "advantages"),
                        a.maybe_tensor(4, "ref_logprobs"), Tensor()};
    const mamw_rows rows = rows_of(logits);
    mamw_policy p = {};
    p.by_sequence = a.truth(8);
    std::tie(inputs[4], p.sequences) = sequences(a.maybe_tensor(9, "offsets"), logits, p.by_sequence);
    describe_policy(p, logits, inputs);
    p.kl_coef = float(a.real(5));
    p.clip_low = float(a.real(6));
    p.clip_high = float(a.real(7));
    p.temperature = float(a.real(10));
    p.ignore_index = a.whole(11);
    p.scale = float(a.real(12));
    size_t need = 0;
    check(mamw_policy_workspace_bytes(&rows, &p, &need), "policy_loss");
    require_gpu(logits);
    const c10::DeviceGuard device(logits.device());
    std::shared_ptr<PolicyLossBackward> node;
    if (wants_grad(logits)) {
        node = node_of<PolicyLossBackward>(logits);
        node->desc = p;
    }
    Tensor logprobs, kl, clipped, workspace;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        workspace = bytes(need, logits);
        logprobs = floats(logits.sizes().slice(0, logits.dim() - 1), logits);
    }
    const Tensor loss = with_node(logits, node, rows, workspace, inputs, [&](void* grad) {
        const Tensor result = floats({3}, logits);
        check(mamw_policy_loss(&rows, &p, ptr<float>(result), ptr<float>(logprobs), grad, ptr(workspace), workspace.numel(),
                               stream_of(logits)),
              "policy_loss");
        kl = result.select(0, 1);
        clipped = result.select(0, 2);
        return result.select(0, 0);
    });
    return pack({loss, logprobs, kl, clipped});
    END_HANDLE_TH_ERRORS
}

// preference_loss(logits, tokens, ref_logprobs, beta, kind, label_smoothing, length_average, offsets, temperature,
//                 ignore_index) -> (loss, logprobs, rewards)
PyObject* preference_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Args a{v, n};
    a.expect(10);
    const Tensor logits = a.tensor(0, "logits"), tokens = a.tensor(1, "tokens");
    Tensor ref = a.maybe_tensor(2, "ref_logprobs");
    const mamw_rows rows = rows_of(logits);
    mamw_preference p = {};
    const auto [offsets, count] = sequences(a.maybe_tensor(7, "offsets"), logits, true);
    TORCH_CHECK_VALUE(count >= 2 && count % 2 == 0, "pairs need an even number of sequences, at least 2 (got ", count,
                      ")");
    if (ref.defined()) {
        type_of(ref, "ref_logprobs", kF32);
        TORCH_CHECK_VALUE(ref.dim() == 1 && ref.size(0) == count && ref.device() == logits.device(),
                          "ref_logprobs must hold one value for each of ", count, " sequences on ", logits.device(),
                          " (got ", ref.sizes(), " on ", ref.device(), ")");
        ref = ref.detach().contiguous();
    }
    p.tokens = per_row(tokens, "tokens", logits, kInts);
    p.ref_logprobs = ref.defined() ? ref.const_data_ptr<float>() : nullptr;
    p.offsets = offsets.defined() ? offsets.const_data_ptr<int64_t>() : nullptr;
    p.sequences = count;
    p.beta = float(a.real(3));
    p.kind = int32_t(a.whole(4));
    p.smoothing = float(a.real(5));
    p.length_average = a.truth(6);
    const double temperature = a.real(8);
    p.temperature = float(temperature);
    p.ignore_index = a.whole(9);
    size_t need = 0;
    check(mamw_preference_workspace_bytes(&rows, &p, &need), "preference_loss");
    require_gpu(logits);
    const bool grad = wants_grad(logits);
    Tensor loss, logprobs, rewards, stats, coef;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        const c10::DeviceGuard device(logits.device());
        const Tensor workspace = bytes(need, logits);
        const Tensor result = floats({3}, logits);
        loss = result.select(0, 0);
        logprobs = floats({count}, logits);
        rewards = floats({count}, logits);
        if (grad) {
            stats = floats({rows.outer, rows.inner, 2}, logits);
            coef = floats(logits.sizes().slice(0, logits.dim() - 1), logits);
        }
        check(mamw_preference_loss(&rows, &p, ptr<float>(result), ptr<float>(logprobs), ptr<float>(rewards),
                                   ptr<float>(stats), ptr<float>(coef), ptr(workspace), workspace.numel(),
                                   stream_of(logits)),
              "preference_loss");
    }
    if (grad) {
        auto node = node_of<PreferenceLossBackward>(logits);
        node->logits = Kept(logits, true);
        node->tokens = Kept(tokens);
        node->rows = rows;
        node->stats = stats;
        node->coef = coef;
        node->temperature = temperature;
        node->ignore_index = p.ignore_index;
        torch::autograd::set_history(loss, node);
    }
    return pack({loss, logprobs, rewards});
    END_HANDLE_TH_ERRORS
}

// distill_loss(logits, teacher_logits, teacher_indices, teacher_lse, mask, temperature, scale) -> (loss,)
PyObject* distill_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Args a{v, n};
    a.expect(7);
    const Tensor logits = a.tensor(0, "logits");
    Tensor inputs[4] = {a.tensor(1, "teacher_logits").detach(), a.tensor(2, "teacher_indices"),
                        a.maybe_tensor(3, "teacher_lse"), a.maybe_tensor(4, "mask")};
    Tensor &teacher = inputs[0], &index = inputs[1];
    const mamw_rows rows = rows_of(logits);
    const int64_t k = teacher.dim() ? teacher.size(-1) : 0;
    TORCH_CHECK_VALUE(k >= 1 && k <= MAMW_MAX_TEACHER, "teacher_logits must have between 1 and ", MAMW_MAX_TEACHER,
                      " values for each row (got ", k, ")");
    if (k > 1 && teacher.stride(-1) != 1) teacher = teacher.contiguous();
    if (k > 1 && index.dim() && index.stride(-1) != 1) index = index.contiguous();
    mamw_distill p = {};
    p.k = k;
    describe_distill(p, logits, inputs);
    p.temperature = float(a.real(5));
    p.scale = float(a.real(6));
    size_t need = 0;
    check(mamw_distill_workspace_bytes(&rows, &p, &need), "distill_loss");
    require_gpu(logits);
    const c10::DeviceGuard device(logits.device());
    std::shared_ptr<DistillLossBackward> node;
    if (wants_grad(logits)) {
        node = node_of<DistillLossBackward>(logits);
        node->desc = p;
    }
    Tensor workspace;
    {
        pybind11::gil_scoped_release no_gil;
        at::AutoDispatchBelowADInplaceOrView below;
        workspace = bytes(need, logits);
    }
    const Tensor loss = with_node(logits, node, rows, workspace, inputs, [&](void* grad) {
        const Tensor result = floats({3}, logits);
        check(mamw_distill_loss(&rows, &p, ptr<float>(result), grad, ptr(workspace), workspace.numel(),
                                stream_of(logits)),
              "distill_loss");
        return result.select(0, 0);
    });
    return pack({loss});
    END_HANDLE_TH_ERRORS
}

template <PyObject* (*kFn)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kFn)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {
    method<token_logprobs>("token_logprobs"),
    method<policy_loss>("policy_loss"),
    method<preference_loss>("preference_loss"),
    method<distill_loss>("distill_loss"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_objectives", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__objectives() {
    THPObjectPtr m(PyModule_Create(&kModule));
    if (!m || PyModule_AddStringConstant(m.get(), "torch_version", TORCH_VERSION) != 0) return nullptr;
    return m.release();
}
