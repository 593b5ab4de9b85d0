// Native host path of the sequence operators (include/dcn_seq.h), in the manner of dcn_torch.cpp: argument checks, output
// allocation, the library call and the graph node of the backward pass, in one C++ call per direction.
//
// One node serves all of them: an operator is a forward function over its input tensors, which says what its backward function
// needs, and that backward function.  Everything kept in between goes through saved variables, so that in-place changes are
// noticed and saved-tensor hooks see it.
#include "dcn_torch.h"

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <mutex>
#include <vector>

#include "../../include/dcn_seq.h"

namespace {

using namespace dcn_host;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Numbers {                         // what a call says beside its tensors
    int64_t ignore = -100;
    int32_t top = 0;
    double temperature = 1.0, eps = 1e-6;
    bool tail = true;
};

struct Operator {
    const char* name;
    const char* node;
    int inputs;                          // slots of the input list
    int differentiable;                  // of them, from the first on
    variable_list (*forward)(const Numbers&, const variable_list& in, bool keep, variable_list& kept);
    // gradients by slot from those of the outputs and what was kept; only what `want` asks for
    variable_list (*backward)(const Numbers&, const variable_list& kept, const variable_list& grads, const std::vector<bool>& want);
};

// ---- checks and layouts ---------------------------------------------------------------------------------------------------
std::string shape_text(at::IntArrayRef s) {
    std::string t;
    for (int64_t v : s) t += (t.empty() ? "" : ", ") + std::to_string(v);
    return "(" + t + ")";
}

int32_t type_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return DCN_SEQ_F32;
        case at::kBFloat16: return DCN_SEQ_BF16;
        case at::kHalf: return DCN_SEQ_F16;
        default: fail(std::string(name) + " must be float32, bfloat16 or float16, got " + dtype_name(t));
    }
}

void on_gpu(const Tensor& t, const char* name) {
    if (!t.is_cuda()) fail(std::string(name) + " must be a CUDA tensor (there is no CPU implementation)");
    if (t.layout() != at::kStrided) fail(std::string(name) + " must be a dense tensor");
}

void beside(const Tensor& t, const char* name, const Tensor& x, const char* xname) {
    if (!t.defined()) return;
    on_gpu(t, name);
    if (t.device() != x.device())
        fail(std::string(name) + " is on " + t.device().str() + " but " + xname + " is on " + x.device().str());
}

void typed(const Tensor& t, const char* name, at::ScalarType want, const char* as = nullptr) {
    if (t.defined() && t.scalar_type() != want)
        fail(std::string(name) + " has dtype " + dtype_name(t) + ", expected torch." + torch::getTHPDtype(want)->name +
             (as != nullptr ? std::string(" as ") + as : ""));
}

void shaped(const Tensor& t, const char* name, at::IntArrayRef want) {
    if (t.defined() && t.sizes() != want)
        fail(std::string(name) + " has shape " + shape_text(t.sizes()) + ", expected " + shape_text(want));
}

Tensor whole_numbers(const Tensor& t, const char* name) {
    if (!t.defined()) return t;
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
        fail(std::string(name) + " must be int64 or int32, got " + dtype_name(t));
    return t.to(at::kLong).contiguous();
}

// Its own values in memory, not those of which it is the negative (the imaginary part of a conjugate)
Tensor in_memory(Tensor t) {
    if (t.defined() && t.is_neg()) return t.resolve_neg();
    return t;
}

variable_list in_memory(const variable_list& v) {
    variable_list r;
    for (const Tensor& t : v) r.push_back(in_memory(t));
    return r;
}

// The last axis dense; any strides over the others
Tensor dense_last(const Tensor& t) {
    return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// [rows, width] with one stride over the rows
Tensor rows_of(const Tensor& t, int64_t rows, int64_t width) {
    return !t.defined() ? t : dense_last(t.dim() == 2 ? t : t.reshape({rows, width}));
}

int64_t row_stride(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* wptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(wptr(t)); }
int64_t* iptr(const Tensor& t) { return static_cast<int64_t*>(wptr(t)); }
void* current_stream(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }
Tensor floats(at::IntArrayRef shape, const Tensor& x) { return at::empty(shape, x.options().dtype(at::kFloat)); }
Tensor maybe(bool yes, const Tensor& like) { return yes ? at::empty(like.sizes(), like.options()) : Tensor(); }

std::vector<int64_t> without_last(const Tensor& t) {
    std::vector<int64_t> v = t.sizes().vec();
    v.pop_back();
    return v;
}

int64_t product(at::IntArrayRef s) {
    int64_t n = 1;
    for (int64_t v : s) n *= v;
    return n;
}

// ---- gated scan: x, gate, state, lengths -> y, last -----------------------------------------------------------------------
dcn_scan scan_of(const Tensor& x, const Tensor& gate, const Tensor& dy) {
    dcn_scan p = {};
    p.dtype = type_of(x, "x");
    p.batch = x.size(0), p.steps = x.size(1), p.channels = x.size(2);
    p.x_batch = x.stride(0), p.x_step = x.stride(1);
    p.gate_batch = gate.stride(0), p.gate_step = gate.stride(1);
    if (dy.defined()) p.dy_batch = dy.stride(0), p.dy_step = dy.stride(1);
    return p;
}

variable_list scan_forward(const Numbers&, const variable_list& in, bool keep, variable_list& kept) {
    on_gpu(in[0], "x");
    type_of(in[0], "x");
    if (in[0].dim() != 3) fail("x has shape " + shape_text(in[0].sizes()) + ", expected (batch, steps, channels)");
    beside(in[1], "gate", in[0], "x");
    beside(in[2], "state", in[0], "x");
    beside(in[3], "lengths", in[0], "x");
    typed(in[1], "gate", in[0].scalar_type(), "x");
    shaped(in[1], "gate", in[0].sizes());
    typed(in[2], "state", at::kFloat);
    shaped(in[2], "state", {in[0].size(0), in[0].size(2)});
    shaped(in[3], "lengths", {in[0].size(0)});
    const Tensor lengths = whole_numbers(in[3], "lengths");
    const Tensor x = dense_last(in[0]), gate = dense_last(in[1]);
    const Tensor state = in[2].defined() ? in[2].contiguous() : in[2];
    const dcn_scan p = scan_of(x, gate, Tensor());
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor y = at::empty(x.sizes(), x.options()), last = floats({p.batch, p.channels}, x);
    const Tensor states = keep ? floats({(int64_t)(dcn_scan_checkpoint_bytes(&p) / sizeof(float))}, x) : Tensor();
    Range range("dcn_scan_forward");
    check(dcn_scan_forward(&p, ptr(x), ptr(gate), fptr(state), iptr(lengths), wptr(y), fptr(last), fptr(states), current_stream(x)),
          "dcn_scan_forward");
    if (keep) kept = {in[0], in[1], lengths, states};
    return {y, last};
}

variable_list scan_backward(const Numbers&, const variable_list& kept, const variable_list& grads, const std::vector<bool>& want) {
    const Tensor x = dense_last(kept[0]), gate = dense_last(kept[1]), dy = dense_last(grads[0]);
    const Tensor dlast = grads[1].defined() ? grads[1].contiguous() : grads[1];
    const dcn_scan p = scan_of(x, gate, dy);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor dx = at::empty(x.sizes(), x.options()), dgate = at::empty(x.sizes(), x.options());
    const Tensor dstate = want[2] ? floats({p.batch, p.channels}, x) : Tensor();
    Range range("dcn_scan_backward");
    check(dcn_scan_backward(&p, ptr(x), ptr(gate), iptr(kept[2]), fptr(kept[3]), ptr(dy), fptr(dlast), wptr(dx), wptr(dgate),
                            fptr(dstate), current_stream(x)),
          "dcn_scan_backward");
    return {want[0] ? dx : Tensor(), want[1] ? dgate : Tensor(), dstate};
}

// ---- gated residual norm: x, block, gate, scale, post_weight, pre_weight -> stream, normed ----------------------------------
dcn_norm norm_of(const Numbers& n, const Tensor& x, const variable_list& in, int64_t rows) {
    dcn_norm p = {};
    p.dtype = type_of(x, "x");
    p.weight_dtype = p.dtype;
    for (int i = 3; i < 6; ++i)
        if (in[i].defined()) p.weight_dtype = type_of(in[i], "weights");
    p.rows = rows;
    p.channels = x.size(-1);
    p.eps = (float)n.eps;
    return p;
}

variable_list norm_forward(const Numbers& n, const variable_list& in, bool keep, variable_list& kept) {
    static const char* const names[] = {"x", "block", "gate", "scale", "post_weight", "pre_weight"};
    on_gpu(in[0], "x");
    type_of(in[0], "x");
    if (in[0].dim() < 1 || in[0].size(-1) < 1 || in[0].size(-1) > 8192)
        fail("x has shape " + shape_text(in[0].sizes()) + ": 1 to 8192 channels are supported");
    if (!(n.eps >= 0.0)) fail("eps must not be negative");
    for (int i = 1; i < 6; ++i) beside(in[i], names[i], in[0], "x");
    for (int i = 1; i < 3; ++i) {
        typed(in[i], names[i], in[0].scalar_type(), "x");
        shaped(in[i], names[i], in[0].sizes());
    }
    for (int i = 2; i < 5; ++i)
        if (in[i].defined() && !in[1].defined()) fail(std::string(names[i]) + " is given without a block");
    at::ScalarType wt = in[0].scalar_type();
    const char* as = "x";
    for (int i = 3; i < 6; ++i) {
        if (!in[i].defined()) continue;
        if (as[0] == 'x' && in[i].scalar_type() == at::kFloat) wt = at::kFloat;
        typed(in[i], names[i], wt, as);
        as = "the other weights";
        shaped(in[i], names[i], {in[0].size(-1)});
    }
    const int64_t rows = product(without_last(in[0]));
    const Tensor x = rows_of(in[0], rows, in[0].size(-1)), block = rows_of(in[1], rows, in[0].size(-1)),
                 gate = rows_of(in[2], rows, in[0].size(-1));
    dcn_norm p = norm_of(n, x, in, rows);
    p.x_row = row_stride(x), p.block_row = row_stride(block), p.gate_row = row_stride(gate);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor normed = at::empty(in[0].sizes(), x.options());
    const Tensor stream = maybe(block.defined(), normed);
    const Tensor stats = keep ? floats({rows, 2}, x) : Tensor();
    const Tensor scale = in[3].defined() ? in[3].contiguous() : in[3], post = in[4].defined() ? in[4].contiguous() : in[4],
                 pre = in[5].defined() ? in[5].contiguous() : in[5];
    Range range("dcn_norm_forward");
    check(dcn_norm_forward(&p, ptr(x), ptr(block), ptr(gate), ptr(scale), ptr(post), ptr(pre), wptr(stream), wptr(normed),
                           fptr(stats), current_stream(x)),
          "dcn_norm_forward");
    if (keep) {
        kept = in;
        kept.push_back(stats);
    }
    if (block.defined()) return {stream, normed};
    return {normed};
}

variable_list norm_backward(const Numbers& n, const variable_list& kept, const variable_list& grads, const std::vector<bool>& want) {
    const bool has_block = kept[1].defined();
    const int64_t c = kept[0].size(-1), rows = product(without_last(kept[0]));
    const Tensor x = rows_of(kept[0], rows, c), block = rows_of(kept[1], rows, c), gate = rows_of(kept[2], rows, c);
    const Tensor dstream = has_block ? rows_of(grads[0], rows, c) : Tensor(), dnormed = rows_of(grads[has_block ? 1 : 0], rows, c);
    Tensor w[3];
    for (int i = 0; i < 3; ++i) w[i] = kept[3 + i].defined() ? kept[3 + i].contiguous() : kept[3 + i];
    dcn_norm p = norm_of(n, x, kept, rows);
    p.x_row = row_stride(x), p.block_row = row_stride(block), p.gate_row = row_stride(gate);
    p.dstream_row = row_stride(dstream), p.dnormed_row = row_stride(dnormed);
    const c10::cuda::CUDAGuard guard(x.device());
    variable_list g(6);
    for (int i = 0; i < 6; ++i)
        if (want[i]) g[i] = at::empty(kept[i].sizes(), kept[i].options());
    const bool weights = want[3] || want[4] || want[5];
    const size_t bytes = weights ? dcn_norm_workspace_bytes(&p) : 0;
    const Tensor ws = bytes > 0 ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
    Range range("dcn_norm_backward");
    check(dcn_norm_backward(&p, ptr(x), ptr(block), ptr(gate), ptr(w[0]), ptr(w[1]), ptr(w[2]), fptr(kept[6]), ptr(dstream),
                            ptr(dnormed), wptr(g[0]), wptr(g[1]), wptr(g[2]), wptr(g[3]), wptr(g[4]), wptr(g[5]), wptr(ws), bytes,
                            current_stream(x)),
          "dcn_norm_backward");
    return g;
}

// ---- rows of logits -------------------------------------------------------------------------------------------------------
dcn_logits logits_of(const Numbers& n, const Tensor& logits, int64_t rows) {
    dcn_logits p = {};
    p.dtype = type_of(logits, "logits");
    p.rows = rows;
    p.vocab = logits.size(-1);
    p.row_stride = row_stride(logits);
    p.temperature = (float)n.temperature;
    return p;
}

void check_logits(const Numbers& n, const Tensor& logits) {
    on_gpu(logits, "logits");
    type_of(logits, "logits");
    if (logits.dim() < 1 || logits.size(-1) < 1)
        fail("logits have shape " + shape_text(logits.sizes()) + ", expected (..., vocabulary)");
    if (!((float)n.temperature >= 1e-3f && (float)n.temperature <= 1e3f)) fail("temperature must lie between 1e-3 and 1e3");
}

// logits, tokens -> logprob, entropy, top_logprobs, top_tokens
variable_list scores_forward(const Numbers& n, const variable_list& in, bool keep, variable_list& kept) {
    check_logits(n, in[0]);
    const std::vector<int64_t> lead = without_last(in[0]);
    beside(in[1], "tokens", in[0], "logits");
    shaped(in[1], "tokens", lead);
    const Tensor tokens = whole_numbers(in[1], "tokens");
    if (n.top < 0 || n.top > DCN_SCORES_MOST_TOP || n.top > in[0].size(-1))
        fail("top is " + std::to_string(n.top) + ": 0 to " + std::to_string((int)DCN_SCORES_MOST_TOP) +
             ", and at most the vocabulary's " + std::to_string(in[0].size(-1)) + ", are supported");
    const int64_t rows = product(lead);
    const Tensor logits = rows_of(in[0], rows, in[0].size(-1));
    const dcn_logits p = logits_of(n, logits, rows);
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor logprob = tokens.defined() ? floats(lead, logits) : Tensor(), entropy = floats(lead, logits);
    std::vector<int64_t> wide = lead;
    wide.push_back(n.top);
    const Tensor best = n.top > 0 ? floats(wide, logits) : Tensor();
    const Tensor best_tokens = n.top > 0 ? at::empty(wide, logits.options().dtype(at::kLong)) : Tensor();
    const Tensor stats = keep ? floats({rows, DCN_LOGITS_STATS}, logits) : Tensor();
    Range range("dcn_scores_forward");
    check(dcn_scores_forward(&p, ptr(logits), iptr(tokens), n.ignore, n.top, fptr(logprob), fptr(entropy), fptr(best),
                             iptr(best_tokens), fptr(stats), current_stream(logits)),
          "dcn_scores_forward");
    if (keep) kept = {in[0], tokens, stats, best_tokens};
    return {logprob, entropy, best, best_tokens};
}

variable_list scores_backward(const Numbers& n, const variable_list& kept, const variable_list& grads, const std::vector<bool>&) {
    const int64_t rows = product(without_last(kept[0]));
    const Tensor logits = rows_of(kept[0], rows, kept[0].size(-1));
    const dcn_logits p = logits_of(n, logits, rows);
    Tensor g[3];
    for (int i = 0; i < 3; ++i)
        if (grads[i].defined()) g[i] = grads[i].contiguous();
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor dlogits = at::empty(kept[0].sizes(), logits.options());
    Range range("dcn_scores_backward");
    check(dcn_scores_backward(&p, ptr(logits), iptr(kept[1]), n.ignore, n.top, iptr(kept[3]), fptr(kept[2]), fptr(g[0]), fptr(g[1]),
                              fptr(g[2]), wptr(dlogits), current_stream(logits)),
          "dcn_scores_backward");
    return {dlogits};
}

// logits, teacher_logprobs, teacher_tokens -> loss
variable_list distill_forward(const Numbers& n, const variable_list& in, bool keep, variable_list& kept) {
    check_logits(n, in[0]);
    if (in[0].size(-1) > DCN_DISTILL_MOST_VOCAB)
        fail("the vocabulary is limited to " + std::to_string((int)DCN_DISTILL_MOST_VOCAB) + " tokens");
    const std::vector<int64_t> lead = without_last(in[0]);
    beside(in[1], "teacher_logprobs", in[0], "logits");
    beside(in[2], "teacher_tokens", in[0], "logits");
    if (in[2].dim() != in[0].dim() || without_last(in[2]) != lead)
        fail("teacher_tokens have shape " + shape_text(in[2].sizes()) + ", expected " + shape_text(lead) + " and the teacher's places");
    shaped(in[1], "teacher_logprobs", in[2].sizes());
    if (in[1].scalar_type() != at::kFloat) typed(in[1], "teacher_logprobs", in[0].scalar_type(), "logits (or torch.float32)");
    const int64_t k = in[2].size(-1), rows = product(lead);
    if (k < 1 || k > DCN_DISTILL_MOST_K)
        fail("the teacher has " + std::to_string(k) + " places: 1 to " + std::to_string((int)DCN_DISTILL_MOST_K) + " are supported");
    const Tensor tokens = whole_numbers(in[2], "teacher_tokens");
    const Tensor logits = rows_of(in[0], rows, in[0].size(-1)), teacher = in[1].contiguous();
    const dcn_logits p = logits_of(n, logits, rows);
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor loss = floats(lead, logits), stats = keep ? floats({rows, DCN_LOGITS_STATS}, logits) : Tensor();
    Range range("dcn_distill_forward");
    check(dcn_distill_forward(&p, ptr(logits), (int32_t)k, ptr(teacher), type_of(teacher, "teacher_logprobs"), iptr(tokens),
                              n.tail ? 1 : 0, fptr(loss), fptr(stats), current_stream(logits)),
          "dcn_distill_forward");
    if (keep) kept = {in[0], teacher.detach(), tokens, stats};
    return {loss};
}

variable_list distill_backward(const Numbers& n, const variable_list& kept, const variable_list& grads, const std::vector<bool>&) {
    const int64_t rows = product(without_last(kept[0]));
    const Tensor logits = rows_of(kept[0], rows, kept[0].size(-1)), dloss = grads[0].contiguous();
    const dcn_logits p = logits_of(n, logits, rows);
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor dlogits = at::empty(kept[0].sizes(), logits.options());
    Range range("dcn_distill_backward");
    check(dcn_distill_backward(&p, ptr(logits), (int32_t)kept[2].size(-1), ptr(kept[1]), type_of(kept[1], "teacher_logprobs"),
                               iptr(kept[2]), n.tail ? 1 : 0, fptr(kept[3]), fptr(dloss), wptr(dlogits), current_stream(logits)),
          "dcn_distill_backward");
    return {dlogits};
}

const Operator kScan = {"gated_scan", "GatedScanFunctionBackward", 4, 3, scan_forward, scan_backward};
const Operator kNorm = {"residual_norm", "ResidualNormFunctionBackward", 6, 6, norm_forward, norm_backward};
const Operator kScores = {"token_scores", "TokenScoresFunctionBackward", 2, 1, scores_forward, scores_backward};
const Operator kDistill = {"distill_topk", "DistillTopkFunctionBackward", 3, 1, distill_forward, distill_backward};

// ---- the graph node -------------------------------------------------------------------------------------------------------
struct SequenceBackward : public Node {
    const Operator* op = nullptr;
    Numbers numbers;
    std::vector<SavedVariable> saved;
    std::vector<bool> has;               // inputs the call had; their edges come in slot order
    bool freed = false;

    std::string name() const override { return op->node; }

    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        if (freed)
            throw std::runtime_error("Trying to backward through the graph a second time (the saved tensors have already "
                                     "been freed). Specify retain_graph=True if you need to backward a second time.");
        std::vector<bool> want(op->differentiable);
        size_t edge = 0;
        bool any = false, differentiated = false;
        for (int s = 0; s < op->differentiable; ++s)
            if (has[s]) want[s] = task_should_compute_output(edge++);
        for (const Tensor& g : grads) {
            any = any || g.defined();
            differentiated = differentiated || (at::GradMode::is_enabled() && g.defined() && g.requires_grad());
        }
        variable_list by_slot(op->differentiable);
        if (any) try {
            const auto self = shared_from_this();
            variable_list kept;
            for (auto& v : saved) kept.push_back(v.unpack(self));
            at::NoGradGuard no_grad;
            by_slot = op->backward(numbers, kept, in_memory(grads), want);
        } catch (const DcnFailure& e) {
            pybind11::gil_scoped_acquire gil;
            PyErr_SetString(g_error, e.text.c_str());
            python_error err;
            err.persist();
            throw std::move(err);
        }
        variable_list out;
        for (int s = 0; s < op->differentiable; ++s)
            if (has[s]) out.push_back(by_slot[s]);
        if (differentiated) {            // gradients of gradients are refused when they are asked for
            auto later = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)out.size());
            for (auto& v : out)
                if (v.defined()) v.requires_grad_(true);
            out = (*later)(std::move(out));
        }
        return out;
    }

    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        freed = true;
        for (auto& v : saved) v.reset_data();
    }
};

variable_list call(const Operator& op, const Numbers& n, const variable_list& in) {
    bool need = false;
    for (int i = 0; i < op.differentiable; ++i) need = need || (in[i].defined() && in[i].requires_grad());
    need = need && at::GradMode::is_enabled();
    for (size_t i = op.differentiable; i < in.size(); ++i)
        if (in[i].defined() && in[i].requires_grad() && at::GradMode::is_enabled())
            fail(std::string("there is no gradient with respect to ") + (&op == &kDistill ? "the teacher" : "this input") +
                 ": detach it");
    variable_list kept;
    if (!need) {
        at::NoGradGuard no_grad;
        return op.forward(n, in, false, kept);
    }
    auto node = std::shared_ptr<SequenceBackward>(new SequenceBackward(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    for (int i = 0; i < op.differentiable; ++i) {
        node->has.push_back(in[i].defined());
        if (in[i].defined())
            edges.push_back(in[i].requires_grad() ? torch::autograd::impl::gradient_edge(in[i]) : torch::autograd::Edge());
    }
    node->set_next_edges(std::move(edges));
    node->op = &op;
    node->numbers = n;
    variable_list out;
    {
        at::NoGradGuard no_grad;
        out = op.forward(n, in, true, kept);
    }
    for (const Tensor& t : kept) node->saved.push_back(SavedVariable(t, false));
    // every output of the forward function is one of the node, so that gradients come back by position
    for (Tensor& t : out) {
        if (t.defined() && t.is_floating_point()) torch::autograd::set_history(t, node);
        else node->add_input_metadata(Node::undefined_input());
    }
    return out;
}

bool inside_transform() {
    return torch::jit::tracer::isTracing() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

bool transformed(const variable_list& in) {
    if (inside_transform()) return true;
    for (const Tensor& v : in)
        if (has_tangent(v)) return true;
    return false;
}

// ---- arguments ------------------------------------------------------------------------------------------------------------
double float_arg(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

int32_t small_arg(PyObject* o) {
    const int64_t v = int_arg(o);
    if (v < -2147483647ll || v > 2147483647ll) fail("value out of range");
    return (int32_t)v;
}

PyObject* wrap(variable_list&& v, bool single) {
    if (single) return THPVariable_Wrap(std::move(v[0]));
    PyObject* t = PyTuple_New((Py_ssize_t)v.size());
    if (t == nullptr) throw python_error();
    for (size_t i = 0; i < v.size(); ++i) {
        PyObject* o = v[i].defined() ? THPVariable_Wrap(std::move(v[i])) : (Py_INCREF(Py_None), Py_None);
        if (o == nullptr) {
            Py_DECREF(t);
            throw python_error();
        }
        PyTuple_SET_ITEM(t, (Py_ssize_t)i, o);
    }
    return t;
}

template <typename F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const DcnFailure& e) {
        PyErr_SetString(g_error, e.text.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// The operator's tensors and numbers from a call's arguments
Numbers numbers_of(const Operator& op, PyObject* const* a, Py_ssize_t n, variable_list& in) {
    Numbers m;
    auto tensors = [&](std::initializer_list<const char*> names, int required) {
        int i = 0;
        for (const char* name : names) {
            in.push_back(i < n ? in_memory(tensor_arg(a[i], name, i >= required)) : Tensor());
            ++i;
        }
    };
    if (&op == &kScan) {
        count_arg(n, 2, 4);
        tensors({"x", "gate", "state", "lengths"}, 2);
    } else if (&op == &kNorm) {
        count_arg(n, 1, 7);
        tensors({"x", "block", "gate", "scale", "post_weight", "pre_weight"}, 1);
        if (n > 6) m.eps = float_arg(a[6]);
    } else if (&op == &kScores) {
        count_arg(n, 1, 5);
        tensors({"logits", "tokens"}, 1);
        if (n > 2) m.top = small_arg(a[2]);
        if (n > 3) m.temperature = float_arg(a[3]);
        if (n > 4) m.ignore = int_arg(a[4]);
    } else {
        count_arg(n, 3, 5);
        tensors({"logits", "teacher_logprobs", "teacher_tokens"}, 3);
        if (n > 3) m.temperature = float_arg(a[3]);
        if (n > 4) {
            const int tail = PyObject_IsTrue(a[4]);
            if (tail < 0) throw python_error();
            m.tail = tail != 0;
        }
    }
    return m;
}

template <const Operator* op>
PyObject* apply(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        variable_list in;
        const Numbers m = numbers_of(*op, a, n, in);
        if (transformed(in)) Py_RETURN_NOTIMPLEMENTED;         // sequence.py takes the other way
        variable_list out;
        {
            pybind11::gil_scoped_release no_gil;
            out = call(*op, m, in);
        }
        return wrap(std::move(out), op == &kDistill);
    });
}

// For the Functions of sequence.py: (outputs, kept) of a forward pass ...
template <const Operator* op>
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        variable_list in, kept, out;
        const Numbers m = numbers_of(*op, a, n, in);
        {
            pybind11::gil_scoped_release no_gil;
            at::NoGradGuard no_grad;
            out = op->forward(m, in, true, kept);
        }
        PyObject* o = wrap(std::move(out), false);
        PyObject* k = wrap(std::move(kept), false);
        return Py_BuildValue("(NN)", o, k);
    });
}

// ... and the gradients by slot: (kept, grads, want, call's arguments)
template <const Operator* op>
PyObject* backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count_arg(n, 4, 4);
        for (int i = 0; i < 4; ++i)
            if (!PyTuple_Check(a[i])) {
                PyErr_SetString(PyExc_TypeError, "expected four tuples");
                throw python_error();
            }
        auto tensors = [](PyObject* t) {
            variable_list v;
            for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(t); ++i) v.push_back(tensor_arg(PyTuple_GET_ITEM(t, i), "saved", true));
            return v;
        };
        const variable_list kept = tensors(a[0]), grads = tensors(a[1]);
        std::vector<bool> want;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[2]); ++i) want.push_back(PyObject_IsTrue(PyTuple_GET_ITEM(a[2], i)) == 1);
        std::vector<PyObject*> args;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[3]); ++i) args.push_back(PyTuple_GET_ITEM(a[3], i));
        variable_list in;
        const Numbers m = numbers_of(*op, args.data(), (Py_ssize_t)args.size(), in);
        bool any = false;
        for (const Tensor& g : grads) any = any || g.defined();
        if ((int)want.size() != op->differentiable || !any) fail("no gradient is asked for");
        variable_list out;
        {
            pybind11::gil_scoped_release no_gil;
            at::NoGradGuard no_grad;
            out = op->backward(m, kept, in_memory(grads), want);
        }
        return wrap(std::move(out), false);
    });
}

// (x, gate, state, slots): one step, the state in place.  kInner: for the Function of sequence.py
template <bool kInner>
PyObject* scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count_arg(n, 3, 4);
        const Tensor x0 = in_memory(tensor_arg(a[0], "x")), gate0 = in_memory(tensor_arg(a[1], "gate"));
        const Tensor state = tensor_arg(a[2], "state"), slots0 = n > 3 ? in_memory(tensor_arg(a[3], "slots", true)) : Tensor();
        if (at::GradMode::is_enabled() && (x0.requires_grad() || gate0.requires_grad() || state.requires_grad()))
            fail("step has no gradient: call it under torch.no_grad(), or take apply");
        if (has_tangent(x0) || has_tangent(gate0) || has_tangent(state))         // (before the state advances)
            fail("step has no derivative: take apply");
        if (!kInner && inside_transform()) Py_RETURN_NOTIMPLEMENTED;
        pybind11::gil_scoped_release no_gil;
        at::NoGradGuard no_grad;
        on_gpu(x0, "x");
        const int32_t type = type_of(x0, "x");
        if (x0.dim() != 2) fail("x has shape " + shape_text(x0.sizes()) + ", expected (rows, channels)");
        beside(gate0, "gate", x0, "x");
        beside(state, "state", x0, "x");
        beside(slots0, "slots", x0, "x");
        typed(gate0, "gate", x0.scalar_type(), "x");
        shaped(gate0, "gate", x0.sizes());
        typed(state, "state", at::kFloat);
        if (state.dim() != 2 || state.size(1) != x0.size(1) || !state.is_contiguous() || state.is_neg())
            fail("state has shape " + shape_text(state.sizes()) + ", expected a contiguous (pool, " + std::to_string(x0.size(1)) + ")");
        shaped(slots0, "slots", {x0.size(0)});
        if (!slots0.defined() && state.size(0) < x0.size(0)) fail("state has fewer rows than x, and no slots are given");
        const Tensor x = dense_last(x0), gate = dense_last(gate0), slots = whole_numbers(slots0, "slots");
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor y = at::empty(x.sizes(), x.options());
        state.unsafeGetTensorImpl()->bump_version();             // (refuses an inference tensor outside inference mode: nothing ran)
        {
            Range range("dcn_scan_step");
            check(dcn_scan_step(type, x.size(0), x.size(1), ptr(x), x.stride(0), ptr(gate), gate.stride(0), fptr(state),
                                state.size(0), iptr(slots), wptr(y), current_stream(x)),
                  "dcn_scan_step");
        }
        pybind11::gil_scoped_acquire gil;
        return THPVariable_Wrap(std::move(y));
    });
}

}  // namespace

PyMethodDef dcn_host::sequence_methods[] = {
    {"gated_scan", DCN_FAST(apply<&kScan>), nullptr},
    {"gated_scan_forward", DCN_FAST(forward<&kScan>), nullptr},
    {"gated_scan_backward", DCN_FAST(backward<&kScan>), nullptr},
    {"gated_scan_step", DCN_FAST(scan_step<false>), nullptr},
    {"gated_scan_step_forward", DCN_FAST(scan_step<true>), nullptr},
    {"residual_norm", DCN_FAST(apply<&kNorm>), nullptr},
    {"residual_norm_forward", DCN_FAST(forward<&kNorm>), nullptr},
    {"residual_norm_backward", DCN_FAST(backward<&kNorm>), nullptr},
    {"token_scores", DCN_FAST(apply<&kScores>), nullptr},
    {"token_scores_forward", DCN_FAST(forward<&kScores>), nullptr},
    {"token_scores_backward", DCN_FAST(backward<&kScores>), nullptr},
    {"distill_topk", DCN_FAST(apply<&kDistill>), nullptr},
    {"distill_topk_forward", DCN_FAST(forward<&kDistill>), nullptr},
    {"distill_topk_backward", DCN_FAST(backward<&kDistill>), nullptr},
    {nullptr, nullptr, 0, nullptr},
};
