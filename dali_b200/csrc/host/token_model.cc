// op:: operators of a token model: layer normalisation, token log probabilities, gradient clipping.  Each is a KernelCall
// (expression.h) that hands its evaluated arguments to an entry point of the C ABI (include/dali_b200.h).
//
// Types: results with the rows' shape have the rows' type; arguments of another type are widened to the one the operator
// computes in (never narrowed).  Shards: rows may be spread over the ranks, their last axis may not; what is summed over the rows is
// combined over the ranks, as a reduction over the sharded axis is.
#include <algorithm>
#include <cmath>

#include "../../../include/dali_b200.h"
#include "../op_host.h"
#include "dali/array/op.h"
#include "dali/array/expression/expression.h"

// ---------------------------------------------------------------- calls and their results
KernelResult::KernelResult(const std::shared_ptr<KernelCall>& call, int index)
    : Expression(N_KERNEL, call->results_[index].shape, call->results_[index].dtype, {}), call_(call), index_(index) {
    for (const Array& a : call->inputs_)
        if (!a.is_stateless()) arguments_.push_back(a);
    shard_ = call->results_[index].shard;
}

std::vector<Array> KernelCall::lazy_results(const std::shared_ptr<KernelCall>& call) {
    std::vector<Array> out;
    call->nodes_.clear();
    for (int i = 0; i < (int)call->results_.size(); ++i) {
        std::shared_ptr<KernelResult> node = std::make_shared<KernelResult>(call, i);
        call->nodes_.push_back(node);
        out.push_back(Array(node));
    }
    return out;
}

Array KernelCall::take(int index) {
    if (computed_.empty() || computed_[index].is_stateless()) {
        const bool all = collective();
        std::vector<Array> in, out;
        Array on;
        for (const Array& a : inputs_) {
            if (a.is_stateless()) { in.push_back(Array()); continue; }
            if (on.is_stateless()) on = a;
            Array b = a;
            if (!b.is_buffer()) b.eval(false);
            in.push_back(b);
        }
        const memory::Device device = on.is_stateless() ? memory::default_preferred_device : on.preferred_device();
        for (int i = 0; i < (int)results_.size(); ++i) {
            const Result& r = results_[i];
            if (i != index && !all && nodes_[i].expired()) { out.push_back(Array()); continue; }
            Array a(r.shape, r.dtype, device);
            a.expression()->shard_ = r.shard;
            out.push_back(a);
        }
        if (!lazy::dry_run()) lazy::device_index(device);      // binds the GPU, or says that there is none
        run(device, in, out);
        ++lazy::stats().kernels;
        lazy::stats().last_variant = name();
        computed_ = out;
    }
    Array mine = computed_[index];
    computed_[index] = Array();
    return mine;
}

namespace {

std::string shape_str(const std::vector<int>& s) {
    std::string o = "[";
    for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
    return o + "]";
}

void require_floating(const Array& a, const std::string& what) {
    DALI_ASSERT(!a.is_stateless(), what + " of a stateless Array");
    DALI_ASSERT(a.dtype() != DTYPE_INT32, what + " takes float, double or bfloat16 arrays (got " + dtype_to_name(a.dtype()) + ")");
}

void note_collective(const std::string& what) {
    ++lazy::stats().collectives;
    lazy::stats().last_collective = what;
}

// A buffer as rows along its last axis with one stride between them (a copy where its strides do not allow that).
struct RowView {
    Array keep;
    int64_t rows = 0, cols = 0, stride = 0;
    const void* data = nullptr;
};
Array as_rows(const Array& a) {
    BufferView* b = as<BufferView>(a);
    if (b->contiguous()) return a;
    if (b->ndim() == 2) {
        const std::vector<int> st = b->normalized_strides();
        if (st[1] == 1 && (st[0] >= b->shape_[1] || b->shape_[0] == 1)) return a;
    }
    Array c = a.ascontiguousarray();
    if (!c.is_buffer()) c.eval(false);
    return c;
}
RowView rows_of(const Array& a, const memory::Device& device) {
    RowView v;
    v.keep = as_rows(a);
    BufferView* b = as<BufferView>(v.keep);
    v.cols = b->ndim() ? b->shape_.back() : 1;
    v.rows = v.cols ? b->numel() / v.cols : 0;
    v.stride = b->contiguous() || v.rows < 2 ? v.cols : b->normalized_strides()[0];
    v.data = (const char*)b->memory_->data(device, memory::AM_READONLY) + b->offset_ * size_of_dtype(b->dtype_);
    return v;
}
// a small argument, contiguous; nullptr for a stateless one.  `keep` holds a copy until the launch has been queued (device
// memory is recycled in stream order).
const void* vector_of(const Array& a, const memory::Device& device, std::vector<Array>* keep) {
    if (a.is_stateless()) return nullptr;
    Array c = a;
    if (!as<BufferView>(c)->contiguous()) {
        c = a.ascontiguousarray();
        if (!c.is_buffer()) c.eval(false);
    }
    keep->push_back(c);
    BufferView* b = as<BufferView>(c);
    return (const char*)b->memory_->data(device, memory::AM_READONLY) + b->offset_ * size_of_dtype(b->dtype_);
}
void* written(const Array& a, const memory::Device& device) {
    return a.is_stateless() ? nullptr : as<BufferView>(a)->memory_->data(device, memory::AM_OVERWRITE);
}

DType widest(std::initializer_list<Array> arrays) {
    DType t = DTYPE_BF16;
    for (const Array& a : arrays) {
        if (a.is_stateless()) continue;
        if (a.dtype() == DTYPE_DOUBLE) return DTYPE_DOUBLE;
        if (a.dtype() == DTYPE_FLOAT) t = DTYPE_FLOAT;
    }
    return t;
}
Array widened(const Array& a, DType t) { return a.is_stateless() || a.dtype() == t ? a : op::unsafe_cast(a, t); }

// ---------------------------------------------------------------- layer norm
struct LayerNormCall : public KernelCall {
    double eps_;
    std::string name() const override { return "layer_norm"; }
    void run(const memory::Device& device, const std::vector<Array>& in, const std::vector<Array>& out) override {
        if (lazy::dry_run()) return;
        std::vector<Array> keep;
        const RowView x = rows_of(in[0], device);
        const void *gamma = vector_of(in[1], device, &keep), *beta = vector_of(in[2], device, &keep);
        const DType t = in[0].dtype(), w = !in[1].is_stateless() ? in[1].dtype() : !in[2].is_stateless() ? in[2].dtype() : t;
        lazy::check(dalib200_layer_norm(lazy::device_index(device), nullptr, t, w, x.rows, x.cols, x.data, x.stride, gamma, beta, eps_,
                                        written(out[0], device), x.cols),
                    "dalib200_layer_norm");
    }
};

struct LayerNormBackwardCall : public KernelCall {
    double eps_;
    DType weights_;
    bool combine_ = false;
    std::string name() const override { return "layer_norm_backward"; }
    bool collective() const override { return combine_; }
    void run(const memory::Device& device, const std::vector<Array>& in, const std::vector<Array>& out) override {
        if (combine_)
            for (int i = 1; i < 3; ++i) note_collective("allreduce sum " + std::to_string(out[i].numel()) + " (gradient of a weight of sharded rows)");
        if (lazy::dry_run()) return;
        std::vector<Array> keep;
        const RowView dy = rows_of(in[0], device), x = rows_of(in[1], device);
        const void* gamma = vector_of(in[2], device, &keep);
        const int dev = lazy::device_index(device);
        void *dx = written(out[0], device), *dg = written(out[1], device), *db = written(out[2], device);
        lazy::check(dalib200_layer_norm_backward(dev, nullptr, in[1].dtype(), weights_, x.rows, x.cols, dy.data, dy.stride, x.data, x.stride,
                                                 gamma, eps_, dx, x.cols, dg, db, nullptr, 0),
                    "dalib200_layer_norm_backward");
        if (!combine_) return;
        for (void* p : {dg, db})
            lazy::check(dalib200_allreduce(dev, nullptr, p, x.cols, weights_, DALIB200_OP_SUM), "dalib200_allreduce");
    }
};

// the type of the rows (`t`) and of the weights beside them
DType weights_type(DType t, std::initializer_list<Array> weights) {
    if (t != DTYPE_BF16) return t;
    for (const Array& w : weights)
        if (!w.is_stateless() && w.dtype() != DTYPE_BF16) return DTYPE_FLOAT;
    return DTYPE_BF16;
}

void check_weight(const Array& w, const Array& x, const char* op, const char* name) {
    if (w.is_stateless()) return;
    require_floating(w, std::string(op) + "'s " + name);
    DALI_ASSERT(w.ndim() == 1 && w.shape()[0] == x.shape().back(),
                std::string(op) + ": " + name + " must be a vector of the last axis' length " + std::to_string(x.shape().back()) +
                    " (got " + name + ".shape = " + shape_str(w.shape()) + ")");
    DALI_ASSERT(!w.shard().sharded(), std::string(op) + ": " + name + " must not be sharded");
}

void check_rows(const Array& x, const char* op) {
    require_floating(x, op);
    DALI_ASSERT(x.ndim() > 0, std::string(op) + " needs an array with a last axis (got a scalar)");
    DALI_ASSERT(x.shard().axis != x.ndim() - 1, std::string(op) + " along the sharded axis is not supported (each rank holds only its part of every row)");
}

// ---------------------------------------------------------------- token log probabilities
struct TokenLogprobsCall : public KernelCall {
    int top_;
    std::string name() const override { return "token_logprobs"; }
    void run(const memory::Device& device, const std::vector<Array>& in, const std::vector<Array>& out) override {
        if (lazy::dry_run()) return;
        std::vector<Array> keep;
        const RowView z = rows_of(in[0], device);
        const void* tokens = vector_of(in[1], device, &keep);
        // a list of alternatives comes whole
        Array values = out[3], index = out[4];
        if (top_ > 0 && values.is_stateless() && !index.is_stateless()) keep.push_back(values = Array(index.shape(), results_[3].dtype, device));
        if (top_ > 0 && index.is_stateless() && !values.is_stateless()) keep.push_back(index = Array(values.shape(), DTYPE_INT32, device));
        const int top = values.is_stateless() ? 0 : top_;
        lazy::check(dalib200_token_logprobs(lazy::device_index(device), nullptr, in[0].dtype(), z.rows, z.cols, z.data, z.stride,
                                            (const int32_t*)tokens, written(out[0], device), written(out[1], device),
                                            written(out[2], device), top, written(values, device), (int32_t*)written(index, device)),
                    "dalib200_token_logprobs");
    }
};

struct TokenLogprobsBackwardCall : public KernelCall {
    std::string name() const override { return "token_logprobs_backward"; }
    void run(const memory::Device& device, const std::vector<Array>& in, const std::vector<Array>& out) override {
        if (lazy::dry_run()) return;
        std::vector<Array> keep;
        const RowView z = rows_of(in[0], device);
        const void* v[5];
        for (int i = 0; i < 5; ++i) v[i] = vector_of(in[i + 1], device, &keep);
        lazy::check(dalib200_token_logprobs_backward(lazy::device_index(device), nullptr, in[0].dtype(), z.rows, z.cols, z.data, z.stride,
                                                     (const int32_t*)v[0], v[1], v[2], v[3], v[4], written(out[0], device), z.cols),
                    "dalib200_token_logprobs_backward");
    }
};

std::vector<int> leading(const Array& a) { return std::vector<int>(a.shape().begin(), a.shape().end() - 1); }

void check_per_row(const Array& a, const Array& logits, const char* op, const char* name) {
    if (a.is_stateless()) return;
    DALI_ASSERT(a.shape() == leading(logits), std::string(op) + ": " + name + " must have one value per row of logits (expected shape " +
                                                  shape_str(leading(logits)) + ", got " + shape_str(a.shape()) + ")");
    DALI_ASSERT(!a.shard().sharded() || a.shard() == logits.shard(), std::string(op) + ": " + name + " is sharded differently from logits");
}
void check_tokens(const Array& tokens, const Array& logits, const char* op) {
    if (tokens.is_stateless()) return;
    DALI_ASSERT(tokens.dtype() == DTYPE_INT32, std::string(op) + ": tokens must be integers (got dtype=" + dtype_to_name(tokens.dtype()) + ").");
    check_per_row(tokens, logits, op, "tokens");
}

// ---------------------------------------------------------------- norms of lists
struct ListCall : public KernelCall {
    bool clip_;
    double max_norm_ = 0;
    std::string name() const override { return clip_ ? "clip_by_global_norm" : "global_norm"; }
    bool collective() const override {
        for (const Array& a : inputs_)
            if (a.shard().sharded()) return true;
        return false;
    }
    // inputs: the list; results: (clipped arrays,) norm
    void run(const memory::Device& device, const std::vector<Array>& in, const std::vector<Array>& out) override {
        std::vector<int> dtypes[2];
        std::vector<int64_t> numel[2];
        std::vector<const void*> from[2];
        std::vector<void*> to;
        std::vector<Array> keep;
        const bool sharded = collective();
        if (sharded) note_collective("allreduce sum 1 f64 (squares of sharded arrays)");
        if (lazy::dry_run()) return;
        const int dev = lazy::device_index(device);
        std::vector<int> all_dtypes;
        std::vector<int64_t> all_numel;
        std::vector<const void*> all_from;
        for (size_t i = 0; i < in.size(); ++i) {
            const void* p = vector_of(in[i], device, &keep);
            const int part = in[i].shard().sharded() ? 1 : 0;
            dtypes[part].push_back(in[i].dtype());
            numel[part].push_back(in[i].numel());
            from[part].push_back(p);
            all_dtypes.push_back(in[i].dtype());
            all_numel.push_back(in[i].numel());
            all_from.push_back(p);
            if (clip_) {
                Array o = out[i];
                if (o.is_stateless()) continue;
                to.push_back(written(o, device));
            }
        }
        // only what is still wanted is scaled; the norm is that of all
        std::vector<int> want_dtypes;
        std::vector<int64_t> want_numel;
        std::vector<const void*> want_from;
        for (size_t i = 0; clip_ && i < in.size(); ++i)
            if (!out[i].is_stateless()) {
                want_dtypes.push_back(all_dtypes[i]);
                want_numel.push_back(all_numel[i]);
                want_from.push_back(all_from[i]);
            }
        Array norm = out.back();
        if (norm.is_stateless()) keep.push_back(norm = Array(std::vector<int>(), results_.back().dtype, device));
        void* pn = written(norm, device);
        const int n = (int)all_from.size();
        if (!sharded && !clip_) {
            lazy::check(dalib200_global_norm(dev, nullptr, n, all_dtypes.data(), all_numel.data(), all_from.data(), norm.dtype(), pn, nullptr, 0),
                        "dalib200_global_norm");
            return;
        }
        if (!sharded && want_from.size() == all_from.size()) {
            lazy::check(dalib200_clip_by_global_norm(dev, nullptr, n, all_dtypes.data(), all_numel.data(), all_from.data(), to.data(), max_norm_,
                                                     norm.dtype(), pn, nullptr, 0),
                        "dalib200_clip_by_global_norm");
            return;
        }
        // the sum of squares by itself: of the whole arrays, and of the shards, which the ranks add up
        Array sums(std::vector<int>({2}), DTYPE_DOUBLE, device);
        double* ps = (double*)written(sums, device);
        for (int part = 0; part < 2; ++part)
            lazy::check(dalib200_sum_squares(dev, nullptr, (int)from[part].size(), dtypes[part].data(), numel[part].data(), from[part].data(),
                                             ps + part, nullptr, 0),
                        "dalib200_sum_squares");
        if (sharded) lazy::check(dalib200_allreduce(dev, nullptr, ps + 1, 1, DTYPE_DOUBLE, DALIB200_OP_SUM), "dalib200_allreduce");
        Array total = op::sum(sums);
        total.eval(false);
        lazy::run_assignment(norm, OPERATOR_T_EQL, op::unsafe_cast(op::sqrt(total), norm.dtype()));
        if (clip_) {
            BufferView* b = as<BufferView>(total);
            const double* pt = (const double*)b->memory_->data(device, memory::AM_READONLY) + b->offset_;
            lazy::check(dalib::scale_to_norm(dev, nullptr, (int)want_from.size(), want_dtypes.data(), want_numel.data(), want_from.data(),
                                             to.data(), pt, max_norm_, norm.dtype()),
                        "dalib200_scale_to_norm");
        }
    }
};

std::shared_ptr<ListCall> list_call(const std::vector<Array>& arrays, bool clip, const char* op) {
    std::shared_ptr<ListCall> call = std::make_shared<ListCall>();
    call->clip_ = clip;
    DType t = DTYPE_FLOAT;
    for (size_t i = 0; i < arrays.size(); ++i) {
        const Array& a = arrays[i];
        require_floating(a, op);
        if (a.dtype() == DTYPE_DOUBLE) t = DTYPE_DOUBLE;
        call->inputs_.push_back(a);
        if (clip) call->results_.push_back({std::to_string(i), a.shape(), a.dtype(), a.shard()});
    }
    call->results_.push_back({"norm", {}, t, Shard()});
    return call;
}

}  // namespace

namespace op {

Array layer_norm(const Array& x, const Array& gamma, const Array& beta, double eps) {
    check_rows(x, "layer_norm");
    check_weight(gamma, x, "layer_norm", "gamma");
    check_weight(beta, x, "layer_norm", "beta");
    DALI_ASSERT(eps >= 0 && std::isfinite(eps), "layer_norm: eps must be a number >= 0");
    const DType t = widest({x}) == DTYPE_DOUBLE || widest({gamma}) == DTYPE_DOUBLE || widest({beta}) == DTYPE_DOUBLE ? DTYPE_DOUBLE : x.dtype();
    const DType w = weights_type(t, {gamma, beta});
    std::shared_ptr<LayerNormCall> call = std::make_shared<LayerNormCall>();
    call->eps_ = eps;
    call->inputs_ = {widened(x, t), widened(gamma, w), widened(beta, w)};
    call->results_ = {{"y", x.shape(), t, x.shard()}};
    return KernelCall::lazy_results(call)[0];
}

std::tuple<Array, Array, Array> layer_norm_backward(const Array& dy, const Array& x, const Array& gamma, double eps) {
    const char* op = "layer_norm_backward";
    check_rows(x, op);
    check_rows(dy, op);
    check_weight(gamma, x, op, "gamma");
    DALI_ASSERT(eps >= 0 && std::isfinite(eps), "layer_norm_backward: eps must be a number >= 0");
    DALI_ASSERT(dy.shape() == x.shape(), "layer_norm_backward: dy must have x's shape (got dy.shape = " + shape_str(dy.shape()) +
                                             ", x.shape = " + shape_str(x.shape()) + ")");
    DALI_ASSERT(dy.shard() == x.shard(), "layer_norm_backward: dy and x are sharded differently");
    const bool sharded = x.shard().sharded();
    const DType t = widest({gamma}) == DTYPE_DOUBLE && !gamma.is_stateless() ? DTYPE_DOUBLE : widest({dy, x});
    // (the ranks' sums are added in fp32 at least)
    const DType w = t == DTYPE_BF16 && sharded ? DTYPE_FLOAT : weights_type(t, {gamma});
    std::shared_ptr<LayerNormBackwardCall> call = std::make_shared<LayerNormBackwardCall>();
    call->eps_ = eps;
    call->weights_ = w;
    call->combine_ = sharded;
    call->inputs_ = {widened(dy, t), widened(x, t), widened(gamma, w)};
    const std::vector<int> cols = {x.shape().back()};
    call->results_ = {{"dx", x.shape(), t, x.shard()}, {"dgamma", cols, w, Shard()}, {"dbeta", cols, w, Shard()}};
    const std::vector<Array> r = KernelCall::lazy_results(call);
    return std::tuple<Array, Array, Array>(r[0], r[1], r[2]);
}

TokenLogprobs token_logprobs(const Array& logits, const Array& tokens, int top) {
    const char* op = "token_logprobs";
    check_rows(logits, op);
    check_tokens(tokens, logits, op);
    const int vocab = logits.shape().back();
    DALI_ASSERT(vocab > 0, "token_logprobs: the vocabulary is empty");
    DALI_ASSERT(top >= 0 && top <= DALIB200_MAX_TOP && top <= vocab,
                "token_logprobs: top must lie between 0 and " + std::to_string(DALIB200_MAX_TOP) + " and not exceed the vocabulary (got " + std::to_string(top) + ")");
    std::shared_ptr<TokenLogprobsCall> call = std::make_shared<TokenLogprobsCall>();
    call->top_ = top;
    call->inputs_ = {logits, tokens};
    const DType t = value_dtype(logits.dtype());
    const std::vector<int> rows = leading(logits);
    std::vector<int> tops = rows;
    tops.push_back(top);
    const Shard s = logits.shard();
    call->results_ = {{"logprob", rows, t, s}, {"entropy", rows, t, s}, {"lse", rows, t, s}, {"top_logprobs", tops, t, s}, {"top_tokens", tops, DTYPE_INT32, s}};
    const std::vector<Array> r = KernelCall::lazy_results(call);
    TokenLogprobs out;
    if (!tokens.is_stateless()) out.logprob = r[0];
    out.entropy = r[1];
    out.lse = r[2];
    if (top > 0) {
        out.top_logprobs = r[3];
        out.top_tokens = r[4];
    }
    return out;
}

Array token_logprobs_backward(const Array& logits, const Array& tokens, const Array& lse, const Array& entropy, const Array& dlogprob,
                              const Array& dentropy) {
    const char* op = "token_logprobs_backward";
    check_rows(logits, op);
    DALI_ASSERT(logits.shape().back() > 0, "token_logprobs_backward: the vocabulary is empty");
    check_tokens(tokens, logits, op);
    DALI_ASSERT(!lse.is_stateless(), "token_logprobs_backward needs lse");
    DALI_ASSERT(!dlogprob.is_stateless() || !dentropy.is_stateless(), "token_logprobs_backward: neither dlogprob nor dentropy is given");
    DALI_ASSERT(dlogprob.is_stateless() || !tokens.is_stateless(), "token_logprobs_backward: dlogprob needs tokens");
    DALI_ASSERT(dentropy.is_stateless() || !entropy.is_stateless(), "token_logprobs_backward: dentropy needs entropy");
    const struct { const Array& a; const char* name; } rows[] = {{lse, "lse"}, {entropy, "entropy"}, {dlogprob, "dlogprob"}, {dentropy, "dentropy"}};
    DType t = logits.dtype();
    for (const auto& r : rows) {
        if (r.a.is_stateless()) continue;
        require_floating(r.a, std::string(op) + "'s " + r.name);
        check_per_row(r.a, logits, op, r.name);
        if (r.a.dtype() == DTYPE_DOUBLE) t = DTYPE_DOUBLE;
    }
    const DType v = value_dtype(t);
    std::shared_ptr<TokenLogprobsBackwardCall> call = std::make_shared<TokenLogprobsBackwardCall>();
    const bool of_token = !dlogprob.is_stateless(), of_entropy = !dentropy.is_stateless();
    call->inputs_ = {widened(logits, t), of_token ? tokens : Array(), widened(lse, v), of_entropy ? widened(entropy, v) : Array(),
                     widened(dlogprob, v), widened(dentropy, v)};
    call->results_ = {{"dlogits", logits.shape(), t, logits.shard()}};
    return KernelCall::lazy_results(call)[0];
}

Array global_norm(const std::vector<Array>& arrays) { return KernelCall::lazy_results(list_call(arrays, false, "global_norm"))[0]; }

std::tuple<std::vector<Array>, Array> clip_by_global_norm(const std::vector<Array>& arrays, double max_norm) {
    DALI_ASSERT(max_norm > 0, "clip_by_global_norm: max_norm must be a number > 0");
    std::shared_ptr<ListCall> call = list_call(arrays, true, "clip_by_global_norm");
    call->max_norm_ = max_norm;
    std::vector<Array> r = KernelCall::lazy_results(call);
    Array norm = r.back();
    r.pop_back();
    return std::tuple<std::vector<Array>, Array>(r, norm);
}

}  // namespace op
