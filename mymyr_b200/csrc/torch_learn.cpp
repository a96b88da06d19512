// The learner's operators over torch tensors: argument checks, outputs and workspaces from torch's allocator, autograd
// nodes, and the calls of the C ABI (mymyr_b200.h). A module of its own (mymyr_b200/lib/_learn.so) rather than ctypes:
// the kernels of a small batch take 4 to 10 us, and a call with its gradient cost 100 us of host time in Python
// against 50 here (of which torch's engine takes 40).

#include "mymyr_b200.h"

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <cmath>
#include <cstring>
#include <stdexcept>
#include <string>
#include <vector>

namespace
{
using at::Tensor;
using OptTensor = std::optional<Tensor>;
namespace ag = torch::autograd;

struct CapacityError : std::length_error
{
    using std::length_error::length_error;
};

void refuse(bool bad, const char* message)
{
    if (bad)
        throw std::invalid_argument(message);
}

void check(b2_status status)
{
    if (status == B2_OK)
        return;
    std::string m(b2_last_error(nullptr, 0) + 1, '\0');
    b2_last_error(m.data(), m.size());
    m.pop_back();
    if (status == B2_INVALID_ARGUMENT || status == B2_UNSUPPORTED)
        throw std::invalid_argument(m);
    if (status == B2_CAPACITY)
        throw CapacityError(m);
    throw std::runtime_error(m);
}

/// The package's context of a device (mymyr_b200.task.default_context). Called with the interpreter's lock.
b2_ctx* context(int device)
{
    static std::array<b2_ctx*, 64> known{};
    refuse(device < 0 || device >= static_cast<int>(known.size()), "more than 64 devices");
    if (!known[device])
    {
        const py::object c = py::module_::import("mymyr_b200.task").attr("default_context")(device);
        known[device] = reinterpret_cast<b2_ctx*>(c.attr("handle").attr("value").cast<uintptr_t>());
    }
    return known[device];
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

int32_t dtype_of(const Tensor& t, const char* message)
{
    switch (t.scalar_type())
    {
        case at::kFloat: return B2_F32;
        case at::kBFloat16: return B2_BF16;
        case at::kHalf: return B2_F16;
        default: throw std::invalid_argument(message);
    }
}

void floating(const Tensor& t, const char* message)
{
    refuse(!t.defined() || !t.is_cuda(), message);
    dtype_of(t, message);
}

int32_t index_bits(const Tensor& t, const Tensor& with, const char* message)
{
    refuse(t.device() != with.device(), message);
    refuse(t.scalar_type() != at::kLong && t.scalar_type() != at::kInt, message);
    return t.scalar_type() == at::kLong ? 64 : 32;
}

at::ScalarType float_type(int32_t dtype)
{
    return dtype == B2_F32 ? at::kFloat : dtype == B2_BF16 ? at::kBFloat16 : at::kHalf;
}

at::ScalarType index_type(int32_t bits) { return bits == 64 ? at::kLong : at::kInt; }

/// A tensor that the backward pass finds saved, if it is of the type, the sizes and on the device that it had: hooks on
/// saved tensors hand back what they will.
const Tensor& as_saved(const Tensor& t, at::ScalarType type, at::IntArrayRef sizes, at::Device device)
{
    refuse(!t.defined() || t.scalar_type() != type || t.device() != device || t.sizes() != sizes,
           "a saved tensor came back with another type, size or device");
    return t;
}

/// Rows with unit column stride.
Tensor unit_columns(const Tensor& t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }

/// A gradient that is no part of a graph: asking for its own gradient is an error, as with once_differentiable.
Tensor no_further(Tensor g)
{
    if (!at::GradMode::is_enabled())
        return g;
    auto error = std::make_shared<ag::DelayedError>("the learner's operators are differentiable once", 1);
    ag::variable_list in{g.requires_grad_(true)};
    return (*error)(std::move(in))[0];
}

// ---------------------------------------------------------------------------------------------- log-probabilities

struct LogProbsCall
{
    b2_ctx* ctx;
    b2_logprobs_args a{};
    Tensor logits, tokens, offsets, mask;  // what `a` points to
    Tensor logprob, entropy, stats, top_logprobs, top_tokens;

    void forward(bool with_stats)
    {
        const auto rows = static_cast<int64_t>(a.rows), top = static_cast<int64_t>(a.top);
        const auto f32 = logits.options().dtype(at::kFloat);
        entropy = at::empty({rows}, f32);
        a.entropy = entropy.data_ptr<float>();
        if (tokens.defined())
        {
            logprob = at::empty({rows}, f32);
            a.logprob = logprob.data_ptr<float>();
        }
        if (top)
        {
            top_logprobs = at::empty({rows, top}, f32);
            top_tokens = at::empty({rows, top}, logits.options().dtype(at::kLong));
            a.top_logprobs = top_logprobs.data_ptr<float>();
            a.top_tokens = top_tokens.data_ptr<int64_t>();
        }
        if (with_stats)
        {
            stats = at::empty({rows, 4}, f32);
            a.stats = stats.data_ptr<float>();
        }
        check(b2_logprobs(ctx, &a, stream_of(logits)));
    }
};

struct LogProbsNode : ag::Function<LogProbsNode>
{
    static ag::variable_list forward(ag::AutogradContext* node, const Tensor& logits, LogProbsCall* call)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        call->forward(true);
        node->save_for_backward({logits, call->tokens, call->offsets, call->mask, call->stats});
        node->saved_data["args"] = std::string(reinterpret_cast<const char*>(&call->a), sizeof(call->a));
        node->saved_data["ctx"] = reinterpret_cast<int64_t>(call->ctx);
        node->saved_data["device"] = static_cast<int64_t>(logits.get_device());
        node->set_materialize_grads(false);
        ag::variable_list out{call->entropy};
        if (call->logprob.defined())
            out.push_back(call->logprob);
        if (call->top_tokens.defined())
        {
            node->mark_non_differentiable({call->top_logprobs, call->top_tokens});
            out.push_back(call->top_logprobs);
            out.push_back(call->top_tokens);
        }
        return out;
    }

    static ag::variable_list backward(ag::AutogradContext* node, ag::variable_list grads)
    {
        const auto saved = node->get_saved_variables();  // throws where one was changed in place since
        b2_logprobs_args a;
        std::memcpy(&a, node->saved_data["args"].toStringRef().data(), sizeof(a));
        // hooks may have moved them and laid them out anew
        const auto rows = static_cast<int64_t>(a.rows), width = static_cast<int64_t>(a.width);
        const bool ragged = a.offsets;
        const at::Device device(at::kCUDA, static_cast<c10::DeviceIndex>(node->saved_data["device"].toInt()));
        const std::vector<int64_t> shape = ragged ? std::vector<int64_t>{width} : std::vector<int64_t>{rows, width};
        const Tensor logits = unit_columns(as_saved(saved[0], float_type(a.dtype), shape, device));
        const Tensor stats = as_saved(saved[4], at::kFloat, {rows, 4}, device).contiguous();
        a.logits = logits.data_ptr();
        a.row_stride = ragged ? 0 : static_cast<uint64_t>(logits.stride(0));
        a.stats = stats.data_ptr<float>();
        Tensor tokens, offsets, mask;
        if (a.tokens)
        {
            tokens = as_saved(saved[1], index_type(a.token_bits), {rows}, device).contiguous();
            a.tokens = tokens.data_ptr();
        }
        if (ragged)
        {
            offsets = as_saved(saved[2], index_type(a.offsets_bits), {rows + 1}, device).contiguous();
            a.offsets = offsets.data_ptr();
        }
        if (a.mask)
        {
            mask = unit_columns(as_saved(saved[3], at::kBool, shape, device));
            a.mask = static_cast<const uint8_t*>(mask.data_ptr());
            a.mask_stride = ragged ? 0 : static_cast<uint64_t>(mask.stride(0));
        }
        const Tensor entropy = grads[0].defined() ? grads[0].contiguous() : Tensor();
        const Tensor logprob = a.tokens && grads[1].defined() ? grads[1].contiguous() : Tensor();
        Tensor grad;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
            check(b2_logprobs_backward(reinterpret_cast<b2_ctx*>(node->saved_data["ctx"].toInt()), &a,
                                       logprob.defined() ? logprob.data_ptr<float>() : nullptr,
                                       entropy.defined() ? entropy.data_ptr<float>() : nullptr, grad.data_ptr(), a.width,
                                       stream_of(logits)));
        }
        return {no_further(grad), Tensor()};
    }
};

/// logprob, entropy, top_logprobs, top_tokens (undefined ones become None).
std::array<OptTensor, 4> logprobs(Tensor logits, OptTensor tokens, OptTensor offsets, OptTensor mask, double temperature,
                                  int64_t top)
{
    floating(logits, "logprobs: logits must be a CUDA tensor of float32, bfloat16 or float16");
    refuse(!(temperature > 0.0) || !std::isfinite(temperature), "logprobs: temperature must be positive and finite");
    refuse(top < 0 || top > B2_TOP_MAX, "logprobs: top must be between 0 and 32");
    LogProbsCall call{context(logits.get_device())};
    const c10::cuda::CUDAGuard guard(logits.device());
    b2_logprobs_args& a = call.a;
    std::vector<int64_t> shape;
    if (offsets)
    {
        a.offsets_bits = index_bits(*offsets, logits, "logprobs: offsets must be int32 or int64, on the logits' device");
        refuse(logits.dim() != 1 || offsets->dim() != 1 || offsets->numel() < 1,
               "logprobs: with offsets [N + 1], logits must be the rows' one vector");
        shape = {offsets->numel() - 1};
        call.offsets = offsets->contiguous();
        a.offsets = call.offsets.data_ptr();
        logits = logits.contiguous();
        a.rows = static_cast<uint64_t>(shape[0]);
        a.width = static_cast<uint64_t>(logits.numel());
    }
    else
    {
        refuse(logits.dim() < 1, "logprobs: logits must have a dimension of tokens");
        shape.assign(logits.sizes().begin(), logits.sizes().end() - 1);
        const int64_t width = logits.size(-1);
        const int64_t rows = c10::multiply_integers(shape);
        if (logits.dim() != 2)
            logits = logits.reshape({rows, width});
        logits = unit_columns(logits);
        a.rows = static_cast<uint64_t>(rows);
        a.width = static_cast<uint64_t>(width);
        a.row_stride = static_cast<uint64_t>(logits.stride(0));
    }
    a.dtype = dtype_of(logits, "");
    a.temperature = static_cast<float>(temperature);
    a.top = static_cast<uint32_t>(top);
    if (tokens)
    {
        a.token_bits = index_bits(*tokens, logits, "logprobs: tokens must be int32 or int64, on the logits' device");
        refuse(tokens->sizes() != at::IntArrayRef(shape), "logprobs: tokens must have the rows' shape");
        call.tokens = tokens->contiguous();
        if (call.tokens.dim() != 1)
            call.tokens = call.tokens.view({static_cast<int64_t>(a.rows)});
        a.tokens = call.tokens.data_ptr();
    }
    if (mask)
    {
        refuse(mask->device() != logits.device() || mask->scalar_type() != at::kBool,
               "logprobs: mask must be a bool tensor on the logits' device");
        refuse(mask->dim() > static_cast<int64_t>(offsets ? 1 : shape.size() + 1),
               "logprobs: mask does not broadcast to the logits");
        Tensor m = *mask;
        if (offsets)
            m = m.expand(logits.sizes()).contiguous();
        else if (m.dim() <= 1)
            m = unit_columns(m.expand({static_cast<int64_t>(a.width)}).expand(logits.sizes()));
        else
        {
            std::vector<int64_t> full = shape;
            full.push_back(static_cast<int64_t>(a.width));
            m = unit_columns(m.expand(full).reshape(logits.sizes()));
        }
        call.mask = m;
        a.mask = static_cast<const uint8_t*>(m.data_ptr());
        a.mask_stride = offsets ? 0 : static_cast<uint64_t>(m.stride(0));
    }
    a.logits = logits.data_ptr();
    call.logits = logits;
    {
        const py::gil_scoped_release unlocked;
        if (logits.requires_grad() && at::GradMode::is_enabled())
        {
            const ag::variable_list out = LogProbsNode::apply(logits, &call);
            call.entropy = out[0];
            if (tokens)
                call.logprob = out[1];
            if (top)
            {
                call.top_logprobs = out[out.size() - 2];
                call.top_tokens = out[out.size() - 1];
            }
        }
        else
            call.forward(false);
        if (shape.size() != 1)
        {
            call.entropy = call.entropy.view(shape);
            if (tokens)
                call.logprob = call.logprob.view(shape);
            if (top)
            {
                shape.push_back(top);
                call.top_logprobs = call.top_logprobs.view(shape);
                call.top_tokens = call.top_tokens.view(shape);
            }
        }
    }
    auto or_none = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return {or_none(call.logprob), or_none(call.entropy), or_none(call.top_logprobs), or_none(call.top_tokens)};
}

// ---------------------------------------------------------------------------------------------- embeddings

Tensor embedding_forward(b2_ctx* ctx, const b2_embedding_args& a, const Tensor& weight)
{
    const Tensor rows = at::empty({static_cast<int64_t>(a.count), weight.size(1)}, weight.options());
    check(b2_embedding(ctx, &a, weight.data_ptr(), static_cast<uint64_t>(weight.stride(0)), rows.data_ptr(),
                       stream_of(weight)));
    return rows;
}

struct EmbeddingNode : ag::Function<EmbeddingNode>
{
    static Tensor forward(ag::AutogradContext* node, const Tensor& weight, const Tensor& tokens, b2_ctx* ctx,
                          const b2_embedding_args* a)
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        node->save_for_backward({tokens});
        node->saved_data["args"] = std::string(reinterpret_cast<const char*>(a), sizeof(*a));
        node->saved_data["ctx"] = reinterpret_cast<int64_t>(ctx);
        return embedding_forward(ctx, *a, weight);
    }

    static ag::variable_list backward(ag::AutogradContext* node, ag::variable_list grads)
    {
        const auto saved = node->get_saved_variables();
        b2_embedding_args a;
        std::memcpy(&a, node->saved_data["args"].toStringRef().data(), sizeof(a));
        const Tensor grad = unit_columns(grads[0]);
        // hooks may have moved them and laid them out anew
        const Tensor tokens =
            as_saved(saved[0], index_type(a.token_bits), {static_cast<int64_t>(a.count)}, grad.device()).contiguous();
        a.tokens = tokens.data_ptr();
        Tensor out;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            out = at::empty({static_cast<int64_t>(a.vocabulary), static_cast<int64_t>(a.width)}, grad.options());
            const size_t size = b2_embedding_workspace(&a);
            const Tensor workspace = at::empty({static_cast<int64_t>(size)}, grad.options().dtype(at::kByte));
            check(b2_embedding_backward(reinterpret_cast<b2_ctx*>(node->saved_data["ctx"].toInt()), &a, grad.data_ptr(),
                                        static_cast<uint64_t>(grad.stride(0)), out.data_ptr(), workspace.data_ptr(),
                                        size, stream_of(grad)));
        }
        return {no_further(out), Tensor(), Tensor(), Tensor()};
    }
};

Tensor embedding(Tensor tokens, Tensor weight, double scale)
{
    floating(weight, "embedding: weight must be a CUDA tensor of float32, bfloat16 or float16");
    refuse(weight.dim() != 2, "embedding: weight must be [V, D]");
    b2_embedding_args a{};
    a.token_bits = index_bits(tokens, weight, "embedding: tokens must be int32 or int64, on the weight's device");
    b2_ctx* const ctx = context(weight.get_device());
    const py::gil_scoped_release unlocked;
    const c10::cuda::CUDAGuard guard(weight.device());
    const Tensor flat = tokens.dim() == 1 ? tokens.contiguous() : tokens.contiguous().view({tokens.numel()});
    weight = unit_columns(weight);
    a.tokens = flat.data_ptr();
    a.dtype = dtype_of(weight, "");
    a.count = static_cast<uint64_t>(flat.numel());
    a.vocabulary = static_cast<uint64_t>(weight.size(0));
    a.width = static_cast<uint64_t>(weight.size(1));
    a.scale = static_cast<float>(scale);
    Tensor rows = weight.requires_grad() && at::GradMode::is_enabled() ? EmbeddingNode::apply(weight, flat, ctx, &a)
                                                                       : embedding_forward(ctx, a, weight);
    if (tokens.dim() == 1)
        return rows;
    std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(weight.size(1));
    return rows.view(shape);
}

// ---------------------------------------------------------------------------------------------- AdamW

void adamw_step(const std::vector<Tensor>& params, const std::vector<OptTensor>& grads, const Tensor& exp_avg,
                const Tensor& exp_avg_sq, const OptTensor& exp_avg_scale, const OptTensor& exp_avg_sq_scale,
                const OptTensor& master, int64_t step, double lr, double beta1, double beta2, double eps,
                double weight_decay, uint32_t seed)
{
    refuse(params.size() != grads.size(), "adamw_step: one gradient for each parameter");
    refuse(!exp_avg.is_cuda(), "adamw_step: the moments must be CUDA tensors");
    refuse(step < 1, "adamw_step: step counts from 1");
    const int32_t bits = exp_avg.scalar_type() == at::kFloat ? 32 : 8;
    const int64_t elements = exp_avg.numel();
    auto array = [&](const Tensor& t, at::ScalarType dtype, int64_t n, const char* message) {
        refuse(t.scalar_type() != dtype || t.device() != exp_avg.device() || t.numel() != n || !t.is_contiguous(), message);
        return t.data_ptr();
    };
    const at::ScalarType kind = bits == 32 ? at::kFloat : at::kFloat8_e4m3fn;
    b2_adamw_args a{};
    a.moment_bits = bits;
    a.blocks = static_cast<uint64_t>(elements / B2_MOMENT_BLOCK);
    const auto blocks = static_cast<int64_t>(a.blocks);
    a.exp_avg = array(exp_avg, kind, elements, "adamw_step: exp_avg must be contiguous, float32 or float8_e4m3fn");
    a.exp_avg_sq = array(exp_avg_sq, kind, elements, "adamw_step: exp_avg_sq must be as exp_avg is");
    if (bits == 8)
    {
        refuse(!exp_avg_scale || !exp_avg_sq_scale, "adamw_step: 8-bit moments need exp_avg_scale and exp_avg_sq_scale");
        const char* message = "adamw_step: scales must be contiguous float32, one for each block of 256 elements";
        a.exp_avg_scale = static_cast<float*>(array(*exp_avg_scale, at::kFloat, blocks, message));
        a.exp_avg_sq_scale = static_cast<float*>(array(*exp_avg_sq_scale, at::kFloat, blocks, message));
    }
    if (master)
        a.master = static_cast<float*>(array(*master, at::kFloat, elements,
                                             "adamw_step: master must be contiguous float32 of the moments' size"));
    a.lr = lr, a.beta1 = beta1, a.beta2 = beta2, a.eps = eps, a.weight_decay = weight_decay;
    a.step = static_cast<uint64_t>(step), a.seed = seed;
    // the tensors by (parameter type, gradient type): a call for each kind
    std::array<std::vector<b2_adamw_tensor>, 9> tables;
    std::vector<Tensor> kept;
    int64_t at = 0;
    for (size_t i = 0; i < params.size(); ++i)
    {
        const Tensor& p = params[i];
        const int64_t n = p.numel(), from = at;
        at += (n + B2_MOMENT_BLOCK - 1) / B2_MOMENT_BLOCK;
        if (!grads[i] || !n)
            continue;
        const Tensor& g = *grads[i];
        refuse(p.device() != exp_avg.device() || g.device() != exp_avg.device(),
               "adamw_step: parameters and gradients must be on the moments' device");
        refuse(!p.is_contiguous(), "adamw_step: parameters must be contiguous");
        refuse(g.sizes() != p.sizes(), "adamw_step: a gradient has its parameter's shape");
        refuse(g.scalar_type() != p.scalar_type() && g.scalar_type() != at::kFloat,
               "adamw_step: a gradient has its parameter's type or float32");
        const char* message = "adamw_step: parameters must be float32, bfloat16 or float16";
        const int32_t p_type = dtype_of(p, message), g_type = dtype_of(g, message);
        const void* data = g.data_ptr();
        if (!g.is_contiguous())
        {
            kept.push_back(g.contiguous());
            data = kept.back().data_ptr();
        }
        tables[p_type * 3 + g_type].push_back({p.data_ptr(), data, static_cast<uint64_t>(n), static_cast<uint32_t>(from), 0});
    }
    refuse(at != blocks || elements % B2_MOMENT_BLOCK,
           "adamw_step: the moments must hold each parameter from a block of 256 elements of its own");
    b2_ctx* const ctx = context(exp_avg.get_device());
    const py::gil_scoped_release unlocked;
    for (int k = 0; k < 9; ++k)
        if (!tables[k].empty())
        {
            a.param_dtype = k / 3, a.grad_dtype = k % 3;
            a.tensors = tables[k].data();
            a.count = static_cast<uint32_t>(tables[k].size());
            check(b2_adamw(ctx, &a, stream_of(exp_avg)));
        }
    for (size_t i = 0; i < params.size(); ++i)
        if (grads[i])
            params[i].unsafeGetTensorImpl()->bump_version();  // autograd sees that they changed
}
}  // namespace

PYBIND11_MODULE(_learn, m)
{
    m.doc() = "The learner's operators over torch tensors (mymyr_b200.learn).";
    py::register_local_exception_translator([](std::exception_ptr p) {
        try
        {
            if (p)
                std::rethrow_exception(p);
        }
        catch (const CapacityError& e)
        {
            py::set_error(py::module_::import("mymyr_b200._lib").attr("CapacityError"), e.what());
        }
    });
    m.def("logprobs", &logprobs);
    m.def("embedding", &embedding);
    m.def("adamw_step", &adamw_step);
}
