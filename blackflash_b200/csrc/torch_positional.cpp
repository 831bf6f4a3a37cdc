// Torch binding of the position-aware operators (blackflash_b200/positional.py): checks,
// outputs, workspaces and autograd nodes in C++ over the C ABI, because a decoding step or a
// short training step takes the GPU less time than the same work takes the interpreter.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <limits>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/blackflash_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int kMaxInt = std::numeric_limits<int>::max();

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return BF_DTYPE_BF16;
        case at::kHalf: return BF_DTYPE_F16;
        case at::kFloat: return BF_DTYPE_F32;
        default: return -1;
    }
}

// Numbers in messages go through std::to_string: streamed into a message as numbers they crash
// the process here, inside the stream's operator<<.
void ok(int rc, const char* what) {
    TORCH_CHECK(rc == BF_OK, what, " failed (code ", std::to_string(rc), "): ", blackflash_last_error());
}

void check(const char* name, const Tensor& t, int64_t dims, const Tensor* like = nullptr, bool fp32 = false) {
    TORCH_CHECK(t.dim() == dims, name, " must have ", std::to_string(dims), " axes");
    const int ty = dtype_of(t);
    TORCH_CHECK(t.is_cuda() && (ty == BF_DTYPE_BF16 || ty == BF_DTYPE_F16 || (fp32 && ty == BF_DTYPE_F32)), name,
                " must be a CUDA tensor of bfloat16", fp32 ? ", float16 or float32" : " or float16");
    TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, "'s last axis must be contiguous");
    if (like)
        TORCH_CHECK(t.scalar_type() == like->scalar_type() && t.device() == like->device(), name,
                    " must have Q's type and device");
    for (int64_t i = 0; i < dims; ++i) TORCH_CHECK(t.size(i) <= kMaxInt, name, " is too large");
}

void check_grouped(const Tensor& q, const Tensor& k, const Tensor& v, const char* kn, const char* vn) {
    check("Q", q, 4);
    TORCH_CHECK(q.size(3) == 64 || q.size(3) == 128, "BlackFlash supports d=64 and d=128");
    check(kn, k, 4, &q);
    check(vn, v, 4, &q);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3), kn, " and ", vn,
                " must have one shape, with Q's batch and d");
    TORCH_CHECK(k.size(1) > 0 && q.size(1) % k.size(1) == 0, "query heads must be a multiple of KV heads");
}

float check_scale(c10::optional<double> scale, int64_t d) {
    const float s = scale ? (float)*scale : (float)(1.0 / std::sqrt((double)d));
    TORCH_CHECK(std::isfinite(s) && s > 0, "scale must be positive and finite");
    return s;
}

void check_window(int64_t window, int64_t sinks) {
    TORCH_CHECK(window >= 1 && sinks >= 0, "need window >= 1 and sinks >= 0");
}
int clamp(int64_t x) { return x < kMaxInt ? (int)x : kMaxInt; }

// The last three strides of [.., heads, tokens, d], and the batch's where there is one.
bf_view view(const Tensor& t) {
    const int64_t n = t.dim();
    return {t.data_ptr(), {n == 4 ? t.stride(0) : 0, t.stride(n - 3), t.stride(n - 2)}};
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

Tensor fresh(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }
Tensor fresh32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
Tensor bytes(long long n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// ---------------------------------------------------------------- sliding window

std::tuple<Tensor, Tensor> window_lse(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                                      c10::optional<double> scale_in, bool want_lse) {
    check_grouped(q, k, v, "K", "V");
    check_window(window, sinks);
    const float scale = check_scale(scale_in, q.size(3));
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor o = fresh(q.sizes(), q), lse;
    if (want_lse) lse = fresh32({q.size(0), q.size(1), q.size(2)}, q);
    if (o.numel() == 0) return {o, lse};
    if (k.size(2) == 0) {
        if (want_lse) lse.fill_(-std::numeric_limits<float>::infinity());
        return {o.zero_(), lse};
    }
    const bf_view vq = view(q), vk = view(k), vv = view(v);
    ok(blackflash_window_fwd(&vq, &vk, &vv, o.data_ptr(), f32(lse), q.size(0), q.size(1), k.size(1), q.size(2), k.size(2),
                             q.size(3), clamp(window), clamp(sinks), scale, dtype_of(q), stream_of(q)),
       "blackflash_window_fwd");
    return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> window_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                                                   const Tensor& d_o, const Tensor& lse, int64_t window, int64_t sinks,
                                                   c10::optional<double> scale_in) {
    check_grouped(q, k, v, "K", "V");
    TORCH_CHECK(q.scalar_type() == at::kBFloat16, "the backward supports bfloat16");
    check_window(window, sinks);
    const float scale = check_scale(scale_in, q.size(3));
    check("O", o, 4, &q);
    check("dO", d_o, 4, &q);
    TORCH_CHECK(o.sizes() == q.sizes() && d_o.sizes() == q.sizes() && o.is_contiguous(),
                "O must be contiguous, O and dO of Q's shape");
    TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.device() == q.device() && lse.is_contiguous() &&
                    lse.sizes() == q.sizes().slice(0, 3),
                "lse must be a contiguous fp32 [B, Hq, Nq] tensor");
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor dq = fresh(q.sizes(), q), dk = fresh(k.sizes(), k), dv = fresh(v.sizes(), v);
    if (q.numel() == 0 || k.numel() == 0) return {dq.zero_(), dk.zero_(), dv.zero_()};
    const int B = q.size(0), Hq = q.size(1), Hkv = k.size(1), Nq = q.size(2), Nkv = k.size(2), d = q.size(3);
    const long long need = blackflash_window_bwd_workspace_bytes(B, Hq, Hkv, Nq, Nkv, d, clamp(window), clamp(sinks));
    if (need < 0) ok(BF_ERR_ARG, "blackflash_window_bwd_workspace_bytes");
    const Tensor ws = bytes(need, q);
    const bf_view vq = view(q), vk = view(k), vv = view(v), vd = view(d_o);
    ok(blackflash_window_bwd(&vq, &vk, &vv, o.data_ptr(), &vd, f32(lse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                             ws.data_ptr(), need, B, Hq, Hkv, Nq, Nkv, d, clamp(window), clamp(sinks), scale, stream_of(q)),
       "blackflash_window_bwd");
    return {dq, dk, dv};
}

// A gradient as the kernels read it: rows contiguous and on 16-byte steps, not broadcast.
Tensor rows(const Tensor& t) {
    bool fine = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; i < t.dim() - 1; ++i)
        fine = fine && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) * t.element_size() % 16 == 0));
    return fine ? t : t.contiguous();
}

// What a backward refuses. A node keeps the stream that it was made on, a leaf's too while any
// graph of the leaf lives; the engine would have the default stream wait for a captured one,
// which ends the capture and, on the engine's thread, the process. It does so for every node that
// this backward goes on to, and for no other: behind views and other operations, but not for
// an input whose gradient was not asked for.
void check_backward() {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "this operator is differentiable once: its backward does not support create_graph=True");
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
    const auto* planned = torch::autograd::get_current_graph_task_exec_info();  // empty: every node
    const auto here = torch::autograd::get_current_node();
    std::vector<const torch::autograd::Node*> todo{here.get()};
    std::unordered_set<const torch::autograd::Node*> known;
    while (!todo.empty()) {
        const auto* node = todo.back();
        todo.pop_back();
        for (const auto& edge : node->next_edges()) {
            auto* next = edge.function.get();
            if (!next || !known.insert(next).second) continue;
            if (planned && !planned->empty()) {
                const auto plan = planned->find(next);
                if (plan == planned->end() || !plan->second.should_execute()) continue;
            }
            const auto stream = next->stream();
            TORCH_CHECK(!stream || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(stream->device_index()),
                        "a backward cannot be captured while a graph of its inputs from the default stream is alive: drop "
                        "that graph first, or make it on another stream");
            todo.push_back(next);
        }
    }
}

struct WindowFn : torch::autograd::Function<WindowFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                          int64_t sinks, c10::optional<double> scale) {
        auto [o, lse] = window_lse(q, k, v, window, sinks, scale, true);
        ctx->save_for_backward({q, k, v, o, lse});
        ctx->saved_data["window"] = window;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return o;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward();
        const variable_list s = ctx->get_saved_variables();
        auto [dq, dk, dv] = window_backward(s[0], s[1], s[2], s[3], rows(grads[0]), s[4], ctx->saved_data["window"].toInt(),
                                            ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toOptional<double>());
        return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
    }
};

Tensor window_with_grad(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                        c10::optional<double> scale) {
    TORCH_CHECK(q.scalar_type() == at::kBFloat16, "the backward supports bfloat16");
    return WindowFn::apply(q, k, v, window, sinks, scale);
}

// ---------------------------------------------------------------- decoding steps

// Without a prefix (kp undefined) the step is blackflash_window_decode's.
std::tuple<Tensor, Tensor> step(const Tensor& q_in, const Tensor& kp, const Tensor& vp, const Tensor& k, const Tensor& v,
                                const Tensor& lengths, int64_t window, int64_t sinks, c10::optional<double> scale_in,
                                bool want_lse) {
    check_grouped(q_in, k, v, "K_cache", "V_cache");
    TORCH_CHECK(lengths.is_cuda() && lengths.scalar_type() == at::kInt && lengths.device() == q_in.device() &&
                    lengths.dim() == 1 && lengths.is_contiguous() && lengths.size(0) == q_in.size(0),
                "lengths must be a contiguous int32 [B] tensor on Q's device");
    check_window(window, sinks);
    const float scale = check_scale(scale_in, q_in.size(3));
    const int B = q_in.size(0), Hq = q_in.size(1), T = q_in.size(2), d = q_in.size(3), Hkv = k.size(1), C = k.size(2);
    int P = 0;
    if (kp.defined()) {
        check("K_prefix", kp, 3, &q_in);
        check("V_prefix", vp, 3, &q_in);
        TORCH_CHECK(kp.sizes() == vp.sizes() && kp.size(0) == Hkv && kp.size(2) == d,
                    "K_prefix and V_prefix must be [Hkv, P, d]");
        P = kp.size(1);
    }
    const c10::cuda::CUDAGuard guard(q_in.device());
    const Tensor q = q_in.contiguous();
    Tensor o = fresh(q.sizes(), q), lse, ws;
    if (want_lse) lse = fresh32({B, Hq, T}, q);
    if (q.numel() == 0 || (P == 0 && C == 0)) {
        if (want_lse) lse.fill_(-std::numeric_limits<float>::infinity());
        return {o.zero_(), lse};
    }
    const long long need = blackflash_decode_workspace_bytes(B, Hq, Hkv, T, P, C, d, clamp(window), clamp(sinks));
    if (need < 0) ok(BF_ERR_ARG, "blackflash_decode_workspace_bytes");
    if (need > 0) ws = bytes(need, q);
    const bf_view vk = view(k), vv = view(v);
    void* w = need > 0 ? ws.data_ptr() : nullptr;
    if (kp.defined()) {
        const bf_view vkp = view(kp), vvp = view(vp);
        ok(blackflash_prefix_decode(q.data_ptr(), &vkp, &vvp, &vk, &vv, lengths.data_ptr<int>(), o.data_ptr(), f32(lse), w,
                                    need, B, Hq, Hkv, T, P, C, d, scale, dtype_of(q), stream_of(q)),
           "blackflash_prefix_decode");
    } else {
        ok(blackflash_window_decode(q.data_ptr(), &vk, &vv, lengths.data_ptr<int>(), o.data_ptr(), f32(lse), w, need, B, Hq,
                                    Hkv, T, C, d, clamp(window), clamp(sinks), scale, dtype_of(q), stream_of(q)),
           "blackflash_window_decode");
    }
    return {o, lse};
}

std::tuple<Tensor, Tensor> window_decode(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths,
                                         int64_t window, int64_t sinks, c10::optional<double> scale, bool want_lse) {
    return step(q, Tensor(), Tensor(), k, v, lengths, window, sinks, scale, want_lse);
}

std::tuple<Tensor, Tensor> prefix_decode(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& k,
                                         const Tensor& v, const Tensor& lengths, c10::optional<double> scale,
                                         bool want_lse) {
    return step(q, kp, vp, k, v, lengths, kMaxInt, 0, scale, want_lse);
}

// ---------------------------------------------------------------- rotary positions

std::tuple<Tensor, Tensor> rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freqs,
                                  bool interleaved, double amplitude, bool inverse) {
    check("Q", q, 4, nullptr, true);
    check("K", k, 4, &q, true);
    const int64_t B = q.size(0), N = q.size(2), d = q.size(3);
    TORCH_CHECK(k.size(0) == B && k.size(2) == N && k.size(3) == d, "K must have Q's batch, tokens and d");
    TORCH_CHECK(positions.device() == q.device() && positions.is_contiguous(),
                "positions must be a contiguous tensor on Q's device");
    const bool p64 = positions.scalar_type() == at::kLong;
    const bool per_batch = positions.dim() == 2;
    TORCH_CHECK((p64 || positions.scalar_type() == at::kInt) &&
                    (per_batch ? positions.size(0) == B && positions.size(1) == N
                               : positions.dim() == 1 && positions.size(0) == N),
                "positions must be int32 or int64, [N] or [B, N]");
    TORCH_CHECK(freqs.device() == q.device() && freqs.is_contiguous() && freqs.scalar_type() == at::kDouble &&
                    freqs.dim() == 1,
                "freqs must be a contiguous fp64 [rotary_dim / 2] tensor on Q's device");
    const int64_t rot = 2 * freqs.numel();
    TORCH_CHECK(d % 2 == 0 && d <= 1024 && rot >= 2 && rot <= d, "need an even d <= 1024 and 1 to d / 2 frequencies");
    TORCH_CHECK(std::isfinite((float)amplitude), "amplitude must be finite");
    const c10::cuda::CUDAGuard guard(q.device());
    Tensor qo = fresh(q.sizes(), q), ko = fresh(k.sizes(), q);
    if (qo.numel() + ko.numel() == 0) return {qo, ko};
    const bf_view vq = view(q), vk = view(k);
    ok(blackflash_rotary(&vq, &vk, qo.data_ptr(), ko.data_ptr(), positions.data_ptr(), p64, per_batch,
                         freqs.data_ptr<double>(), B, q.size(1), k.size(1), N, d, rot, interleaved, (float)amplitude, inverse,
                         dtype_of(q), stream_of(q)),
       "blackflash_rotary");
    return {qo, ko};
}

// A gradient as the rotary kernel reads it: last axis contiguous, whole pairs.
Tensor pairs(const Tensor& t) {
    bool fine = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % (2 * t.element_size()) == 0;
    for (int64_t i = 0; i < t.dim() - 1; ++i) fine = fine && (t.size(i) <= 1 || t.stride(i) % 2 == 0);
    return fine ? t : t.contiguous();
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& positions,
                                 const Tensor& freqs, bool interleaved, double amplitude) {
        ctx->save_for_backward({positions, freqs});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["amplitude"] = amplitude;
        auto [qo, ko] = rotary(q, k, positions, freqs, interleaved, amplitude, false);
        return {qo, ko};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        check_backward();
        // The map is linear, so its gradient is its transpose: the same turn backwards.
        const variable_list s = ctx->get_saved_variables();
        auto [dq, dk] = rotary(pairs(grads[0]), pairs(grads[1]), s[0], s[1], ctx->saved_data["interleaved"].toBool(),
                               ctx->saved_data["amplitude"].toDouble(), true);
        return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> rotary_with_grad(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freqs,
                                            bool interleaved, double amplitude) {
    const variable_list out = RotaryFn::apply(q, k, positions, freqs, interleaved, amplitude);
    return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Position-aware attention operators over libblackflash_b200.so";
    m.def("window_lse", &window_lse);
    m.def("window_backward", &window_backward);
    m.def("window_with_grad", &window_with_grad);
    m.def("window_decode", &window_decode);
    m.def("prefix_decode", &prefix_decode);
    m.def("rotary", &rotary);
    m.def("rotary_with_grad", &rotary_with_grad);
}
