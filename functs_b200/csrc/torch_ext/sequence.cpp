#include "sequence.h"

#include <ATen/core/grad_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cstring>
#include <vector>

#include "../../../include/functs_b200.h"

namespace functs_b200 {

bool carriesTangent(const at::Tensor& t) { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined(); }
bool wantsDerivative(const at::Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || carriesTangent(t) || !t.has_storage(); }

namespace {

int32_t dtypeOf(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return FB_DTYPE_F32;
        case at::kHalf: return FB_DTYPE_F16;
        case at::kBFloat16: return FB_DTYPE_BF16;
        default: TORCH_CHECK_TYPE(false, name, " must be torch.float32, torch.float16 or torch.bfloat16, got ", t.scalar_type());
    }
    return -1;
}

// An input: on `device`, of `dtype`, and not one that wants a gradient.
void checkInput(const at::Tensor& t, const at::Device& device, at::ScalarType dtype, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor (functs_b200 has no CPU path)");
    TORCH_CHECK_VALUE(t.device() == device, name, " must be on ", device, ", not on ", t.device());
    TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK_NOT_IMPLEMENTED(!(t.requires_grad() && at::GradMode::is_enabled()), name,
                                " requires a gradient, and this operator has none: call it under torch.no_grad()");
    TORCH_CHECK_NOT_IMPLEMENTED(!carriesTangent(t), name, " carries a tangent, and this operator has no derivative");
    TORCH_CHECK_NOT_IMPLEMENTED(t.has_storage(), name, " is a tensor of a transform (torch.func), which this operator does not have");
}
void checkSizes(const at::Tensor& t, at::IntArrayRef sizes, const char* name) {
    TORCH_CHECK_VALUE(t.sizes() == sizes, name, " must be of sizes ", sizes, ", not ", t.sizes());
}

// Where a kernel says that a wait of its own ran out, for callers that give no status word: in pinned host memory, a word for each device, asked
// at that device's next call.  (Slots and tokens that are out of range are the caller's; without a status word they are skipped as documented,
// and not reported.)
constexpr int kMostDevices = 64, kWordsApart = 16;  // (a line of 64 bytes each)
int32_t* ownStatusWord(const at::Device& device) {
    static int32_t* const words = [] {
        void* p = nullptr;
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // (the first call may be one that is captured)
        cudaThreadExchangeStreamCaptureMode(&mode);
        const cudaError_t rc = cudaHostAlloc(&p, kMostDevices * kWordsApart * sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (rc != cudaSuccess) {
            cudaGetLastError();
            return static_cast<int32_t*>(nullptr);
        }
        std::memset(p, 0, kMostDevices * kWordsApart * sizeof(int32_t));
        return static_cast<int32_t*>(p);
    }();
    if (words == nullptr || device.index() < 0 || device.index() >= kMostDevices) return nullptr;
    int32_t* const word = words + device.index() * kWordsApart;
    if ((*static_cast<volatile int32_t*>(word) & FB_STATUS_WAIT_TIMEOUT) != 0) {
        *static_cast<volatile int32_t*>(word) = 0;
        TORCH_CHECK(false, "linear_attention: a bounded device-side wait ran out in an earlier call on ", device, "; its outputs mean nothing");
    }
    return word;
}

int32_t* statusWord(const MaybeTensor& status, const at::Device& device, bool own) {
    if (!status.has_value()) return own ? ownStatusWord(device) : nullptr;
    TORCH_CHECK_VALUE(status->scalar_type() == at::kInt && status->numel() >= 1 && (status->device() == device || status->is_pinned()),
                      "status must be an int32 tensor on ", device, " or in pinned memory");
    return status->data_ptr<int32_t>();
}

// (a view that negates when it is read, as of a conjugate's imaginary part, is written out)
at::Tensor channelsAdjacent(const at::Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t.resolve_neg() : t.contiguous().resolve_neg(); }
at::Tensor packed(const at::Tensor& t) { return t.contiguous().resolve_neg(); }

int32_t narrow(int64_t n, const char* what) {
    TORCH_CHECK_VALUE(n <= INT32_MAX, what, " (", n, ") is too large");
    return static_cast<int32_t>(n);
}

void checkRc(int rc, const char* what) {
    TORCH_CHECK_VALUE(rc != FB_ERR_INVALID_ARGUMENT, functs_b200_last_error());
    TORCH_CHECK(rc == FB_OK, "functs_b200 ", what, ": ", functs_b200_last_error());
}

// strides of [B, T, H, D], or of [B, H, D] as of one token
void strides(const at::Tensor& t, int64_t (&s)[3]) {
    s[0] = t.stride(0);
    s[1] = t.dim() == 4 ? t.stride(1) : 0;
    s[2] = t.stride(t.dim() - 2);
}

// the checks and the launch that whole prompts and single tokens share; `state` is defined, `fresh`: it holds nothing yet
void run(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay, double scale, const at::Tensor& state,
         bool fresh, const MaybeTensor& slots, const MaybeTensor& lengths, const at::Tensor& out, const MaybeTensor& status, int64_t tokens) {
    const int64_t B = q.size(0), H = q.size(-2);
    const at::Device device = q.device();
    const at::Tensor qc = channelsAdjacent(q), kc = channelsAdjacent(k), vc = channelsAdjacent(v), decay = packed(log_decay);
    functs_b200_linear_attention_args a = {};
    a.dtype = dtypeOf(q, "q");
    a.batch = narrow(B, "batch");
    a.tokens = narrow(tokens, "tokens");
    a.heads = narrow(H, "heads");
    a.kv_heads = narrow(k.size(-2), "kv_heads");
    a.dk = narrow(q.size(-1), "dk");
    a.dv = narrow(v.size(-1), "dv");
    a.num_slots = narrow(state.size(0), "num_slots");
    a.q = qc.data_ptr(), a.k = kc.data_ptr(), a.v = vc.data_ptr(), a.out = out.data_ptr();
    strides(qc, a.q_stride), strides(kc, a.k_stride), strides(vc, a.v_stride), strides(out, a.out_stride);
    a.log_decay = decay.data_ptr<float>();
    a.state_in = fresh ? nullptr : state.data_ptr<float>();
    a.state_out = state.data_ptr<float>();
    at::Tensor slots_c, lengths_c;
    if (slots.has_value()) {
        slots_c = packed(*slots);
        a.slots = slots_c.data_ptr<int32_t>();
    }
    if (lengths.has_value()) {
        lengths_c = packed(*lengths);
        a.lengths = lengths_c.data_ptr<int32_t>();
    }
    a.status = statusWord(status, device, /*own=*/tokens > 1);
    a.scale = static_cast<float>(scale);
    at::Tensor scratch;
    const int64_t bytes = functs_b200_linear_attention_scratch_bytes(&a);
    if (bytes > 0) scratch = at::empty({bytes}, q.options().dtype(at::kByte));
    checkRc(functs_b200_linear_attention(&a, bytes > 0 ? scratch.data_ptr() : nullptr, at::cuda::getCurrentCUDAStream().stream()),
            "linear_attention");
}

// what q, k, v, log_decay, slots, lengths and a given state have to be; dims: 4 with tokens, 3 for one token per sequence
void checkAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay, const at::Tensor* state,
                    const MaybeTensor& slots, const MaybeTensor& lengths, int64_t dims) {
    TORCH_CHECK_VALUE(q.dim() == dims && k.dim() == dims && v.dim() == dims, dims == 4 ? "q, k and v must be [B, T, heads, channels]"
                                                                                        : "q, k and v must be [B, heads, channels]");
    const at::Device device = q.device();
    dtypeOf(q, "q");
    checkInput(q, device, q.scalar_type(), "q");
    checkInput(k, device, q.scalar_type(), "k");
    checkInput(v, device, q.scalar_type(), "v");
    checkInput(log_decay, device, at::kFloat, "log_decay");
    const int64_t B = q.size(0), H = q.size(-2), Hk = k.size(-2), Dk = q.size(-1), Dv = v.size(-1);
    TORCH_CHECK_VALUE(H >= 1 && Hk >= 1 && H % Hk == 0, "heads (", H, ") must be a multiple of the key and value heads (", Hk, ")");
    TORCH_CHECK_VALUE(Dk >= 1 && Dk <= 128 && Dv >= 1 && Dv <= 128, "heads must have 1 to 128 channels, got ", Dk, " and ", Dv);
    TORCH_CHECK_VALUE(k.size(0) == B && v.size(0) == B && v.size(-2) == Hk && k.size(-1) == Dk && (dims == 3 || (k.size(1) == q.size(1) && v.size(1) == q.size(1))),
                      "q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not fit one another");
    checkSizes(log_decay, {H}, "log_decay");
    if (state != nullptr) {
        checkInput(*state, device, at::kFloat, "state");
        TORCH_CHECK_VALUE(!state->is_neg(), "state must not be a negated view");
        TORCH_CHECK_VALUE(state->dim() == 4 && state->size(1) == H && state->size(2) == Dk && state->size(3) == Dv && state->is_contiguous(),
                          "state must be a contiguous [slots, ", H, ", ", Dk, ", ", Dv, "] tensor");
        TORCH_CHECK_VALUE(slots.has_value() || state->size(0) == B, "without slots, state must hold ", B, " states");
    } else {
        TORCH_CHECK_VALUE(!slots.has_value(), "slots name rows of a state: give one");
    }
    if (slots.has_value()) {
        checkInput(*slots, device, at::kInt, "slots");
        checkSizes(*slots, {B}, "slots");
    }
    if (lengths.has_value()) {
        checkInput(*lengths, device, at::kInt, "lengths");
        checkSizes(*lengths, {B}, "lengths");
    }
}

// A kernel has written `t`: autograd, which may have saved it for a backward pass, has to know.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The memory from a tensor's first element to its last.
struct Span {
    uintptr_t first = 0, end = 0;
    explicit Span(const at::Tensor* t) {
        if (t == nullptr || t->numel() == 0) return;
        int64_t last = 0;
        const auto sizes = t->sizes(), strides = t->strides();
        for (size_t d = 0; d < sizes.size(); ++d) last += (sizes[d] - 1) * strides[d];
        first = reinterpret_cast<uintptr_t>(t->const_data_ptr());
        end = first + (last + 1) * t->element_size();
    }
    bool apart(const Span& o) const { return end <= o.first || o.end <= first || first == end || o.first == o.end; }
};

// Whether no two elements of `t` can be the same: every stride steps over all that the smaller ones reach.
bool elementsApart(const at::Tensor& t) {
    std::vector<std::pair<int64_t, int64_t>> by_stride;
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1) by_stride.emplace_back(t.stride(d), t.size(d));
    std::sort(by_stride.begin(), by_stride.end());
    int64_t reach = 0;
    for (const auto& [stride, size] : by_stride) {
        if (stride <= reach) return false;
        reach += (size - 1) * stride;
    }
    return true;
}

// What is written (the output, a given state) lies apart from all that is read while it is, and from one another.
void checkWritten(const at::Tensor* out, const at::Tensor* state, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& log_decay, const MaybeTensor& slots, const MaybeTensor& lengths, const MaybeTensor& status) {
    const Span to(out), kept(state);
    TORCH_CHECK_VALUE(to.apart(kept), "out must not share memory with the state");
    const auto check = [&](const at::Tensor* t) {
        const Span read(t);
        TORCH_CHECK_VALUE(kept.apart(read), "state must not share memory with the inputs");
        TORCH_CHECK_VALUE(to.apart(read), "out must not share memory with the inputs (from its first element to its last)");
    };
    for (const at::Tensor* t : {&q, &k, &v, &log_decay}) check(t);
    for (const MaybeTensor* t : {&slots, &lengths, &status})
        if (t->has_value()) check(&**t);
}

at::Tensor output(const MaybeTensor& out, const at::Tensor& q, const at::Tensor& v) {
    std::vector<int64_t> sizes = q.sizes().vec();
    sizes.back() = v.size(-1);
    if (!out.has_value()) return at::empty(sizes, q.options());
    checkInput(*out, q.device(), q.scalar_type(), "out");
    TORCH_CHECK_VALUE(!out->is_neg(), "out must not be a negated view");
    checkSizes(*out, sizes, "out");
    TORCH_CHECK_VALUE(out->size(-1) == 1 || out->stride(-1) == 1, "out must have adjacent channels");
    TORCH_CHECK_VALUE(elementsApart(*out), "out must not overlap itself");
    return *out;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> linearAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                   double scale, const MaybeTensor& state, const MaybeTensor& slots,
                                                   const MaybeTensor& lengths, const MaybeTensor& out, const MaybeTensor& status) {
    const at::Tensor* given = state.has_value() ? &*state : nullptr;
    checkAttention(q, k, v, log_decay, given, slots, lengths, 4);
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor o = output(out, q, v);
    checkWritten(out.has_value() ? &o : nullptr, given, q, k, v, log_decay, slots, lengths, status);
    const at::Tensor s = given != nullptr ? *given : at::empty({q.size(0), q.size(2), q.size(3), v.size(3)}, q.options().dtype(at::kFloat));
    run(q, k, v, log_decay, scale, s, given == nullptr, slots, lengths, o, status, q.size(1));
    if (given != nullptr) written(s);
    if (out.has_value()) written(o);
    return {o, s};
}

at::Tensor linearAttentionStep(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                               const at::Tensor& state, double scale, const MaybeTensor& slots, const MaybeTensor& out,
                               const MaybeTensor& status) {
    checkAttention(q, k, v, log_decay, &state, slots, std::nullopt, 3);
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor o = output(out, q, v);
    checkWritten(out.has_value() ? &o : nullptr, &state, q, k, v, log_decay, slots, std::nullopt, status);
    run(q, k, v, log_decay, scale, state, false, slots, std::nullopt, o, status, 1);
    written(state);
    if (out.has_value()) written(o);
    return o;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> tokenLogprobs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top,
                                                                         const MaybeTensor& status) {
    TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) >= 1, "logits must be [rows, vocab]");
    const at::Device device = logits.device();
    const int32_t dtype = dtypeOf(logits, "logits");
    checkInput(logits, device, logits.scalar_type(), "logits");
    checkInput(tokens, device, at::kLong, "tokens");
    const int64_t R = logits.size(0), V = logits.size(1);
    checkSizes(tokens, {R}, "tokens");
    TORCH_CHECK_VALUE(top >= 0 && top <= FB_LOGPROBS_MAX_TOP && top <= V, "top must be 0 to ", FB_LOGPROBS_MAX_TOP, " and at most the vocabulary (", V,
                      "), got ", top);
    c10::cuda::CUDAGuard guard(device);
    const at::Tensor x = channelsAdjacent(logits), ids = packed(tokens);
    const auto f32 = logits.options().dtype(at::kFloat);
    at::Tensor lp = at::empty({R}, f32), entropy = at::empty({R}, f32), top_lp = at::empty({R, top}, f32),
               top_ids = at::empty({R, top}, f32.dtype(at::kLong));
    checkRc(functs_b200_token_logprobs(x.data_ptr(), dtype, x.stride(0), ids.data_ptr<int64_t>(), narrow(R, "rows"), narrow(V, "vocab"),
                                       static_cast<int32_t>(top), lp.data_ptr<float>(), entropy.data_ptr<float>(), top_lp.data_ptr<float>(),
                                       top_ids.data_ptr<int64_t>(), statusWord(status, device, /*own=*/false), at::cuda::getCurrentCUDAStream().stream()),
            "token_logprobs");
    return {lp, entropy, top_lp, top_ids};
}

}  // namespace functs_b200
