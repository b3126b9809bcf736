// The short causal convolution over time of every channel on its own:  y[t] = bias + sum_j w[j] x[t - W + 1 + j],  silu on request.
//
// A pass over the rows: every input is read once and every output written once, but for the W - 1 rows in front of a thread's tokens, which it
// reads again (from L2).  A thread has V adjacent channels (of 16 or 8 bytes where the rows lie on such boundaries) and a run of tokens, whose last W - 1
// inputs it keeps in registers; sums are in fp32, in the order of the formula, two channels an instruction.  Bound by HBM beside two exponential-unit
// results an element (30 us of 8 x 2048 tokens of 4096 channels in bf16, which take 56 in all: 4.8 TB/s; by single products 83, with eight
// channels a thread 60, four tokens ahead 61, at four blocks an SM instead of five 59: five leave 96 registers a thread, and at width 4 36 bytes are spilled).  In fp32
// half as many tokens take 46 us, 5.8 TB/s; 4095 channels, whose rows no vector fits, 106.  192 single tokens of 4096 channels 4.5 us (9.3 by the prompts' kernel).
#include <type_traits>

#include "activation.cuh"
#include "linattn.cuh"

namespace fb {

using ConvArgs = functs_b200_causal_conv_args;

constexpr int kConvThreads = 128;
constexpr int kConvMinRun = 8;

// V adjacent channels of a row: as they lie in memory, and in 32 bits, by twos
template <typename T, int V>
struct __align__(sizeof(T) * V) ConvPack {
    T v[V];
};
template <typename T, int V>
struct ConvRow {
    static constexpr int P = (V + 1) / 2;
    static __device__ __forceinline__ void get(const ConvPack<T, V>& p, uint64_t (&x)[P]) {
        if constexpr (V == 1) {
            x[0] = pair_of(lin_float(p.v[0]), 0.0f);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < P; ++i) x[i] = pair_of(lin_float(p.v[2 * i]), lin_float(p.v[2 * i + 1]));
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(p.v)[i];
                if constexpr (std::is_same<T, __half>::value) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                    x[i] = pair_of(f.x, f.y);
                } else {
                    x[i] = pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
                }
            }
        }
    }
    static __device__ __forceinline__ ConvPack<T, V> put(const uint64_t (&x)[P]) {
        ConvPack<T, V> p;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float2 f = pair_get(x[i]);
            p.v[2 * i] = lin_from<T>(f.x);
            if (2 * i + 1 < V) p.v[2 * i + 1] = lin_from<T>(f.y);
        }
        return p;
    }
};

// a thread's V x W weights, which lie side by side: by 16 bytes where they can
template <typename T, int W, int V>
struct __align__(16) ConvTaps {
    T v[V * W];
    __device__ __forceinline__ void get(const T* p) {
        if (V * W * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(V * W * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < V * W; ++i) v[i] = p[i];
        }
    }
};

// run: tokens of a CTA (at least W - 1: only the CTAs of the first run reach in front of token 0).  A sequence's CTAs of the first run also write
// its new state: they alone read the old one, each thread the channels that it writes.  AHEAD: tokens whose loads are on their way at once.
template <typename T, int W, int V, int AHEAD>
__global__ void __launch_bounds__(kConvThreads, V > 1 && W <= 4 ? (sizeof(T) == 2 ? 5 : 4) : 3) causal_conv_kernel(const ConvArgs a, int run) {
    using Pack = ConvPack<T, V>;
    using Row = ConvRow<T, V>;
    constexpr int P = Row::P;
    const int c = (blockIdx.x * kConvThreads + threadIdx.x) * V, b = blockIdx.z, t0 = blockIdx.y * run;
    int bits;
    const int slot = lin_slot(a.slots, a.num_slots, b, threadIdx.x & 31, bits);
    if (bits != 0 && a.status != nullptr && threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(a.status, bits);
    if (c >= a.channels) return;
    const int length = slot < 0 ? 0 : a.lengths == nullptr ? a.tokens : min(max(a.lengths[b], 0), a.tokens);
    const int64_t state = static_cast<int64_t>(slot < 0 ? 0 : slot) * (W - 1) * a.channels + c;
    const T* state_in = a.state_in == nullptr ? nullptr : static_cast<const T*>(a.state_in) + state;
    const T* x = static_cast<const T*>(a.x) + b * a.x_stride[0] + c;
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + c;
    const auto at = [](const T* p) { return *reinterpret_cast<const Pack*>(p); };
    const int end = min(t0 + run, a.tokens), last = min(end, length);
    if (t0 < last) {
        Pack next[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) next[k] = t0 + k < last ? at(x + (t0 + k) * a.x_stride[1]) : Pack{};
        uint64_t w[W][P], bias[P], in[W - 1 + AHEAD][P];
        ConvTaps<T, W, V> taps;
        taps.get(static_cast<const T*>(a.weight) + static_cast<int64_t>(c) * W);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const bool two = 2 * i + 1 < V;
            const T* q = static_cast<const T*>(a.bias) + c + 2 * i;
            bias[i] = a.bias == nullptr ? 0ull : pair_of(lin_float(q[0]), two ? lin_float(q[1]) : 0.0f);
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = pair_of(lin_float(taps.v[2 * i * W + j]), two ? lin_float(taps.v[(2 * i + 1) * W + j]) : 0.0f);
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const int t = t0 - (W - 1) + j;
            Pack p = {};
            if (t >= 0) p = at(x + t * a.x_stride[1]);
            else if (state_in != nullptr) p = at(state_in + static_cast<int64_t>(W - 1 + t) * a.channels);
            Row::get(p, in[j]);
        }
        const T* from = x + (t0 + AHEAD) * a.x_stride[1];
        T* to = out + t0 * a.out_stride[1];
        const bool silu = a.silu != 0;
        for (int t = t0; t < last; t += AHEAD) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                Row::get(next[k], in[W - 1 + k]);
                if (t + AHEAD + k < last) next[k] = at(from);
                from += a.x_stride[1];
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                uint64_t y[P];
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    y[i] = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) y[i] = pair_fma(w[j][i], in[j + k][i], y[i]);
                    if (silu) {
                        const float2 f = pair_get(y[i]);
                        y[i] = pair_of(act_silu(f.x), V > 1 ? act_silu(f.y) : 0.0f);
                    }
                }
                if (t + k < last) *reinterpret_cast<Pack*>(to) = Row::put(y);
                to += a.out_stride[1];
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
#pragma unroll
                for (int i = 0; i < P; ++i) in[j][i] = in[j + AHEAD][i];
            }
        }
    }
    for (int t = max(t0, length); t < end; ++t) *reinterpret_cast<Pack*>(out + t * a.out_stride[1]) = Pack{};
    if (blockIdx.y == 0 && slot >= 0) {
        // row k of the new state is input length - (W - 1) + k: one of the prompt, or the old state's row length + k, which is not written yet
        T* state_out = static_cast<T*>(a.state_out) + state;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            Pack p = {};
            if (length + k >= W - 1) p = at(x + (length + k - (W - 1)) * a.x_stride[1]);
            else if (state_in != nullptr) p = at(state_in + static_cast<int64_t>(length + k) * a.channels);
            *reinterpret_cast<Pack*>(state_out + static_cast<int64_t>(k) * a.channels) = p;
        }
    }
}

// One token per sequence: the rows of the state and the token, all on their way before anything is looked up.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(const ConvArgs a) {
    using Pack = ConvPack<T, V>;
    using Row = ConvRow<T, V>;
    constexpr int P = Row::P;
    const int c = (blockIdx.x * kConvThreads + threadIdx.x) * V, b = blockIdx.y;
    const bool lives = c < a.channels;
    const int named = a.slots == nullptr ? b : a.slots[b];
    const bool inside = named >= 0 && named < a.num_slots;
    const int64_t state = static_cast<int64_t>(inside ? named : 0) * (W - 1) * a.channels + c;
    // (a state may be read whether the slot is this sequence's or an earlier one's)
    Pack rows[W];
    ConvTaps<T, W, V> taps;
    Pack bias = {};
#pragma unroll
    for (int j = 0; j < W; ++j) rows[j] = Pack{};
    if (lives) {
        rows[W - 1] = *reinterpret_cast<const Pack*>(static_cast<const T*>(a.x) + b * a.x_stride[0] + c);
        if (inside && a.state_in != nullptr) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) rows[j] = *reinterpret_cast<const Pack*>(static_cast<const T*>(a.state_in) + state + static_cast<int64_t>(j) * a.channels);
        }
        taps.get(static_cast<const T*>(a.weight) + static_cast<int64_t>(c) * W);
        if (a.bias != nullptr) {
            const T* q = static_cast<const T*>(a.bias) + c;
            if (reinterpret_cast<uintptr_t>(q) % sizeof(Pack) == 0) {
                bias = *reinterpret_cast<const Pack*>(q);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) bias.v[i] = q[i];
            }
        }
    }
    int bits;
    const int slot = lin_slot(a.slots, a.num_slots, b, threadIdx.x & 31, bits);
    if (bits != 0 && a.status != nullptr && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(a.status, bits);
    if (!lives) return;
    uint64_t y[P], in[P];
    Row::get(bias, y);
#pragma unroll
    for (int j = 0; j < W; ++j) {
        Row::get(rows[j], in);
#pragma unroll
        for (int i = 0; i < P; ++i)
            y[i] = pair_fma(pair_of(lin_float(taps.v[2 * i * W + j]), 2 * i + 1 < V ? lin_float(taps.v[(2 * i + 1) * W + j]) : 0.0f), in[i], y[i]);
    }
    if (a.silu) {
#pragma unroll
        for (int i = 0; i < P; ++i) y[i] = pair_of(act_silu(pair_get(y[i]).x), act_silu(pair_get(y[i]).y));
    }
    *reinterpret_cast<Pack*>(static_cast<T*>(a.out) + b * a.out_stride[0] + c) = slot >= 0 ? Row::put(y) : Pack{};
    if (slot < 0) return;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) *reinterpret_cast<Pack*>(static_cast<T*>(a.state_out) + state + static_cast<int64_t>(j) * a.channels) = rows[j + 1];
}

template <typename T, int W, int V>
static int launch_conv(const ConvArgs& a, cudaStream_t st) {
    const int tiles = (a.channels + kConvThreads * V - 1) / (kConvThreads * V);
    // long runs read few rows twice, short ones fill the chip
    int run = 64;
    while (run > kConvMinRun && static_cast<int64_t>(tiles) * a.batch * ((a.tokens + run - 1) / run) < 8 * kNumSMs) run /= 2;
    while ((a.tokens + run - 1) / run >= 65536) run *= 2;
    const int runs = a.tokens > run ? (a.tokens + run - 1) / run : 1;
    return launch_after(causal_conv_kernel<T, W, V, V == 1 ? 4 : 8>, dim3(tiles, runs, a.batch), dim3(kConvThreads), 0, st, false, "causal_conv", a, run);
}

template <typename T, int W, int V>
static int launch_conv_step(const ConvArgs& a, cudaStream_t st) {
    const int tiles = (a.channels + kConvThreads * V - 1) / (kConvThreads * V);
    return launch_after(causal_conv_step_kernel<T, W, V>, dim3(tiles, a.batch), dim3(kConvThreads), 0, st, false, "causal_conv", a);
}

template <typename T, int W>
static int launch_conv(const ConvArgs& a, cudaStream_t st) {
    constexpr int V = 4, VS = W <= 4 ? 16 / sizeof(T) : 4;  // for prompts, for single tokens
    const int64_t strides = a.x_stride[0] | a.x_stride[1] | a.out_stride[0] | a.out_stride[1] | a.channels;
    const uintptr_t pointers = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.state_in) |
                               reinterpret_cast<uintptr_t>(a.state_out);
    const auto fits = [&](int v) { return strides % v == 0 && pointers % (v * sizeof(T)) == 0; };
    if (a.tokens == 1 && a.lengths == nullptr) return fits(VS) ? launch_conv_step<T, W, VS>(a, st) : launch_conv_step<T, W, 1>(a, st);
    return fits(V) ? launch_conv<T, W, V>(a, st) : launch_conv<T, W, 1>(a, st);
}

template <typename T>
static int launch_conv(const ConvArgs& a, cudaStream_t st) {
    switch (a.width) {
        case 2: return launch_conv<T, 2>(a, st);
        case 3: return launch_conv<T, 3>(a, st);
        case 4: return launch_conv<T, 4>(a, st);
        case 5: return launch_conv<T, 5>(a, st);
        case 6: return launch_conv<T, 6>(a, st);
        case 7: return launch_conv<T, 7>(a, st);
        default: return launch_conv<T, 8>(a, st);
    }
}

}  // namespace fb

extern "C" int functs_b200_causal_conv(const functs_b200_causal_conv_args* args, void* stream) {
    using namespace fb;
    FB_REQUIRE(args != nullptr, "causal_conv: null pointer");
    const ConvArgs& a = *args;
    FB_REQUIRE(a.dtype >= FB_DTYPE_F32 && a.dtype <= FB_DTYPE_BF16, "causal_conv: unknown dtype %d", a.dtype);
    FB_REQUIRE(a.batch >= 0 && a.batch < 65536 && a.tokens >= 0 && a.tokens <= (1 << 30), "causal_conv: batch must be 0 .. 65535, tokens 0 .. %d", 1 << 30);
    FB_REQUIRE(a.channels >= 1 && a.channels <= (1 << 24), "causal_conv: channels must be 1 .. %d", 1 << 24);
    FB_REQUIRE(a.width >= 2 && a.width <= 8, "causal_conv: width (%d) must be 2 .. 8", a.width);
    FB_REQUIRE(a.num_slots >= 0, "causal_conv: num_slots must not be negative");
    FB_REQUIRE(a.slots != nullptr || a.num_slots == a.batch, "causal_conv: without slots there are as many states as sequences");
    if (a.batch == 0) return FB_OK;
    FB_REQUIRE(a.weight != nullptr && a.state_out != nullptr, "causal_conv: null pointer");
    FB_REQUIRE(a.tokens == 0 || (a.x != nullptr && a.out != nullptr), "causal_conv: null pointer");
    const uintptr_t elements = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.bias) |
                               reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.state_in) | reinterpret_cast<uintptr_t>(a.state_out);
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.lengths) | reinterpret_cast<uintptr_t>(a.status);
    FB_REQUIRE(elements % (a.dtype == FB_DTYPE_F32 ? 4 : 2) == 0 && words % 4 == 0, "causal_conv: pointers must lie on a boundary of their type");
    const cudaStream_t st = as_stream(stream);
    if (a.dtype == FB_DTYPE_F32) return launch_conv<float>(a, st);
    if (a.dtype == FB_DTYPE_F16) return launch_conv<__half>(a, st);
    return launch_conv<__nv_bfloat16>(a, st);
}
