// Selective scan: a diagonal state space whose step, input and output depend on the token.
//
//   d = softplus(dt[t][c] + bias[c]);  h[c][n] = exp(d A[c][n]) h[c][n] + d x[t][c] B[t][n];  y = sum_n C[t][n] h[c][n] + D[c] x[t][c]
//
// States never leave registers between tokens: a lane has PER of a channel's (four or eight), so that a channel's states lie in LANES lanes of a warp, and
// warps know nothing of one another.  A decay is an exponential of d (A log2 e): off by 1.4e-7 at most and 5e-8 on average, which over a memory
// of a thousand tokens makes 6e-7 of a state (token by token in fp32 with a library's exponential 4.5e-7).
//
// What a token costs a warp of 16 channels of 16 states: eight exponentials (64 cycles of a scheduler), 16 products by pairs (34 cycles), eight loads from
// shared memory and shuffles, and some 35 instructions to prepare and finish it, 70 in all.  Exponentials are 16 per cycle and SM, and 19 a channel with the step's
// and the gate's, which bounds 8 x 1024 tokens of 4096 channels at 141 us.  They take 232: a warp's instructions wait for one another, and there are
// only 3.5 warps for a scheduler (issue 57 %, exponentials 55 %, shared memory 58 %).  With one thing left out at a time, all of one build: without the exponentials 218,
// without loads of B and C 221, without shuffles 205; with tiles copied when they are needed, not ahead, 333.  DRAM would take 42.
//
// Few channels and many tokens: sequences are cut into parts.  One launch goes through all parts but the last from a state of zero and leaves what each
// adds and the sum of its steps; in the second every part makes its start of what the parts before it left, h = exp(A sum d) h + end, and forms the outputs.
//
// Tried, us for 8 sequences of up to 2048 tokens (half of them padding) of 4096 channels: tiles prepared and finished by a whole block between barriers 342
// (four lanes a channel, 541 before its products went by pairs and its loads ahead); sequences in their given order 376 (in order of length 248); 16
// states a lane 355 (a warp for 32 channels: too few); the next tokens prepared while one group is walked through, steps handed over through
// shared memory 418; 80 registers a thread instead of 168 324.
#include <type_traits>

#include "activation.cuh"
#include "linattn.cuh"

namespace fb {

using ScanArgs = functs_b200_selective_scan_args;

constexpr int kScanMaxStates = 64;
// four adjacent elements, as one word
template <typename T>
struct ScanRow;
template <>
struct ScanRow<float> {
    using Word = uint4;
    static __device__ __forceinline__ Word zero() { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ Word one(const float* p, int n) {
        return make_uint4(n > 0 ? __float_as_uint(p[0]) : 0, n > 1 ? __float_as_uint(p[1]) : 0, n > 2 ? __float_as_uint(p[2]) : 0, n > 3 ? __float_as_uint(p[3]) : 0);
    }
    static __device__ __forceinline__ void get(Word w, float (&x)[4]) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ Word put(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <typename T>
struct ScanRow16 {
    using Word = uint2;
    static __device__ __forceinline__ Word zero() { return make_uint2(0, 0); }
    static __device__ __forceinline__ Word one(const T* p, int n) {
        const auto at = [&](int k) { return k < n ? static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[k]) : 0u; };
        return make_uint2(at(0) | (at(1) << 16), at(2) | (at(3) << 16));
    }
};
template <>
struct ScanRow<__nv_bfloat16> : ScanRow16<__nv_bfloat16> {
    static __device__ __forceinline__ void get(Word w, float (&x)[4]) {
        x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xFFFF0000u);
        x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xFFFF0000u);
    }
    static __device__ __forceinline__ Word put(const float (&x)[4]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
template <>
struct ScanRow<__half> : ScanRow16<__half> {
    static __device__ __forceinline__ void get(Word w, float (&x)[4]) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
    static __device__ __forceinline__ Word put(const float (&x)[4]) {
        const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
};
// `n` of four adjacent elements are there; vec: they lie on a boundary of four
template <typename T>
__device__ __forceinline__ typename ScanRow<T>::Word scan_get(const T* p, int n, bool vec) {
    return vec ? *reinterpret_cast<const typename ScanRow<T>::Word*>(p) : ScanRow<T>::one(p, n);
}

// the states of a lane, zeros behind the last, as pairs
template <int PER>
__device__ __forceinline__ void scan_load(const float* p, int n, int states, bool vec, uint64_t (&x)[PER / 2]) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (vec) {
            if (n + i < states) v = *reinterpret_cast<const float4*>(p + n + i);
        } else {
            if (n + i < states) v.x = p[n + i];
            if (n + i + 1 < states) v.y = p[n + i + 1];
            if (n + i + 2 < states) v.z = p[n + i + 2];
            if (n + i + 3 < states) v.w = p[n + i + 3];
        }
        x[i / 2] = pair_of(v.x, v.y), x[i / 2 + 1] = pair_of(v.z, v.w);
    }
}
template <int PER>
__device__ __forceinline__ void scan_store(float* p, int n, int states, bool vec, const uint64_t (&x)[PER / 2]) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
        const float2 a = pair_get(x[i / 2]), b = pair_get(x[i / 2 + 1]);
        if (vec) {
            if (n + i < states) *reinterpret_cast<float4*>(p + n + i) = make_float4(a.x, a.y, b.x, b.y);
        } else {
            if (n + i < states) p[n + i] = a.x;
            if (n + i + 1 < states) p[n + i + 1] = a.y;
            if (n + i + 2 < states) p[n + i + 2] = b.x;
            if (n + i + 3 < states) p[n + i + 3] = b.y;
        }
    }
}

// A log2 e, two at a time, for exponentials of 2.  No further from 0 than a float goes: a rate of -inf (or one whose product is) forgets at a step above 0 all
// the same, and a step of 0, which also stands for tokens behind the last, leaves a state as it is.  A NaN stays one.
__device__ __forceinline__ uint64_t scan_rate(uint64_t a) {
    const float2 r = pair_get(pair_mul(a, pair_of(kActLog2e, kActLog2e)));
    const auto limited = [](float x) { return -max_nan(-max_nan(x, -3.402823466e38f), -3.402823466e38f); };
    return pair_of(limited(r.x), limited(r.y));
}

struct ScanPlan {
    int32_t tiles, parts, part_tokens;  // channel tiles of a group; parts of a sequence
    bool vec_rows, vec_bc, vec_states;  // whether rows of channels, rows of B and C, states lie on boundaries of 16 bytes
    float* ends;                        // [batch][parts][channels][states]: the start, then what each part leaves
    float* sums;                        // [batch][parts][channels]: of a part's steps, behind the part itself (0: none)
};

constexpr int kScanWarps = 4;   // of a CTA, each for itself
constexpr int kScanTile = 16;   // tokens of a tile

template <typename T, int LANES, int PER>
struct ScanShape {
    static constexpr int CHANNELS = 32 / LANES, STATES = LANES * PER;  // of a warp
    static constexpr int OWN = LANES <= 4 ? 4 : 2, GROUP = OWN * LANES;  // tokens of a group that a lane prepares, and all
    static constexpr bool CONVERT = sizeof(T) == 2;                         // B and C are kept in 32 bits
};
// what a warp has in shared memory
template <typename T, int LANES, int PER>
struct __align__(16) ScanShared {
    using S = ScanShape<T, LANES, PER>;
    struct __align__(16) Stage {
        T row[3][kScanTile][S::CHANNELS];  // x, dt, z
        T bc[2][kScanTile][S::STATES];
    } stage[2];
    float bc[S::CONVERT ? 2 : 1][S::CONVERT ? kScanTile : 1][S::STATES];
};

template <int BYTES>
__device__ __forceinline__ void scan_copy(void* to, const void* from, bool there) {  // (zeros where it is not)
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? BYTES : 0), "n"(BYTES) : "memory");
}

// A tile's rows into shared memory: WIDTH elements of every token, of which `width` are there; zeros behind them and behind the last token.
template <typename T, int WIDTH>
__device__ __forceinline__ void scan_rows(T (&to)[kScanTile][WIDTH], const T* from, int64_t stride, int tokens, int width, bool vec, int lane) {
    constexpr int BYTES = WIDTH * sizeof(T) < 16 ? WIDTH * sizeof(T) : 16, N = BYTES / sizeof(T), PIECES = WIDTH / N;
    if (vec && width == WIDTH) {
#pragma unroll
        for (int i = lane; i < kScanTile * PIECES; i += 32) {
            const int t = i / PIECES, k = i % PIECES * N;
            scan_copy<BYTES>(&to[t][k], from + (t < tokens ? t : 0) * stride + k, t < tokens);
        }
    } else {
#pragma unroll 4
        for (int i = lane; i < kScanTile * WIDTH; i += 32) {
            const int t = i / WIDTH, k = i % WIDTH;
            to[t][k] = t < tokens && k < width ? from[t * stride + k] : lin_from<T>(0.0f);
        }
    }
}

// The same for whole tiles on boundaries of 16 bytes, a tile after the other: a lane's place in the first row that it copies, which moves on.
template <typename T, int WIDTH>
struct ScanFeed {
    static constexpr int BYTES = WIDTH * sizeof(T) < 16 ? WIDTH * sizeof(T) : 16, N = BYTES / sizeof(T), PIECES = WIDTH / N, ROWS = 32 / PIECES;
    const T* at;
    __device__ __forceinline__ void start(const T* from, int64_t stride, int lane) { at = from + lane / PIECES * stride + lane % PIECES * N; }
    __device__ __forceinline__ void copy(T (&to)[kScanTile][WIDTH], int64_t stride, int lane) {
#pragma unroll
        for (int t = 0; t < kScanTile; t += ROWS) {
            if (ROWS <= kScanTile || lane / PIECES < kScanTile) scan_copy<BYTES>(&to[t + lane / PIECES][lane % PIECES * N], at, true);
            at += (ROWS < kScanTile ? ROWS : kScanTile) * stride;
        }
    }
};

// The place-th longest sequence (of equal ones the first), so that short ones fill up behind long ones; the place-th where there are more than 32.
__device__ __forceinline__ int scan_sequence(const ScanArgs& a, int place, int lane) {
    if (a.lengths == nullptr || a.batch > 32) return place;
    const int length = lane < a.batch ? min(max(a.lengths[lane], 0), a.tokens) : -1;
    int ahead = 0;
    for (int i = 0; i < a.batch; ++i) {
        const int other = __shfl_sync(kFullMask, length, i);
        ahead += other > length || (other == length && i < lane);
    }
    return __ffs(__ballot_sync(kFullMask, lane < a.batch && ahead == place)) - 1;
}

// A warp has CHANNELS channels of one group of a sequence, each of them in LANES lanes of PER states.  Tiles of tokens come into shared memory a tile
// ahead.  Of LANES tokens a lane prepares one (step, input), hands it to the channel's other lanes, and gets the token's sum over the states back
// from them to finish and store it.  Lanes that have the same states of different channels are neighbours: a load of 16 bytes that
// they share takes two cycles of the SM, four where they take turns.  ENDS: only the states and the sums of the steps are wanted.
template <typename T, int LANES, int PER, bool ENDS>
__global__ void __launch_bounds__(32 * kScanWarps, 3) scan_kernel(const ScanArgs a, const ScanPlan plan) {
    using S = ScanShape<T, LANES, PER>;
    constexpr int PAIRS = PER / 2;
    extern __shared__ __align__(16) unsigned char scan_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = blockIdx.y, b = scan_sequence(a, blockIdx.z, lane);
    ScanShared<T, LANES, PER>& sh = reinterpret_cast<ScanShared<T, LANES, PER>*>(scan_smem)[warp];
    const int tile = blockIdx.x * kScanWarps + warp, g = tile / plan.tiles, per_group = a.channels / a.groups;
    if (g >= a.groups) return;
    const int first = (tile % plan.tiles) * S::CHANNELS, c0 = g * per_group + first, channels = min(S::CHANNELS, per_group - first);
    const int mine = lane % S::CHANNELS, share = lane / S::CHANNELS, n0 = share * PER;
    const bool lives = mine < channels;
    int bits;
    const int slot = lin_slot(a.slots, a.num_slots, b, lane, bits);
    if (!ENDS && bits != 0 && a.status != nullptr && threadIdx.x == 0 && blockIdx.x == 0 && part == 0) atomicOr(a.status, bits);
    const int length = slot < 0 ? 0 : a.lengths == nullptr ? a.tokens : min(max(a.lengths[b], 0), a.tokens);
    const int begin = part * plan.part_tokens, end = min(length, begin + plan.part_tokens);
    const int64_t state = (static_cast<int64_t>(slot < 0 ? 0 : slot) * a.channels + c0 + mine) * a.states;
    const int64_t scratch = static_cast<int64_t>(b) * plan.parts * a.channels + c0 + mine;  // part p's: + p * channels
    const T* x = static_cast<const T*>(a.x) + b * a.x_stride[0] + c0;
    const T* dt = static_cast<const T*>(a.dt) + b * a.dt_stride[0] + c0;
    const T* z = ENDS || a.z == nullptr ? nullptr : static_cast<const T*>(a.z) + b * a.z_stride[0] + c0;
    const T* bm = static_cast<const T*>(a.B) + b * a.b_stride[0] + g * a.b_stride[2];
    const T* cm = static_cast<const T*>(a.C) + b * a.c_stride[0] + g * a.c_stride[2];
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + c0;
    const bool feeds = plan.vec_rows && plan.vec_bc && channels == S::CHANNELS && a.states == S::STATES;
    ScanFeed<T, S::CHANNELS> feed_x, feed_dt, feed_z;
    ScanFeed<T, S::STATES> feed_b, feed_c;
    feed_x.start(x + begin * a.x_stride[1], a.x_stride[1], lane), feed_dt.start(dt + begin * a.dt_stride[1], a.dt_stride[1], lane);
    feed_z.start(z + begin * a.z_stride[1], a.z_stride[1], lane);
    feed_b.start(bm + begin * a.b_stride[1], a.b_stride[1], lane), feed_c.start(cm + begin * a.c_stride[1], a.c_stride[1], lane);
    const auto fetch = [&](int t0, int stage) {
        const int n = end - t0;
        auto& to = sh.stage[stage];
        if (feeds && n >= kScanTile) {
            feed_x.copy(to.row[0], a.x_stride[1], lane);
            feed_dt.copy(to.row[1], a.dt_stride[1], lane);
            if (z != nullptr) feed_z.copy(to.row[2], a.z_stride[1], lane);
            feed_b.copy(to.bc[0], a.b_stride[1], lane);
            if (!ENDS) feed_c.copy(to.bc[1], a.c_stride[1], lane);
        } else {
            scan_rows<T, S::CHANNELS>(to.row[0], x + t0 * a.x_stride[1], a.x_stride[1], n, channels, plan.vec_rows, lane);
            scan_rows<T, S::CHANNELS>(to.row[1], dt + t0 * a.dt_stride[1], a.dt_stride[1], n, channels, plan.vec_rows, lane);
            if (z != nullptr) scan_rows<T, S::CHANNELS>(to.row[2], z + t0 * a.z_stride[1], a.z_stride[1], n, channels, plan.vec_rows, lane);
            scan_rows<T, S::STATES>(to.bc[0], bm + t0 * a.b_stride[1], a.b_stride[1], n, a.states, plan.vec_bc, lane);
            if (!ENDS) scan_rows<T, S::STATES>(to.bc[1], cm + t0 * a.c_stride[1], a.c_stride[1], n, a.states, plan.vec_bc, lane);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (begin < end) fetch(begin, 0);
    uint64_t h[PAIRS] = {}, rate[PAIRS] = {};
    float bias = 0.0f, direct = 0.0f;
    if (lives && slot >= 0) {
        scan_load<PER>(a.A + static_cast<int64_t>(c0 + mine) * a.states, n0, a.states, false, rate);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) rate[i] = scan_rate(rate[i]);
        if (a.dt_bias != nullptr) bias = a.dt_bias[c0 + mine];
        if (!ENDS && a.D != nullptr) direct = a.D[c0 + mine];
        if (plan.parts == 1 || (ENDS && part == 0)) {
            if (a.state_in != nullptr) scan_load<PER>(a.state_in + state, n0, a.states, plan.vec_states, h);
            if (ENDS) scan_store<PER>(plan.ends + scratch * a.states, n0, a.states, plan.vec_states, h);
        }
    }
    if (!ENDS && plan.parts > 1) {
        pdl_wait();
        if (lives && begin < max(end, 1)) {
            // what the parts before leave: the first goes on from the start itself
            scan_load<PER>(plan.ends + (scratch + static_cast<int64_t>(part > 0 ? 1 : 0) * a.channels) * a.states, n0, a.states, plan.vec_states, h);
            for (int p = 2; p <= part; ++p) {
                uint64_t left[PAIRS];
                const int64_t at = scratch + static_cast<int64_t>(p) * a.channels;
                scan_load<PER>(plan.ends + at * a.states, n0, a.states, plan.vec_states, left);
                // (a power by its cube root: where a part's tokens let a state grow the power itself may pass 32 bits, and the state, small or 0 before, need not)
                const float third = plan.sums[at] * (1.0f / 3.0f);
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) {
                    const float2 e = pair_get(pair_mul(rate[i], pair_of(third, third)));
                    const uint64_t root = pair_of(act_ex2(-max_nan(-e.x, -127.0f)), act_ex2(-max_nan(-e.y, -127.0f)));
                    h[i] = pair_fma(root, pair_mul(root, pair_mul(root, h[i])), left[i]);
                }
            }
        }
    }
    const bool softplus = a.softplus != 0, gated = z != nullptr;
    const int64_t out_step = LANES * a.out_stride[1];
    double all = 0.0;  // of the steps
    int stage = 0;
    for (int t0 = begin; t0 < end; t0 += kScanTile, stage ^= 1) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        if (t0 + kScanTile < end) fetch(t0 + kScanTile, stage ^ 1);
        auto& now = sh.stage[stage];
        const float *bs, *cs;
        if constexpr (S::CONVERT) {
#pragma unroll
            for (int i = lane; i < (ENDS ? 1 : 2) * kScanTile * S::STATES / 4; i += 32) {
                float v[4];
                ScanRow<T>::get(reinterpret_cast<const typename ScanRow<T>::Word*>(now.bc)[i], v);
                reinterpret_cast<float4*>(sh.bc)[i] = make_float4(v[0], v[1], v[2], v[3]);
            }
            __syncwarp();
            bs = &sh.bc[0][0][n0], cs = &sh.bc[1][0][n0];
        } else {
            bs = reinterpret_cast<const float*>(&now.bc[0][0][n0]), cs = reinterpret_cast<const float*>(&now.bc[1][0][n0]);
        }
        // Of a group of tokens a lane prepares and finishes OWN, LANES apart.  `tokens`: of the tile; behind the last nothing happens, as with a step of 0.
        float sum = 0.0f;
        const auto walk = [&](auto whole, int tokens) {
            constexpr bool WHOLE = decltype(whole)::value;
            [[maybe_unused]] T* to = out + (t0 + share) * a.out_stride[1] + mine;
#pragma unroll 1
            for (int t = 0; t < (WHOLE ? kScanTile : tokens); t += S::GROUP) {
                float xs[S::OWN], d[S::OWN], dx[S::OWN], y[S::GROUP];
#pragma unroll
                for (int k = 0; k < S::OWN; ++k) {
                    const int own = t + k * LANES + share;
                    xs[k] = lin_float(now.row[0][own][mine]);
                    const float raw = lin_float(now.row[1][own][mine]) + bias, soft = act_softplus(raw);
                    d[k] = softplus ? soft : raw;
                    dx[k] = d[k] * xs[k];
                    if (!WHOLE && own >= tokens) d[k] = dx[k] = 0.0f;
                    if (ENDS) sum += d[k];
                }
#pragma unroll
                for (int j = 0; j < S::GROUP; ++j) {
                    const int at = (t + j) * S::STATES;
                    float dj = d[j / LANES], dxj = dx[j / LANES];
                    if constexpr (LANES > 1) {
                        const int from = j % LANES * S::CHANNELS + mine;
                        dj = __shfl_sync(kFullMask, dj, from), dxj = __shfl_sync(kFullMask, dxj, from);
                    }
                    const uint64_t dd = pair_of(dj, dj), ddx = pair_of(dxj, dxj);
                    uint64_t parts = 0;
#pragma unroll
                    for (int i = 0; i < PAIRS; i += 2) {
                        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(bs + at + 2 * i);
                        h[i] = pair_fma(pair_ex2(pair_mul(dd, rate[i])), h[i], pair_mul(ddx, q.x));
                        h[i + 1] = pair_fma(pair_ex2(pair_mul(dd, rate[i + 1])), h[i + 1], pair_mul(ddx, q.y));
                        if constexpr (!ENDS) {
                            const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(cs + at + 2 * i);
                            parts = i == 0 ? pair_mul(r.x, h[0]) : pair_fma(r.x, h[i], parts);
                            parts = pair_fma(r.y, h[i + 1], parts);
                        }
                    }
                    y[j] = pair_get(parts).x + pair_get(parts).y;
                }
                if constexpr (!ENDS) {
#pragma unroll
                    for (int k = 0; k < S::OWN; ++k) {
                        const int own = t + k * LANES + share;
                        // the sums over the channel's lanes, each lane its own token's
                        float* v = y + k * LANES;
#pragma unroll
                        for (int o = LANES / 2; o > 0; o /= 2) {
                            const bool upper = (share & o) != 0;
#pragma unroll
                            for (int l = 0; l < o; ++l) {
                                const float other = __shfl_xor_sync(kFullMask, upper ? v[l] : v[l + o], o * S::CHANNELS);
                                v[l] = (upper ? v[l + o] : v[l]) + other;
                            }
                        }
                        const float open = act_silu(lin_float(now.row[2][own][mine]));
                        const float all = fmaf(direct, xs[k], v[0]);
                        if (lives && (WHOLE || own < tokens)) *to = lin_from<T>(gated ? all * open : all);
                        to += out_step;
                    }
                }
            }
        };
        if (end - t0 >= kScanTile) walk(std::true_type(), kScanTile);
        else walk(std::false_type(), end - t0);
        if (ENDS) all += static_cast<double>(sum);
        __syncwarp();
    }
    if constexpr (ENDS) {
        pdl_launch_dependents();
#pragma unroll
        for (int o = S::CHANNELS; o < 32; o *= 2) all += __shfl_xor_sync(kFullMask, all, o);
        if (lives) {
            const int64_t at = scratch + static_cast<int64_t>(part + 1) * a.channels;
            scan_store<PER>(plan.ends + at * a.states, n0, a.states, plan.vec_states, h);
            if (share == 0) plan.sums[at] = static_cast<float>(all);
        }
    } else {
        const int last = min(a.tokens, begin + plan.part_tokens);
        for (int t = max(begin, length) + share; t < last; t += LANES)
            if (lives) out[t * a.out_stride[1] + mine] = lin_from<T>(0.0f);
        const bool keeps = length == 0 ? part == 0 : begin < length && end == length;  // the part with the last token
        if (keeps && slot >= 0 && lives) scan_store<PER>(a.state_out + state, n0, a.states, plan.vec_states, h);
    }
}

// One token per sequence: a pass over the states, LANES lanes a channel, eight states a lane.  A CTA goes through `each` sequences with the same
// channels, so that their rates are read once and addresses only move on.
// Bound by the states' traffic and its latency (of the 13 cycles between a warp's instructions 6.5 are waits for a load): 192 sequences of 4096 channels of 16 states 31 us
// from HBM (3.5 TB/s; 24.5 where the states are in L2), 35 with fp32 inputs, whose registers spill (52 bytes of 64 registers).  What
// is on its way at once are the warps' loads, so more warps are worth more than a warp's loads ahead: two sequences ahead in five CTAs an SM 33, three in
// four 36, four through shared memory by asynchronous copies 30; the next piece of four states beside its neighbour lanes' 32.6; four states a
// lane, with addresses worked out anew for every sequence (260 instructions for 16 bytes of each lane), 40.  (With the depth of 1 written out, not as kStepAhead, the
// loop comes out otherwise: that call 29 us, 300 sequences of 1536 channels 18.1 for 16.9, 512 of 1024 20.7 for 19.9.)
constexpr int kStepThreads = 128, kStepMostEach = 32, kStepAhead = 1, kStepCtas = 8, kStepPer = 8;
template <typename T, int LANES>
__global__ void __launch_bounds__(kStepThreads, kStepCtas) scan_step_kernel(const ScanArgs a, const ScanPlan plan, int each) {
    constexpr int CHANNELS = kStepThreads / LANES, PAIRS = kStepPer / 2;
    using Row = ScanRow<T>;
    __shared__ int s_named[kStepMostEach], s_slot[kStepMostEach];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.x / plan.tiles, per_group = a.channels / a.groups, first = (blockIdx.x % plan.tiles) * CHANNELS;
    const int mine = first + tid / LANES, n0 = (tid % LANES) * kStepPer, c = g * per_group + mine;
    const bool lives = mine < per_group;
    const int b0 = blockIdx.y * each, count = min(each, a.batch - b0);
    if (tid < count) s_named[tid] = a.slots == nullptr ? b0 + tid : a.slots[b0 + tid];
    // where the next sequence's are
    const T* x_at = static_cast<const T*>(a.x) + b0 * a.x_stride[0] + c;
    const T* dt_at = static_cast<const T*>(a.dt) + b0 * a.dt_stride[0] + c;
    const T* z_at = static_cast<const T*>(a.z) + b0 * a.z_stride[0] + c;
    const T* b_at = static_cast<const T*>(a.B) + b0 * a.b_stride[0] + g * a.b_stride[2] + n0;
    const T* c_at = static_cast<const T*>(a.C) + b0 * a.c_stride[0] + g * a.c_stride[2] + n0;
    T* out_at = static_cast<T*>(a.out) + b0 * a.out_stride[0] + c;
    const int64_t row = static_cast<int64_t>(a.channels) * a.states, place = static_cast<int64_t>(c) * a.states;
    uint64_t h[kStepAhead][PAIRS], rate[PAIRS] = {};
    T x[kStepAhead], dt[kStepAhead], z[kStepAhead];
    typename Row::Word bv[kStepAhead][2], cv[kStepAhead][2];
    // sequence i's: its state too, which may be read whether the slot is this sequence's or an earlier one's
    const auto fetch = [&](int i, int k) {
        const int named = s_named[i];
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) h[k][p] = 0;
        if (a.state_in != nullptr && named >= 0 && named < a.num_slots)
            scan_load<kStepPer>(a.state_in + named * row + place, n0, a.states, plan.vec_states, h[k]);
        x[k] = *x_at, dt[k] = *dt_at;
        x_at += a.x_stride[0], dt_at += a.dt_stride[0];
        if (a.z != nullptr) z[k] = *z_at, z_at += a.z_stride[0];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            bv[k][p] = cv[k][p] = Row::zero();
            if (n0 + 4 * p < a.states) {
                bv[k][p] = scan_get(b_at + 4 * p, a.states - n0 - 4 * p, plan.vec_bc);
                cv[k][p] = scan_get(c_at + 4 * p, a.states - n0 - 4 * p, plan.vec_bc);
            }
        }
        b_at += a.b_stride[0], c_at += a.c_stride[0];
    };
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStepAhead; ++k)
        if (lives && k < count) fetch(k, k);
    float bias = 0.0f, direct = 0.0f;
    if (lives) {
        scan_load<kStepPer>(a.A + place, n0, a.states, plan.vec_states && reinterpret_cast<uintptr_t>(a.A) % 16 == 0, rate);
        if (a.dt_bias != nullptr) bias = a.dt_bias[c];
        if (a.D != nullptr) direct = a.D[c];
    }
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) rate[p] = scan_rate(rate[p]);
    for (int i = warp; i < count; i += kStepThreads / 32) {
        int bits;
        const int slot = lin_slot(a.slots, a.num_slots, b0 + i, lane, bits);
        if (lane == 0) s_slot[i] = slot;
        if (bits != 0 && a.status != nullptr && lane == 0 && blockIdx.x == 0) atomicOr(a.status, bits);
    }
    __syncthreads();
    for (int i0 = 0; i0 < count; i0 += kStepAhead) {
#pragma unroll
        for (int k = 0; k < kStepAhead; ++k) {
            const int i = i0 + k;
            if (i >= count) break;
            const int slot = s_slot[i];
            float y = 0.0f, xf = 0.0f;
            if (lives) {
                xf = lin_float(x[k]);
                float d = lin_float(dt[k]) + bias;
                if (a.softplus != 0) d = act_softplus(d);
                const uint64_t dd = pair_of(d, d), dx = pair_of(d * xf, d * xf);
                uint64_t sum = 0;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float bf[4], cf[4];
                    Row::get(bv[k][p], bf);
                    Row::get(cv[k][p], cf);
                    uint64_t &u = h[k][2 * p], &v = h[k][2 * p + 1];
                    u = pair_fma(pair_ex2(pair_mul(rate[2 * p], dd)), u, pair_mul(dx, pair_of(bf[0], bf[1])));
                    v = pair_fma(pair_ex2(pair_mul(rate[2 * p + 1], dd)), v, pair_mul(dx, pair_of(bf[2], bf[3])));
                    sum = p == 0 ? pair_mul(u, pair_of(cf[0], cf[1])) : pair_fma(u, pair_of(cf[0], cf[1]), sum);
                    sum = pair_fma(v, pair_of(cf[2], cf[3]), sum);
                }
                y = pair_get(sum).x + pair_get(sum).y;
            }
#pragma unroll
            for (int o = 1; o < LANES; o *= 2) y += __shfl_xor_sync(kFullMask, y, o);
            if (lives) {
                if (slot >= 0) scan_store<kStepPer>(a.state_out + slot * row + place, n0, a.states, plan.vec_states, h[k]);
                if (n0 == 0) {
                    if (a.D != nullptr) y = fmaf(direct, xf, y);
                    if (a.z != nullptr) y *= act_silu(lin_float(z[k]));
                    *out_at = lin_from<T>(slot >= 0 ? y : 0.0f);
                }
                out_at += a.out_stride[0];
                if (i + kStepAhead < count) fetch(i + kStepAhead, k);
            }
        }
    }
}

// How a prompt is cut up: states of a lane, and parts where whole sequences leave most of the chip without a warp.
struct ScanCut {
    int per, lanes, parts, part_tokens;
};
// Chosen by a model of the time.  A token takes a warp alone 54 ns with four states a lane and 82 with eight, and a scheduler with several warps 33 and
// 63 for each (1 x 4096 tokens of 512 channels 218 and 335 us, 8 x 1024 of 4096 233 and 225).  A pass for the parts' ends is three quarters of
// a pass for outputs (2 parts of the former 188 and 299, 16 of them 39 and 47; 24 of 1 x 8192 of 2048 channels 182, one 699).
static ScanCut scan_cut(const ScanArgs& a) {
    ScanCut best = {};
    double least = 0.0;
    for (int per = 4; per <= 8; per *= 2) {
        ScanCut cut = {per, 1, 1, 1 << 30};
        while (cut.lanes * per < a.states) cut.lanes *= 2;
        if (cut.lanes > 8 || (per > 4 && a.states <= 4)) continue;
        const double alone = per == 4 ? 54e-3 : 82e-3, shared = per == 4 ? 33e-3 : 63e-3;
        const int64_t warps = (static_cast<int64_t>(a.channels / a.groups) * cut.lanes + 31) / 32 * a.groups * a.batch;
        const auto token = [&](int64_t w) {
            const double each = shared * static_cast<double>((w + 4 * kNumSMs - 1) / (4 * kNumSMs));
            return each > alone ? each : alone;
        };
        for (int parts = 1; parts <= 48 && (parts == 1 || parts * 2 * kScanTile <= a.tokens); parts += parts < 4 ? 1 : parts < 16 ? 4 : 8) {
            const double time = static_cast<double>(a.tokens) / parts * (token(warps * parts) + (parts > 1 ? 0.75 * token(warps * (parts - 1)) : 0.0)) +
                                (parts > 1 ? 2.0 + 0.2 * parts : 0.0);
            if (least > 0.0 && time >= least) continue;
            least = time;
            best = cut;
            if (parts > 1) {
                best.part_tokens = ((a.tokens + parts - 1) / parts + kScanTile - 1) / kScanTile * kScanTile;
                best.parts = (a.tokens + best.part_tokens - 1) / best.part_tokens;
            }
        }
    }
    return best;
}
static int64_t scan_scratch(const ScanArgs& a, const ScanCut& cut) {
    return cut.parts == 1 ? 0 : static_cast<int64_t>(a.batch) * cut.parts * a.channels * (a.states + 1) * 4;
}

template <typename T>
static ScanPlan scan_plan(const ScanArgs& a) {
    ScanPlan plan = {};
    plan.parts = 1, plan.part_tokens = 1 << 30;
    const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    constexpr int N = 16 / sizeof(T);
    int64_t strides = a.x_stride[0] | a.x_stride[1] | a.dt_stride[0] | a.dt_stride[1] | (a.channels / a.groups);
    if (a.z != nullptr) strides |= a.z_stride[0] | a.z_stride[1];
    plan.vec_rows = strides % N == 0 && (at(a.x) | at(a.dt) | at(a.z)) % 16 == 0;
    plan.vec_states = a.states % 4 == 0 && (at(a.state_in) | at(a.state_out)) % 16 == 0;
    plan.vec_bc = (a.b_stride[0] | a.b_stride[1] | a.b_stride[2] | a.c_stride[0] | a.c_stride[1] | a.c_stride[2] | a.states) % N == 0 &&
                  (at(a.B) | at(a.C)) % 16 == 0;
    return plan;
}

template <typename T, int LANES, int PER>
static int launch_scan(const ScanArgs& a, const ScanCut& cut, void* scratch, cudaStream_t st) {
    ScanPlan plan = scan_plan<T>(a);
    plan.tiles = (a.channels / a.groups + 32 / LANES - 1) / (32 / LANES);
    const int64_t blocks = (static_cast<int64_t>(plan.tiles) * a.groups + kScanWarps - 1) / kScanWarps;
    constexpr int smem = kScanWarps * sizeof(ScanShared<T, LANES, PER>);
    if (smem > 48 * 1024) FB_TRY(check_cuda(cudaFuncSetAttribute(scan_kernel<T, LANES, PER, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "selective_scan"));
    if (cut.parts > 1) {
        FB_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "selective_scan: scratch must lie on a boundary of 16 bytes");
        plan.parts = cut.parts, plan.part_tokens = cut.part_tokens;
        plan.ends = static_cast<float*>(scratch);
        plan.sums = plan.ends + static_cast<int64_t>(a.batch) * cut.parts * a.channels * a.states;
        if (smem > 48 * 1024) FB_TRY(check_cuda(cudaFuncSetAttribute(scan_kernel<T, LANES, PER, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "selective_scan"));
        FB_TRY(launch_after(scan_kernel<T, LANES, PER, true>, dim3(static_cast<unsigned>(blocks), plan.parts - 1, a.batch), dim3(32 * kScanWarps), smem, st, false,
                            "selective_scan", a, plan));
    }
    return launch_after(scan_kernel<T, LANES, PER, false>, dim3(static_cast<unsigned>(blocks), plan.parts, a.batch), dim3(32 * kScanWarps), smem, st, plan.parts > 1,
                        "selective_scan", a, plan);
}

template <typename T, int LANES>
static int launch_step(const ScanArgs& a, cudaStream_t st) {
    ScanPlan plan = scan_plan<T>(a);
    plan.tiles = (a.channels / a.groups + kStepThreads / LANES - 1) / (kStepThreads / LANES);
    const int64_t blocks = static_cast<int64_t>(plan.tiles) * a.groups;
    plan.vec_bc = ((a.b_stride[0] | a.b_stride[2] | a.c_stride[0] | a.c_stride[2] | a.states) % 4) == 0 &&
                  (reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C)) % (4 * sizeof(T)) == 0;
    // all CTAs at once, as many as the SMs hold, each with as few sequences as that leaves
    const int64_t rows = blocks < kStepCtas * kNumSMs ? kStepCtas * kNumSMs / blocks : 1;
    int64_t each = (a.batch + rows - 1) / rows;
    if (each > kStepMostEach) each = kStepMostEach;
    return launch_after(scan_step_kernel<T, LANES>, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>((a.batch + each - 1) / each)), dim3(kStepThreads), 0, st, false,
                        "selective_scan", a, plan, static_cast<int>(each));
}

template <typename T>
static int launch_scan(const ScanArgs& a, void* scratch, cudaStream_t st) {
    if (a.tokens == 1 && a.lengths == nullptr) {
        if (a.states <= 8) return launch_step<T, 1>(a, st);
        if (a.states <= 16) return launch_step<T, 2>(a, st);
        if (a.states <= 32) return launch_step<T, 4>(a, st);
        return launch_step<T, 8>(a, st);
    }
    const ScanCut cut = scan_cut(a);
    if (cut.per == 8) {
        if (cut.lanes == 1) return launch_scan<T, 1, 8>(a, cut, scratch, st);
        if (cut.lanes == 2) return launch_scan<T, 2, 8>(a, cut, scratch, st);
        if (cut.lanes == 4) return launch_scan<T, 4, 8>(a, cut, scratch, st);
        return launch_scan<T, 8, 8>(a, cut, scratch, st);
    }
    if (cut.lanes == 1) return launch_scan<T, 1, 4>(a, cut, scratch, st);
    if (cut.lanes == 2) return launch_scan<T, 2, 4>(a, cut, scratch, st);
    if (cut.lanes == 4) return launch_scan<T, 4, 4>(a, cut, scratch, st);
    return launch_scan<T, 8, 4>(a, cut, scratch, st);
}

}  // namespace fb

extern "C" int64_t functs_b200_selective_scan_scratch_bytes(const functs_b200_selective_scan_args* a) {
    using namespace fb;
    if (a == nullptr || a->batch <= 0 || a->tokens <= 0 || a->channels <= 0 || a->groups <= 0 || a->channels % a->groups != 0 || a->states <= 0 ||
        a->states > kScanMaxStates)
        return 0;
    return scan_scratch(*a, scan_cut(*a));
}

extern "C" int functs_b200_selective_scan(const functs_b200_selective_scan_args* args, void* scratch, void* stream) {
    using namespace fb;
    FB_REQUIRE(args != nullptr, "selective_scan: null pointer");
    const ScanArgs& a = *args;
    FB_REQUIRE(a.dtype >= FB_DTYPE_F32 && a.dtype <= FB_DTYPE_BF16, "selective_scan: unknown dtype %d", a.dtype);
    FB_REQUIRE(a.batch >= 0 && a.batch < 65536 && a.tokens >= 0 && a.tokens <= (1 << 30), "selective_scan: batch must be 0 .. 65535, tokens 0 .. %d", 1 << 30);
    FB_REQUIRE(a.channels >= 1 && a.channels <= (1 << 24) && a.groups >= 1 && a.channels % a.groups == 0,
               "selective_scan: channels (%d) must be a multiple of groups (%d), and at most %d", a.channels, a.groups, 1 << 24);
    FB_REQUIRE(a.states >= 1 && a.states <= kScanMaxStates, "selective_scan: states (%d) must be 1 .. %d", a.states, kScanMaxStates);
    FB_REQUIRE(a.num_slots >= 0, "selective_scan: num_slots must not be negative");
    FB_REQUIRE(a.slots != nullptr || a.num_slots == a.batch, "selective_scan: without slots there are as many states as sequences");
    if (a.batch == 0) return FB_OK;
    FB_REQUIRE(a.A != nullptr && a.state_out != nullptr, "selective_scan: null pointer");
    FB_REQUIRE(a.tokens == 0 || (a.x != nullptr && a.dt != nullptr && a.B != nullptr && a.C != nullptr && a.out != nullptr), "selective_scan: null pointer");
    const uintptr_t elements = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dt) | reinterpret_cast<uintptr_t>(a.z) |
                               reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C) | reinterpret_cast<uintptr_t>(a.out);
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.D) | reinterpret_cast<uintptr_t>(a.dt_bias) |
                            reinterpret_cast<uintptr_t>(a.state_in) | reinterpret_cast<uintptr_t>(a.state_out) | reinterpret_cast<uintptr_t>(a.slots) |
                            reinterpret_cast<uintptr_t>(a.lengths) | reinterpret_cast<uintptr_t>(a.status);
    FB_REQUIRE(elements % (a.dtype == FB_DTYPE_F32 ? 4 : 2) == 0 && words % 4 == 0, "selective_scan: pointers must lie on a boundary of their type");
    const cudaStream_t st = as_stream(stream);
    if (a.dtype == FB_DTYPE_F32) return launch_scan<float>(a, scratch, st);
    if (a.dtype == FB_DTYPE_F16) return launch_scan<__half>(a, scratch, st);
    return launch_scan<__nv_bfloat16>(a, scratch, st);
}
