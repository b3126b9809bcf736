// Attention with a decaying state over prompts, a chunk of 64 tokens at a time on the tensor cores.
//
// Within a chunk whose first token follows the state S (l = decay, i and j count from 0, n = its tokens):
//   out_i = scale * ( l^(i+1) S^T q_i  +  sum_{j <= i} l^(i-j) (q_i . k_j) v_j )          S' = l^n S + sum_j l^(n-1-j) k_j v_j^T
// which is four products:  G = Q K^T,  X = S^T Q^T,  Y = V^T P^T with P = G masked and decayed,  U = K^T W with W = decayed V.
// S stays in registers in fp32 and is decayed and added there (the tensor core truncates when it adds); the decay is a sum of two floats,
// because its rounding would be the same for every chunk.
//
// Operands have 8 bits, so what has more is a sum of parts: S and P of two (what they make is rounded to 16 bits at once, 2^-17 apart),
// W of three (it makes the state, which is fp32).  Q, K and V are their own part in bf16, two in fp16 (exact), three in fp32; products of
// parts that are below the result's precision are left out, and the small ones are added first.
//
// One layout serves all products: core matrices of 8 tokens x 16 bytes (8 channels), channel groups 1024 bytes apart.  Read along channels
// a tile is a K-major operand of rows = tokens, read along tokens an MN-major operand of rows = channels, with the two strides of the
// descriptor exchanged.  All products have M = 128 rows; where there are 64, the others are whatever follows in shared memory, and their
// results, which are rows of their own, are not looked at.
//
// NaN and infinities: a masked entry of P is 0 by selection, but 0 * V is not 0 for a V that is not finite, so such entries are taken as 0 in
// Y (not in W) and the outputs of their channel, from their token on, are set to NaN.
#include <type_traits>

#include "linattn.cuh"
#include "tcgen05.cuh"

namespace fb {

constexpr int kLtThreads = 256;
constexpr int kLtChunk = 64;
constexpr uint32_t kLtWaitLimit = 4000000u;
constexpr uint32_t kLtTmemCols = 512;
// TMEM columns of the four products
constexpr uint32_t kLtG = 0, kLtX = 64, kLtY = 128, kLtU = 192;

template <typename T, int DK_, int DV_>
struct LtCfg {
    static constexpr int DK = DK_, DV = DV_;
    static constexpr bool kAsync = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int NX = kAsync ? 1 : std::is_same<T, __half>::value ? 2 : 3;  // parts of q, k, v
    static constexpr int NS = std::is_same<T, float>::value ? 3 : 2;                // parts of S and P
    static constexpr int NW = 3;                                                    // parts of W
    static constexpr int kStages = kAsync ? 2 : 1;
    static constexpr int kTileK = kLtChunk * DK * 2, kTileV = kLtChunk * DV * 2, kPartS = DK * DV * 2, kPartP = kLtChunk * kLtChunk * 2;
    static constexpr int kStage = NX * (2 * kTileK + kTileV);
    static constexpr int oS = kStages * kStage, oW = oS + NS * kPartS, oP = oW + NW * kTileV, oMisc = oP + NS * kPartP;
};

struct LtMisc {
    uint64_t bar_g, bar_u, bar_y;
    uint32_t tmem;
    int dead;          // a wait ran out
    int any_bad;       // the chunk has a V that is not finite
    int b;
    float power_lo;    // what power[64] leaves of decay^64
    float power[kLtChunk + 1];
    int first_bad[128];  // per channel: the first such token of the chunk
};

__device__ __forceinline__ void lt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}

__device__ __forceinline__ uint32_t lt_pack(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// Eight values as N parts of eight bf16 each; part p goes to at + p * stride.
template <int N>
__device__ __forceinline__ void lt_store_parts(unsigned char* at, int stride, float (&x)[8]) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = lt_pack(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4*>(at + p * stride) = make_uint4(u[0], u[1], u[2], u[3]);
        if (p + 1 < N) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __fsub_rn(x[2 * i], __uint_as_float(u[i] << 16));
                x[2 * i + 1] = __fsub_rn(x[2 * i + 1], __uint_as_float(u[i] & 0xFFFF0000u));
            }
        }
    }
}

__device__ __forceinline__ void lt_cp16(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// Eight channels of one row in fp32, zeros behind `valid`.
template <typename T>
__device__ __forceinline__ void lt_load8(const T* p, int valid, bool aligned, float (&x)[8]) {
    if (aligned && valid == 8) {
        if (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = lin_float(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < valid ? lin_float(p[i]) : 0.0f;
    }
}

// (8-channel group, token) of the `i`-th of a tile's 16-byte pieces: eight tokens beside one another, then four groups
__device__ __forceinline__ void lt_piece(int i, int groups, int& group, int& token) {
    const int lane = i & 31, w = i >> 5, per = groups / 4;  // groups is a multiple of 4
    group = (w % per) * 4 + (lane >> 3);
    token = (w / per) * 8 + (lane & 7);
}
__device__ __forceinline__ int lt_offset(int group, int token) { return group * 1024 + (token >> 3) * 128 + (token & 7) * 16; }

template <typename T, int DK, int DV>
__global__ void __launch_bounds__(kLtThreads, 1) linattn_chunk_kernel(const LinArgs a, int tiles, bool aligned) {
    using C = LtCfg<T, DK, DV>;
    extern __shared__ __align__(1024) unsigned char smem[];
    LtMisc& m = *reinterpret_cast<LtMisc*>(smem + C::oMisc);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile = blockIdx.x % tiles, h = (blockIdx.x / tiles) % a.heads, order = blockIdx.x / (tiles * a.heads);
    const int hk = h / (a.heads / a.kv_heads), col0 = tile * DV, dv = min(DV, a.dv - col0);

    // long sequences first, so that the last CTAs are short ones
    if (tid == 0) m.b = order;
    __syncthreads();
    if (a.lengths != nullptr && a.batch <= kLtThreads) {
        if (tid < a.batch) {
            const int mine = lin_length(a, tid);
            int before = 0;
            for (int j = 0; j < a.batch; ++j) {
                const int other = lin_length(a, j);
                before += other > mine || (other == mine && j < tid);
            }
            if (before == order) m.b = tid;
        }
        __syncthreads();
    }
    const int b = m.b;
    int bits;
    const int slot = lin_slot(a, b, lane, bits);
    if (bits != 0 && a.status != nullptr && tid == 0 && tile == 0) atomicOr(a.status, bits);
    const int length = slot < 0 ? 0 : lin_length(a, b);
    const int64_t state_at = (static_cast<int64_t>(slot < 0 ? 0 : slot) * a.heads + h) * a.dk * a.dv + col0;
    const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[2];
    const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
    const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2] + col0;
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[2] + col0;

    // rows behind the sequence
    for (int64_t i = tid; i < static_cast<int64_t>(a.tokens - length) * dv; i += kLtThreads) {
        const int64_t t = i / dv;
        out[(length + t) * a.out_stride[1] + (i - t * dv)] = lin_from<T>(0.0f);
    }
    if (slot < 0) return;

    // S: thread -> row (its TMEM lane) and half of the columns
    constexpr int SC = DV / 2;
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const bool has_row = row < a.dk;
    float s[SC];
    {
        const float* at = a.state_in + state_at + static_cast<int64_t>(row) * a.dv + half * SC;
#pragma unroll
        for (int c = 0; c < SC; ++c) s[c] = a.state_in != nullptr && has_row && half * SC + c < dv ? at[c] : 0.0f;
    }
    const double log_decay = static_cast<double>(fmaxf(a.log_decay[h], -1e30f));
    if (tid <= kLtChunk) {
        const double p = exp(log_decay * tid);
        m.power[tid] = static_cast<float>(p);
        if (tid == kLtChunk) m.power_lo = static_cast<float>(p - static_cast<double>(static_cast<float>(p)));
    }
    if (tid < 128) m.first_bad[tid] = kLtChunk;
    if (tid == 0) {
        mbar_init(&m.bar_g, 1);
        mbar_init(&m.bar_u, 1);
        mbar_init(&m.bar_y, 1);
        fence_barrier_init();
        m.dead = m.any_bad = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&m.tmem)), "r"(kLtTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = m.tmem, lane_base = tmem + ((static_cast<uint32_t>(warp & 3) * 32u) << 16);
    // instruction descriptors: fp32 accumulators, bf16 operands, M = 128; N, and which operands are MN-major
    constexpr uint32_t kD = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24), kMnA = 1u << 15, kMnB = 1u << 16;
    constexpr uint32_t kIdescG = kD | ((kLtChunk / 8) << 17), kIdescX = kD | kMnA | ((kLtChunk / 8) << 17), kIdescU = kD | kMnA | kMnB | ((DV / 8) << 17);

    const int chunks = (length + kLtChunk - 1) / kLtChunk;
    // brings chunk c into its stage
    const auto fetch = [&](int c) {
        unsigned char* st = smem + (c % C::kStages) * C::kStage;
        const int t0 = c * kLtChunk, n = min(kLtChunk, length - t0);
        if (C::kAsync && aligned) {
#pragma unroll
            for (int i = tid; i < kLtChunk * DK / 8; i += kLtThreads) {
                int g, t;
                lt_piece(i, DK / 8, g, t);
                const int bytes = t < n ? max(0, min(16, (a.dk - g * 8) * 2)) : 0;
                const int at = lt_offset(g, t);
                lt_cp16(st + at, bytes > 0 ? q + (t0 + t) * a.q_stride[1] + g * 8 : q, bytes);
                lt_cp16(st + C::kTileK + at, bytes > 0 ? k + (t0 + t) * a.k_stride[1] + g * 8 : k, bytes);
            }
#pragma unroll
            for (int i = tid; i < kLtChunk * DV / 8; i += kLtThreads) {
                int g, t;
                lt_piece(i, DV / 8, g, t);
                const int bytes = t < n ? max(0, min(16, (dv - g * 8) * 2)) : 0;
                lt_cp16(st + 2 * C::kTileK + lt_offset(g, t), bytes > 0 ? v + (t0 + t) * a.v_stride[1] + g * 8 : v, bytes);
            }
        } else {
            for (int i = tid; i < kLtChunk * DK / 8; i += kLtThreads) {
                int g, t;
                lt_piece(i, DK / 8, g, t);
                const int valid = t < n ? max(0, min(8, a.dk - g * 8)) : 0;
                const int at = lt_offset(g, t);
                float x[8];
                lt_load8(q + (t0 + t) * a.q_stride[1] + g * 8, valid, aligned, x);
                lt_store_parts<C::NX>(st + at, C::kTileK, x);
                lt_load8(k + (t0 + t) * a.k_stride[1] + g * 8, valid, aligned, x);
                lt_store_parts<C::NX>(st + C::NX * C::kTileK + at, C::kTileK, x);
            }
            for (int i = tid; i < kLtChunk * DV / 8; i += kLtThreads) {
                int g, t;
                lt_piece(i, DV / 8, g, t);
                const int valid = t < n ? max(0, min(8, dv - g * 8)) : 0;
                const int at = lt_offset(g, t);
                float x[8];
                lt_load8(v + (t0 + t) * a.v_stride[1] + g * 8, valid, aligned, x);
                if (!C::kAsync) {  // W from the values themselves
                    const float w = m.power[t < n ? n - 1 - t : 0];
                    float y[8];
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        y[e] = x[e] * w;
                        bad |= !(fabsf(x[e]) <= 3.4028234663852886e38f);
                    }
                    if (bad) {
                        m.any_bad = 1;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (!(fabsf(x[e]) <= 3.4028234663852886e38f)) {
                                atomicMin(&m.first_bad[g * 8 + e], t);
                                x[e] = 0.0f;
                            }
                    }
                    lt_store_parts<C::NW>(smem + C::oW + at, C::kTileV, y);
                }
                lt_store_parts<C::NX>(st + 2 * C::NX * C::kTileK + at, C::kTileV, x);
            }
        }
    };

    if (C::kStages == 2 && chunks > 0) fetch(0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int c = 0; c < chunks; ++c) {
        const uint32_t parity = c & 1;
        const int t0 = c * kLtChunk, n = min(kLtChunk, length - t0);
        unsigned char* st = smem + (c % C::kStages) * C::kStage;
        const uint32_t sq = smem_u32(st), sk = sq + C::NX * C::kTileK, sv = sk + C::NX * C::kTileK, ss = smem_u32(smem + C::oS),
                       sw = smem_u32(smem + C::oW), sp = smem_u32(smem + C::oP);
        if (C::kStages == 2) {
            if (c + 1 < chunks) fetch(c + 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            fetch(c);
        }
        fence_proxy_async();
        __syncthreads();
        if (tid == 0) {  // G = Q K^T
            tc_fence_after();
            bool add = false;
#pragma unroll
            for (int sum = C::NX - 1; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p)
#pragma unroll
                    for (int i = 0; i < DK / 16; ++i) {
                        lt_mma(tmem + kLtG, make_smem_desc(sq + p * C::kTileK + i * 2048, 1024, 128),
                               make_smem_desc(sk + (sum - p) * C::kTileK + i * 2048, 1024, 128), kIdescG, add);
                        add = true;
                    }
            tc_commit(&m.bar_g);
        }
        if (C::kAsync) {  // W = decayed V
            for (int i = tid; i < kLtChunk * DV / 8; i += kLtThreads) {
                int g, t;
                lt_piece(i, DV / 8, g, t);
                const int at = lt_offset(g, t);
                uint4* vp = reinterpret_cast<uint4*>(st + 2 * C::kTileK + at);
                const uint4 u = *vp;
                const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
                const float w = m.power[t < n ? n - 1 - t : 0];
                float x[8];
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bad |= (w4[e] & 0x7F80u) == 0x7F80u || (w4[e] & 0x7F800000u) == 0x7F800000u;
                    x[2 * e] = __uint_as_float(w4[e] << 16) * w;
                    x[2 * e + 1] = __uint_as_float(w4[e] & 0xFFFF0000u) * w;
                }
                if (bad) {
                    m.any_bad = 1;
                    uint32_t fix[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        fix[e] = w4[e];
                        if ((w4[e] & 0x7F80u) == 0x7F80u) fix[e] &= 0xFFFF0000u, atomicMin(&m.first_bad[g * 8 + 2 * e], t);
                        if ((w4[e] & 0x7F800000u) == 0x7F800000u) fix[e] &= 0xFFFFu, atomicMin(&m.first_bad[g * 8 + 2 * e + 1], t);
                    }
                    *vp = make_uint4(fix[0], fix[1], fix[2], fix[3]);
                }
                lt_store_parts<C::NW>(smem + C::oW + at, C::kTileV, x);
            }
        }
        // S as an operand: rows dk, groups of 8 columns DK * 16 bytes apart
        if (row < DK) {
#pragma unroll
            for (int g = 0; g < SC / 8; ++g) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[g * 8 + e];
                lt_store_parts<C::NS>(smem + C::oS + (half * (SC / 8) + g) * (DK * 16) + (row >> 3) * 128 + (row & 7) * 16, C::kPartS, x);
            }
        }
        fence_proxy_async();
        __syncthreads();
        if (tid == 0) {
            tc_fence_after();
            bool add = false;
            // X = S^T Q^T
#pragma unroll
            for (int sum = C::NS - 1; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p) {
                    if (sum - p >= C::NX) continue;
#pragma unroll
                    for (int i = 0; i < DK / 16; ++i) {
                        lt_mma(tmem + kLtX, make_smem_desc(ss + p * C::kPartS + i * 256, 128, DK * 16),
                               make_smem_desc(sq + (sum - p) * C::kTileK + i * 2048, 1024, 128), kIdescX, add);
                        add = true;
                    }
                }
            // U = K^T W
            add = false;
#pragma unroll
            for (int sum = C::NW - 1; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p) {
                    if (sum - p >= C::NX) continue;
#pragma unroll
                    for (int i = 0; i < kLtChunk / 16; ++i) {
                        lt_mma(tmem + kLtU, make_smem_desc(sk + (sum - p) * C::kTileK + i * 256, 128, 1024),
                               make_smem_desc(sw + p * C::kTileV + i * 256, 128, 1024), kIdescU, add);
                        add = true;
                    }
                }
            tc_commit(&m.bar_u);
        }
        // P: rows = tokens i, in the first two warps of each half
        if ((warp & 3) < 2) {
            if (!mbar_wait_bounded(&m.bar_g, parity, kLtWaitLimit)) m.dead = 1;
            tc_fence_after();
            float g[32];
            tc_ld_32cols(lane_base + kLtG + half * 32, g);
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int j = half * 32 + o * 8 + e;
                    x[e] = j <= row ? g[o * 8 + e] * m.power[row - j < 0 ? 0 : row - j] : 0.0f;
                }
                lt_store_parts<C::NS>(smem + C::oP + (half * 4 + o) * 1024 + (row >> 3) * 128 + (row & 7) * 16, C::kPartP, x);
            }
            fence_proxy_async();
            tc_fence_before();
        }
        __syncthreads();
        if (m.dead) break;
        if (tid == 0) {  // Y = V^T P^T
            tc_fence_after();
            bool add = false;
#pragma unroll
            for (int sum = C::NS - 1; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p) {
                    if (sum - p >= C::NX) continue;
#pragma unroll
                    for (int i = 0; i < kLtChunk / 16; ++i) {
                        lt_mma(tmem + kLtY, make_smem_desc(sv + (sum - p) * C::kTileV + i * 256, 128, 1024),
                               make_smem_desc(sp + p * C::kPartP + i * 2048, 1024, 128), kIdescX, add);
                        add = true;
                    }
                }
            tc_commit(&m.bar_y);
        }
        if (!mbar_wait_bounded(&m.bar_u, parity, kLtWaitLimit)) m.dead = 1;
        tc_fence_after();
        {
            const float pn = m.power[n], pn_lo = n == kLtChunk ? m.power_lo : 0.0f;
#pragma unroll
            for (int g = 0; g < SC / 32; ++g) {
                float u[32];
                tc_ld_32cols(lane_base + kLtU + half * SC + g * 32, u);
#pragma unroll
                for (int e = 0; e < 32; ++e) s[g * 32 + e] = fmaf(pn, s[g * 32 + e], fmaf(pn_lo, s[g * 32 + e], u[e]));
            }
        }
        if (!mbar_wait_bounded(&m.bar_y, parity, kLtWaitLimit)) m.dead = 1;
        tc_fence_after();
        {
            float x[32], y[32];
            tc_ld_32cols(lane_base + kLtX + half * 32, x);
            tc_ld_32cols(lane_base + kLtY + half * 32, y);
            const int first_bad = m.any_bad ? m.first_bad[row] : kLtChunk;
            if (row < dv) {
                T* at = out + (t0 + half * 32) * a.out_stride[1] + row;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int t = half * 32 + i;
                    float o = fmaf(m.power[t + 1], x[i], y[i]) * a.scale;
                    if (t >= first_bad) o = __int_as_float(0x7fffffff);
                    if (t < n) *at = lin_from<T>(o);
                    at += a.out_stride[1];
                }
            }
        }
        tc_fence_before();
        __syncthreads();
        if (m.dead) break;
        if (m.any_bad) {  // (the next chunk's marks come behind a barrier)
            if (tid < 128) m.first_bad[tid] = kLtChunk;
            __syncthreads();
            if (tid == 0) m.any_bad = 0;
            __syncthreads();
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (m.dead && tid == 0 && a.status != nullptr) atomicOr(a.status, FB_STATUS_WAIT_TIMEOUT);
    if (has_row) {
        float* at = a.state_out + state_at + static_cast<int64_t>(row) * a.dv + half * SC;
#pragma unroll
        for (int c = 0; c < SC; ++c)
            if (half * SC + c < dv) at[c] = s[c];
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kLtTmemCols) : "memory");
}

template <typename T, int DK, int DV>
static int launch_chunk(const LinArgs& a, cudaStream_t st) {
    using C = LtCfg<T, DK, DV>;
    constexpr int bytes = C::oMisc + static_cast<int>(sizeof(LtMisc));
    static_assert(bytes <= 232448, "shared memory");
    const int tiles = (a.dv + DV - 1) / DV;
    const int64_t ctas = static_cast<int64_t>(a.batch) * a.heads * tiles;
    FB_REQUIRE(ctas < (1ll << 31), "linear_attention: batch * heads is too large");
    bool aligned = true;
    const void* base[3] = {a.q, a.k, a.v};
    const int64_t* stride[3] = {a.q_stride, a.k_stride, a.v_stride};
    for (int i = 0; i < 3; ++i) {
        aligned = aligned && reinterpret_cast<uintptr_t>(base[i]) % 16 == 0;
        for (int j = 0; j < 3; ++j) aligned = aligned && stride[i][j] * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    }
    FB_TRY(check_cuda(cudaFuncSetAttribute(linattn_chunk_kernel<T, DK, DV>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "linear_attention"));
    return launch_after(linattn_chunk_kernel<T, DK, DV>, dim3(static_cast<unsigned>(ctas)), dim3(kLtThreads), bytes, st, false, "linear_attention",
                        a, tiles, aligned);
}

template <typename T>
static int launch_chunk(const LinArgs& a, cudaStream_t st) {
    constexpr int wide = std::is_same<T, float>::value ? 64 : 128;  // (fp32 operands of 128 x 128 do not fit shared memory)
    if (a.dk <= 64) return a.dv <= 64 ? launch_chunk<T, 64, 64>(a, st) : launch_chunk<T, 64, wide>(a, st);
    return a.dv <= 64 ? launch_chunk<T, 128, 64>(a, st) : launch_chunk<T, 128, wide>(a, st);
}

int launch_linattn_chunk(const LinArgs& a, cudaStream_t st) {
    if (a.dtype == FB_DTYPE_F32) return launch_chunk<float>(a, st);
    if (a.dtype == FB_DTYPE_F16) return launch_chunk<__half>(a, st);
    return launch_chunk<__nv_bfloat16>(a, st);
}

}  // namespace fb
