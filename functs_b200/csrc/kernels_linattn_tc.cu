// Attention with a decaying state over prompts, a chunk of 64 tokens at a time on the tensor cores.
//
// Within a chunk whose first token follows the state S (l = decay, i and j count from 0, n = its tokens):
//   out_i = scale * ( l^(i+1) S^T q_i  +  sum_{j <= i} l^(i-j) (q_i . k_j) v_j )          S' = l^n S + sum_j l^(n-1-j) k_j v_j^T
// which is four products:  G = Q K^T,  X = S^T Q^T,  Y = V^T P^T with P = G masked and decayed,  U = K^T W with W = decayed V.
// S is decayed and added to in fp32 outside the tensor core (which truncates when it adds).
//
// Operands have 8 bits, so what has more is a sum of parts: S and P of two (what they make is rounded to 16 bits at once, 2^-17 apart;
// three where the outputs are fp32), W of three (it makes the state, which is fp32: two would leave 2^-16 of each term, with three it is 2e-7 off).  Q, K and V are
// their own part in bf16, two in fp16 (exact), three in fp32; products of parts that are below the result's precision are left out, and the
// small ones are added first.
//
// X, Y and U are formed transposed, with the channels of V as rows, so that S^T is an operand in TMEM (in shared memory it cost 128 KB of
// writes and reads per chunk, and shared memory's bandwidth was the bound), and stores of S and of the outputs are coalesced.  All products
// have M = 128 rows; where there are 64, the others are whatever follows in memory, and their results, which are rows of their own, are not
// looked at.  Q, K and V lie as rows of 64 channels (128 bytes, swizzled), read along channels (K-major) or along tokens (MN-major); W and P,
// which threads write, as core matrices of 8 rows x 16 bytes.
//
// Roles, so that loads, conversions, products and stores of neighbouring chunks overlap (one CTA per SM):
//   S   8 warps: S' = l^n S + U in TMEM, a channel of V per thread, half of the channels of K; S' as operand parts
//   W   W from V (and, where tiles cannot be had by TMA, or are split into parts, the tiles themselves)
//   O   the outputs from X and Y
//   P   P from G: four warps (there are 64 rows)
//   beside these, one warp issues U and G, one X and Y, so that the tensor core has work while either waits, and one issues the copies.
// G of the next chunk is formed in U's columns as soon as they have been read, so P is ready long before its product's turn.
//
// What bounds it: 128 x 128 heads in bf16 take 2.8 us per chunk and SM, where HBM would let 64 tokens pass in 1.5.  The chunk's 44 products
// alone take 2100 cycles (2700 where a lane is chosen by comparison instead of election), and more beside the other warps, whose reads and
// writes of shared memory they share; the warps' 13 850 instructions of a chunk issue at 2.4 of 4 per cycle, and no pipe is busy more than 41 % of
// the time.  The roles wait for one another: U for W, S for U, X for S, the outputs for X, chunk after chunk (when a chunk took 4.2 us, leaving
// out the work of one role saved 3 to 13 %, of four together 34 %).  16 x 2048 tokens of 16 heads 186 us (2.9 TB/s), 8192 tokens of 16 heads 93,
// 16 uneven prompts of up to 2048 tokens 108.  In fp16 and fp32 the threads split every tile into parts: 4.4 us per chunk of 64 x 64 heads,
// 10.4 of 128 x 128, which shared memory holds once.
// Tried and slower: G in columns of its own behind X, so that it does not wait for U to be read (2.95 and 3.3 us per chunk against 2.75);
// S read eight columns at a time with the next eight on their way (2.82); the roles' loops unrolled (4.5: instruction cache); one lane of a
// warp waiting for all (6.5); all of a chunk's phases by all warps between block barriers (6.8).
//
// NaN and infinities: a masked entry of P is 0 by selection, but 0 * V is not 0 for a V that is not finite, so such entries are taken as 0 in
// Y (not in W) and the outputs of their channel, from their token on, are set to NaN.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "linattn.cuh"
#include "tcgen05.cuh"

namespace fb {

constexpr int kLtChunk = 64;
constexpr int kLtRanked = 128;  // sequences, as many as a CTA has threads for at least
constexpr int kLtWarpsS = 8, kLtWarpsP = 8;  // (of the P group four make P, two issue products, one copies)
constexpr uint32_t kLtWaitLimit = 200000u, kLtWaitLimitDropped = 5000u;
// Development switch (functs_b200_debug_set "linattn_drop_state"): in this thread's calls nobody says that S is there, so that the waits for it,
// and for what follows from it, run out.
static thread_local int t_lt_drop = 0;
void linattn_set_drop_state(int on) { t_lt_drop = on ? 1 : 0; }
// TMEM columns: U (and, between two of them, G), X, Y, S^T in fp32 and as two operand parts of DK / 2 columns, or as three parts, which are exact
constexpr uint32_t kLtU = 0, kLtG = 0, kLtX = 128, kLtY = 192, kLtS = 256, kLtTmemCols = 512;

template <typename T, int DK_, int DV_>
struct LtCfg {
    static constexpr int DK = DK_, DV = DV_;
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int NX = kBf16 ? 1 : std::is_same<T, __half>::value ? 2 : 3;  // parts of q, k, v
    static constexpr int NS = std::is_same<T, float>::value ? 3 : 2;               // parts of S and P
    static constexpr int NW = 3;                                                   // parts of W
    static constexpr int kWarpsW = 8, kWarpsO = kBf16 ? 8 : 4;
    static constexpr int kFirstW = kLtWarpsS, kFirstO = kFirstW + kWarpsW, kFirstP = kFirstO + kWarpsO, kThreads = 32 * (kFirstP + kLtWarpsP);
    static_assert(kFirstO % 4 == 0 && kFirstP % 4 == 0, "a warp's TMEM lanes go by its number");
    static constexpr int kTileK = kLtChunk * DK * 2, kTileV = kLtChunk * DV * 2, kPartP = kLtChunk * kLtChunk * 2;
    static constexpr int kStage = 2 * NX * kTileK, oK = NX * kTileK;  // Q, and K behind it
    // stages of Q and K, and of W: two where they fit; of V in bf16 three (it is read a chunk ahead, for W)
    static constexpr int kStages = 2 * (kStage + (NX + NW) * kTileV) + NS * kPartP <= 224 * 1024 ? 2 : 1;
    static constexpr int kStagesV = kBf16 ? 3 : kStages;
    static constexpr int oV = kStages * kStage, oW = oV + kStagesV * NX * kTileV, oP = oW + kStages * NW * kTileV, oMisc = oP + NS * kPartP;
    static constexpr uint32_t kParts = NS == 3 ? kLtS : kLtS + 128;  // TMEM columns of the parts of S^T
};

struct LtMisc {
    uint64_t full[2], full_v[3], v_whole[3], empty[2], w_full[2], w_free[2];  // stages; v_whole: V with zeros where it must have them
    uint64_t g_full, g_read, u_full, u_free, s_full, x_full, p_full, y_full, xy_free;
    uint64_t none_left[2];                         // of the two warps that issue products: theirs are done
    uint32_t tmem;
    int dead;                                      // a wait ran out
    uint32_t wait_limit;                           // tries of a wait
    int b;
    float power_next, power_gap, power_off;        // the float beyond power[64] on decay^64's side, how far, and how far decay^64 is (relative)
    float power[kLtChunk + 4];                        // decay^i
    float scaled_front[kLtChunk], scaled[kLtChunk + 4];  // scale * decay^i, and in front of it what masked entries of P read
    __align__(16) float scaled_next[kLtChunk];        // scale * decay^(i+1)
    uint2 weight[kLtChunk];                        // decay^i as three bf16 parts, each twice: w0 w0, w1 w1 (w2 below)
    uint32_t weight2[kLtChunk];
    int bad;                                       // the first token with a V that is not finite
    int first_bad[128];                            // the same per channel (behind it the channel's state is not finite either)
};

struct LtPlan {
    int segs;        // parts of a sequence
    int seg_tokens;  // a multiple of the chunk
    int mode;        // 0: whole sequences; 1: the state that each part adds, 2: outputs of the parts
    int boundary;    // of which all rows lie: 16, 8, 4 or 2 bytes
    float* states;   // [batch * heads][segs][dk][dv]
    float2* decays;  // [batch * heads][segs]: of each part, as a sum of two floats
    uint32_t wait_limit;  // tries of a wait
    int drop_state;       // the switch below
};

// ---- small pieces ---------------------------------------------------------------------------------------------------

__device__ __forceinline__ void lt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// One lane of a whole warp.  (Where the compiler knows that one thread alone is active, it keeps descriptors in uniform registers: 2094
// cycles to issue a chunk's 44 products instead of 2732 behind `lane == 0`.)
__device__ __forceinline__ bool lt_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// tiles of rows of 128 bytes with the 128-byte swizzle: the 8-row groups `sbo` apart, the next 64 channels (MN-major) `lbo`
__device__ __forceinline__ uint64_t lt_desc_swizzled(uint32_t addr, uint32_t lbo, uint32_t sbo) { return make_smem_desc(addr, lbo, sbo) | (2ull << 61); }

__device__ __forceinline__ void lt_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// 16 TMEM columns of the thread's lane; 8 columns
__device__ __forceinline__ void lt_ld(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void lt_ld(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
// (the values are operands of the wait, so that nothing uses them before it)
__device__ __forceinline__ void lt_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void lt_ld_wait(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
__device__ __forceinline__ void lt_st(uint32_t taddr, const float (&x)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"f"(x[0]),
        "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]), "f"(x[8]), "f"(x[9]), "f"(x[10]), "f"(x[11]), "f"(x[12]),
        "f"(x[13]), "f"(x[14]), "f"(x[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void lt_st(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void lt_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One box of 64 channels x 64 tokens of a head.
__device__ __forceinline__ void lt_tma(void* dst, const CUtensorMap* map, int channel, int token, int head, int seq, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(channel), "r"(token), "r"(head), "r"(seq), "r"(smem_u32(bar))
        : "memory");
}

// Waits for a phase; gives up when the limit runs out or somebody else has given up.
// (the hardware holds the thread for up to some ten microseconds: asking again and again took issue slots from the warps that work)
__device__ __forceinline__ bool lt_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool lt_wait_one(LtMisc& m, uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < m.wait_limit; ++i) {
        if (lt_try(bar, parity)) return true;
        if ((i & 7u) == 7u && *reinterpret_cast<volatile int*>(&m.dead)) return false;
    }
    *reinterpret_cast<volatile int*>(&m.dead) = 1;
    return false;
}
__device__ __forceinline__ bool lt_wait(LtMisc& m, uint64_t* bar, uint32_t parity) {
    const bool ok = lt_wait_one(m, bar, parity);
    return __all_sync(kFullMask, ok) != 0;
}
// A warp's shared-memory writes are operands from here on: one arrival.
__device__ __forceinline__ void lt_arrive_operands(uint64_t* bar, int lane) {
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}
// A warp has read its TMEM columns: one arrival.
__device__ __forceinline__ void lt_arrive_read(uint64_t* bar, int lane) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// A bf16 part of two values: of two parts both are rounded (2^-8 of its power of two is left for the second, 2^-17 lost, at most);
// of three the first two are the values' upper halves, taken out of them, which is exact and does not overflow, and the last what is left, rounded.
template <int N>
__device__ __forceinline__ uint32_t lt_part(float& x, float& y, int p) {
    if (p + 1 == N || N == 2) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
        const uint32_t u = *reinterpret_cast<const uint32_t*>(&r);
        if (p + 1 < N) {
            x = __fsub_rn(x, __uint_as_float(u << 16));
            y = __fsub_rn(y, __uint_as_float(u & 0xFFFF0000u));
        }
        return u;
    }
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    x = __fsub_rn(x, __uint_as_float(a & 0xFFFF0000u));
    y = __fsub_rn(y, __uint_as_float(b & 0xFFFF0000u));
    return __byte_perm(a, b, 0x7632);
}
// Eight values as N parts of eight bf16 each, part p at `at + p * stride`.
template <int N>
__device__ __forceinline__ void lt_store_parts(unsigned char* at, int stride, float (&x)[8]) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = lt_part<N>(x[2 * i], x[2 * i + 1], p);
        *reinterpret_cast<uint4*>(at + p * stride) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// Eight channels of one row in fp32, zeros behind `valid`; in the largest loads that the rows' boundary allows.
template <typename T, typename P>
__device__ __forceinline__ void lt_load8_as(const T* p, float (&x)[8]) {
    constexpr int N = sizeof(P) / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += N) {
        const P u = reinterpret_cast<const P*>(p)[i / N];
#pragma unroll
        for (int j = 0; j < N; ++j) x[i + j] = lin_float(reinterpret_cast<const T*>(&u)[j]);
    }
}
template <typename T>
__device__ __forceinline__ void lt_load8(const T* p, int valid, int boundary, float (&x)[8]) {
    if (valid == 8 && boundary == 16) lt_load8_as<T, uint4>(p, x);
    else if (valid == 8 && boundary == 8) lt_load8_as<T, uint2>(p, x);
    else if (sizeof(T) == 2 && valid == 8 && boundary == 4) lt_load8_as<T, uint32_t>(p, x);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < valid ? lin_float(p[i]) : 0.0f;
    }
}
// Eight bf16 values times a weight of three parts, as three parts, in bf16 arithmetic: with a fused multiply-add that rounds once, products
// and their errors are exact.  v w0 = p + r and v w1 = t0 + t1; r + t0 = s + e (D. Knuth, The Art of Computer Programming, volume 2, 4.2.2,
// theorem B); the parts are p, s and e + t1 + v w2, which is rounded below 2^-25 of the product.
__device__ __forceinline__ void lt_weigh(unsigned char* at, int stride, const uint32_t (&v)[4], const uint32_t (&w)[3]) {
    const auto bf = [](const uint32_t& u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
    uint32_t part[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 x = bf(v[i]), w0 = bf(w[0]), w1 = bf(w[1]);
        const __nv_bfloat162 p = __hmul2_rn(x, w0), r = __hfma2(x, w0, __hneg2(p)), t0 = __hmul2_rn(x, w1), t1 = __hfma2(x, w1, __hneg2(t0));
        const __nv_bfloat162 s = __hadd2_rn(r, t0), rest = __hsub2_rn(s, r);
        const __nv_bfloat162 e = __hadd2_rn(__hsub2_rn(r, __hsub2_rn(s, rest)), __hsub2_rn(t0, rest));
        const __nv_bfloat162 q = __hadd2_rn(e, __hfma2(x, bf(w[2]), t1));
        part[0][i] = *reinterpret_cast<const uint32_t*>(&p);
        part[1][i] = *reinterpret_cast<const uint32_t*>(&s);
        part[2][i] = *reinterpret_cast<const uint32_t*>(&q);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(at + k * stride) = make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
}
// (a swizzled tile: rows of 64 channels; a plain one: groups of 8 channels 1024 bytes apart)
__device__ __forceinline__ int lt_swizzled(int group, int token) { return (group >> 3) * 8192 + token * 128 + (((group ^ token) & 7) << 4); }
__device__ __forceinline__ int lt_plain(int group, int token) { return group * 1024 + (token >> 3) * 128 + (token & 7) * 16; }
__device__ __forceinline__ bool lt_finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

// ---- the kernel -----------------------------------------------------------------------------------------------------

// LOADS: how the rows are read.  By TMA; by loads of 16 bytes; or by those that plan.boundary allows (a kernel of its own: their code beside
// the others' costs: 16 x 2048 tokens of 16 heads of 64 in fp32 279 us; when it was taken out 297, with it 317).
enum LtLoads { kLtTma, kLtWide, kLtAny };
template <typename T, int DK, int DV, LtLoads LOADS>
__global__ void __launch_bounds__(LtCfg<T, DK, DV>::kThreads, 1)
linattn_chunk_kernel(const LinArgs a, const LtPlan plan, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v) {
    constexpr bool TMA = LOADS == kLtTma;
    using C = LtCfg<T, DK, DV>;
    constexpr int kWarpsW = C::kWarpsW;
    extern __shared__ __align__(1024) unsigned char smem[];
    LtMisc& m = *reinterpret_cast<LtMisc*>(smem + C::oMisc);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seg = blockIdx.x % plan.segs, rest = blockIdx.x / plan.segs;
    const int h = rest % a.heads, order = rest / a.heads, hk = h / (a.heads / a.kv_heads);

    if (plan.mode == 1) pdl_launch_dependents();
    // Long sequences first, so that the last CTAs are short ones.  Every CTA ranks all of them, so not beyond kLtRanked: uneven sequences of 4 to 8
    // heads of 128 in bf16, 128 of up to 1024 tokens 121 us (in the order given 134), 96 with few long ones 89 (119), 128 of up to 256 108 (104);
    // but 200 of up to 128 154 ranked and 123 in the order given, 600 of 512 325 and 171, 1000 of 64 1530 and 253.
    if (tid == 0) m.b = order;
    __syncthreads();
    if (a.lengths != nullptr && a.batch <= kLtRanked) {
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
    if (bits != 0 && a.status != nullptr && tid == 0 && seg == 0) atomicOr(a.status, bits);
    const int length = slot < 0 ? 0 : lin_length(a, b);
    const int seg0 = plan.segs > 1 ? seg * plan.seg_tokens : 0;                                        // first token of this part
    const int seg_end = plan.segs > 1 && seg + 1 < plan.segs ? min(length, seg0 + plan.seg_tokens) : length;
    const bool outputs = plan.mode != 1;
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[2];
    if (outputs) {  // rows behind the sequence, those that fall in this part
        const int z0 = max(length, seg0), z1 = plan.segs > 1 && seg + 1 < plan.segs ? min(a.tokens, seg0 + plan.seg_tokens) : a.tokens;
        lin_clear(out, a.out_stride[1], z0, z1, a.dv);
    }
    if (slot < 0 || (plan.mode == 2 && seg_end <= seg0)) return;
    const int chunks = max(0, seg_end - seg0 + kLtChunk - 1) / kLtChunk;

    const double log_decay = static_cast<double>(lin_log_decay(a, h));
    if (tid <= kLtChunk) {
        const double p = exp(log_decay * tid);
        m.power[tid] = static_cast<float>(p);
        m.scaled[tid] = static_cast<float>(p * static_cast<double>(a.scale));
        if (tid > 0) m.scaled_next[tid - 1] = m.scaled[tid];
        if (tid < kLtChunk) {
            double left = p;
            uint32_t w[3];
            for (int i = 0; i < 3; ++i) {
                const __nv_bfloat16 part = __float2bfloat16_rn(static_cast<float>(left));
                left -= static_cast<double>(__bfloat162float(part));
                const __nv_bfloat162 twice = __halves2bfloat162(part, part);
                w[i] = *reinterpret_cast<const uint32_t*>(&twice);
            }
            m.weight[tid] = make_uint2(w[0], w[1]);
            m.weight2[tid] = w[2];
        } else {
            const float near = static_cast<float>(p), off = static_cast<float>(p - static_cast<double>(near));
            const float next = __uint_as_float(__float_as_uint(near) + (off > 0.0f ? 1u : 0xffffffffu));
            m.power_next = off != 0.0f && near > 0.0f ? next : near;
            m.power_gap = near > 0.0f ? fabsf(next - near) / near : 1.0f;
            m.power_off = near > 0.0f ? fabsf(off) / near : 0.0f;
        }
    }
    if (plan.mode == 1 && tid == kLtChunk + 1) {  // the decay of the whole part
        const double p = exp(log_decay * static_cast<double>(max(0, seg_end - seg0)));
        const float near = static_cast<float>(p);
        plan.decays[(static_cast<int64_t>(b) * a.heads + h) * plan.segs + seg] = make_float2(near, static_cast<float>(p - static_cast<double>(near)));
    }
    if (tid < 128) m.first_bad[tid] = 0x7fffffff;
    if (tid < kLtChunk) m.scaled_front[tid] = 0.0f;
    if (tid == 0) {
        for (int i = 0; i < C::kStagesV; ++i) mbar_init(&m.full_v[i], 1), mbar_init(&m.v_whole[i], kWarpsW);
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&m.full[i], TMA ? 1 : kWarpsW);
            mbar_init(&m.empty[i], outputs ? 2 : 1);
            mbar_init(&m.w_full[i], kWarpsW);
            mbar_init(&m.w_free[i], 1);
        }
        mbar_init(&m.g_full, 1), mbar_init(&m.u_full, 1), mbar_init(&m.x_full, 1), mbar_init(&m.y_full, 1);
        mbar_init(&m.none_left[0], 1), mbar_init(&m.none_left[1], 1);
        mbar_init(&m.p_full, 4);
        mbar_init(&m.g_read, 4);
        mbar_init(&m.u_free, kLtWarpsS);
        mbar_init(&m.s_full, kLtWarpsS);
        mbar_init(&m.xy_free, C::kWarpsO);
        fence_barrier_init();
        m.dead = 0;
        m.wait_limit = plan.wait_limit;
        m.bad = 0x7fffffff;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&m.tmem)), "r"(kLtTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (plan.mode == 2) pdl_wait();  // (the parts' states)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = m.tmem, lane_base = tmem + ((static_cast<uint32_t>(warp & 3) * 32u) << 16);

    if (warp < kLtWarpsS) {
        // ---- S: row = channel of V
        constexpr int kHalf = DK / 2;
        const int row = (warp & 3) * 32 + lane, k0 = (warp >> 2) * kHalf;
        const bool has_row = row < a.dv;
        const int64_t cell = static_cast<int64_t>(k0) * a.dv + row;
        const int64_t own = (static_cast<int64_t>(slot) * a.heads + h) * a.dk * a.dv + cell;
        const int64_t part = ((static_cast<int64_t>(b) * a.heads + h) * plan.segs + seg) * a.dk * a.dv + cell;
        const float* from = plan.mode == 2 ? plan.states + part : plan.mode == 0 && a.state_in != nullptr ? a.state_in + own : nullptr;
        float* to = plan.mode == 2 ? nullptr : plan.mode == 1 ? plan.states + part : a.state_out + own;
        // (loops stay loops here and below: unrolled, the roles' code did not fit the instruction cache, and a third of all stalls was for it)
        const auto keep_parts = [&](int g, float (&s)[16]) {
#pragma unroll
            for (int p = 0; p < C::NS; ++p) {
                uint32_t u[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = lt_part<C::NS>(s[2 * e], s[2 * e + 1], p);
                lt_st(lane_base + C::kParts + p * kHalf + (k0 + g) / 2, u);
            }
        };
        const auto at_end = [&](int g, const float (&s)[16]) {
            if (to == nullptr || !has_row) return;
            float* at = to + static_cast<int64_t>(g) * a.dv;
#pragma unroll
            for (int e = 0; e < 16; ++e, at += a.dv)
                if (k0 + g + e < a.dk) *at = s[e];
        };
        if (from == nullptr && chunks > 0) {  // (little code: fetched cold, the loop below takes 2 us)
            // the columns that this warp itself reads: U does not wait for S, so nothing orders other warps' columns before its first reading
            const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (C::NS == 2) {
#pragma unroll 1
                for (int g = 0; g < kHalf; g += 8) lt_st(lane_base + kLtS + k0 + g, zero);
            }
#pragma unroll 1
            for (int p = 0; p < C::NS; ++p) {
#pragma unroll 1
                for (int g = 0; g < kHalf / 2; g += 8) lt_st(lane_base + C::kParts + p * kHalf + k0 / 2 + g, zero);
            }
        } else {
#pragma unroll 1
            for (int g = 0; g < kHalf; g += 16) {
                float s[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = from != nullptr && has_row && k0 + g + e < a.dk ? from[static_cast<int64_t>(g + e) * a.dv] : 0.0f;
                if (chunks == 0) at_end(g, s);
                if (C::NS == 2) lt_st(lane_base + kLtS + k0 + g, s);
                keep_parts(g, s);
            }
        }
        lt_st_wait();
        if (!plan.drop_state) lt_arrive_read(&m.s_full, lane);
        // The decay of a chunk is one of the two floats beside it, by turns, so that their product stays within half a step of the decay's
        // power: rounded the same way every time it would be off by 2^-25 per chunk.
        float drift = 0.0f;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {  // S behind chunk c
            const bool last = c + 1 == chunks;
            if (!lt_wait(m, &m.u_full, c & 1)) break;
            if (C::NS == 3 && outputs && !last && !lt_wait(m, &m.x_full, c & 1)) break;  // (the parts are S itself)
            tc_fence_after();
            const int n = min(kLtChunk, seg_end - seg0 - c * kLtChunk);
            float pn = m.power[n];
            if (n == kLtChunk) {
                drift += m.power_off;
                if (2.0f * drift >= m.power_gap) {
                    drift -= m.power_gap;
                    pn = m.power_next;
                }
            }
#pragma unroll 1
            for (int g = 0; g < kHalf; g += 16) {
                float s[16];
                uint32_t ru[16];
                lt_ld(lane_base + kLtU + k0 + g, ru);
                if (C::NS == 3) {
                    uint32_t p0[8], p1[8], p2[8];
                    lt_ld(lane_base + C::kParts + (k0 + g) / 2, p0);
                    lt_ld(lane_base + C::kParts + kHalf + (k0 + g) / 2, p1);
                    lt_ld(lane_base + C::kParts + 2 * kHalf + (k0 + g) / 2, p2);
                    lt_ld_wait(p0);
                    lt_ld_wait(p1);
                    lt_ld_wait(p2);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {  // (exact: the parts are 24 bits)
                        s[2 * e] = __uint_as_float(p0[e] << 16) + (__uint_as_float(p1[e] << 16) + __uint_as_float(p2[e] << 16));
                        s[2 * e + 1] = __uint_as_float(p0[e] & 0xFFFF0000u) + (__uint_as_float(p1[e] & 0xFFFF0000u) + __uint_as_float(p2[e] & 0xFFFF0000u));
                    }
                } else {
                    uint32_t rs[16];
                    lt_ld(lane_base + kLtS + k0 + g, rs);
                    lt_ld_wait(rs);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __uint_as_float(rs[e]);
                }
                lt_ld_wait(ru);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = fmaf(pn, s[e], __uint_as_float(ru[e]));
                if (last) at_end(g, s);
                else if (C::NS == 3) keep_parts(g, s);
                else lt_st(lane_base + kLtS + k0 + g, s);
            }
            lt_arrive_read(&m.u_free, lane);
            if (last) break;
            if (C::NS == 2 && outputs) {  // its parts, when the product before is done with the last ones
                if (!lt_wait(m, &m.x_full, c & 1)) break;
                tc_fence_after();
                lt_st_wait();
#pragma unroll 1
                for (int g = 0; g < kHalf; g += 16) {
                    uint32_t rs[16];
                    float s[16];
                    lt_ld(lane_base + kLtS + k0 + g, rs);
                    lt_ld_wait(rs);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __uint_as_float(rs[e]);
                    keep_parts(g, s);
                }
            }
            lt_st_wait();
            lt_arrive_read(&m.s_full, lane);  // (not behind the last: it would be a phase ahead of the products' wait for this one)
        }
    } else if (warp < C::kFirstO) {
        // ---- W (and tiles)
        constexpr int threads = 32 * kWarpsW;
        const int rank = warp - C::kFirstW, id = rank * 32 + lane;
        const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[2] + seg0 * a.q_stride[1];
        const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2] + seg0 * a.k_stride[1];
        const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2] + seg0 * a.v_stride[1];
        uint32_t w[3] = {0, 0, 0};  // the weight of this thread's token
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            const int t0 = c * kLtChunk, n = min(kLtChunk, seg_end - seg0 - t0), stage = c % C::kStages;
            const uint32_t turn = (c / C::kStages) & 1;
            unsigned char *st = smem + stage * C::kStage, *vt = smem + C::oV + (c % C::kStagesV) * C::NX * C::kTileV;
            if (TMA) {
                if (!lt_wait(m, &m.full_v[c % C::kStagesV], (c / C::kStagesV) & 1)) break;
                // W's place is free when the product before that has it is done.  That product has read its K too, so the wait for K below
                // is for this chunk's: V alone is two chunks ahead of Q and K, and a barrier that is still in the phase of the chunk
                // before in this stage lets a wait for the other parity through.
                if (c >= C::kStages && !lt_wait(m, &m.w_free[stage], turn ^ 1u)) break;
                // rows behind the sequence are somebody's: K (here) and V (below) must be zero there; Q's make rows that nobody reads
                if (n < kLtChunk && !lt_wait(m, &m.full[stage], turn)) break;
                for (int i = id; i < (kLtChunk - n) * (DK / 8); i += threads)
                    *reinterpret_cast<uint4*>(st + C::oK + lt_swizzled(i % (DK / 8), n + i / (DK / 8))) = make_uint4(0, 0, 0, 0);
            } else {
                if (c >= C::kStages && !lt_wait(m, &m.empty[stage], turn ^ 1u)) break;
                // the next chunk's rows, into L2
                for (int i = id; i < 3 * kLtChunk; i += threads) {
                    const int t = t0 + kLtChunk + (i & (kLtChunk - 1));
                    if (t >= seg_end - seg0) continue;
                    const char* row = reinterpret_cast<const char*>(i < kLtChunk ? k + t * a.k_stride[1] : i < 2 * kLtChunk ? v + t * a.v_stride[1] : q + t * a.q_stride[1]);
                    const int bytes = (i < kLtChunk || i >= 2 * kLtChunk ? a.dk : a.dv) * static_cast<int>(sizeof(T));
                    for (int at = 0; at < bytes; at += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + at));
                }
                static_assert(TMA || kLtChunk * DK / 8 / threads % 2 == 0, "pieces");
#pragma unroll 1
                for (int i0 = 0; i0 < kLtChunk * DK / 8 / threads; i0 += 2) {
                    float x[2][8], y[2][8];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int i = id + (i0 + j) * threads, g = i % (DK / 8), t = i / (DK / 8);
                        const int valid = t < n ? max(0, min(8, a.dk - g * 8)) : 0;
                        lt_load8(k + (t0 + t) * a.k_stride[1] + g * 8, valid, LOADS == kLtWide ? 16 : plan.boundary, y[j]);
                        if (outputs) lt_load8(q + (t0 + t) * a.q_stride[1] + g * 8, valid, LOADS == kLtWide ? 16 : plan.boundary, x[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int i = id + (i0 + j) * threads, at = lt_swizzled(i % (DK / 8), i / (DK / 8));
                        if (outputs) lt_store_parts<C::NX>(st + at, C::kTileK, x[j]);
                        lt_store_parts<C::NX>(st + C::oK + at, C::kTileK, y[j]);
                    }
                }
            }
            // V, and W
            if (!TMA && c >= C::kStages && !lt_wait(m, &m.w_free[stage], turn ^ 1u)) break;
            unsigned char* wt = smem + C::oW + stage * C::NW * C::kTileV;
            // a warp's piece: 16 bytes of eight tokens beside one another, four groups of channels.  A thread keeps to its tokens.
            constexpr int kGroups = DV / 32;
            if constexpr (TMA) {
                // (a short loop: the roles' code has to stay in the instruction cache together)
                static_assert(kWarpsW == 8, "a warp has eight tokens");
                const int t = rank * 8 + (lane & 7);
                if (c == 0 || n < kLtChunk) {
                    const int back = t < n ? n - 1 - t : 0;
                    w[0] = m.weight[back].x, w[1] = m.weight[back].y, w[2] = m.weight2[back];
                }
                unsigned char *from = vt + lt_swizzled(lane >> 3, t), *to = wt + lt_plain(lane >> 3, t);
                const auto at_of = [&](int g) { return from + (((t & 4) != 0 ? -64 : 64) * (g & 1)) + (g >> 1) * 8192; };  // (four groups on is one bit of the swizzle)
                uint4 next = *reinterpret_cast<const uint4*>(at_of(0));
                uint32_t high = 0;
#pragma unroll 1
                for (int g = 0; g < kGroups; ++g) {
                    if (t >= n) *reinterpret_cast<uint4*>(at_of(g)) = next = make_uint4(0, 0, 0, 0);
                    const uint32_t w4[4] = {next.x, next.y, next.z, next.w};
                    if (g + 1 < kGroups) next = *reinterpret_cast<const uint4*>(at_of(g + 1));
                    lt_weigh(to + g * 4096, C::kTileV, w4, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) high = __vmaxu2(high, w4[e] & 0x7FFF7FFFu);
                }
                if ((high & 0xFFFFu) >= 0x7F80u || high >= 0x7F800000u) {
                    atomicMin(&m.bad, t0 + t);
#pragma unroll 1
                    for (int d = 0; d < DV / 4; ++d) {  // (this thread's channels, one by one)
                        const int g = (d >> 3) * 4 + (lane >> 3);
                        uint16_t* at = reinterpret_cast<uint16_t*>(vt + lt_swizzled(g, t)) + (d & 7);
                        if ((*at & 0x7F80u) != 0x7F80u) continue;
                        *at = 0;
                        atomicMin(&m.first_bad[g * 8 + (d & 7)], t0 + t);
                    }
                }
            } else {
                const int t = rank * 8 + (lane & 7);
                const float weight = m.power[t < n ? n - 1 - t : 0];
#pragma unroll 1
                for (int g0 = 0; g0 < kGroups; g0 += 2) {  // two pieces on their way together
                    float x[2][8], y[8];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int g = (g0 + j) * 4 + (lane >> 3);
                        lt_load8(v + (t0 + t) * a.v_stride[1] + g * 8, t < n ? max(0, min(8, a.dv - g * 8)) : 0, LOADS == kLtWide ? 16 : plan.boundary, x[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int g = (g0 + j) * 4 + (lane >> 3);
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = x[j][e] * weight;
                        lt_store_parts<C::NW>(wt + lt_plain(g, t), C::kTileV, y);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            if (lt_finite(x[j][e])) continue;
                            atomicMin(&m.bad, t0 + t);
                            atomicMin(&m.first_bad[g * 8 + e], t0 + t);
                            x[j][e] = 0.0f;
                        }
                        lt_store_parts<C::NX>(vt + lt_swizzled(g, t), C::kTileV, x[j]);
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                if (!TMA) mbar_arrive(&m.full[stage]);
                mbar_arrive(&m.w_full[stage]);
                mbar_arrive(&m.v_whole[c % C::kStagesV]);  // (one per stage of V: this warp may be two chunks ahead of the product that waits)
            }
        }
    } else if (warp < C::kFirstP) {
        // ---- the outputs: row = channel of V, a share of the tokens
        constexpr int kShare = kLtChunk / (C::kWarpsO / 4);
        const int row = (warp & 3) * 32 + lane, token0 = ((warp - C::kFirstO) >> 2) * kShare;
        if (outputs) {
            out += seg0 * a.out_stride[1] + row;
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
                if (!lt_wait(m, &m.y_full, c & 1)) break;
                tc_fence_after();
                const int first = *reinterpret_cast<volatile int*>(&m.bad) < (c + 1) * kLtChunk ? m.first_bad[row] - c * kLtChunk : kLtChunk;
                const int t0 = c * kLtChunk + token0, n = row < a.dv ? min(kShare, seg_end - seg0 - t0) : 0;
                T* at = out + t0 * a.out_stride[1];
                const bool whole = n == kShare;
#pragma unroll 1
                for (int u = 0; u < kShare; u += 8) {
                    uint32_t x[8], y[8];
                    lt_ld(lane_base + kLtX + token0 + u, x);
                    lt_ld(lane_base + kLtY + token0 + u, y);
                    float power[8];
                    *reinterpret_cast<float4*>(power) = *reinterpret_cast<const float4*>(m.scaled_next + token0 + u);
                    *reinterpret_cast<float4*>(power + 4) = *reinterpret_cast<const float4*>(m.scaled_next + token0 + u + 4);
                    lt_ld_wait(x);
                    lt_ld_wait(y);
                    if (u + 8 == kShare) lt_arrive_read(&m.xy_free, lane);
                    T o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = lin_from<T>(fmaf(power[i], __uint_as_float(x[i]), __uint_as_float(y[i])));
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) at[i * a.out_stride[1]] = o[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (u + i < n) at[i * a.out_stride[1]] = o[i];
                    }
                    at += 8 * a.out_stride[1];
                }
                if (first < token0 + kShare) {
#pragma unroll 1
                    for (int u = max(0, first - token0); u < min(kShare, n); ++u) out[(t0 + u) * a.out_stride[1]] = lin_from<T>(__int_as_float(0x7fffffff));
                }
            }
        }
    } else if ((warp & 3) < 2) {
        // ---- P: row = token i; half of the tokens j
        const int row = (warp & 3) * 32 + lane, half = (warp - C::kFirstP) >> 2;
        if (outputs) {
            unsigned char* at = smem + C::oP + half * 4 * 1024 + (row >> 3) * 128 + (row & 7) * 16;
            const int d0 = row - half * 32;
            const bool nothing = half > (warp & 3), whole = half < (warp & 3);  // tokens behind all of the rows, in front of all
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
                if (!lt_wait(m, &m.g_full, c & 1)) break;
                tc_fence_after();
                uint32_t g[2][16];
                if (!nothing) {
                    lt_ld(lane_base + kLtG + half * 32, g[0]);
                    lt_ld(lane_base + kLtG + half * 32 + 16, g[1]);
                    lt_ld_wait(g[0]);
                    lt_ld_wait(g[1]);
                }
                lt_arrive_read(&m.g_read, lane);
                if (c > 0 && !lt_wait(m, &m.y_full, (c - 1) & 1)) break;  // (the product before has read P)
                if (nothing) {
#pragma unroll 1
                    for (int f = 0; f < 4 * C::NS; ++f) *reinterpret_cast<uint4*>(at + (f & 3) * 1024 + (f >> 2) * C::kPartP) = make_uint4(0, 0, 0, 0);
                } else {
                    const float* power = m.scaled + d0;
#pragma unroll 1
                    for (int f = 0; f < 32; f += 16) {
#pragma unroll
                        for (int r = 0; r < 16; r += 8) {
                            float x[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(g[0][r + e]) * power[-f - r - e];
                            if (!whole) {
#pragma unroll
                                for (int e = 0; e < 8; ++e) x[e] = d0 - f >= r + e ? x[e] : 0.0f;
                            }
                            lt_store_parts<C::NS>(at + (f + r) / 8 * 1024, C::kPartP, x);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) g[0][e] = g[1][e];
                    }
                }
                lt_arrive_operands(&m.p_full, lane);
            }
        }
    } else if (warp == C::kFirstP + 2 || warp == C::kFirstP + 6) {
        // ---- the products
        {
            // instruction descriptors: fp32 accumulators, bf16 operands, M = 128; N, and which operands are MN-major
            constexpr uint32_t kD = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24), kMnA = 1u << 15, kMnB = 1u << 16;
            constexpr uint32_t kIdescG = kD | ((kLtChunk / 8) << 17), kIdescX = kIdescG, kIdescY = kIdescG | kMnA,
                               kIdescU = kD | kMnA | kMnB | ((DK / 8) << 17);
            const uint32_t base = smem_u32(smem);
            const uint64_t dp = make_smem_desc(base + C::oP, 1024, 128);
            const auto wait = [&](uint64_t* bar, uint32_t parity) { return lt_wait(m, bar, parity); };
            // The products of parts p of one operand and r of the other with p + r < parts, the small ones first; mma(p, r, i, add) is one step
            // of four along the sum.  (The loops stay loops: as straight code this warp waited for its instructions.)
            const auto parts = [&](int na, int nb, int count, int quads, auto&& mma) {
                bool add = false;
#pragma unroll 1
                for (int sum = count - 1; sum >= 0; --sum)
#pragma unroll 1
                    for (int p = max(0, sum - nb + 1); p <= min(sum, na - 1); ++p)
#pragma unroll 1
                        for (int quad = 0; quad < quads; ++quad)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                mma(p, sum - p, quad, i, add);
                                add = true;
                            }
            };
            const auto stage_at = [&](int c) { return base + (c % C::kStages) * C::kStage; };
            const auto stage_here = [&](int c) { return wait(&m.full[c % C::kStages], (c / C::kStages) & 1); };
            if (warp == C::kFirstP + 6) {
                const auto make_g = [&](int c) {  // G = Q K^T
                    tc_fence_after();
                    if (lt_elect()) {
                        const uint64_t dq = lt_desc_swizzled(stage_at(c), 16, 1024), dk = lt_desc_swizzled(stage_at(c) + C::oK, 16, 1024);
                        parts(C::NX, C::NX, C::NX, DK / 64, [&](int p, int r, int quad, int i, bool add) {
                            const int step = quad * 8192 + i * 32;
                            lt_mma(tmem + kLtG, dq + ((p * C::kTileK + step) >> 4), dk + ((r * C::kTileK + step) >> 4), kIdescG, add);
                        });
                        tc_commit(&m.g_full);
                    }
                    __syncwarp();
                };
                bool ok = true;
                if (outputs && chunks > 0) {
                    ok = stage_here(0);
                    if (ok) make_g(0);
                }
#pragma unroll 1
                for (int c = 0; c < chunks && ok; ++c) {
                    if (!wait(&m.w_full[c % C::kStages], (c / C::kStages) & 1)) break;
                    if (!(outputs ? wait(&m.g_read, c & 1) : stage_here(c) && (c == 0 || wait(&m.u_free, (c - 1) & 1)))) break;
                    tc_fence_after();
                    if (lt_elect()) {  // U^T = W^T K
                        const uint64_t dk = lt_desc_swizzled(stage_at(c) + C::oK, 8192, 1024),
                                       dw = make_smem_desc(base + C::oW + (c % C::kStages) * C::NW * C::kTileV, 128, 1024);
                        parts(C::NW, C::NX, C::NW, 1, [&](int p, int r, int, int i, bool add) {
                            lt_mma(tmem + kLtU, dw + ((p * C::kTileV + i * 256) >> 4), dk + ((r * C::kTileK + i * 2048) >> 4), kIdescU, add);
                        });
                        tc_commit(&m.u_full);
                        tc_commit(&m.w_free[c % C::kStages]);
                        tc_commit(&m.empty[c % C::kStages]);
                    }
                    __syncwarp();
                    if (outputs && c + 1 < chunks) {
                        ok = stage_here(c + 1) && wait(&m.u_free, c & 1);
                        if (ok) make_g(c + 1);
                    }
                }
            } else if (outputs) {
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    if (!stage_here(c) || !wait(&m.s_full, c & 1) || (c > 0 && !wait(&m.xy_free, (c - 1) & 1))) break;
                    tc_fence_after();
                    if (lt_elect()) {  // X^T = S^T Q^T
                        const uint64_t dq = lt_desc_swizzled(stage_at(c), 16, 1024);
                        parts(C::NS, C::NX, C::NS, DK / 64, [&](int p, int r, int quad, int i, bool add) {
                            lt_mma_tmem(tmem + kLtX, tmem + C::kParts + p * (DK / 2) + quad * 32 + i * 8,
                                        dq + ((r * C::kTileK + quad * 8192 + i * 32) >> 4), kIdescX, add);
                        });
                        tc_commit(&m.x_full);
                    }
                    __syncwarp();
                    if (!wait(&m.p_full, c & 1) || !wait(&m.v_whole[c % C::kStagesV], (c / C::kStagesV) & 1)) break;
                    tc_fence_after();
                    if (lt_elect()) {  // Y^T = V^T P^T
                        const uint64_t dv = lt_desc_swizzled(base + C::oV + (c % C::kStagesV) * C::NX * C::kTileV, 8192, 1024);
                        parts(C::NS, C::NX, C::NS, 1, [&](int p, int r, int, int i, bool add) {
                            lt_mma(tmem + kLtY, dv + ((r * C::kTileV + i * 2048) >> 4), dp + ((p * C::kPartP + i * 2048) >> 4), kIdescY, add);
                        });
                        tc_commit(&m.y_full);
                        tc_commit(&m.empty[c % C::kStages]);
                    }
                    __syncwarp();
                }
            }
            // none of its products is under way when the CTA ends, not even where somebody gave up (TMEM is freed, and barriers end with it)
            uint64_t* none_left = &m.none_left[warp == C::kFirstP + 6 ? 0 : 1];
            if (lt_elect()) tc_commit(none_left);
            __syncwarp();
            for (uint32_t i = 0; i < plan.wait_limit && !lt_try(none_left, 0); ++i) {}
        }
    } else if (TMA && warp == C::kFirstP + 3 && lane == 0) {
        // ---- the copies: Q and K of a chunk and V of the next
        int issued = 0, issued_v = 0;
        const auto copy_v = [&](int c) {
            uint64_t* bar = &m.full_v[c % C::kStagesV];
            mbar_arrive_expect_tx(bar, C::kTileV);
            for (int i = 0; i < DV / 64; ++i)
                lt_tma(smem + C::oV + (c % C::kStagesV) * C::kTileV + i * 8192, &map_v, i * 64, seg0 + c * kLtChunk, hk, b, bar);
            issued_v = c + 1;
        };
        if (chunks > 0) copy_v(0);
        for (int c = 0; c < chunks; ++c) {
            const int stage = c % C::kStages;
            if (c >= C::kStages && !lt_wait_one(m, &m.empty[stage], ((c / C::kStages) & 1) ^ 1u)) break;
            unsigned char* st = smem + stage * C::kStage;
            mbar_arrive_expect_tx(&m.full[stage], (outputs ? 2 : 1) * C::kTileK);
            for (int i = 0; i < DK / 64; ++i) {
                if (outputs) lt_tma(st + i * 8192, &map_q, i * 64, seg0 + c * kLtChunk, h, b, &m.full[stage]);
                lt_tma(st + C::oK + i * 8192, &map_k, i * 64, seg0 + c * kLtChunk, hk, b, &m.full[stage]);
            }
            issued = c + 1;
            if (c + 1 < chunks) copy_v(c + 1);
        }
        // no copy is in flight when the CTA ends, not even where somebody gave up
        for (int c = max(0, issued - C::kStages); c < issued; ++c) mbar_wait_bounded(&m.full[c % C::kStages], (c / C::kStages) & 1, kLtWaitLimit);
        for (int c = max(0, issued_v - C::kStagesV); c < issued_v; ++c)
            mbar_wait_bounded(&m.full_v[c % C::kStagesV], (c / C::kStagesV) & 1, kLtWaitLimit);
    }
    tc_fence_before();
    __syncthreads();
    if (m.dead && tid == 0 && a.status != nullptr) atomicOr(a.status, FB_STATUS_WAIT_TIMEOUT);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kLtTmemCols) : "memory");
}

// ---- host side ------------------------------------------------------------------------------------------------------

// The driver's encoder of tensor maps, found through the runtime (the library does not link the driver).
using LtEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static LtEncode lt_encoder() {
    static const LtEncode fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
            p = nullptr;
        cudaGetLastError();
        return reinterpret_cast<LtEncode>(p);
    }();
    return fn;
}

// Whether [seq, token, head, channel] can be copied in boxes, and the map for it.
static bool lt_encode(CUtensorMap* map, const void* base, const int64_t* stride, int channels, int tokens, int heads, int batch) {
    const LtEncode fn = lt_encoder();
    if (fn == nullptr) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(batch)};
    const int64_t by_dim[3] = {stride[1], stride[2], stride[0]};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; ++i) {
        const int64_t bytes = by_dim[i] * 2;
        strides[i] = dims[i + 1] == 1 ? 16 : static_cast<cuuint64_t>(bytes);
        if (dims[i + 1] > 1 && (bytes <= 0 || bytes >= (1ll << 40))) return false;
    }
    const cuuint32_t box[4] = {64, kLtChunk, 1, 1}, step[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The states in front of a sequence's parts, from what each part adds, and the state behind the last one.  One thread per cell of S.  The decay
// of a part is a sum of two floats: rounded to one, it would be off the same way for every part (2.3e-6 of a state that passed 64 of them).
__global__ void __launch_bounds__(256) linattn_carry_kernel(const LinArgs a, float* states, float2* decays, int segs, int seg_tokens) {
    // (plain pointers: both are written by the kernel before, and nothing may read them ahead of the wait for it)
    const int64_t cells = static_cast<int64_t>(a.dk) * a.dv, cell = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int h = blockIdx.y % a.heads, b = blockIdx.y / a.heads, lane = threadIdx.x & 31;
    int bits;
    const int slot = lin_slot(a, b, lane, bits);
    pdl_wait();
    if (slot < 0 || cell >= cells) return;
    const int length = lin_length(a, b);
    const int64_t own = (static_cast<int64_t>(slot) * a.heads + h) * cells + cell, first = (static_cast<int64_t>(b) * a.heads + h) * segs;
    float* part = states + first * cells + cell;
    float s = a.state_in != nullptr ? a.state_in[own] : 0.0f;
    for (int i = 0; i < segs; ++i) {
        const float added = part[i * cells];
        const float2 decay = decays[first + i];
        part[i * cells] = s;
        if (i * seg_tokens < length) s = fmaf(decay.x, s, fmaf(decay.y, s, added));  // (no tokens, no decay: not even one that is NaN)
    }
    a.state_out[own] = s;
}

// How many parts a sequence is cut into, by the time that it would take (in us; fitted to 66 sizes with 1 to 32 parts, and
// within a hundredth of the best of those at 65 of them: 256 tokens of 8 heads of 64 in fp32 take 23.3 whole and 21.7 in four parts).  Cutting costs a second reading of K and V, a start of both kernels for every wave of parts, and the states in between; it
// pays where whole sequences leave SMs without work.  128 x 128 heads in bf16: 8192 tokens of 16 heads 354 whole and 93 in nine parts, 1024
// tokens 47 and 33 in eight; but 8 x 1024 tokens of 8 heads 50 and 65 in two, 3 x 640 tokens of 16 heads 33 and 54 in three.
static void lt_cut(const LinArgs& a, int64_t rows, int& segs, int& seg_tokens) {
    const int chunks = (a.tokens + kLtChunk - 1) / kLtChunk;
    segs = 1;
    seg_tokens = 0;
    if (rows > 65535) return;
    const bool bf16 = a.dtype == FB_DTYPE_BF16;
    const double chunk = bf16 ? 2.6 : a.dk <= 64 && a.dv <= 64 ? 4.2 : 10.0, again = chunk * (bf16 ? 1.4 : 1.65);
    const double start = 12.0 + 6.0 * a.dk * a.dv / (kLinMaxDim * kLinMaxDim);
    const auto waves = [](int64_t ctas) { return ctas <= kNumSMs ? 1.0 : 1.1 * static_cast<double>((ctas + kNumSMs - 1) / kNumSMs); };
    double best = waves(rows) * (chunks * chunk + 5.0);
    for (int n = 2; n <= 64 && n <= chunks; ++n) {
        const int each = (chunks + n - 1) / n;
        const int parts = (chunks + each - 1) / each;
        const double cost = waves(rows * parts) * (each * again + start) + 6.0;
        if (cost < best) {
            best = cost;
            segs = parts;
            seg_tokens = each * kLtChunk;
        }
    }
}

// floats of the parts' states; their decays lie behind them
static int64_t lt_state_floats(const LinArgs& a, int segs) {
    return (static_cast<int64_t>(a.batch) * a.heads * segs * a.dk * a.dv + 3) / 4 * 4;
}
int64_t linattn_chunk_scratch_bytes(const LinArgs& a) {
    int segs, seg_tokens;
    lt_cut(a, static_cast<int64_t>(a.batch) * a.heads, segs, seg_tokens);
    return segs == 1 ? 0 : lt_state_floats(a, segs) * 4 + static_cast<int64_t>(a.batch) * a.heads * segs * 8;
}

template <auto kernel>
static int launch_chunk(dim3 grid, int threads, int bytes, cudaStream_t st, const LinArgs& a, LtPlan plan, const CUtensorMap* maps) {
    static std::atomic<uint64_t> ready{0};  // devices whose attribute is set (of this instantiation's kernel)
    int device = 0;
    FB_TRY(check_cuda(cudaGetDevice(&device), "linear_attention"));
    const uint64_t bit = 1ull << (device & 63);
    if (device >= 64 || (ready.load(std::memory_order_relaxed) & bit) == 0) {
        FB_TRY(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "linear_attention"));
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    if (plan.segs == 1) return launch_after(kernel, grid, dim3(threads), bytes, st, false, "linear_attention", a, plan, maps[0], maps[1], maps[2]);
    plan.mode = 1;
    FB_TRY(launch_after(kernel, grid, dim3(threads), bytes, st, false, "linear_attention", a, plan, maps[0], maps[1], maps[2]));
    const dim3 carry(static_cast<unsigned>((a.dk * a.dv + 255) / 256), static_cast<unsigned>(a.batch * a.heads));
    FB_TRY(launch_after(linattn_carry_kernel, carry, dim3(256), 0, st, true, "linear_attention", a, plan.states, plan.decays, plan.segs, plan.seg_tokens));
    plan.mode = 2;
    return launch_after(kernel, grid, dim3(threads), bytes, st, true, "linear_attention", a, plan, maps[0], maps[1], maps[2]);
}

template <typename T, int DK, int DV>
static int launch_chunk(const LinArgs& a, void* scratch, cudaStream_t st) {
    using C = LtCfg<T, DK, DV>;
    constexpr int bytes = C::oMisc + static_cast<int>(sizeof(LtMisc));
    static_assert(bytes <= 232448, "shared memory");
    LtPlan plan = {};
    plan.drop_state = t_lt_drop;
    plan.wait_limit = t_lt_drop ? kLtWaitLimitDropped : kLtWaitLimit;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.heads;
    lt_cut(a, rows, plan.segs, plan.seg_tokens);
    FB_REQUIRE(plan.segs == 1 || (scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0), "linear_attention: scratch must be given, 16-byte aligned");
    plan.states = static_cast<float*>(scratch);
    if (plan.segs > 1) plan.decays = reinterpret_cast<float2*>(plan.states + lt_state_floats(a, plan.segs));
    const int64_t ctas = static_cast<int64_t>(a.batch) * a.heads * plan.segs;
    FB_REQUIRE(ctas < (1ll << 31), "linear_attention: batch * heads is too large");
    const void* base[3] = {a.q, a.k, a.v};
    const int64_t* stride[3] = {a.q_stride, a.k_stride, a.v_stride};
    uint64_t lies = 16;
    for (int i = 0; i < 3; ++i) {
        const int64_t sizes[3] = {a.batch, a.tokens, i == 0 ? a.heads : a.kv_heads};
        lies |= reinterpret_cast<uintptr_t>(base[i]);
        for (int j = 0; j < 3; ++j) lies |= sizes[j] == 1 ? 0 : static_cast<uint64_t>(stride[i][j]) * sizeof(T);
    }
    plan.boundary = static_cast<int>(lies & (~lies + 1));
    CUtensorMap maps[3] = {};
    const bool tma = C::kBf16 && plan.boundary == 16 && lt_encode(&maps[0], a.q, a.q_stride, a.dk, a.tokens, a.heads, a.batch) &&
               lt_encode(&maps[1], a.k, a.k_stride, a.dk, a.tokens, a.kv_heads, a.batch) &&
               lt_encode(&maps[2], a.v, a.v_stride, a.dv, a.tokens, a.kv_heads, a.batch);
    const dim3 grid(static_cast<unsigned>(ctas));
    if constexpr (C::kBf16) {
        if (tma) return launch_chunk<linattn_chunk_kernel<T, DK, DV, kLtTma>>(grid, C::kThreads, bytes, st, a, plan, maps);
    } else {
        if (plan.boundary == 16) return launch_chunk<linattn_chunk_kernel<T, DK, DV, kLtWide>>(grid, C::kThreads, bytes, st, a, plan, maps);
    }
    return launch_chunk<linattn_chunk_kernel<T, DK, DV, kLtAny>>(grid, C::kThreads, bytes, st, a, plan, maps);
}

template <typename T>
static int launch_chunk(const LinArgs& a, void* scratch, cudaStream_t st) {
    if (a.dk <= 64) return a.dv <= 64 ? launch_chunk<T, 64, 64>(a, scratch, st) : launch_chunk<T, 64, 128>(a, scratch, st);
    return a.dv <= 64 ? launch_chunk<T, 128, 64>(a, scratch, st) : launch_chunk<T, 128, 128>(a, scratch, st);
}

int launch_linattn_chunk(const LinArgs& a, void* scratch, cudaStream_t st) {
    if (a.dtype == FB_DTYPE_F32) return launch_chunk<float>(a, scratch, st);
    if (a.dtype == FB_DTYPE_F16) return launch_chunk<__half>(a, scratch, st);
    return launch_chunk<__nv_bfloat16>(a, scratch, st);
}

}  // namespace fb
