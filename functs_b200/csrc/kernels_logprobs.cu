// Log probabilities of given tokens, entropies and the best alternatives: one pass over the logits.
//
//   With the row's maximum m,  s = sum 2^d  and  t = sum 2^d d  with  d = (x - m) log2 e  give  log sum exp(x) = m + ln s  and
//   entropy = ln s - ln2 t / s.
// Every thread takes the largest element that it has met as its reference, so that d is small where 2^d is large (an exponent of 40 is off by
// 2^-20: a row whose best lies that far above the others and above its thread's reference came out 2.7e-6 off, above 0).  That element itself
// stays out of the sums: in them it would round the small ones away, and against the row's maximum its own power is exact, 1 where it is
// the maximum.  So s >= 1 and t <= 0, no log probability is above 0 and no entropy below.  A thread looks for a larger element once in four
// vectors; the loop is a fused multiply-add, an exponential and two sums per element.
//
// Alternatives: each thread also keeps the maximum of its elements.  The top-th largest of some of those maxima (the largest of every warp)
// bounds the top-th largest element from below, so only the few threads whose maximum reaches it have candidates: their elements are read
// again (from L2), and what reaches the bound is ordered by rank counting.  Elements equal to the bound are listed too, or, where there are many (a masked row with few
// finite logits, a constant row), taken by one ordered scan that stops as soon as it has enough.  More candidates than the list holds
// (rows whose large values sit in few threads) select the bound again by radix, exactly.
//
// A row is one CTA, or a cluster of up to eight whose parts meet in the first one's shared memory; a short row is a warp.
//
// Bound by HBM beside exponentials and issue where rows are many (4096 rows of 32000 in bf16 and in fp16 52 us, 5.0 TB/s, in fp32 89, 5.9 TB/s)
// and by latency where they are few (one row of 32000 in fp32 4.5 us, with five alternatives 7.1: the choice is eight block barriers).
// Three blocks of 512 threads an SM are worth 40 registers a thread: with 50, two of them, 600 rows of 50001 in bf16 with 20 alternatives take
// 31 us (24.7), 2410 of 12838 in fp16 with five 41 (31.5).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace fb {

constexpr int kLpMaxThreads = 512;
constexpr int kLpMaxTop = FB_LOGPROBS_MAX_TOP;
constexpr int kLpMaxParts = 8;               // CTAs per row
constexpr int kLpTopParts = 4;               // the same with alternatives
constexpr int kLpList = 1024;                // candidates above the bound; as many equal to it
constexpr int kLpBusy = 128;                 // threads whose elements are looked through one by one
constexpr float kLpLog2e = 1.44269504088896340736f;
constexpr double kLpLog2eOff = 1.0 / static_cast<double>(kLpLog2e) - 0.69314718055994530942;  // what rounding log2 e takes from ln 2
constexpr float kLpFloor = -3.4e8f;          // stands for no element: the sums of what lies below it are taken by lp_again
constexpr float kLpFarValue = 268435456.0f;  // 2^28: where x log2e is rounded by 16 and more, see lp_again

struct LpArgs {
    const void* logits;
    int64_t row_stride;
    const int64_t* tokens;
    int32_t vocab, top;
    float *logprobs, *entropy, *top_logprobs;
    int64_t* top_ids;
    int32_t* status;
};

// Order of values as unsigned numbers: NaN above all, both zeros the same, never 0 (which stands for no element).
__device__ __forceinline__ uint32_t lp_order(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t order) {
    if (order == 0xFFFFFFFFu) return __uint_as_float(0x7FFFFFFFu);
    return __uint_as_float((order & 0x80000000u) ? (order & 0x7FFFFFFFu) : ~order);
}
__device__ __forceinline__ uint64_t lp_key(uint32_t order, uint32_t id) { return (static_cast<uint64_t>(order) << 32) | (0xFFFFFFFFu - id); }

__device__ __forceinline__ float lp_ex2(float x) {  // (of 0 exactly 1)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& u, float (&x)[4]) {
        x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    template <int K>
    static __device__ __forceinline__ float most(const uint4 (&u)[K]) {
        float m = __uint_as_float(u[0].x);
#pragma unroll
        for (int k = 0; k < K; ++k)
            m = max_nan(max_nan(m, max_nan(__uint_as_float(u[k].x), __uint_as_float(u[k].y))), max_nan(__uint_as_float(u[k].z), __uint_as_float(u[k].w)));
        return m;
    }
};
template <>
struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& u, float (&x)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    template <int K>
    static __device__ __forceinline__ float most(const uint4 (&u)[K]) {
        const auto two = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
        __nv_bfloat162 m = two(u[0].x);
#pragma unroll
        for (int k = 0; k < K; ++k) m = __hmax2_nan(__hmax2_nan(m, __hmax2_nan(two(u[k].x), two(u[k].y))), __hmax2_nan(two(u[k].z), two(u[k].w)));
        return max_nan(__low2float(m), __high2float(m));
    }
};
template <>
struct LpVec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& u, float (&x)[8]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
    template <int K>
    static __device__ __forceinline__ float most(const uint4 (&u)[K]) {
        const auto two = [](const uint32_t& w) { return *reinterpret_cast<const __half2*>(&w); };
        __half2 m = two(u[0].x);
#pragma unroll
        for (int k = 0; k < K; ++k) m = __hmax2_nan(__hmax2_nan(m, __hmax2_nan(two(u[k].x), two(u[k].y))), __hmax2_nan(two(u[k].z), two(u[k].w)));
        return max_nan(__low2float(m), __high2float(m));
    }
};

// sums of a warp, of a part of a row, of a row: against its own largest element
struct __align__(16) LpSums {
    float most;  // the largest element (NaN if there is one, -inf if there is none)
    float s, t;
    __device__ __forceinline__ void none() { most = __int_as_float(0xff800000), s = t = 0.0f; }
};

// Whether sums against a rounded x log2e do not do for this largest element (finite, and far from 0).
__device__ __forceinline__ bool lp_far(float most) { return fabsf(most) >= kLpFarValue && fabsf(most) <= 3.402823466e38f; }
// elements against the largest one, by a difference that is exact where it matters
template <int N>
__device__ __forceinline__ void lp_take_near(const float (&x)[N], float most, float& s, float& t) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = fmaxf((x[i] - most) * kLpLog2e, -1000.0f), e = lp_ex2(d);
        s += e;
        t = fmaf(e, d, t);
    }
}

// a row: log sum exp = base + log_s
struct LpRow {
    double base, log_s;
    bool empty;
    __device__ __forceinline__ float logprob(float x) const {
        return empty ? __int_as_float(0xff800000) : static_cast<float>((static_cast<double>(x) - base) - log_s);
    }
};

struct LpThread {
    float most;       // the largest element (NaN if there is one)
    float held, ref;  // the largest above the floor, which is not in the sums, and the reference that they are against: held log2e, rounded
    float s, t;

    __device__ __forceinline__ void start() { most = __int_as_float(0xff800000), held = kLpFloor, ref = kLpFloor * kLpLog2e, s = t = 0.0f; }
    // x is the one to hold, and what was held goes into the sums
    __device__ __forceinline__ void hold(float x) {
        const float own = fmaf(held, kLpLog2e, -ref), e = lp_ex2(own), to = x * kLpLog2e, d = ref - to, f = lp_ex2(d);
        s += e;
        t = fmaf(e, own, t);
        t = f > 0.0f ? f * fmaf(d, s, t) : 0.0f;  // (so far below that nothing of them is left: they need not be numbers)
        s = f > 0.0f ? f * s : 0.0f;
        held = x, ref = to;
    }
    // The elements of K vectors (get(k, x) gives one), of which `m` is the largest.
    template <int N, int K, class F>
    __device__ __forceinline__ void take(float m, F get) {
        most = max_nan(most, m);
        float own = 0.0f, own_t = 0.0f;
        if (m > held) {
            hold(m);
            const float d = fmaf(m, kLpLog2e, -ref);
            own = lp_ex2(d), own_t = own * d;
        }
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float x[N];
            get(k, x);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = fmaxf(fmaf(x[i], kLpLog2e, -ref), -1000.0f);  // (-inf: its power is 0, and 0 * d must be; a NaN is in `most`)
                x[i] = lp_ex2(d);
                t = fmaf(x[i], d, t);
            }
#pragma unroll
            for (int w = N / 2; w > 0; w /= 2) {  // (by halves: `own` is among them, and rounds the others three times instead of seven)
#pragma unroll
                for (int i = 0; i < w; ++i) x[i] += x[i + w];
            }
            sum += x[0];
        }
        s += sum - own;
        t -= own_t;
    }
    __device__ __forceinline__ void take_one(float x) {
        take<1, 1>(x, [&](int, float (&y)[1]) { y[0] = x; });
    }
    template <class V, int K>
    __device__ __forceinline__ void take_vectors(const uint4 (&u)[K]) {
        take<V::N, K>(V::most(u), [&](int k, float (&x)[V::N]) { V::get(u[k], x); });
    }
    // The warp's sums, in all lanes.  (Where its largest element is far from 0 they mean nothing: lp_again takes them.)
    __device__ __forceinline__ LpSums warp_sums() const {
        LpSums all;
        all.most = most;
        for (int d = 16; d > 0; d /= 2) all.most = max_nan(all.most, __shfl_xor_sync(kFullMask, all.most, d));
        all.s = all.t = 0.0f;
        if (held > kLpFloor) {
            const float d = fmaxf((held - all.most) * kLpLog2e, -1000.0f), below = fmaf(-all.most, kLpLog2e, ref), f = lp_ex2(below), rest = fmaxf(s, 0.0f);
            all.s = lp_ex2(d), all.t = all.s * d;
            if (f > 0.0f) all.s = fmaf(f, rest, all.s), all.t += fminf(f * fmaf(below, rest, t), 0.0f);
        }
        for (int d = 16; d > 0; d /= 2) {
            all.s += __shfl_xor_sync(kFullMask, all.s, d);
            all.t += __shfl_xor_sync(kFullMask, all.t, d);
        }
        return all;
    }
};

template <bool TOP>
struct LpShared {
    LpSums sums[kLpMaxThreads / 32];
    LpSums part[kLpMaxParts];                 // of the row's CTAs (in the first one)
    uint64_t most[TOP ? 2 * kLpMaxTop : 1];   // the largest of the threads' maxima, warp by warp
    uint64_t above[TOP ? kLpList : 1], equal[TOP ? kLpList : 1];  // candidates
    uint64_t best[kLpMaxTop];                 // this CTA's, in order
    uint64_t parts_best[TOP ? kLpTopParts * kLpMaxTop : 1];  // of the row's CTAs (in the first one)
    uint64_t row_best[kLpMaxTop];             // the row's
    LpRow whole;
    int64_t token;                            // the token to score and its logit, fetched at the start (registers that the loop needs)
    float token_logit;
    uint32_t hist[256];
    uint32_t warp_count[kLpMaxThreads / 32];
    int busy[kLpBusy];                        // threads that have candidates
    int num_threads, num_above, num_equal;
    uint32_t bound, digit, wanted;
};

__device__ __forceinline__ uint32_t lp_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t lp_first(const void* p) {  // the same place in the row's first CTA
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
__device__ __forceinline__ void lp_put(uint32_t at, float x, float y, float z) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(x), "f"(y), "f"(z), "f"(0.0f) : "memory");
}
__device__ __forceinline__ void lp_put(uint32_t at, uint64_t v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }

// Writes a row's two numbers.
__device__ __forceinline__ LpRow lp_finish(const LpArgs& a, int64_t r, const LpSums& sums, int64_t token, float token_logit) {
    LpRow row;
    row.empty = sums.most == __int_as_float(0xff800000);
    row.base = static_cast<double>(sums.most);
    // (log2 e in 32 bits is 1.3e-8 too small, so every power a little too large: to first order t says how much in all.  The largest element's
    // own, which is 1, is not: where the others are lost beside it, what t has of them is not to be taken off.)
    double s = fmax(fma(kLpLog2eOff, static_cast<double>(sums.t), static_cast<double>(sums.s)), 1.0);
    if (!(sums.most <= 3.402823466e38f)) s = static_cast<double>(__int_as_float(0x7fffffff));  // a NaN or an infinity
    row.log_s = log(s);
    float lp = row.logprob(token_logit);
    if (token < 0) lp = 0.0f;
    if (token >= a.vocab) {
        lp = __int_as_float(0x7fffffff);
        if (a.status != nullptr) atomicOr(a.status, FB_STATUS_INDEX_RANGE);
    }
    a.logprobs[r] = lp;
    a.entropy[r] = row.empty ? 0.0f : static_cast<float>(row.log_s - static_cast<double>(sums.t) / (s * static_cast<double>(kLpLog2e)));
    return row;
}

// The elements of a part of a row: vectors, and single ones in front of (first part) and behind (last part) the row's 16-byte boundaries.
template <typename T>
struct LpPart {
    const T* row;
    int head, vec_id, num_vec, tail, tail_id;  // ids: of the first vector's first element, of the tail's first
    __device__ __forceinline__ int id_of(int v) const { return vec_id + v * LpVec<T>::N; }
    __device__ __forceinline__ uint4 vec(int v) const { return *reinterpret_cast<const uint4*>(row + id_of(v)); }
    __device__ __forceinline__ int count() const { return head + num_vec * LpVec<T>::N + tail; }
    __device__ __forceinline__ int id_at(int e) const {  // of the part's e-th element
        if (e < head) return e;
        e -= head;
        return e < num_vec * LpVec<T>::N ? vec_id + e : tail_id + (e - num_vec * LpVec<T>::N);
    }
    __device__ __forceinline__ uint32_t order(int id) const { return lp_order(LpVec<T>::one(row + id)); }
};

// number of entries of a list in descending order that are above `key`
__device__ __forceinline__ int lp_above(const uint64_t* list, int n, uint64_t key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}
// the sums of `count` lanes (a power of two) together, in all of them
__device__ __forceinline__ void lp_join_lanes(LpSums& sums, int count) {
    const float own = sums.most;
    for (int d = count / 2; d > 0; d /= 2) sums.most = max_nan(sums.most, __shfl_xor_sync(kFullMask, sums.most, d));
    const float below = own == __int_as_float(0xff800000) ? -1000.0f : fmaxf((own - sums.most) * kLpLog2e, -1000.0f), f = lp_ex2(below);
    sums.t = f * fmaf(below, sums.s, sums.t);
    sums.s = f * sums.s;
    for (int d = count / 2; d > 0; d /= 2) {
        sums.s += __shfl_xor_sync(kFullMask, sums.s, d);
        sums.t += __shfl_xor_sync(kFullMask, sums.t, d);
    }
}

// calls f(order, id) for the elements that this thread has
template <typename T, class F>
__device__ __forceinline__ void lp_each(const LpPart<T>& p, F f) {
    constexpr int N = LpVec<T>::N;
    const int who = threadIdx.x, threads = blockDim.x;
    for (int v = who; v < p.num_vec; v += threads) {
        float x[N];
        LpVec<T>::get(p.vec(v), x);
#pragma unroll
        for (int i = 0; i < N; ++i) f(lp_order(x[i]), p.id_of(v) + i);
    }
    if (who < p.head) f(p.order(who), who);
    if (who < p.tail) f(p.order(p.tail_id + who), p.tail_id + who);
}

// A part whose largest element is 2^28 or more from 0, once more: there x log2e is rounded by so much that powers of the remainder overflow
// (and -inf, where a mask is the type's lowest value).  Nothing else comes here: masked elements below a row of usual ones count as nothing.
// (A call: inlined, the loop over usual rows came out slower, 4096 rows of 32000 in bf16 65 us and 57 when that was tried.)
template <typename T, bool TOP>
__device__ __noinline__ void lp_again(LpShared<TOP>& sh, const LpPart<T>& p) {
    constexpr int N = LpVec<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    float most = sh.sums[0].most;
    for (int w = 1; w < warps; ++w) most = max_nan(most, sh.sums[w].most);
    if (!lp_far(most)) return;
    __syncthreads();
    float s = 0.0f, t = 0.0f;
    for (int v = tid; v < p.num_vec; v += threads) {
        float x[N];
        LpVec<T>::get(p.vec(v), x);
        lp_take_near(x, most, s, t);
    }
    if (tid < p.head) lp_take_near({LpVec<T>::one(p.row + tid)}, most, s, t);
    if (tid < p.tail) lp_take_near({LpVec<T>::one(p.row + p.tail_id + tid)}, most, s, t);
    for (int d = 16; d > 0; d /= 2) {
        s += __shfl_xor_sync(kFullMask, s, d);
        t += __shfl_xor_sync(kFullMask, t, d);
    }
    if (lane == 0) sh.sums[warp] = {most, s, t};
    __syncthreads();
}

// The `top` best of the part (keys 0 behind them if it has fewer), best first, in sh.best.  most: of this thread's elements.
template <typename T>
__device__ void lp_select(LpShared<true>& sh, const LpPart<T>& p, int top, float most) {
    constexpr int N = LpVec<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    const uint32_t mine = tid < p.num_vec || tid < p.head || tid < p.tail ? lp_order(most) : 0u;
    if (tid < top) sh.best[tid] = 0;
    if (tid == 0) sh.num_threads = sh.num_above = sh.num_equal = 0, sh.bound = 0;
    // a bound: the top-th largest of the warps' (top / warps) largest lanes, by counting
    const int having = (min(threads, max(p.num_vec, max(p.head, p.tail))) + 31) / 32;  // warps that have elements
    const int share = having > 0 ? min(32, (top + having - 1) / having) : 0, listed = share * having;
    uint32_t left = mine;
    for (int i = 0; i < share && warp < having; ++i) {
        const uint32_t largest = __reduce_max_sync(kFullMask, left);
        if (lane == __ffs(__ballot_sync(kFullMask, left == largest)) - 1) {
            sh.most[warp * share + i] = lp_key(largest, tid);
            left = 0;
        }
    }
    __syncthreads();
    if (tid < listed) {
        const uint64_t key = sh.most[tid];
        int rank = 0;
        for (int j = 0; j < listed; ++j) rank += sh.most[j] > key;
        if (rank == top - 1) sh.bound = static_cast<uint32_t>(key >> 32);  // (0 where fewer threads than that have elements: all count)
    }
    __syncthreads();
    uint32_t bound = sh.bound;
    if (mine != 0 && mine >= bound) {
        const int at = atomicAdd(&sh.num_threads, 1);
        if (at < kLpBusy) sh.busy[at] = tid;
    }
    __syncthreads();
    const auto list = [&](uint32_t order, int id) {
        if (order < bound) return;
        if (order > bound) {
            const int at = atomicAdd(&sh.num_above, 1);
            if (at < kLpList) sh.above[at] = lp_key(order, id);
        } else {
            const int at = atomicAdd(&sh.num_equal, 1);
            if (at < kLpList) sh.equal[at] = lp_key(order, id);
        }
    };
    const int busy = sh.num_threads;
    if (busy <= kLpBusy) {
        // (every piece of theirs on its way at once: one wait for L2)
        const int each = (p.num_vec + threads - 1) / threads + 1;
        for (int i = tid; i < busy * each; i += threads) {
            const int who = sh.busy[i / each], k = i % each, v = who + k * threads;
            if (k + 1 < each) {
                if (v >= p.num_vec) continue;
                float x[N];
                LpVec<T>::get(p.vec(v), x);
#pragma unroll
                for (int e = 0; e < N; ++e) list(lp_order(x[e]), p.id_of(v) + e);
            } else {
                if (who < p.head) list(p.order(who), who);
                if (who < p.tail) list(p.order(p.tail_id + who), p.tail_id + who);
            }
        }
    } else {
        lp_each(p, list);
    }
    __syncthreads();
    if (sh.num_above > kLpList) {
        // too many: the top-th largest element itself, eight bits at a time
        uint32_t prefix = 0, mask = 0, wanted = top;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += threads) sh.hist[i] = 0;
            __syncthreads();
            lp_each(p, [&](uint32_t order, int) {
                if ((order & mask) == prefix) atomicAdd(&sh.hist[(order >> shift) & 255u], 1u);
            });
            __syncthreads();
            if (tid == 0) {
                uint32_t seen = 0;
                int digit = 255;
                for (; digit > 0 && seen + sh.hist[digit] < wanted; --digit) seen += sh.hist[digit];
                sh.digit = digit;
                sh.wanted = wanted - seen;
            }
            __syncthreads();
            prefix |= sh.digit << shift;
            mask |= 255u << shift;
            wanted = sh.wanted;
        }
        __syncthreads();
        bound = prefix;
        if (tid == 0) sh.num_above = sh.num_equal = 0;
        __syncthreads();
        lp_each(p, list);
        __syncthreads();
    }
    const int above = sh.num_above, equal = sh.num_equal;
    for (int i = tid; i < above; i += threads) {
        const uint64_t key = sh.above[i];
        int rank = 0;
        for (int j = 0; j < above; ++j) rank += sh.above[j] > key;
        if (rank < top) sh.best[rank] = key;
    }
    int need = max(0, min(top - above, equal)), place = above;
    if (equal <= kLpList) {
        if (need > 0) {
            for (int i = tid; i < equal; i += threads) {
                const uint64_t key = sh.equal[i];
                int rank = 0;
                for (int j = 0; j < equal; ++j) rank += sh.equal[j] > key;
                if (rank < need) sh.best[place + rank] = key;
            }
        }
    } else {
        // many are equal to the bound: the first of them, by a scan in order
        const int total = p.count();
        for (int base = 0; base < total && need > 0; base += threads * N) {
            uint32_t hit = 0;
            for (int i = 0; i < N; ++i) {
                const int e = base + tid * N + i;
                if (e < total && p.order(p.id_at(e)) == bound) hit |= 1u << i;
            }
            int before = __popc(hit);
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int o = __shfl_up_sync(kFullMask, before, d);
                if (lane >= d) before += o;
            }
            if (lane == 31) sh.warp_count[warp] = before;
            __syncthreads();
            before -= __popc(hit);
            int all = 0;
            for (int w = 0; w < warps; ++w) {
                if (w < warp) before += sh.warp_count[w];
                all += sh.warp_count[w];
            }
            for (int i = 0; i < N; ++i) {
                if (!((hit >> i) & 1u)) continue;
                if (before < need) sh.best[place + before] = lp_key(bound, p.id_at(base + tid * N + i));
                ++before;
            }
            __syncthreads();
            place += min(all, need);
            need -= min(all, need);
        }
    }
    __syncthreads();
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpMaxThreads, 3) logprobs_kernel(const LpArgs a, int parts) {
    constexpr int N = LpVec<T>::N;
    __shared__ LpShared<TOP> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    const int rank = parts > 1 ? static_cast<int>(lp_cluster_rank()) : 0;
    const int64_t r = blockIdx.x / parts;
    LpPart<T> p;
    p.row = static_cast<const T*>(a.logits) + r * a.row_stride;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p.row) & 15u) / sizeof(T));
    const int head = min(a.vocab, off == 0 ? 0 : N - off), vecs = (a.vocab - head) / N, share = (vecs + parts - 1) / parts;
    const int first = min(vecs, rank * share);
    p.head = rank == 0 ? head : 0;
    p.vec_id = head + first * N;
    p.num_vec = min(share, vecs - first);
    p.tail_id = head + vecs * N;
    p.tail = rank == parts - 1 ? a.vocab - p.tail_id : 0;
    if (rank == 0 && tid == 0) {
        const int64_t token = a.tokens[r];
        sh.token = token;
        sh.token_logit = token >= 0 && token < a.vocab ? LpVec<T>::one(p.row + token) : 0.0f;
    }

    if (parts > 1) lp_cluster_arrive();  // (waited for before the first CTA is written to)
    LpThread th;
    th.start();
    if (tid < p.head) th.take_one(LpVec<T>::one(p.row + tid));
    if (tid < p.tail) th.take_one(LpVec<T>::one(p.row + p.tail_id + tid));
    int v = tid;
    for (; v + 3 * threads < p.num_vec; v += 4 * threads) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = p.vec(v + i * threads);
        th.take_vectors<LpVec<T>>(u);
    }
    for (; v < p.num_vec; v += threads) {
        const uint4 u[1] = {p.vec(v)};
        th.take_vectors<LpVec<T>>(u);
    }
    const float most = th.most;
    // the block's sums
    LpSums sums = th.warp_sums();
    if (lane == 0) sh.sums[warp] = sums;
    if (__syncthreads_or(lane == 0 && lp_far(sums.most))) lp_again<T, TOP>(sh, p);
    if (warp == 0) {
        sums.none();
        if (lane < warps) sums = sh.sums[lane];
        lp_join_lanes(sums, 16);
    }
    if constexpr (TOP) lp_select<T>(sh, p, a.top, most);
    if (parts > 1) {
        // what the parts have meets in the first one's shared memory
        lp_cluster_wait();  // (it runs)
        if (tid == 0) lp_put(lp_first(&sh.part[rank]), sums.most, sums.s, sums.t);
        if (TOP && tid < a.top) lp_put(lp_first(&sh.parts_best[rank * a.top + tid]), sh.best[tid]);
        lp_cluster_arrive();
        lp_cluster_wait();
        if (rank != 0) return;
        if (warp == 0) {
            sums = sh.part[lane & (parts - 1)];
            lp_join_lanes(sums, parts);
        }
    }
    if (tid == 0) sh.whole = lp_finish(a, r, sums, sh.token, sh.token_logit);
    if (TOP) {
        const uint64_t* best = sh.best;
        if (parts > 1) {
            // every part's list is in order: a candidate's place is the number of larger ones, found by halving
            for (int i = tid; i < parts * a.top; i += threads) {
                const int c = i / a.top;
                const uint64_t key = sh.parts_best[i];
                int place = 0;
                for (int o = 0; o < parts; ++o) place += o == c ? i - c * a.top : lp_above(sh.parts_best + o * a.top, a.top, key);
                if (key != 0 && place < a.top) sh.row_best[place] = key;
            }
            best = sh.row_best;
        }
        __syncthreads();
        for (int i = tid; i < a.top; i += threads) {
            const uint64_t key = best[i];
            a.top_logprobs[r * a.top + i] = sh.whole.logprob(lp_value(static_cast<uint32_t>(key >> 32)));
            a.top_ids[r * a.top + i] = static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
        }
    }
}

// Rows of up to 1024 logits: a warp each, its elements in registers, the best taken one by one.
constexpr int kLpShort = 1024, kLpShortRows = 4;
template <typename T, int COUNT>
__global__ void __launch_bounds__(32 * kLpShortRows) logprobs_short_kernel(const LpArgs a, int rows) {
    const int lane = threadIdx.x & 31;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kLpShortRows + (threadIdx.x >> 5);
    if (r >= rows) return;
    const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
    const int64_t token = a.tokens[r];
    const float token_logit = token >= 0 && token < a.vocab ? LpVec<T>::one(row + token) : 0.0f;
    float x[COUNT];  // element i * 32 + lane; -inf where there is none
#pragma unroll
    for (int i = 0; i < COUNT; ++i) x[i] = i * 32 + lane < a.vocab ? LpVec<T>::one(row + i * 32 + lane) : __int_as_float(0xff800000);
    LpThread th;
    th.start();
    float m = x[0];
#pragma unroll
    for (int i = 1; i < COUNT; ++i) m = max_nan(m, x[i]);
    th.take<8, COUNT / 8>(m, [&](int k, float (&y)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[k * 8 + i];
    });
    LpSums sums = th.warp_sums();
    if (lp_far(sums.most)) {  // (see lp_again)
        float s = 0.0f, t = 0.0f;
        lp_take_near(x, sums.most, s, t);
        for (int d = 16; d > 0; d /= 2) {
            s += __shfl_xor_sync(kFullMask, s, d);
            t += __shfl_xor_sync(kFullMask, t, d);
        }
        sums.s = s, sums.t = t;
    }
    LpRow whole = {};
    if (lane == 0) whole = lp_finish(a, r, sums, token, token_logit);
    uint32_t order[COUNT], most = 0;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        order[i] = i * 32 + lane < a.vocab ? lp_order(x[i]) : 0u;
        most = max(most, order[i]);
    }
    for (int k = 0; k < a.top; ++k) {
        const uint32_t best = __reduce_max_sync(kFullMask, most);
        uint32_t id = 0xFFFFFFFFu;
        if (most == best) {
#pragma unroll
            for (int i = COUNT - 1; i >= 0; --i)
                if (order[i] == best) id = i * 32 + lane;
        }
        id = __reduce_min_sync(kFullMask, id);
        if (lane == static_cast<int>(id & 31u)) {  // taken
            most = 0;
#pragma unroll
            for (int i = 0; i < COUNT; ++i) {
                if (i == static_cast<int>(id >> 5)) order[i] = 0;
                most = max(most, order[i]);
            }
        }
        if (lane == 0) {
            a.top_logprobs[r * a.top + k] = whole.logprob(lp_value(best));
            a.top_ids[r * a.top + k] = id;
        }
    }
}

template <typename T>
static int launch_logprobs_short(const LpArgs& a, int rows, cudaStream_t st) {
    const dim3 grid((rows + kLpShortRows - 1) / kLpShortRows), block(32 * kLpShortRows);
    if (a.vocab <= 256) return launch_after(logprobs_short_kernel<T, 8>, grid, block, 0, st, false, "token_logprobs", a, rows);
    return launch_after(logprobs_short_kernel<T, kLpShort / 32>, grid, block, 0, st, false, "token_logprobs", a, rows);
}

template <typename T, bool TOP>
static int launch_logprobs(const LpArgs& a, int rows, cudaStream_t st) {
    const int vecs = a.vocab / LpVec<T>::N;
    // One CTA per row, unless rows are few and long.  Without alternatives a part of 512 vectors at least (one row of 32000 fp32 logits 4.4 us in
    // eight parts or four, 4.9 in one).  With alternatives the parts' lists have to meet: four parts from 8192 vectors on (8 rows of 65536 in
    // bf16 from HBM 10.9 us in one, 9.8 in four; of 131072 16.2 and 10.8), fewer vectors in one (one row of 32000 in fp32 7.4, in four 8.2).
    // With several rows per SM 256 threads a row (4096 rows of 32000 in bf16: 52.5 us, with 512 threads 62.4), else 512 (256 rows of 131072
    // with 20 alternatives 23.1, with 256 threads 32.1).
    const int most = !TOP ? kLpMaxParts : vecs >= 8192 ? kLpTopParts : 1;
    int parts = 1;
    while (parts < most && static_cast<int64_t>(rows) * parts * 2 <= kNumSMs && vecs / (parts * 2) >= 512) parts *= 2;
    const int each = vecs / parts;
    const int threads = each >= 1024 ? (rows >= 4 * kNumSMs ? 256 : 512) : each >= 512 ? 256 : 128;  // (a row has 128 vectors at least, a part 512)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * parts);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    FB_TRY(check_cuda(cudaLaunchKernelEx(&cfg, logprobs_kernel<T, TOP>, a, parts), "token_logprobs"));
    count_launch();
    return FB_OK;
}

template <typename T>
static int launch_logprobs(const LpArgs& a, int rows, cudaStream_t st) {
    if (a.vocab <= kLpShort) return launch_logprobs_short<T>(a, rows, st);
    return a.top > 0 ? launch_logprobs<T, true>(a, rows, st) : launch_logprobs<T, false>(a, rows, st);
}

}  // namespace fb

extern "C" int functs_b200_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, const int64_t* tokens, int32_t rows,
                                          int32_t vocab, int32_t top, float* logprobs, float* entropy, float* top_logprobs,
                                          int64_t* top_ids, int32_t* status, void* stream) {
    using namespace fb;
    FB_REQUIRE(dtype >= FB_DTYPE_F32 && dtype <= FB_DTYPE_BF16, "token_logprobs: unknown dtype %d", dtype);
    FB_REQUIRE(rows >= 0 && rows <= (1 << 24), "token_logprobs: rows must be 0 .. %d", 1 << 24);
    FB_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "token_logprobs: vocab must be 1 .. %d", 1 << 30);
    FB_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= vocab, "token_logprobs: top must be 0 .. %d and at most vocab", kLpMaxTop);
    if (rows == 0) return FB_OK;
    FB_REQUIRE(logits != nullptr && tokens != nullptr && logprobs != nullptr && entropy != nullptr, "token_logprobs: null pointer");
    FB_REQUIRE(top == 0 || (top_logprobs != nullptr && top_ids != nullptr), "token_logprobs: null pointer");
    FB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == FB_DTYPE_F32 ? 4 : 2) == 0, "token_logprobs: logits must lie on a boundary of their type");
    const uintptr_t words = reinterpret_cast<uintptr_t>(logprobs) | reinterpret_cast<uintptr_t>(entropy) | reinterpret_cast<uintptr_t>(top_logprobs) |
                            reinterpret_cast<uintptr_t>(status);
    FB_REQUIRE(words % 4 == 0 && (reinterpret_cast<uintptr_t>(tokens) | reinterpret_cast<uintptr_t>(top_ids)) % 8 == 0,
               "token_logprobs: pointers must lie on a boundary of their type");
    const LpArgs a = {logits, row_stride, tokens, vocab, top, logprobs, entropy, top_logprobs, top_ids, status};
    const cudaStream_t st = as_stream(stream);
    if (dtype == FB_DTYPE_F32) return launch_logprobs<float>(a, rows, st);
    if (dtype == FB_DTYPE_F16) return launch_logprobs<__half>(a, rows, st);
    return launch_logprobs<__nv_bfloat16>(a, rows, st);
}
