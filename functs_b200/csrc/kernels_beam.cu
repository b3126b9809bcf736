// Beam search: the best continuations of every group of beams, and the states of the beams that go on.
//
// Selection.  score(k, v) = scores[k] + x_k[v] - log sum exp x_k.  Within a beam the order is that of its logits, so only the `top` best of each row
// can be among the group's: one pass over a row gives its sum and those (as token_logprobs has it; few long rows are cut into parts), then a block per
// group joins the parts' sums and lists and merges the rows' lists: a candidate's place is the number of better ones.
//
// The order is that of the scores in 64 bits.  A row's logarithm out of the pass is off by some 2^-19 at most (5e-8 as measured), the same for all of
// its candidates, so only neighbours from different rows that lie nearer to one another than that can be the wrong way round.  Where there are any
// among the best (one call of 64 groups of 8 in ten), the rows in question are summed again in 64 bits by the group's block, and the lists
// merged again: 14 us more for every row of 50001, bound by the block's SM, which does some 16 products in 64 bits a cycle (with the library's
// exponentials, four at a time, 25); 8 beams that are alike 129 us, 64 of 32000 in fp32 1450.  Tried for that: a cluster of eight blocks a group that shares the rows, 14 us instead of 50 for two of them, but 3.5 us
// more for every call of many groups.
//
// Two launches, 9.5 us for 4 rows of 32000 in fp32 (7 the pass and the choice, whose block barriers are the latency, the rest the merging); 64 groups of 8 rows of
// 50001 in bf16 24 us, 2.1 TB/s (27 with a few near neighbours): a row's choice follows its pass, which a block loads nothing behind.  In 16 bits the rows' kernel spills 24 to 28
// bytes of 40 registers.  64 beams with 64 candidates 440 us: places by halving, a chain of loads.  Tried, when those were 10 and 25.5: rows of a group as a cluster
// that merges in its first block's shared memory 10.5 and 32.7 (all blocks stay until the slowest has finished), 256 threads a row 14 and 28.
#include "logprobs.cuh"

namespace fb {

constexpr int kBeamMaxBeams = FB_BEAM_MAX_BEAMS, kBeamMaxTop = FB_BEAM_MAX_TOP;
constexpr int kBeamMergeThreads = 256;
constexpr int kBeamInParts = 128;  // candidates of a group whose rows are in parts, at most
static_assert(kBeamMaxBeams <= kBeamMergeThreads - kBeamInParts, "the rows' sums are for the other threads");

enum BeamKind : int32_t { kBeamLive = 0, kBeamFlat = 1, kBeamNan = 2, kBeamEnded = 3 };  // flat: -inf for all

struct BeamRow {
    double base, log_s;  // log sum exp = base + log_s
    int32_t kind;
};
// what a block leaves of its part of a row, beside its best candidates
struct __align__(16) BeamPart {
    LpSums sums;
    float off;  // how far the logarithm of the sum may be from its value
};

struct BeamArgs {
    const void* logits;
    int64_t group_stride, beam_stride, end_token;
    const float* scores;
    const uint8_t* ended;
    int32_t beams, vocab, top, listed;  // listed: candidates of a part, the smaller of top and vocab
    int32_t parts;                      // blocks of a row
    float* out_scores;
    int64_t *parents, *tokens;
    BeamPart* left;  // [rows, parts]
    uint64_t* keys;  // [rows, parts, listed]: see lp_key, best first; 0 behind the last
};

// What can be said of a row before its logits are looked at: a live one's are.
__device__ __forceinline__ int beam_kind(const BeamArgs& a, int64_t row) {
    const float score = a.scores[row];
    if (!(score <= 3.402823466e38f)) return kBeamNan;
    if (score < -3.402823466e38f) return kBeamFlat;
    return a.ended != nullptr && a.ended[row] != 0 ? kBeamEnded : kBeamLive;
}

template <typename T>
__device__ __forceinline__ const T* beam_row(const BeamArgs& a, int64_t row) {
    return static_cast<const T*>(a.logits) + (row / a.beams) * a.group_stride + (row % a.beams) * a.beam_stride;
}

// A block per part of a row.
template <typename T>
__global__ void __launch_bounds__(kLpMaxThreads, 3) beam_rows_kernel(const BeamArgs a) {
    __shared__ LpShared<true> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int64_t row = blockIdx.x / a.parts;
    if (beam_kind(a, row) != kBeamLive) return;
    const LpPart<T> p = lp_part(beam_row<T>(a, row), a.vocab, static_cast<int>(blockIdx.x % a.parts), a.parts);
    const LpThread th = lp_pass(p);
    LpSums sums = th.warp_sums();
    if (lane == 0) sh.sums[warp] = sums;
    const bool far = __syncthreads_or(lane == 0 && lp_far(sums.most));
    if (far) lp_again<T, true>(sh, p);
    if (warp == 0) {
        sums.none();
        if (lane < warps) sums = sh.sums[lane];
        lp_join_lanes(sums, 16);
        // Powers are off by 2^-22.5 and by the rounding of their exponents, some 2^-22 in all; a thread adds up what four vectors give, 2^-24 of the sum
        // each time (far from 0 every element's own).
        const int adds = (p.count() + blockDim.x - 1) / blockDim.x;
        if (lane == 0) a.left[blockIdx.x] = {sums, far ? (adds + 32) * 0x1p-24f : 0x1p-20f + (adds / 16 + 16) * 0x1p-24f};
    }
    lp_select<T>(sh, p, a.listed, th.most);
    pdl_launch_dependents();
    for (int i = tid; i < a.listed; i += blockDim.x) a.keys[static_cast<int64_t>(blockIdx.x) * a.listed + i] = sh.best[i];
}

constexpr int kBeamPowers = 256;  // (2^8: see beam_exp)
constexpr int kBeamLoads = 32;
struct BeamShared {
    BeamRow row[kBeamMaxBeams];
    float score[kBeamMaxBeams], off[kBeamMaxBeams];
    uint8_t again[kBeamMaxBeams];
    double part[kBeamMergeThreads / 32], power[kBeamPowers];
    uint64_t in_parts[kBeamInParts];  // keys of a group whose rows are in parts
    int any;
};

// A float as a double by its bits (one below the normal range as some 1e-38): a conversion is slow.
__device__ __forceinline__ double beam_double(float x) {
    const uint32_t u = __float_as_uint(x);
    return __hiloint2double(static_cast<int>((u & 0x80000000u) | (((u & 0x7FFFFFFFu) >> 3) + (896u << 20))), static_cast<int>(u << 29));
}
// exp(x - base), x <= base, for sums in 64 bits.  With y = x - base, k = y 256 / ln 2 rounded to a whole number and r = y - k ln 2 / 256, |r| <= 0.0014, it is 2^(k / 256),
// from a table of kBeamPowers powers, times the first terms of exp(r)'s Taylor series (4e-17 are left out).  Eight products in 64 bits, of which an SM does 16 a
// cycle.  What lies 600 or more below base, -inf too, counts as nothing: by the difference, since next to a base far from 0 there may be no float 600 below.
__device__ __forceinline__ double beam_exp(float x, float base, const double* power) {
    const float apart = x - base;
    const float whole = fmaf(fmaxf(apart, -600.0f), kBeamPowers * kLpLog2e, 12582912.0f);  // 1.5 * 2^23: a sum with it is a whole number, in its last bits
    const int k = __float_as_int(whole) - __float_as_int(12582912.0f);
    const double y = beam_double(x) - beam_double(base), r = fma(beam_double(whole - 12582912.0f), -0.69314718055994530942 / kBeamPowers, y);
    double p = fma(1.0 / 24.0, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0) * power[k & (kBeamPowers - 1)];
    p = __hiloint2double(__double2hiint(p) + (k >> 8) * (1 << 20), __double2loint(p));
    return apart > -600.0f ? p : 0.0;
}

// entries of a list in descending order that are above `x`, or, where `equal`, not below it
__device__ __forceinline__ int beam_above(const double* list, int n, double x, bool equal) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > x || (equal && list[mid] == x)) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The candidates' scores (a NaN as +inf, which no other has), and who is at each place: order[place] = candidate.  Lists follow one another by beam: of equal
// scores the lowest beam comes first, and of one beam's the largest logit, then the lowest token, which is a list's own order.  (Next to a score far from 0 logits
// that differ make the same score.)
constexpr int kBeamCount = 512;  // candidates whose places are counted one by one: a halving is a chain of loads
__device__ __forceinline__ void beam_place(const BeamArgs& a, const BeamShared& sh, const uint64_t* keys, double* score, int* order) {
    const int count = a.beams * a.listed;
    for (int c = threadIdx.x; c < count; c += kBeamMergeThreads) {
        const int k = c / a.listed, i = c % a.listed;
        const BeamRow& row = sh.row[k];
        double s = -INFINITY;
        if (row.kind == kBeamLive) {
            s = static_cast<double>(sh.score[k]) + ((static_cast<double>(lp_value(static_cast<uint32_t>(keys[c] >> 32))) - row.base) - row.log_s);
        } else if (row.kind == kBeamNan) {
            s = INFINITY;
        } else if (row.kind == kBeamEnded && i == 0) {
            s = static_cast<double>(sh.score[k]);
        }
        score[c] = s;
    }
    __syncthreads();
    if (count <= kBeamCount) {
        for (int c = threadIdx.x; c < count; c += kBeamMergeThreads) {
            const double own = score[c];
            int place = 0;
#pragma unroll 8
            for (int o = 0; o < count; ++o) {
                const double other = score[o];
                place += other > own || (other == own && o < c);
            }
            order[place] = c;
        }
    } else {
        for (int c = threadIdx.x; c < count; c += kBeamMergeThreads) {
            const int list = c / a.listed;
            const double own = score[c];
            int place = c % a.listed;
            for (int o = 0; o < a.beams; ++o)
                if (o != list) place += beam_above(score + o * a.listed, a.listed, own, o < list);
            order[place] = c;
        }
    }
    __syncthreads();
}

// A block per group: its rows' sums, then the best of their lists.
template <typename T>
__global__ void __launch_bounds__(kBeamMergeThreads) beam_merge_kernel(const BeamArgs a) {
    extern __shared__ __align__(16) unsigned char beam_smem[];
    __shared__ BeamShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, count = a.beams * a.listed;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.beams;
    double* score = reinterpret_cast<double*>(beam_smem);
    uint64_t* keys = reinterpret_cast<uint64_t*>(score + count);  // of every row, best first
    int* order = reinterpret_cast<int*>(keys + count);
    int kind = kBeamLive;
    if (tid < a.beams) {
        kind = beam_kind(a, first + tid);
        sh.score[tid] = a.scores[first + tid];
        sh.again[tid] = 0;
    }
    if (tid == 0) sh.any = 0;
    for (int c = tid; c < count; c += kBeamMergeThreads) order[c] = c;  // (a candidate whatever the scores)
    pdl_wait();
    if (a.parts == 1) {
        for (int c = tid; c < count; c += kBeamMergeThreads) keys[c] = a.keys[first * a.listed + c];
    } else if (tid >= kBeamMergeThreads - kBeamInParts) {
        // a row's lists become one, by their keys (upper warps: beside the rows' sums)
        const int c = tid - (kBeamMergeThreads - kBeamInParts), span = a.parts * a.listed, k = c / span;
        const bool there = k < a.beams;
        uint64_t key = 0;
        if (there) key = sh.in_parts[c] = a.keys[first * span + c];
        asm volatile("bar.sync 1, %0;" ::"n"(kBeamInParts) : "memory");
        int place = 0;
        for (int o = k * span; there && o < (k + 1) * span; ++o) place += sh.in_parts[o] > key;
        if (there && place < a.listed) keys[k * a.listed + place] = key;
    }
    if (tid < a.beams) {
        BeamRow row = {0.0, 0.0, kind};
        float off = 0.0f;
        if (kind == kBeamLive) {
            const BeamPart* left = a.left + (first + tid) * a.parts;
            LpSums sums = left[0].sums;
            off = left[0].off;
            for (int p = 1; p < a.parts; ++p) {
                const LpSums own = sums, more = left[p].sums;
                off = fmaxf(off, left[p].off);
                sums.most = max_nan(own.most, more.most);
                sums.s = sums.t = 0.0f;
                for (const LpSums& one : {own, more}) {
                    if (one.most == __int_as_float(0xff800000)) continue;
                    const float below = fmaxf((one.most - sums.most) * kLpLog2e, -1000.0f), f = lp_ex2(below);
                    sums.t = fmaf(f, fmaf(below, one.s, one.t), sums.t);
                    sums.s = fmaf(f, one.s, sums.s);
                }
            }
            if (a.parts > 1) off += a.parts * 0x1p-22f;
            double s;
            const LpRow got = lp_row(sums, s);
            row.base = got.base, row.log_s = got.log_s;
            if (got.empty) row.kind = kBeamFlat;
            else if (!(sums.most <= 3.402823466e38f)) row.kind = kBeamNan;
        }
        sh.row[tid] = row;
        sh.off[tid] = row.kind == kBeamLive ? off : 0.0f;
    }
    __syncthreads();
    beam_place(a, sh, keys, score, order);
    float off = 0.0f;
    for (int k = 0; k < a.beams; ++k) off = fmaxf(off, sh.off[k]);
    const double near = 2.0 * static_cast<double>(off);
    // neighbours that may be the wrong way round; behind the last place as long as they lie as near (or where a score's own rounding may part or join them)
    const auto check = [&](int p) {
        const int c = order[p], d = order[p + 1];
        if (!(score[c] < INFINITY && score[d] > -INFINITY && score[c] - score[d] <= near + (fabs(score[c]) + fabs(score[d])) * 0x1p-52)) return false;
        const int k = c / a.listed, o = d / a.listed;
        if (k != o) sh.again[k] = sh.again[o] = 1, sh.any = 1;
        return true;
    };
    for (int p = tid; p < a.top - 1; p += kBeamMergeThreads) check(p);
    if (tid == 0) {
        for (int p = a.top - 1; p + 1 < count && check(p); ++p) {}
    }
    __syncthreads();
    if (sh.any != 0) {
        for (int i = tid; i < kBeamPowers; i += kBeamMergeThreads) sh.power[i] = exp(i * (0.69314718055994530942 / kBeamPowers));
        __syncthreads();
        for (int k = 0; k < a.beams; ++k) {
            if (sh.again[k] == 0 || sh.row[k].kind != kBeamLive) continue;
            const T* row = beam_row<T>(a, first + k);
            const float base = static_cast<float>(sh.row[k].base);  // (the largest logit)
            // (elements by their number, whatever boundary a row lies on: rows that are the same have the same sum; many on their way at once)
            double some[4] = {};
            for (int v = tid; v < a.vocab; v += kBeamLoads * kBeamMergeThreads) {
                float x[kBeamLoads];
#pragma unroll
                for (int e = 0; e < kBeamLoads; ++e) {
                    const int at = v + e * kBeamMergeThreads;
                    x[e] = at < a.vocab ? LpVec<T>::one(row + at) : __int_as_float(0xff800000);
                }
#pragma unroll
                for (int e = 0; e < kBeamLoads; ++e) some[e % 4] += beam_exp(x[e], base, sh.power);
            }
            double s = (some[0] + some[1]) + (some[2] + some[3]);
            for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(kFullMask, s, d);
            __syncthreads();
            if (lane == 0) sh.part[warp] = s;
            __syncthreads();
            if (tid == 0) {
                s = 0.0;
                for (int w = 0; w < kBeamMergeThreads / 32; ++w) s += sh.part[w];
                sh.row[k].log_s = log(s);
            }
        }
        __syncthreads();
        beam_place(a, sh, keys, score, order);
    }
    for (int p = tid; p < a.top; p += kBeamMergeThreads) {
        const int c = order[p], k = c / a.listed, i = c % a.listed;
        const int settled = sh.row[k].kind;
        int64_t token = i;
        if (settled == kBeamLive) token = static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(keys[c]));
        if (settled == kBeamEnded) token = i == 0 ? a.end_token : i <= a.end_token ? i - 1 : i;
        const int64_t at = static_cast<int64_t>(blockIdx.x) * a.top + p;
        a.out_scores[at] = settled == kBeamNan ? __int_as_float(0x7fffffff) : static_cast<float>(score[c]);
        a.parents[at] = k;
        a.tokens[at] = token;
    }
}

// Blocks of a row at most: few rows leave most SMs without one.
static int beam_most_parts(int64_t groups, int beams) {
    int parts = 1;
    while (parts < 8 && groups * beams * parts * 2 <= kNumSMs && beams * parts * 2 <= kBeamMaxBeams) parts *= 2;
    return parts;
}

template <typename T>
static int launch_beam(BeamArgs& a, int groups, cudaStream_t st) {
    const int64_t rows = static_cast<int64_t>(groups) * a.beams;
    const int vecs = a.vocab / LpVec<T>::N;
    // a part has 2048 vectors at least (one row of 32000 in fp32 is two, one of 65536 in 16 bits four), and a group 128 candidates at most: merging them is what
    // parts cost (8 rows of 131072 in bf16 with 16 candidates, when every part's list was merged by scores: 64 lists 96 us, 32 24, 8 22; with 8 candidates, two parts
    // a row, 12.9)
    const int most = beam_most_parts(groups, a.beams);
    a.parts = 1;
    while (a.parts < most && vecs / (a.parts * 2) >= 2048 && a.beams * a.parts * 2 * a.listed <= kBeamInParts) a.parts *= 2;
    a.left = reinterpret_cast<BeamPart*>(a.keys);
    a.keys = reinterpret_cast<uint64_t*>(a.left + rows * a.parts);
    // 512 threads a block are three blocks an SM.  384 are four: long rows in one wave instead of two (512 rows of 131072 in bf16 47 us and 56, of 50001
    // 25.5 and 25.8; of 32000 18.5 and 16.8).
    const int each = vecs / a.parts;
    const bool wave = rows * a.parts > 3 * kNumSMs && rows * a.parts <= 4 * kNumSMs && each >= 6144;
    const int threads = wave ? 384 : each >= 1024 ? 512 : each >= 512 ? 256 : 128;
    FB_TRY(launch_after(beam_rows_kernel<T>, dim3(static_cast<unsigned>(rows * a.parts)), dim3(threads), 0, st, false, "beam_select", a));
    const size_t smem = static_cast<size_t>(a.beams) * a.listed * (sizeof(double) + sizeof(uint64_t) + sizeof(int));
    if (smem > 40 * 1024)
        FB_TRY(check_cuda(cudaFuncSetAttribute(beam_merge_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)), "beam_select"));
    return launch_after(beam_merge_kernel<T>, dim3(groups), dim3(kBeamMergeThreads), smem, st, true, "beam_select", a);
}

// ---- the states of the beams that go on ---------------------------------------------------------------------------------

constexpr int kReorderThreads = 256, kReorderPools = 32, kReorderMostBeams = 1 << 20;
constexpr int64_t kReorderPiece = 16 * 1024;  // bytes of a row that a CTA copies

struct ReorderArgs {
    const int64_t* parents;
    const int32_t* slots;
    int32_t* new_slots;
    int32_t* status;
    int32_t beams, num_slots, count;
    int32_t pieces;                  // of all pools' rows
    int32_t end[kReorderPools];      // the piece behind a pool's last
    void* data[kReorderPools];
    int64_t row_bytes[kReorderPools];
};

// Copies `bytes` from one place to another, the whole block.
template <typename W>
__device__ __forceinline__ void reorder_copy(void* to, const void* from, int64_t bytes) {
    constexpr int AHEAD = 4;
    const int n = static_cast<int>(bytes / sizeof(W));
    for (int i = threadIdx.x; i < n; i += AHEAD * kReorderThreads) {
        W x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (i + k * kReorderThreads < n) x[k] = static_cast<const W*>(from)[i + k * kReorderThreads];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (i + k * kReorderThreads < n) static_cast<W*>(to)[i + k * kReorderThreads] = x[k];
    }
}

// A CTA copies one piece of the rows of one group.  No copy's source is another's destination: sources are slots of beams with children, destinations
// of beams without, and no slot stands twice in the table.
__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const ReorderArgs a) {
    __shared__ int s_slot[kBeamMaxBeams], s_parent[kBeamMaxBeams], s_free[kBeamMaxBeams], s_from[kBeamMaxBeams];
    __shared__ int s_bits;
    const int tid = threadIdx.x, k = a.beams, pieces = max(a.pieces, 1);
    const int64_t g = blockIdx.x / pieces, first = g * k;
    int piece = blockIdx.x % pieces;
    if (tid == 0) s_bits = 0;
    __syncthreads();
    if (tid < k) {
        const int slot = a.slots[first + tid];
        const int64_t parent = a.parents[first + tid];
        s_slot[tid] = slot;
        s_parent[tid] = static_cast<int>(parent);
        if (slot < 0 || slot >= a.num_slots || parent < 0 || parent >= k) atomicOr(&s_bits, FB_STATUS_INDEX_RANGE);
    }
    __syncthreads();
    const bool none = s_slot[0] < 0;
    bool twice = false;
    for (int64_t e = tid; e < first + k && !none; e += kReorderThreads) {
        const int slot = a.slots[e];
        for (int j = e < first ? 0 : static_cast<int>(e - first) + 1; j < k; ++j) twice |= slot == s_slot[j];
    }
    if (twice) atomicOr(&s_bits, FB_STATUS_INDEX_TWICE);
    __syncthreads();
    const int bits = s_bits;
    const bool writes = piece == 0;
    if (none || bits != 0) {
        if (writes && tid < k) a.new_slots[first + tid] = s_slot[tid];
        if (writes && tid == 0 && !none && a.status != nullptr) atomicOr(a.status, bits);
        return;
    }
    int later = 0, rank = 0;  // whether an earlier beam has the same parent; how many such, or free slots, come before
    if (tid < k) {
        bool goes_on = false;
        for (int j = 0; j < k; ++j) goes_on |= s_parent[j] == tid;
        s_free[tid] = goes_on ? 0 : 1;
        for (int j = 0; j < tid; ++j) later |= s_parent[j] == s_parent[tid];
        s_from[tid] = later;
    }
    __syncthreads();
    int copies = 0, free_rank = 0, is_free = 0;
    for (int j = 0; j < k; ++j) copies += s_from[j];
    if (tid < k) {
        is_free = s_free[tid];
        for (int j = 0; j < tid; ++j) rank += s_from[j], free_rank += s_free[j];
    }
    __syncthreads();
    if (is_free) s_free[free_rank] = s_slot[tid];  // (the slots that come free, in order)
    __syncthreads();
    if (tid < k) {
        const int from = s_slot[s_parent[tid]];
        if (writes) a.new_slots[first + tid] = later ? s_free[rank] : from;
        if (later) s_from[rank] = from;
    }
    __syncthreads();
    if (a.pieces == 0) return;
    int pool = 0;
    while (piece >= a.end[pool]) ++pool;
    if (pool > 0) piece -= a.end[pool - 1];
    const int64_t row = a.row_bytes[pool], at = piece * kReorderPiece, bytes = min(kReorderPiece, row - at);
    char* const data = static_cast<char*>(a.data[pool]) + at;
    const uintptr_t boundary = reinterpret_cast<uintptr_t>(data) | static_cast<uintptr_t>(row);
    for (int c = 0; c < copies; ++c) {
        char* to = data + s_free[c] * row;
        const char* from = data + s_from[c] * row;
        if (boundary % 16 == 0) reorder_copy<uint4>(to, from, bytes);
        else if (boundary % 4 == 0) reorder_copy<uint32_t>(to, from, bytes);
        else reorder_copy<uint8_t>(to, from, bytes);
    }
}

}  // namespace fb

extern "C" int64_t functs_b200_beam_select_scratch_bytes(int32_t groups, int32_t beams, int32_t top) {
    if (groups <= 0 || beams <= 0 || top <= 0) return 0;
    return static_cast<int64_t>(groups) * beams * fb::beam_most_parts(groups, beams) * (static_cast<int64_t>(sizeof(fb::BeamPart)) + static_cast<int64_t>(top) * 8);
}

extern "C" int functs_b200_beam_select(const void* logits, int32_t dtype, int64_t group_stride, int64_t beam_stride, const float* scores,
                                       const uint8_t* ended, int64_t end_token, int32_t groups, int32_t beams, int32_t vocab, int32_t top,
                                       float* out_scores, int64_t* parents, int64_t* tokens, void* scratch, void* stream) {
    using namespace fb;
    FB_REQUIRE(dtype >= FB_DTYPE_F32 && dtype <= FB_DTYPE_BF16, "beam_select: unknown dtype %d", dtype);
    FB_REQUIRE(groups >= 0 && groups <= (1 << 20), "beam_select: groups must be 0 .. %d", 1 << 20);
    FB_REQUIRE(beams >= 1 && beams <= kBeamMaxBeams, "beam_select: beams must be 1 .. %d", kBeamMaxBeams);
    FB_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "beam_select: vocab must be 1 .. %d", 1 << 30);
    FB_REQUIRE(top >= 1 && top <= kBeamMaxTop && top <= static_cast<int64_t>(beams) * vocab, "beam_select: top must be 1 .. %d and at most beams * vocab",
               kBeamMaxTop);
    FB_REQUIRE(ended == nullptr || (end_token >= 0 && end_token < vocab), "beam_select: end_token must be in the vocabulary");
    if (groups == 0) return FB_OK;
    FB_REQUIRE(logits != nullptr && scores != nullptr && out_scores != nullptr && parents != nullptr && tokens != nullptr && scratch != nullptr,
               "beam_select: null pointer");
    FB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == FB_DTYPE_F32 ? 4 : 2) == 0 &&
                   (reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(out_scores)) % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(tokens)) % 8 == 0 && reinterpret_cast<uintptr_t>(scratch) % 16 == 0,
               "beam_select: pointers must lie on a boundary of their type, scratch on one of 16 bytes");
    BeamArgs a = {logits, group_stride, beam_stride, end_token, scores, ended, beams, vocab, top, top < vocab ? top : vocab, 1, out_scores, parents, tokens, nullptr,
                  static_cast<uint64_t*>(scratch)};
    const cudaStream_t st = as_stream(stream);
    if (dtype == FB_DTYPE_F32) return launch_beam<float>(a, groups, st);
    if (dtype == FB_DTYPE_F16) return launch_beam<__half>(a, groups, st);
    return launch_beam<__nv_bfloat16>(a, groups, st);
}

extern "C" int functs_b200_beam_reorder(const functs_b200_state_pool* pools, int32_t count, int32_t num_slots, const int64_t* parents,
                                        const int32_t* slots, int32_t* new_slots, int32_t groups, int32_t beams, int32_t* status, void* stream) {
    using namespace fb;
    FB_REQUIRE(groups >= 0 && groups <= (1 << 20), "beam_reorder: groups must be 0 .. %d", 1 << 20);
    FB_REQUIRE(beams >= 1 && beams <= kBeamMaxBeams, "beam_reorder: beams must be 1 .. %d", kBeamMaxBeams);
    FB_REQUIRE(count >= 0 && num_slots >= 0, "beam_reorder: sizes must not be negative");
    if (groups == 0) return FB_OK;
    FB_REQUIRE(parents != nullptr && slots != nullptr && new_slots != nullptr && (count == 0 || pools != nullptr), "beam_reorder: null pointer");
    FB_REQUIRE(reinterpret_cast<uintptr_t>(parents) % 8 == 0 &&
                   (reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(new_slots) | reinterpret_cast<uintptr_t>(status)) % 4 == 0,
               "beam_reorder: pointers must lie on a boundary of their type");
    for (int32_t i = 0; i < count; ++i) {
        FB_REQUIRE(pools[i].row_bytes >= 0 && pools[i].row_bytes <= (1ll << 40), "beam_reorder: row_bytes must be 0 .. 2^40");
        FB_REQUIRE(pools[i].row_bytes == 0 || num_slots == 0 || pools[i].data != nullptr, "beam_reorder: null pointer");
    }
    // (every CTA compares its group's slots with all that stand before them: 1.3 ms for 2048 groups of 64, 70 ms for 2^14 of them, 0.9 s for 2^20 groups of one; 2^20 of
    // 64 would be minutes)
    FB_REQUIRE(static_cast<int64_t>(groups) * beams <= kReorderMostBeams, "beam_reorder: the table is too large: %d groups of %d beams, of %d beams in all at most", groups,
               beams, kReorderMostBeams);
    int32_t next = 0;
    do {
        ReorderArgs a = {parents, slots, new_slots, status, beams, num_slots};
        int64_t pieces = 0;
        for (; next < count && a.count < kReorderPools; ++next) {
            if (pools[next].row_bytes == 0) continue;
            pieces += (pools[next].row_bytes + kReorderPiece - 1) / kReorderPiece;
            FB_REQUIRE((pieces > 0 ? pieces : 1) * groups < (1ll << 31), "beam_reorder: the states are too large");
            a.data[a.count] = pools[next].data, a.row_bytes[a.count] = pools[next].row_bytes, a.end[a.count] = static_cast<int32_t>(pieces);
            ++a.count;
        }
        a.pieces = static_cast<int32_t>(pieces);
        FB_TRY(launch_after(beam_reorder_kernel, dim3(static_cast<unsigned>((pieces > 0 ? pieces : 1) * groups)), dim3(kReorderThreads), 0, as_stream(stream), false,
                            "beam_reorder", a));
    } while (next < count);
    return FB_OK;
}
