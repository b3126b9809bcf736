// Attention with a decaying state, token by token:  S = decay * S + k v^T,  out = scale * S^T q.
//
// Serves single tokens, which are a pass over the states (bound by their traffic: 8 bytes per cell), and prompts of few tokens (bound by
// what one CTA issues for a token, 0.3 us: shuffles and sums over the rows of S, while few heads leave most SMs without a CTA).  Longer prompts go chunk by chunk.  A state never leaves registers between tokens.
#include <type_traits>

#include "linattn.cuh"

namespace fb {

constexpr int kRecurThreads = 256;
constexpr int kRecurTokens = 16;  // tokens staged at a time

// One token of 16 states of 128 x 128 3.9 us, of 1536 42 (4.8 TB/s), of 8192 187 (5.75 TB/s).
//
// A CTA owns 32 columns of one state: thread -> (column group tid % CG, rows tid / CG + i * RG), so a warp reads whole sectors of four rows, and every thread keeps its part of S in registers over all tokens.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRecurThreads) linattn_recurrent_kernel(const LinArgs a, int tiles) {
    constexpr int CG = 8, RG = kRecurThreads / CG, ROWS = kLinMaxDim / RG, COLS = 4 * CG, WARPS = kRecurThreads / 32;
    __shared__ float s_q[kRecurTokens][kLinMaxDim], s_k[kRecurTokens][kLinMaxDim], s_v[kRecurTokens][COLS];
    __shared__ float s_part[kRecurTokens][WARPS][COLS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile = blockIdx.x % tiles, bh = blockIdx.x / tiles, h = bh % a.heads, b = bh / a.heads;
    const int hk = h / (a.heads / a.kv_heads);
    const int cg = tid % CG, rg = tid / CG, col0 = tile * COLS, c0 = col0 + cg * 4;
    const int cols = min(COLS, a.dv - col0);
    int bits;
    const int slot = lin_slot(a, b, lane, bits);
    if (bits != 0 && a.status != nullptr && tid == 0) atomicOr(a.status, bits);
    const int length = slot < 0 ? 0 : lin_length(a, b);
    // The decay as a sum of two: its rounding would be the same at every token and add up (2e-6 of the state after 63 tokens; now 1e-7).
    const double exact = exp(static_cast<double>(a.log_decay[h]));
    const float decay = static_cast<float>(exact), decay_lo = static_cast<float>(exact - static_cast<double>(decay));
    const int64_t state = (static_cast<int64_t>(slot < 0 ? 0 : slot) * a.heads + h) * a.dk * a.dv;

    float s[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = rg + i * RG;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
        if (slot >= 0 && a.state_in != nullptr && r < a.dk) {
            const float* at = a.state_in + state + static_cast<int64_t>(r) * a.dv + c0;
            if (VEC) {
                if (c0 < a.dv) {
                    const float4 x = *reinterpret_cast<const float4*>(at);
                    s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < a.dv) s[i][j] = at[j];
            }
        }
    }
    const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[2];
    const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
    const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2] + col0;
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[2] + col0;
    // rows that nothing reads stay zero
    const int staged = min(kRecurTokens, length);
    if (a.dk < kLinMaxDim) {
        for (int i = tid; i < staged * kLinMaxDim; i += kRecurThreads) (&s_q[0][0])[i] = (&s_k[0][0])[i] = 0.0f;
    }
    if (cols < COLS) {
        for (int i = tid; i < staged * COLS; i += kRecurThreads) (&s_v[0][0])[i] = 0.0f;
    }
    __syncthreads();
    for (int t0 = 0; t0 < length; t0 += kRecurTokens) {
        const int n = min(kRecurTokens, length - t0);
        for (int i = tid; i < n * a.dk; i += kRecurThreads) {
            const int t = i / a.dk, d = i - t * a.dk;
            s_q[t][d] = lin_float(q[(t0 + t) * a.q_stride[1] + d]);
            s_k[t][d] = lin_float(k[(t0 + t) * a.k_stride[1] + d]);
        }
        for (int i = tid; i < n * cols; i += kRecurThreads) {
            const int t = i / cols, d = i - t * cols;
            s_v[t][d] = lin_float(v[(t0 + t) * a.v_stride[1] + d]);
        }
        __syncthreads();
#pragma unroll 4
        for (int t = 0; t < n; ++t) {  // (tokens overlap: only S ties one to the next)
            const float4 vv = *reinterpret_cast<const float4*>(&s_v[t][cg * 4]);
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const float kr = s_k[t][rg + i * RG], qr = s_q[t][rg + i * RG];
                s[i][0] = fmaf(kr, vv.x, fmaf(decay, s[i][0], decay_lo * s[i][0]));
                s[i][1] = fmaf(kr, vv.y, fmaf(decay, s[i][1], decay_lo * s[i][1]));
                s[i][2] = fmaf(kr, vv.z, fmaf(decay, s[i][2], decay_lo * s[i][2]));
                s[i][3] = fmaf(kr, vv.w, fmaf(decay, s[i][3], decay_lo * s[i][3]));
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = fmaf(qr, s[i][j], o[j]);
            }
#pragma unroll
            for (int d = CG; d < 32; d *= 2) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] += __shfl_xor_sync(kFullMask, o[j], d);
            }
            if (lane < CG) *reinterpret_cast<float4*>(&s_part[t][warp][cg * 4]) = make_float4(o[0], o[1], o[2], o[3]);
        }
        __syncthreads();
        for (int i = tid; i < n * COLS; i += kRecurThreads) {
            const int t = i / COLS, d = i % COLS;
            float o = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) o += s_part[t][w][d];
            if (d < cols) out[(t0 + t) * a.out_stride[1] + d] = lin_from<T>(o * a.scale);
        }
    }
    lin_clear(out, a.out_stride[1], length, a.tokens, cols);
    if (slot < 0) return;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = rg + i * RG;
        if (r >= a.dk) continue;
        float* at = a.state_out + state + static_cast<int64_t>(r) * a.dv + c0;
        if (VEC) {
            if (c0 < a.dv) *reinterpret_cast<float4*>(at) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + j < a.dv) at[j] = s[i][j];
        }
    }
}

// One token, many states: a CTA has a whole state, LANES lanes a row of it, so that 64 KB are on their way at once and one slot is looked up.
constexpr int kStepThreads = 256;
// A lane has four columns of a row, beside one another (VEC: rows of whole 16 bytes) or LANES apart.
template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(kStepThreads) linattn_step_kernel(const LinArgs a) {
    constexpr int WARPS = kStepThreads / 32, PER = 32 / LANES, STEP = WARPS * PER, ROWS = kLinMaxDim / STEP;
    __shared__ float s_q[kLinMaxDim], s_k[kLinMaxDim];
    __shared__ __align__(16) float s_part[WARPS][LANES * 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x % a.heads, b = blockIdx.x / a.heads, hk = h / (a.heads / a.kv_heads);
    const int row = warp * PER + lane / LANES, col = (lane % LANES) * (VEC ? 4 : 1);
    constexpr int kNext = VEC ? 1 : LANES;  // columns between two of a lane's
    const bool has_col = col < a.dv;
    const int named = a.slots == nullptr ? b : a.slots[b];
    const bool inside = named >= 0 && named < a.num_slots;
    const int64_t state = (static_cast<int64_t>(inside ? named : 0) * a.heads + h) * a.dk * a.dv;
    // the state first: it may be read whether the slot is this sequence's or an earlier one's
    float4 s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = row + i * STEP;
        s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (inside && has_col && r < a.dk && a.state_in != nullptr) {
            const float* at = a.state_in + state + static_cast<int64_t>(r) * a.dv + col;
            if (VEC) s[i] = *reinterpret_cast<const float4*>(at);
            else {
                s[i].x = at[0];
                if (col + kNext < a.dv) s[i].y = at[kNext];
                if (col + 2 * kNext < a.dv) s[i].z = at[2 * kNext];
                if (col + 3 * kNext < a.dv) s[i].w = at[3 * kNext];
            }
        }
    }
    const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[2];
    const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
    const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2];
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[2];
    if (tid < kLinMaxDim) s_q[tid] = tid < a.dk ? lin_float(q[tid]) : 0.0f;
    else s_k[tid - kLinMaxDim] = tid - kLinMaxDim < a.dk ? lin_float(k[tid - kLinMaxDim]) : 0.0f;
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = col + j * kNext < a.dv ? lin_float(v[col + j * kNext]) : 0.0f;
    int bits;
    const int slot = lin_slot(a, b, lane, bits);
    if (bits != 0 && a.status != nullptr && tid == 0) atomicOr(a.status, bits);
    const double exact = exp(static_cast<double>(a.log_decay[h]));  // (a sum of two floats: see above)
    const float decay = static_cast<float>(exact), decay_lo = static_cast<float>(exact - static_cast<double>(decay));
    __syncthreads();
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const float kr = s_k[row + i * STEP], qr = s_q[row + i * STEP];
        s[i].x = fmaf(kr, x[0], fmaf(decay, s[i].x, decay_lo * s[i].x));
        s[i].y = fmaf(kr, x[1], fmaf(decay, s[i].y, decay_lo * s[i].y));
        s[i].z = fmaf(kr, x[2], fmaf(decay, s[i].z, decay_lo * s[i].z));
        s[i].w = fmaf(kr, x[3], fmaf(decay, s[i].w, decay_lo * s[i].w));
        o[0] = fmaf(qr, s[i].x, o[0]), o[1] = fmaf(qr, s[i].y, o[1]), o[2] = fmaf(qr, s[i].z, o[2]), o[3] = fmaf(qr, s[i].w, o[3]);
        const int r = row + i * STEP;
        if (slot >= 0 && has_col && r < a.dk) {
            float* at = a.state_out + state + static_cast<int64_t>(r) * a.dv + col;
            if (VEC) *reinterpret_cast<float4*>(at) = s[i];
            else {
                at[0] = s[i].x;
                if (col + kNext < a.dv) at[kNext] = s[i].y;
                if (col + 2 * kNext < a.dv) at[2 * kNext] = s[i].z;
                if (col + 3 * kNext < a.dv) at[3 * kNext] = s[i].w;
            }
        }
    }
#pragma unroll
    for (int d = LANES; d < 32; d *= 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += __shfl_xor_sync(kFullMask, o[j], d);
    }
    if (lane < LANES) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s_part[warp][col + j * kNext] = o[j];
    }
    __syncthreads();
    if (tid < a.dv) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) y += s_part[w][tid];
        out[tid] = lin_from<T>(slot >= 0 ? y * a.scale : 0.0f);
    }
}

// Whether a prompt goes chunk by chunk (kernels_linattn_tc.cu) or token by token.  A chunk takes 11.6 us per wave of heads however few tokens it
// has.  Token by token it is 3.5 us and 0.3 per token while the column tiles are on an SM each, 0.25 per token and tile of an SM beyond
// that: 8 heads of 64, 24 tokens 9.3 (12.0 as a chunk); 128 heads of 128, 8 tokens 11.4 (11.9), 24 tokens 24.8; 1024 heads, 8 tokens 71 (83).
static bool lin_by_chunks(const LinArgs& a) {
    const int64_t heads = static_cast<int64_t>(a.batch) * a.heads, tiles = heads * ((a.dv + 31) / 32);
    const double chunk = 11.6 * static_cast<double>((heads + kNumSMs - 1) / kNumSMs);
    const double token = 0.25 * static_cast<double>(tiles) / kNumSMs;
    return a.tokens > 1 && 3.5 + a.tokens * (token > 0.3 ? token : 0.3) > chunk;
}

template <typename T, bool VEC>
static int launch_step(const LinArgs& a, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.batch) * a.heads), block(kStepThreads);
    if (a.dv <= 32) return launch_after(linattn_step_kernel<T, 8, VEC>, grid, block, 0, st, false, "linear_attention", a);
    if (a.dv <= 64) return launch_after(linattn_step_kernel<T, 16, VEC>, grid, block, 0, st, false, "linear_attention", a);
    return launch_after(linattn_step_kernel<T, 32, VEC>, grid, block, 0, st, false, "linear_attention", a);
}

template <typename T>
static int launch_recurrent(const LinArgs& a, cudaStream_t st) {
    const bool vec = a.dv % 4 == 0 && reinterpret_cast<uintptr_t>(a.state_in) % 16 == 0 && reinterpret_cast<uintptr_t>(a.state_out) % 16 == 0;
    const int64_t bh = static_cast<int64_t>(a.batch) * a.heads;
    const int tiles = (a.dv + 31) / 32;
    FB_REQUIRE(bh * tiles < (1ll << 31), "linear_attention: batch * heads is too large");
    // Whole states where they are small (48 of 64 x 64 3.2 us, in column tiles 4.1) or fill half of the SMs (128 x 128: 16 states 4.6, in
    // tiles 3.9; 64 4.8 and 4.7; 112 5.1 and 6.1; 256 7.1 and 9.7; 1536 42 and 53; of 128 x 39, 2856 31 and 51)
    if (a.tokens == 1 && a.lengths == nullptr && (a.dk * a.dv <= 64 * 64 || bh >= kNumSMs / 2))
        return vec ? launch_step<T, true>(a, st) : launch_step<T, false>(a, st);
    const dim3 grid(static_cast<unsigned>(bh * tiles));
    if (vec) return launch_after(linattn_recurrent_kernel<T, true>, grid, dim3(kRecurThreads), 0, st, false, "linear_attention", a, tiles);
    return launch_after(linattn_recurrent_kernel<T, false>, grid, dim3(kRecurThreads), 0, st, false, "linear_attention", a, tiles);
}

}  // namespace fb

extern "C" int64_t functs_b200_linear_attention_scratch_bytes(const functs_b200_linear_attention_args* a) {
    using namespace fb;
    if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->dk <= 0 || a->dv <= 0 || !lin_by_chunks(*a)) return 0;
    return linattn_chunk_scratch_bytes(*a);
}

extern "C" int functs_b200_linear_attention(const functs_b200_linear_attention_args* args, void* scratch, void* stream) {
    using namespace fb;
    FB_REQUIRE(args != nullptr, "linear_attention: null pointer");
    const LinArgs& a = *args;
    FB_REQUIRE(a.dtype >= FB_DTYPE_F32 && a.dtype <= FB_DTYPE_BF16, "linear_attention: unknown dtype %d", a.dtype);
    FB_REQUIRE(a.batch >= 0 && a.tokens >= 0 && a.tokens <= (1 << 30) && a.heads > 0 && a.kv_heads > 0 && a.heads % a.kv_heads == 0,
               "linear_attention: sizes must not be negative, and heads (%d) a multiple of kv_heads (%d)", a.heads, a.kv_heads);
    FB_REQUIRE(a.dk >= 1 && a.dk <= kLinMaxDim && a.dv >= 1 && a.dv <= kLinMaxDim, "linear_attention: dk (%d) and dv (%d) must be 1 .. %d", a.dk,
               a.dv, kLinMaxDim);
    FB_REQUIRE(a.slots != nullptr || a.num_slots == a.batch, "linear_attention: without slots there are as many states as sequences");
    FB_REQUIRE(a.num_slots >= 0, "linear_attention: num_slots must not be negative");
    if (a.batch == 0) return FB_OK;
    FB_REQUIRE(a.log_decay != nullptr && a.state_out != nullptr, "linear_attention: null pointer");
    FB_REQUIRE(a.tokens == 0 || (a.q != nullptr && a.k != nullptr && a.v != nullptr && a.out != nullptr), "linear_attention: null pointer");
    const uintptr_t elements = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                               reinterpret_cast<uintptr_t>(a.out);
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.log_decay) | reinterpret_cast<uintptr_t>(a.state_in) | reinterpret_cast<uintptr_t>(a.state_out) |
                            reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.lengths) | reinterpret_cast<uintptr_t>(a.status);
    FB_REQUIRE(elements % (a.dtype == FB_DTYPE_F32 ? 4 : 2) == 0 && words % 4 == 0, "linear_attention: pointers must lie on a boundary of their type");
    const cudaStream_t st = as_stream(stream);
    if (lin_by_chunks(a)) return launch_linattn_chunk(a, scratch, st);
    if (a.dtype == FB_DTYPE_F32) return launch_recurrent<float>(a, st);
    if (a.dtype == FB_DTYPE_F16) return launch_recurrent<__half>(a, st);
    return launch_recurrent<__nv_bfloat16>(a, st);
}
