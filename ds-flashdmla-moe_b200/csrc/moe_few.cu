// A whole MoE FFN layer for the few tokens of a decode step (T <= 128): gate, top-k, the chosen experts' SwiGLU MLPs, the
// shared expert and the weighted sum (README.md:17-20 of the reference names the parts; it ships no source for them).
//
//   z[t, e]  = sum_i x[t, i] Wg[i, e]                                  the k largest win, ties: lower expert
//   w[t, j]  = exp(z_j - z_0) / sum_j' exp(z_j' - z_0)                 softmax over the winners = p_j / sum of the selected p
//   out[t]   = sum_j w[t, j] (silu(x[t] W1[e_j]) * (x[t] W3[e_j])) W2[e_j]  (+ the shared expert with weight 1)
//
// There is no capacity: no assignment is dropped.
//
// The logits are summed in 64 bits, so which experts win does not depend on the order of a sum (two logits that differ by a
// rounding of a 32-bit sum would otherwise pick different experts in different kernels).
//
// Bound: the weights of the experts that win, 6 d f bytes each, read once for all tokens.  One launch of the gate kernel and one of
// the layer kernel (moe_few_tc.cuh) for bf16 and widths that are multiples of 64, five launches on CUDA cores for the rest.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"
#include "ptx.cuh"

namespace fdmla {
namespace few {

constexpr int MAX_T = 128;

__device__ __forceinline__ float silu(float x) { return x / (1.f + __expf(-x)); }

// ---- gate: logits in 64 bits -------------------------------------------------------------------------------------------
// Block (32 experts, one of gridDim.y slices of d, TOK tokens): a lane owns an expert, a warp every 16th of ROWS rows at a time,
// whose loads are all in flight at once.  part[s, t, e] holds slice s's share of the logit.  All blocks together also clear the
// counters of the kernel behind.  For one token 512 rows and one block per SM (64 registers, as two blocks would leave, spill and
// cost 3 us of 23 .. 150); for more 128 rows, 8 tokens and two blocks (256 rows
// spill).
constexpr int GATE_THREADS = 512, GATE_TOK = 8, MAX_SLICES = 32;

template <typename T, int TOK, int ROWS>
__global__ void __launch_bounds__(GATE_THREADS, TOK == 1 ? 1 : 2) gate_kernel(const T *__restrict__ x, const float *__restrict__ Wg,
                                                            double *__restrict__ part, unsigned *__restrict__ counters,
                                                            int n_counters, int n_tok, int d, int E) {
    // activations as [row][token] (one token of padding against bank conflicts), later the warps' sums as [warp][token][expert]
    constexpr int LDX = TOK == 1 ? 1 : TOK + 1, WARPS = GATE_THREADS / 32;
    __shared__ double s_x[ROWS * LDX > WARPS * TOK * 32 ? ROWS * LDX : WARPS * TOK * 32];
    ptx::launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int e = blockIdx.x * 32 + lane, t0 = blockIdx.z * TOK;
    {
        const int block = (blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
        const int blocks = gridDim.x * gridDim.y * gridDim.z;
        for (int i = block * GATE_THREADS + threadIdx.x; i < n_counters; i += blocks * GATE_THREADS) counters[i] = 0u;
    }
    const int lo = (int)((long long)d * blockIdx.y / gridDim.y), hi = (int)((long long)d * (blockIdx.y + 1) / gridDim.y);
    double acc[TOK];
#pragma unroll
    for (int j = 0; j < TOK; ++j) acc[j] = 0.0;
    for (int r0 = lo; r0 < hi; r0 += ROWS) {
        const int rows = hi - r0 < ROWS ? hi - r0 : ROWS;
        float wv[ROWS / 16];
#pragma unroll
        for (int i = 0; i < ROWS / 16; ++i) {
            const int r = warp + 16 * i;
            wv[i] = (r < rows && e < E) ? __ldg(Wg + (size_t)(r0 + r) * E + e) : 0.f;
        }
        __syncthreads();
        {   // a warp stages 1 / (16 / TOK) of a token's rows; all loads in flight
            const int j = warp % TOK, part0 = (warp / TOK) * 32 + lane;
            float v[ROWS * TOK / GATE_THREADS];
#pragma unroll
            for (int i = 0; i < ROWS * TOK / GATE_THREADS; ++i) {
                const int r = part0 + i * (GATE_THREADS / TOK);
                v[i] = (r < rows && t0 + j < n_tok) ? to_f32(x[(size_t)(t0 + j) * d + r0 + r]) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < ROWS * TOK / GATE_THREADS; ++i) s_x[(part0 + i * (GATE_THREADS / TOK)) * LDX + j] = (double)v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ROWS / 16; ++i) {
            const int r = warp + 16 * i;
            if (r >= rows) break;
            const double wd = (double)wv[i];
#pragma unroll
            for (int j = 0; j < TOK; ++j) acc[j] = fma(s_x[r * LDX + j], wd, acc[j]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TOK; ++j) s_x[(warp * TOK + j) * 32 + lane] = acc[j];
    __syncthreads();
    if (warp < TOK && e < E && t0 + warp < n_tok) {          // warp j sums token j
        double z = 0.0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) z += s_x[(w * TOK + warp) * 32 + lane];
        part[((size_t)blockIdx.y * n_tok + t0 + warp) * E + e] = z;
    }
}

template <typename T>
static int launch_gate(const void *x, const float *Wg, double *part, unsigned *counters, int n_counters, int n_tok, int d, int E,
                       int slices, cudaStream_t s) {
    const dim3 grid((E + 31) / 32, slices, (n_tok + GATE_TOK - 1) / GATE_TOK);
    if (n_tok == 1) gate_kernel<T, 1, 512><<<grid, GATE_THREADS, 0, s>>>(static_cast<const T *>(x), Wg, part, counters, n_counters, n_tok, d, E);
    else gate_kernel<T, GATE_TOK, 128><<<grid, GATE_THREADS, 0, s>>>(static_cast<const T *>(x), Wg, part, counters, n_counters, n_tok, d, E);
    return check_launch();
}

// slices of d: one round of blocks, at least 64 rows each
static int gate_slices(int n_tok, int d, int E) {
    const int blocks = ((E + 31) / 32) * ((n_tok + GATE_TOK - 1) / GATE_TOK);
    int s = (n_tok == 1 ? 1 : 2) * kNumSMs / blocks;
    if (s > MAX_SLICES) s = MAX_SLICES;
    if (s > d / 64) s = d / 64;
    return s < 1 ? 1 : s;
}

// Logits as integers of the same order; a NaN is below every number (it never wins while a number is left).  0 marks a winner.
__device__ __forceinline__ unsigned long long logit_key(double z) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(z + 0.0);     // -0 and 0 tie
    return isnan(z) ? 1ull : ((u >> 63) ? ~u : (u | (1ull << 63)));
}
__device__ __forceinline__ double key_logit(unsigned long long key) {
    return __longlong_as_double((long long)((key >> 63) ? (key & ~(1ull << 63)) : ~key));
}

// The k winners of one token by one warp; key [E] (shared memory) is overwritten.  `nan`: some logit of the token is NaN, and
// so are its weights then, as those of a softmax over the logits would be.  Every lane keeps the best of its experts, a round
// is three warp reductions (high half, low half, index) and a new scan by the lane that lost its best.
__device__ __forceinline__ void topk_warp(unsigned long long *key, int E, int k, bool nan, int32_t *idx, float *w,
                                          int lane) {
    unsigned long long best = 0;
    int at = 0x7fffffff;
    auto scan = [&]() {
        best = 0;
        at = 0x7fffffff;
        for (int e = lane; e < E; e += 32)
            if (key[e] > best) { best = key[e]; at = e; }
    };
    scan();
    double z0 = 0.0;
    float my_w = 0.f, sum = 0.f;
    int my_i = 0;
    for (int j = 0; j < k; ++j) {
        const uint32_t hi = (uint32_t)(best >> 32), top = __reduce_max_sync(0xffffffffu, hi);
        const uint32_t lo = hi == top ? (uint32_t)best : 0u, low = __reduce_max_sync(0xffffffffu, lo);
        const int i = (int)__reduce_min_sync(0xffffffffu, hi == top && (uint32_t)best == low ? (uint32_t)at : 0x7fffffffu);
        const double z = key_logit(((unsigned long long)top << 32) | low);
        if (at == i) { key[i] = 0ull; scan(); }
        if (j == 0) z0 = z;
        const float pj = nan ? CUDART_NAN_F : expf((float)(z - z0));
        sum += pj;
        if (lane == j) { my_w = pj; my_i = i; }
    }
    if (lane < k) { idx[lane] = my_i; w[lane] = my_w / sum; }
}

// Sort keys of one token's logits into key [E]: sums of the slices, in order, for two experts at a time with eight loads each in
// flight (32 each take 1 us longer for the few slices of a narrow layer and gain nothing for wide ones).  Returns whether this
// thread saw a NaN.
__device__ __forceinline__ bool token_keys(const double *__restrict__ part, int slices, size_t stride, int E, unsigned long long *key) {
    bool nan = false;
    for (int e0 = threadIdx.x; e0 < E; e0 += 2 * blockDim.x) {
        const int e1 = e0 + blockDim.x < E ? e0 + blockDim.x : e0;
        double z[2] = {0.0, 0.0};
        for (int s0 = 0; s0 < slices; s0 += 8) {
            double v[2][8];
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const double *row = part + (size_t)(s0 + s) * stride;
                v[0][s] = s0 + s < slices ? row[e0] : 0.0;
                v[1][s] = s0 + s < slices ? row[e1] : 0.0;
            }
#pragma unroll
            for (int s = 0; s < 8; ++s) { z[0] += v[0][s]; z[1] += v[1][s]; }
        }
        key[e0] = logit_key(z[0]);
        key[e1] = logit_key(z[1]);               // the same expert again where there is no second one
        nan |= isnan(z[0]) || isnan(z[1]);
    }
    return nan;
}

// ---- the layer on CUDA cores: any type, any width ------------------------------------------------------------------------
__global__ void __launch_bounds__(128) route_kernel(const double *__restrict__ part, int slices, int32_t *__restrict__ idx,
                                                    float *__restrict__ w, int n_tok, int E, int k) {
    extern __shared__ unsigned long long s_key[];
    const int t = blockIdx.x;
    const bool nan = __syncthreads_or(token_keys(part + (size_t)t * E, slices, (size_t)n_tok * E, E, s_key));
    if (threadIdx.x < 32) topk_warp(s_key, E, k, nan, idx + (size_t)t * k, w + (size_t)t * k, threadIdx.x);
}

// Tokens (and the slots j of their choices) of expert e, in token order; expert E is the shared one (every token).
// Assignment (t, j) is row t k + j of the intermediate results, the shared expert's row of token t is n_tok k + t.
__device__ __forceinline__ int expert_rows(const int32_t *idx, int e, int E, int n_tok, int k, int *s_tok, int *s_row, int *s_n) {
    if (threadIdx.x == 0) *s_n = 0;
    __syncthreads();
    for (int t0 = 0; t0 < n_tok; t0 += 32) {                  // warp 0 walks the tokens in order
        if (threadIdx.x >= 32) break;
        const int t = t0 + threadIdx.x;
        int row = -1;
        if (t < n_tok) {
            if (e == E) row = n_tok * k + t;
            else for (int j = 0; j < k; ++j) if (idx[(size_t)t * k + j] == e) row = t * k + j;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, row >= 0);
        const int base = *s_n;
        if (row >= 0) {
            const int o = base + __popc(hit & ((1u << threadIdx.x) - 1));
            s_tok[o] = t;
            s_row[o] = row;
        }
        __syncwarp();
        if (threadIdx.x == 0) *s_n = base + __popc(hit);
        __syncwarp();
    }
    __syncthreads();
    return *s_n;
}

// Block: 64 output columns of one expert, four slices of the reduction, four tokens at a time.  Reads an expert's weights once per
// four of its tokens with two bytes per lane and load: bound by the latency of those loads (the layer at T = 1, d = 7168, E = 256,
// f = 2048 in bf16: 1.44 ms, 0.55 TB/s).
constexpr int SIMT_COLS = 64, SIMT_TOK = 4;

// UP: h[row, c] = silu(x W1) (x W3);  otherwise: y[row, c] = h W2
template <typename T, typename In, bool UP>
__global__ void __launch_bounds__(256) expert_kernel(const In *__restrict__ in, const T *__restrict__ Wa, const T *__restrict__ Wb,
                                                     const T *__restrict__ Sa, const T *__restrict__ Sb, float *__restrict__ out,
                                                     const int32_t *__restrict__ idx, int n_tok, int red, int cols, int E, int k) {
    __shared__ int s_tok[MAX_T], s_row[MAX_T], s_n;
    __shared__ float s_red[4][SIMT_COLS][2 * SIMT_TOK + 1];
    const int e = blockIdx.y;
    const int n = expert_rows(idx, e, E, n_tok, k, s_tok, s_row, &s_n);
    if (n == 0) return;
    const T *A = e == E ? Sa : Wa + (size_t)e * red * cols;
    const T *B = UP ? (e == E ? Sb : Wb + (size_t)e * red * cols) : nullptr;
    const int cl = threadIdx.x & (SIMT_COLS - 1), slice = threadIdx.x / SIMT_COLS, c = blockIdx.x * SIMT_COLS + cl;
    for (int g = 0; g < n; g += SIMT_TOK) {
        float a[SIMT_TOK] = {}, b[SIMT_TOK] = {};
        size_t src[SIMT_TOK];
#pragma unroll
        for (int j = 0; j < SIMT_TOK; ++j) {
            const int i = g + j < n ? g + j : g;
            src[j] = (size_t)(UP ? s_tok[i] : s_row[i]) * red;
        }
        if (c < cols) {
            for (int i = slice; i < red; i += 4) {
                const float wa = to_f32(A[(size_t)i * cols + c]);
                const float wb = UP ? to_f32(B[(size_t)i * cols + c]) : 0.f;
#pragma unroll
                for (int j = 0; j < SIMT_TOK; ++j) {
                    const float v = to_f32(in[src[j] + i]);
                    a[j] = fmaf(v, wa, a[j]);
                    if (UP) b[j] = fmaf(v, wb, b[j]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SIMT_TOK; ++j) { s_red[slice][cl][j] = a[j]; s_red[slice][cl][SIMT_TOK + j] = b[j]; }
        __syncthreads();
        // slice j of the threads finishes token g + j
        if (g + slice < n && c < cols) {
            float va = 0.f, vb = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) { va += s_red[s][cl][slice]; vb += s_red[s][cl][SIMT_TOK + slice]; }
            out[(size_t)s_row[g + slice] * cols + c] = UP ? silu(va) * vb : va;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const float *__restrict__ y, const float *__restrict__ w, T *__restrict__ out,
                                                  int n_tok, int d, int k, int shared) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)n_tok * d) return;
    const int t = (int)(i / d), c = (int)(i - (long long)t * d);
    float v = shared ? y[((size_t)n_tok * k + t) * d + c] : 0.f;
    for (int j = 0; j < k; ++j) v = fmaf(w[(size_t)t * k + j], y[((size_t)t * k + j) * d + c], v);
    out[i] = from_f32<T>(v);
}

// ---- workspace ---------------------------------------------------------------------------------------------------------
static inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
    size_t part, idx, w, h, y, total;
};
static Layout portable_layout(int n_tok, int d, int f, int E, int k, int shared) {
    Layout L{};
    size_t o = 0;
    const size_t rows = (size_t)n_tok * (k + shared);
    L.part = o; o += up256((size_t)gate_slices(n_tok, d, E) * n_tok * E * sizeof(double));
    L.idx = o;  o += up256((size_t)n_tok * k * 4);
    L.w = o;    o += up256((size_t)n_tok * k * 4);
    L.h = o;    o += up256(rows * f * 4);
    L.y = o;    o += up256(rows * d * 4);
    L.total = o;
    return L;
}

struct Args {
    const void *x; const float *Wg; const void *W1, *W3, *W2, *S1, *S3, *S2; void *out;
    int n_tok, d, f, E, k, shared;
};

template <typename T>
static int run_portable(const Args &a, uint8_t *ws, cudaStream_t s) {
    const Layout L = portable_layout(a.n_tok, a.d, a.f, a.E, a.k, a.shared);
    double *part = reinterpret_cast<double *>(ws + L.part);
    int32_t *idx = reinterpret_cast<int32_t *>(ws + L.idx);
    float *w = reinterpret_cast<float *>(ws + L.w), *h = reinterpret_cast<float *>(ws + L.h), *y = reinterpret_cast<float *>(ws + L.y);
    const int slices = gate_slices(a.n_tok, a.d, a.E);
    if (launch_gate<T>(a.x, a.Wg, part, nullptr, 0, a.n_tok, a.d, a.E, slices, s) != FDMLA_OK) return FDMLA_ERR_CUDA;
    route_kernel<<<a.n_tok, 128, a.E * sizeof(double), s>>>(part, slices, idx, w, a.n_tok, a.E, a.k);
    expert_kernel<T, T, true><<<dim3((a.f + SIMT_COLS - 1) / SIMT_COLS, a.E + a.shared), 256, 0, s>>>(
        static_cast<const T *>(a.x), static_cast<const T *>(a.W1), static_cast<const T *>(a.W3), static_cast<const T *>(a.S1),
        static_cast<const T *>(a.S3), h, idx, a.n_tok, a.d, a.f, a.E, a.k);
    expert_kernel<T, float, false><<<dim3((a.d + SIMT_COLS - 1) / SIMT_COLS, a.E + a.shared), 256, 0, s>>>(
        h, static_cast<const T *>(a.W2), nullptr, static_cast<const T *>(a.S2), nullptr, y, idx, a.n_tok, a.f, a.d, a.E, a.k);
    sum_kernel<T><<<(unsigned)(((long long)a.n_tok * a.d + 255) / 256), 256, 0, s>>>(y, w, static_cast<T *>(a.out), a.n_tok, a.d, a.k, a.shared);
    return check_launch();
}

}  // namespace few
}  // namespace fdmla

#include "moe_few_tc.cuh"

using namespace fdmla;

static bool few_shape_ok(int T, int d, int f, int E, int k) {
    return T <= few::MAX_T && k <= E && k <= 32 && E <= 2048 && d <= (1 << 20) && f <= (1 << 20);
}

extern "C" size_t fdmla_moe_few_workspace_bytes(int T, int d, int f, int E, int k, int shared, int dtype) {
    if (T <= 0 || d <= 0 || f <= 0 || E <= 0 || k <= 0 || !few_shape_ok(T, d, f, E, k)) return 0;
    // the larger of the two families' needs: which one runs also depends on fdmla_set_backend and on the pointers
    const size_t simt = few::portable_layout(T, d, f, E, k, shared != 0).total;
    if (!few::tc_supported(d, f, E, dtype)) return simt;
    const size_t tc = few::tc_layout(T, d, f, E, k, shared != 0).total;
    return tc > simt ? tc : simt;
}

extern "C" int fdmla_moe_few(const void *x, const float *Wg, const void *W1, const void *W3, const void *W2, const void *S1,
                             const void *S3, const void *S2, void *out, void *workspace, size_t workspace_bytes, int T, int d,
                             int f, int E, int k, int dtype, void *stream) {
    if (T < 0 || d <= 0 || f <= 0 || E <= 0 || k <= 0 || (dtype != FDMLA_F32 && dtype != FDMLA_BF16)) return FDMLA_ERR_INVALID;
    const int shared = S1 != nullptr;
    if (shared != (S3 != nullptr) || shared != (S2 != nullptr)) return FDMLA_ERR_INVALID;
    if (!few_shape_ok(T, d, f, E, k)) return FDMLA_ERR_UNSUPPORTED;
    if (T == 0) return FDMLA_OK;
    if (!x || !Wg || !W1 || !W3 || !W2 || !out) return FDMLA_ERR_INVALID;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
        workspace_bytes < fdmla_moe_few_workspace_bytes(T, d, f, E, k, shared, dtype)) return FDMLA_ERR_WORKSPACE;
    const few::Args a{x, Wg, W1, W3, W2, S1, S3, S2, out, T, d, f, E, k, shared};
    cudaStream_t s = (cudaStream_t)stream;
    const bool tc = few::tc_supported(d, f, E, dtype) && few::tc_aligned(a);
    if (fdmla_get_backend() == FDMLA_BACKEND_TENSOR && !tc) return FDMLA_ERR_UNSUPPORTED;
    if (tc && tensor_kernels_allowed()) {
        note_kernel("tcgen05");
        return few::run_tensor(a, static_cast<uint8_t *>(workspace), s);
    }
    note_kernel("portable");
    return dtype == FDMLA_F32 ? few::run_portable<float>(a, static_cast<uint8_t *>(workspace), s)
                              : few::run_portable<__nv_bfloat16>(a, static_cast<uint8_t *>(workspace), s);
}
