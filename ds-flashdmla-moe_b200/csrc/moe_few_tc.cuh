// The MoE layer for few tokens on the tensor cores: one persistent kernel behind the gate kernel (included by moe_few.cu).
//
// Everything is bound by reading the weights of the experts that won, so the weights are the M side of the products (128
// weight columns per tile) and ALL tokens of the call the N side (16 .. 128 columns): an expert's weights pass through shared
// memory once, whatever the number of its tokens, and a token that did not choose the expert costs a column of zeros, not a
// gather.
//   stage 1   D1 = W1_e^T x^T, D3 = W3_e^T x^T; h[e, t] = gate[t, e] silu(D1) D3, 0 for tokens that did not choose e
//   stage 2   out^T = sum_e W2_e^T h_e^T: one accumulator for all experts of the call (the shared expert is one more with gate
//             weight 1), so there is no scatter, no combine pass and one rounding of the result.  h carries the gate weight and
//             is rounded to bf16 for the tensor cores: a relative error of at most 2^-8 per element, as without the weight.
//
// The work of either stage is cut into equal contiguous runs of 64-deep steps, one run per CTA; a tile that two or more CTAs
// share is left as fp32 pieces in scratch and summed, piece by piece in order, by the CTA that finishes last (tickets; the
// result does not depend on who that is).  Grid barriers (cooperative launch: all CTAs are resident) stand behind the top-k and
// between the stages; the producer warp fills its ring with stage 2's weights before the second barrier, so HBM does not idle.
//
// Warp 0 issues the copies, warp 1 the MMAs, warps 2-5 read the accumulators (thread = weight column).  All waits are bounded
// (codes 41-44 of fdmla_device_error_flag).
#pragma once

namespace fdmla {

bool make_tensor_map_bf16(CUtensorMap *m, const void *base, long long rows, int cols, int box_rows);
bool make_tensor_map_bf16_chunked(CUtensorMap *m, const void *base, long long rows, int cols, int box_rows, int box_chunks);

namespace few {

constexpr int TC_THREADS = 192;
constexpr int A_BYTES = 2 * 128 * 64 * 2;             // 32 KB of weights a stage: W1 and W3 [64 x 128], or two steps of W2
constexpr int MAX_E = 2048;
enum { ERR_PRODUCER = 41, ERR_MMA = 42, ERR_EPILOGUE = 43, ERR_GRID = 44 };
__device__ int g_few_error = 0;

// NP: tokens of the call rounded up to the width of the MMA's N side.  The ring takes what shared memory has left: 196 to
// 216 KB; about 50 KB in flight per SM cover the latency of HBM at full bandwidth.
template <int NP> struct Cfg {
    static constexpr int B_STEP = NP * 128;           // 64 activations of every token
    static constexpr int STAGE = A_BYTES + 2 * B_STEP;
    static constexpr int STAGES = NP == 16 ? 6 : (NP == 32 ? 5 : (NP == 64 ? 4 : 3));
    static constexpr int COLS = 4 * NP;               // tensor memory: two buffers of (D1, D3)
    static constexpr int SMEM = 1024 + STAGES * STAGE + 6144;
    static_assert(SMEM <= kMaxSmemPerBlock, "shared memory overflow");
};

struct TcShared {                                     // behind the ring
    uint64_t bars[2 * 6 + 4];
    uint32_t tmem, bitmap[MAX_E / 32];
    int n_active, last, dead;
    float gate[MAX_T];
    uint16_t list[MAX_E];
};
static_assert(sizeof(TcShared) <= 6144, "TcShared outgrew its space");

struct TcProblem {
    int n_tok, d, f, E, k, shared, slices;
    int ft, kc1, nt, fs;                              // 128-wide tiles of f, 64-deep steps of d, 128-wide tiles of d, 128-deep pairs of steps of f
    const double *part;
    int32_t *idx;
    float *w;
    unsigned *bars, *tickets1, *tickets2;             // zero at launch
    __nv_bfloat16 *h;                                 // [active expert, token, f]
    float *pieces;                                    // [2 per CTA][2 n_tok][128]
    __nv_bfloat16 *out;
};

// One stage's work: `per` units (ring stages) a tile, units 0 .. total - 1 dealt out in contiguous runs to the first `ctas` CTAs.
struct Runs {
    unsigned total, per, ctas;
    __device__ __forceinline__ Runs(unsigned tiles, unsigned per_, unsigned grid) : total(tiles * per_), per(per_), ctas(grid < total ? grid : total) {}
    __device__ __forceinline__ unsigned start(unsigned c) const { return c >= ctas ? total : (unsigned)((unsigned long long)total * c / ctas); }
    __device__ __forceinline__ unsigned owner(unsigned u) const { return (unsigned)((((unsigned long long)u + 1) * ctas - 1) / total); }
};

__device__ __forceinline__ bool grid_wait(const unsigned *bar, unsigned n) {
    for (uint32_t it = 0; it < (16u << 20); ++it) {
        if (ptx::ld_acquire_gpu(bar) >= n) return true;
        __nanosleep(32);
    }
    return false;
}

template <int NP>
__global__ void __launch_bounds__(TC_THREADS, 1)
layer_kernel(const TcProblem p, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmH,
             const __grid_constant__ CUtensorMap tmW1, const __grid_constant__ CUtensorMap tmW3, const __grid_constant__ CUtensorMap tmW2,
             const __grid_constant__ CUtensorMap tmS1, const __grid_constant__ CUtensorMap tmS3, const __grid_constant__ CUtensorMap tmS2) {
    using namespace ptx;
    using C = Cfg<NP>;
    constexpr int STAGES = C::STAGES, STAGE = C::STAGE, B_STEP = C::B_STEP;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    TcShared &sh = *reinterpret_cast<TcShared *>(ring + STAGES * STAGE);
    const uint32_t bar0 = smem_u32(sh.bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto ACC_FULL = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
    auto ACC_EMPTY = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        sh.dead = *reinterpret_cast<volatile int *>(&g_few_error) != 0;      // an earlier launch gave up a wait: do nothing
        for (int s = 0; s < STAGES; ++s) { mbar_init(FULL(s), 1); mbar_init(EMPTY(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(ACC_FULL(a), 1); mbar_init(ACC_EMPTY(a), 128); }
        fence_mbar_init();
    }
    if (warp == 1) { tmem_alloc(smem_u32(&sh.tmem), C::COLS); tmem_relinquish(); }
    for (int i = tid; i < MAX_E / 32; i += TC_THREADS) sh.bitmap[i] = 0u;

    // ---- top-k: one token per CTA; the slices of its logits are summed in order, in shared memory that the ring uses later ----
    double *s_z = reinterpret_cast<double *>(ring);
    for (int t = blockIdx.x; t < p.n_tok; t += gridDim.x) {
        for (int e = tid; e < p.E; e += TC_THREADS) {
            double v = 0.0;
            for (int s = 0; s < p.slices; ++s) v += p.part[((size_t)s * p.n_tok + t) * p.E + e];
            s_z[e] = v;
        }
        __syncthreads();
        if (warp == 0) topk_warp(s_z, p.E, p.k, p.idx + (size_t)t * p.k, p.w + (size_t)t * p.k, lane);
        __syncthreads();
    }
    fence_proxy_async_all();
    __syncthreads();
    if (tid == 0 && !sh.dead) {
        __threadfence();
        atomicAdd(p.bars, 1u);
        if (!grid_wait(p.bars, gridDim.x)) { sh.dead = 1; atomicCAS(&g_few_error, 0, ERR_GRID); }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    const bool dead = sh.dead != 0;
    // ---- the experts that won, ascending; the shared one is the last ---------------------------------------------------------
    if (!dead)
        for (int i = tid; i < p.n_tok * p.k; i += TC_THREADS) {
            const int e = __ldcg(p.idx + i);
            atomicOr(&sh.bitmap[e >> 5], 1u << (e & 31));
        }
    __syncthreads();
    if (warp == 0) {
        uint32_t b0 = sh.bitmap[2 * lane], b1 = sh.bitmap[2 * lane + 1];
        const int n = __popc(b0) + __popc(b1);
        int at = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += u;
        }
        if (lane == 31) sh.n_active = at;
        at -= n;
        for (; b0; b0 &= b0 - 1) sh.list[at++] = (uint16_t)(64 * lane + __ffs(b0) - 1);
        for (; b1; b1 &= b1 - 1) sh.list[at++] = (uint16_t)(64 * lane + 32 + __ffs(b1) - 1);
    }
    __syncthreads();
    const unsigned routed = sh.n_active, active = routed + p.shared;
    const Runs r1(active * p.ft, p.kc1, gridDim.x), r2(p.nt, active * p.fs, gridDim.x);
    const unsigned cta = blockIdx.x;
    const unsigned u1_lo = dead ? 0 : r1.start(cta), u1_hi = dead ? 0 : r1.start(cta + 1);
    const unsigned u2_lo = dead ? 0 : r2.start(cta), u2_hi = dead ? 0 : r2.start(cta + 1);
    const int f_steps = p.f / 64;

    if (warp == 0) {
        // ================================ producer ================================
        const bool elected = elect_one();
        if (lane == 0) { prefetch_tmap(&tmX); prefetch_tmap(&tmW1); prefetch_tmap(&tmW3); prefetch_tmap(&tmW2); prefetch_tmap(&tmH); }
        bool ok = !dead;
        int s = 0, use = 0;
        for (unsigned u = u1_lo; u < u1_hi && ok;) {
            const unsigned tile = u / r1.per, a = tile / p.ft, i = tile - a * p.ft, k0 = u - tile * r1.per;
            const unsigned k1 = min(r1.per, k0 + (u1_hi - u));
            const bool own = a >= routed;
            const CUtensorMap *m1 = own ? &tmS1 : &tmW1, *m3 = own ? &tmS3 : &tmW3;
            const int row0 = own ? 0 : (int)sh.list[a] * p.d;
            for (unsigned kc = k0; kc < k1 && ok; ++kc) {
                if (use > 0) ok = mbar_wait(EMPTY(s), (use - 1) & 1);
                if (ok && elected) {
                    const uint32_t dst = smem_u32(ring + s * STAGE);
                    mbar_arrive_expect_tx(FULL(s), A_BYTES + B_STEP);
                    tma_load_3d(dst, m1, 0, row0 + (int)kc * 64, (int)i * 2, FULL(s));
                    tma_load_3d(dst + A_BYTES / 2, m3, 0, row0 + (int)kc * 64, (int)i * 2, FULL(s));
                    tma_load_2d(dst + A_BYTES, &tmX, (int)kc * 64, 0, FULL(s));
                }
                if (++s == STAGES) { s = 0; ++use; }
            }
            u += k1 - k0;
        }
        // stage 2: weights of the first units ahead of the barrier, the activations h behind it
        auto load = [&](unsigned u, int slot, bool weights, bool acts) {
            const unsigned j = u / r2.per, q = u - j * r2.per, a = q / p.fs, c2 = q - a * p.fs;
            const bool own = a >= routed;
            const int row0 = (own ? 0 : (int)sh.list[a] * p.f) + (int)c2 * 128;
            const int nk = min(2, f_steps - 2 * (int)c2);
            const uint32_t dst = smem_u32(ring + slot * STAGE);
            if (weights) {
                mbar_arrive_expect_tx(FULL(slot), nk * (A_BYTES / 2 + B_STEP));
                for (int c = 0; c < nk; ++c)
                    tma_load_3d(dst + c * (A_BYTES / 2), own ? &tmS2 : &tmW2, 0, row0 + c * 64, (int)j * 2, FULL(slot));
            }
            if (acts)
                for (int c = 0; c < nk; ++c)
                    tma_load_2d(dst + A_BYTES + c * B_STEP, &tmH, (int)c2 * 128 + c * 64, (int)a * p.n_tok, FULL(slot));
        };
        const unsigned ahead = min(u2_hi - u2_lo, (unsigned)STAGES);
        const int s_first = s;
        for (unsigned i = 0; i < ahead && ok; ++i) {
            if (use > 0) ok = mbar_wait(EMPTY(s), (use - 1) & 1);
            if (ok && elected) load(u2_lo + i, s, true, false);
            if (++s == STAGES) { s = 0; ++use; }
        }
        if (ok && !grid_wait(p.bars + 1, gridDim.x)) { ok = false; if (lane == 0) atomicCAS(&g_few_error, 0, ERR_GRID); }
        ok = __all_sync(0xffffffffu, ok);
        fence_proxy_async_all();                       // h was written with ordinary stores
        if (ok && elected)
            for (unsigned i = 0; i < ahead; ++i) load(u2_lo + i, (s_first + (int)i) % STAGES, false, true);
        for (unsigned u = u2_lo + ahead; u < u2_hi && ok; ++u) {
            ok = mbar_wait(EMPTY(s), (use - 1) & 1);
            if (ok && elected) load(u, s, true, true);
            if (++s == STAGES) { s = 0; ++use; }
        }
        if (!ok && !dead && lane == 0) atomicCAS(&g_few_error, 0, ERR_PRODUCER);
        __syncwarp();
    } else if (warp == 1) {
        // ================================ MMA issuer ================================
        const bool elected = elect_one();
        constexpr uint32_t idesc = make_idesc_bf16(128, NP, 1, 0);
        bool ok = !dead;
        int s = 0, n_done = 0;
        uint32_t ph = 0;
#pragma unroll 1
        for (int stage = 1; stage <= 2; ++stage) {
            const unsigned per = stage == 1 ? r1.per : r2.per, hi = stage == 1 ? u1_hi : u2_hi;
            for (unsigned u = stage == 1 ? u1_lo : u2_lo; u < hi;) {
                if (!__all_sync(0xffffffffu, ok)) break;
                const unsigned k0 = u % per, k1 = min(per, k0 + (hi - u));
                const int acc = n_done & 1;
                const uint32_t d0 = tmem + acc * 2 * NP;
                if (n_done >= 2) {
                    ok = mbar_wait(ACC_EMPTY(acc), ((n_done >> 1) - 1) & 1);
                    tc_fence_after_sync();
                }
                for (unsigned kc = k0; kc < k1; ++kc) {
                    ok = ok && mbar_wait(FULL(s), ph);
                    tc_fence_after_sync();
                    if (elected && ok) {
                        const uint32_t a = smem_u32(ring + s * STAGE), b = a + A_BYTES;
                        if (stage == 1) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint64_t db = make_smem_desc(b + k * 32, 16, 1024, kLayoutSw128);
                                mma_bf16_ss(d0, make_smem_desc(a + k * 2048, 8192, 1024, kLayoutSw128), db, idesc, kc != k0 || k != 0);
                                mma_bf16_ss(d0 + NP, make_smem_desc(a + A_BYTES / 2 + k * 2048, 8192, 1024, kLayoutSw128), db, idesc, kc != k0 || k != 0);
                            }
                        } else {
                            const int steps = min(2, f_steps - 2 * (int)(kc % p.fs));
                            for (int c = 0; c < steps; ++c)
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    mma_bf16_ss(d0, make_smem_desc(a + c * (A_BYTES / 2) + k * 2048, 8192, 1024, kLayoutSw128),
                                                make_smem_desc(b + c * B_STEP + k * 32, 16, 1024, kLayoutSw128), idesc, kc != k0 || c != 0 || k != 0);
                        }
                        mma_commit(EMPTY(s));
                        if (kc == k1 - 1) mma_commit(ACC_FULL(acc));
                    }
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
                ++n_done;
                u += k1 - k0;
            }
        }
        if (!ok && !dead && lane == 0) atomicCAS(&g_few_error, 0, ERR_MMA);
        __syncwarp();
    } else {
        // ================================ epilogue ================================
        const int L = (warp & 3) * 32 + lane;          // TMEM lane = weight column of the tile
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const int n_tok = p.n_tok;
        const size_t piece_floats = (size_t)2 * n_tok * 128;
        bool ok = !dead;
        int n_done = 0;
        // gate weight of every token for active expert a; negative: the token did not choose it
        auto set_gate = [&](unsigned a) {
            named_bar_sync(1, 128);                    // the table's previous readers are done
            if (L < n_tok) {
                float g = a >= routed ? 1.f : -1.f;
                if (a < routed) {
                    const int e = sh.list[a];
                    for (int j = 0; j < p.k; ++j)
                        if (__ldcg(p.idx + (size_t)L * p.k + j) == e) g = __ldcg(p.w + (size_t)L * p.k + j);
                }
                sh.gate[L] = g;
            }
            named_bar_sync(1, 128);
        };
        auto put_h = [&](unsigned a, int col, int t, float v1, float v3) {
            const float g = sh.gate[t];
            if (col < p.f) p.h[((size_t)a * n_tok + t) * p.f + col] = __float2bfloat16_rn(g < 0.f ? 0.f : g * silu(v1) * v3);
        };
        auto put_out = [&](int col, int t, float v) {
            if (col < p.d) p.out[(size_t)t * p.d + col] = __float2bfloat16_rn(v);
        };
#pragma unroll 1
        for (int stage = 1; stage <= 2; ++stage) {
            const Runs &r = stage == 1 ? r1 : r2;
            const unsigned lo = stage == 1 ? u1_lo : u2_lo, hi = stage == 1 ? u1_hi : u2_hi;
            for (unsigned u = lo; u < hi;) {
                const unsigned tile = u / r.per, k0 = u - tile * r.per, k1 = min(r.per, k0 + (hi - u));
                const unsigned a = stage == 1 ? tile / p.ft : 0;
                const int col = (int)(stage == 1 ? tile - a * p.ft : tile) * 128 + L;
                const bool whole = k1 - k0 == r.per;
                const int acc = n_done & 1;
                if (stage == 1 && whole) set_gate(a);
                if (ok) ok = mbar_wait(ACC_FULL(acc), (n_done >> 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after_sync();
                const uint32_t d0 = tmem + lane_base + acc * 2 * NP;
                float *piece = p.pieces + (2 * (size_t)cta + (tile == lo / r.per ? 0 : 1)) * piece_floats + L;
#pragma unroll 1
                for (int c = 0; c < NP && c < n_tok; c += 16) {
                    uint32_t v1[16], v3[16];
                    if (ok) {
                        tmem_ld16(d0 + c, v1);
                        if (stage == 1) tmem_ld16(d0 + NP + c, v3);
                        tmem_wait_ld();
                    }
                    if (!ok) continue;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int t = c + j;
                        if (t >= n_tok) continue;
                        const float x1 = __uint_as_float(v1[j]), x3 = __uint_as_float(v3[j]);
                        if (!whole) {
                            piece[(size_t)t * 128] = x1;
                            if (stage == 1) piece[(size_t)(n_tok + t) * 128] = x3;
                        } else if (stage == 1) put_h(a, col, t, x1, x3);
                        else put_out(col, t, x1);
                    }
                }
                tc_fence_before_sync();
                mbar_arrive(ACC_EMPTY(acc));
                ++n_done;
                u += k1 - k0;
                if (whole) continue;
                // a shared tile: whoever brings the last piece sums them all, in order
                __threadfence();
                named_bar_sync(1, 128);
                const unsigned c_lo = r.owner(tile * r.per), c_hi = r.owner(tile * r.per + r.per - 1);
                if (L == 0) sh.last = atomicAdd((stage == 1 ? p.tickets1 : p.tickets2) + tile, 1u) == c_hi - c_lo;
                named_bar_sync(1, 128);
                if (!sh.last) continue;
                __threadfence();
                if (stage == 1) set_gate(a);
                if (!ok) continue;
                // the first CTA's run reaches the tile after others unless it starts with it; the rest start inside it
                const float *first = p.pieces + (2 * (size_t)c_lo + (r.start(c_lo) / r.per == tile ? 0 : 1)) * piece_floats + L;
                for (int t = 0; t < n_tok; ++t) {
                    float x1 = __ldcg(first + (size_t)t * 128), x3 = stage == 1 ? __ldcg(first + (size_t)(n_tok + t) * 128) : 0.f;
#pragma unroll 4
                    for (unsigned c = c_lo + 1; c <= c_hi; ++c) {
                        const float *q = p.pieces + 2 * (size_t)c * piece_floats + L;
                        x1 += __ldcg(q + (size_t)t * 128);
                        if (stage == 1) x3 += __ldcg(q + (size_t)(n_tok + t) * 128);
                    }
                    if (stage == 1) put_h(a, col, t, x1, x3);
                    else put_out(col, t, x1);
                }
            }
            if (stage == 1) {
                fence_proxy_async_all();               // h is read by bulk copies
                __threadfence();
                named_bar_sync(1, 128);
                if (L == 0 && !dead) atomicAdd(p.bars + 1, 1u);
            }
        }
        if (!ok && !dead) atomicCAS(&g_few_error, 0, ERR_EPILOGUE);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) { tc_fence_after_sync(); tmem_dealloc(tmem, C::COLS); }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
static int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
        cudaGetLastError();
        sms = kNumSMs;
    }
    return sms;
}

struct TcLayout {
    size_t part, idx, w, counters, h, pieces, total;
    int n_counters, active_max, grid;
};
static TcLayout tc_layout(int n_tok, int d, int f, int E, int k, int shared) {
    TcLayout L{};
    L.grid = sm_count();
    L.active_max = (n_tok * k < E ? n_tok * k : E) + shared;
    L.n_counters = 2 + L.active_max * ((f + 127) / 128) + (d + 127) / 128;
    size_t o = 0;
    L.part = o;     o += up256((size_t)gate_slices(n_tok, d, E) * n_tok * E * sizeof(double));
    L.idx = o;      o += up256((size_t)n_tok * k * 4);
    L.w = o;        o += up256((size_t)n_tok * k * 4);
    L.counters = o; o += up256((size_t)L.n_counters * 4);
    L.h = o;        o += up256((size_t)L.active_max * n_tok * f * 2);
    L.pieces = o;   o += up256((size_t)2 * L.grid * 2 * n_tok * 128 * 4);
    L.total = o;
    return L;
}

static bool tc_supported(int d, int f, int E, int dtype) {
    return dtype == FDMLA_BF16 && d % 64 == 0 && f % 64 == 0 && (long long)E * d < (1LL << 31) && (long long)E * f < (1LL << 31) &&
           (long long)(E + 1) * ((f + 127) / 128) * (d / 64) < (1LL << 31) && (long long)(E + 1) * ((d + 127) / 128) * ((f + 127) / 128) < (1LL << 31);
}
static bool tc_aligned(const Args &a) {
    return ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.W1) | reinterpret_cast<uintptr_t>(a.W3) |
             reinterpret_cast<uintptr_t>(a.W2) | reinterpret_cast<uintptr_t>(a.S1) | reinterpret_cast<uintptr_t>(a.S3) |
             reinterpret_cast<uintptr_t>(a.S2)) & 15) == 0;
}

template <int NP>
static int launch_layer(const TcProblem &p, const Args &a, int grid, int active_max, cudaStream_t s) {
    CUtensorMap tmX, tmH, tm[6];
    if (!make_tensor_map_bf16(&tmX, a.x, a.n_tok, a.d, NP) ||
        !make_tensor_map_bf16(&tmH, p.h, (long long)active_max * a.n_tok, a.f, NP)) return FDMLA_ERR_CUDA;
    const void *base[6] = {a.W1, a.W3, a.W2, a.S1, a.S3, a.S2};
    for (int i = 0; i < 6; ++i) {
        if (i >= 3 && !a.shared) { tm[i] = tm[i - 3]; continue; }
        const long long rows = (i % 3 == 2 ? a.f : a.d) * (long long)(i < 3 ? a.E : 1);
        if (!make_tensor_map_bf16_chunked(&tm[i], base[i], rows, i % 3 == 2 ? a.d : a.f, 64, 2)) return FDMLA_ERR_CUDA;
    }
    if (cudaFuncSetAttribute(layer_kernel<NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NP>::SMEM) != cudaSuccess) {
        cudaGetLastError();
        return FDMLA_ERR_CUDA;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = Cfg<NP>::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeCooperative;
    at.val.cooperative = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, layer_kernel<NP>, p, tmX, tmH, tm[0], tm[1], tm[2], tm[3], tm[4], tm[5]) != cudaSuccess) {
        cudaGetLastError();
        return FDMLA_ERR_CUDA;
    }
    return check_launch();
}

static int run_tensor(const Args &a, uint8_t *ws, cudaStream_t s) {
    const TcLayout L = tc_layout(a.n_tok, a.d, a.f, a.E, a.k, a.shared);
    TcProblem p{};
    p.n_tok = a.n_tok; p.d = a.d; p.f = a.f; p.E = a.E; p.k = a.k; p.shared = a.shared;
    p.slices = gate_slices(a.n_tok, a.d, a.E);
    p.ft = (a.f + 127) / 128; p.kc1 = a.d / 64; p.nt = (a.d + 127) / 128; p.fs = (a.f + 127) / 128;
    double *part = reinterpret_cast<double *>(ws + L.part);
    unsigned *counters = reinterpret_cast<unsigned *>(ws + L.counters);
    p.part = part;
    p.idx = reinterpret_cast<int32_t *>(ws + L.idx);
    p.w = reinterpret_cast<float *>(ws + L.w);
    p.bars = counters; p.tickets1 = counters + 2; p.tickets2 = p.tickets1 + (size_t)L.active_max * p.ft;
    p.h = reinterpret_cast<__nv_bfloat16 *>(ws + L.h);
    p.pieces = reinterpret_cast<float *>(ws + L.pieces);
    p.out = static_cast<__nv_bfloat16 *>(a.out);
    gate_kernel<__nv_bfloat16><<<dim3((a.E + 31) / 32, p.slices, (a.n_tok + GATE_TOK - 1) / GATE_TOK), GATE_THREADS, 0, s>>>(
        static_cast<const __nv_bfloat16 *>(a.x), a.Wg, part, counters, L.n_counters, a.n_tok, a.d, a.E);
    if (check_launch() != FDMLA_OK) return FDMLA_ERR_CUDA;
    if (a.n_tok <= 16) return launch_layer<16>(p, a, L.grid, L.active_max, s);
    if (a.n_tok <= 32) return launch_layer<32>(p, a, L.grid, L.active_max, s);
    if (a.n_tok <= 64) return launch_layer<64>(p, a, L.grid, L.active_max, s);
    return launch_layer<128>(p, a, L.grid, L.active_max, s);
}

}  // namespace few

int few_error_flag(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, few::g_few_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && v != 0) {
        const int zero = 0;
        if (cudaMemcpyToSymbol(few::g_few_error, &zero, sizeof(int)) != cudaSuccess) return -1;
    }
    return v;
}

}  // namespace fdmla
