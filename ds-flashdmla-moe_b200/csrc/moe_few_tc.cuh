// The MoE layer for few tokens on the tensor cores: one persistent kernel behind the gate kernel (included by moe_few.cu).
//
// Everything is bound by reading the weights of the experts that won, so the weights are the M side of the products (128
// weight columns per tile) and the tokens the N side: an expert's weights pass through shared memory once, whatever the number
// of its tokens.
//   stage 1   D1 = W1_e^T x^T, D3 = W3_e^T x^T for all tokens of the call (16 .. 128 columns; no gather), of which the columns of
//             the tokens that chose e give rows of h = silu(D1) D3, rounded to bf16 because the MMAs take both operands in one
//             type (the result's relative error against 64 bits is 0.0024 instead of the 0.0017 of its own rounding)
//   stage 2   y^T = W2_e^T h_e^T over e's rows of h (groups of at most 64)
//   stage 3   out[t] = sum over t's choices of w y, plus the shared expert's y, rounded once
//
// Work is handed out in items, in the order in which they lie in memory (neighbouring CTAs read neighbouring columns of the same
// rows): the first by CTA number, the rest from a counter, because CTAs that read the same number of bytes finish up to a
// quarter apart.  A tile is cut along its reduction into `split` items when there are few tiles; the fp32 pieces are summed in order
// behind the next barrier, by all CTAs.  Grid barriers (cooperative launch: all CTAs are resident) stand behind the top-k and
// between the stages; ahead of stage 2 the producer warp fills its ring with weights and has the next ones brought into L2, so
// HBM does not idle.
//
// Warp 0 issues the copies, warp 1 the MMAs, warps 2-5 read the accumulators (thread = weight column).  All waits are bounded
// (codes 41-44 of fdmla_device_error_flag).
//
// Measured with the gate kernel, replayed from a CUDA graph, d = 7168, f = 2048, E = 256, top-8 and a shared expert: T = 1 147 us
// (793 MB, 5.4 TB/s), T = 128 3.34 ms (22.3 GB, 6.7 TB/s; 3.4 to 3.8 ms when several layers' weights take turns); d = 4096, f = 1024, E = 64: T = 1 62 us, T = 64 288 us (5.7 TB/s).
// A step that is not bandwidth: gate 6 us, top-k and tables 6 us, 2 us per grid barrier.
#pragma once

#include <type_traits>

namespace fdmla {

bool make_tensor_map_bf16(CUtensorMap *m, const void *base, long long rows, int cols, int box_rows);
bool make_tensor_map_bf16_chunked(CUtensorMap *m, const void *base, long long rows, int cols, int box_rows, int box_chunks);

namespace few {

constexpr int TC_THREADS = 192;
constexpr int A_BYTES = 2 * 128 * 64 * 2;             // 32 KB of weights a stage: W1 and W3 [64 x 128], or two steps of W2
constexpr int MAX_E = 2048;
enum { ERR_PRODUCER = 41, ERR_MMA = 42, ERR_EPILOGUE = 43, ERR_GRID = 44 };
__device__ int g_few_error = 0;

// NP: tokens of the call rounded up to the width of the MMA's N side in stage 1.  The ring takes 192 to 216 KB of shared memory;
// about 50 KB in flight per SM cover the latency of HBM at full bandwidth.
constexpr int GROUP = 64;                             // rows of h in one accumulator of stage 2
constexpr int QUEUE = 16;                             // items under way: at most 6 ring stages + 2 accumulators + 2
constexpr unsigned NO_ITEM = 0xffffffffu;
constexpr int N_COUNTERS = 6;

template <int NP> struct TcShared {                   // behind the ring
    static constexpr int ROWS = NP * 32, EXPERTS = ROWS < MAX_E ? ROWS : MAX_E;      // k <= 32
    uint64_t bars[2 * 6 + 4 + QUEUE];
    uint32_t tmem, queue[QUEUE], ahead[6], scan[16];
    int n_routed, n_groups, last, dead;
    int32_t idx[32];                                  // a single token's choices and their weights
    float w[32];
    uint16_t expert[EXPERTS];                         // routed experts, ascending
    uint16_t first[EXPERTS + 1];                      // their first rows of h
    uint16_t group[EXPERTS + 2 + ROWS / GROUP];       // routed expert (or n_routed: the shared one) | second group << 15
    uint16_t row[ROWS];                               // of every choice (t, j)
    uint8_t token[ROWS];                              // of every row of h
};
template <int NP> struct Cfg {
    static constexpr int GN = NP < GROUP ? NP : GROUP;
    static constexpr int B_BYTES = (NP > 2 * GN ? NP : 2 * GN) * 128;   // 64 activations of all tokens / 2 x 64 of a group
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = NP == 16 ? 6 : (NP == 32 ? 5 : 4);
    static constexpr int COLS = 4 * NP;               // tensor memory: two buffers of (D1, D3)
    static constexpr int SMEM = 1024 + STAGES * STAGE + (int)sizeof(TcShared<NP>);
    static_assert(SMEM <= kMaxSmemPerBlock, "shared memory overflow");
    static_assert(STAGES * STAGE >= 16384 + MAX_E * 18 + 2 * TcShared<NP>::ROWS, "the tables behind the top-k overflow the ring");
};

struct TcProblem {
    int n_tok, d, f, E, k, shared, slices;
    int ft, kc1, nt, fs;                              // 128-wide tiles of f, 64-deep steps of d, 128-wide tiles of d, 128-deep pairs of steps of f
    int split_cap, rows;                              // most items per tile that the scratch holds; rows of h
    const double *part;
    int32_t *idx;
    float *w;
    unsigned *bars, *next;                            // [4] grid barriers, [2] item counters: zero at launch
    __nv_bfloat16 *h;                                 // [rows, f], the shared expert's rows last
    float *pieces;                                    // stage 1: [split][rows][2][ft 128]; stage 2: y [split][rows][d]
    __nv_bfloat16 *out;
};

// Items of a stage: tiles x split, `per` units (ring stages) a tile.  About a dozen items per CTA even out the CTAs' speeds; an
// item has two units at least.
struct Items {
    unsigned per, split, total;
    __device__ __forceinline__ Items(unsigned tiles, unsigned per_, unsigned cap) : per(per_) {
        unsigned s = (12 * gridDim.x + tiles - 1) / tiles;
        s = min(min(s, cap), per / 2);
        split = max(s, 1u);
        total = tiles * split;
    }
    __device__ __forceinline__ unsigned begin(unsigned s) const { return per * s / split; }
};

__device__ __forceinline__ bool grid_wait(const unsigned *bar, unsigned n) {
    for (uint32_t it = 0; it < (8u << 20); ++it)
        if (ptx::ld_acquire_gpu(bar) >= n) return true;
    return false;
}

template <int NP, bool LAT>
__global__ void __launch_bounds__(TC_THREADS, 1)
layer_kernel(const TcProblem p, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmH,
             const __grid_constant__ CUtensorMap tmW1, const __grid_constant__ CUtensorMap tmW3, const __grid_constant__ CUtensorMap tmW2,
             const __grid_constant__ CUtensorMap tmS1, const __grid_constant__ CUtensorMap tmS3, const __grid_constant__ CUtensorMap tmS2) {
    using namespace ptx;
    using C = Cfg<NP>;
    constexpr int STAGES = C::STAGES, STAGE = C::STAGE;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    TcShared<NP> &sh = *reinterpret_cast<TcShared<NP> *>(ring + STAGES * STAGE);
    const uint32_t bar0 = smem_u32(sh.bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto ACC_FULL = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
    auto ACC_EMPTY = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
    auto QUEUED = [&](int q) { return bar0 + 8u * (2 * STAGES + 4 + q); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int choices = p.n_tok * p.k;

    if (tid == 0) {
        sh.dead = *reinterpret_cast<volatile int *>(&g_few_error) != 0;      // an earlier launch gave up a wait: do nothing
        for (int s = 0; s < STAGES; ++s) { mbar_init(FULL(s), 1); mbar_init(EMPTY(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(ACC_FULL(a), 1); mbar_init(ACC_EMPTY(a), 128); }
        for (int q = 0; q < QUEUE; ++q) mbar_init(QUEUED(q), 1);
        sh.last = 0;
        fence_mbar_init();
    }
    if (warp == 1) { tmem_alloc(smem_u32(&sh.tmem), C::COLS); tmem_relinquish(); }
    wait_for_primary();                                // the gate kernel's logits and zeroed counters

    // ---- top-k: a token per CTA, in shared memory that the ring uses later ---------------------------------------------------
    unsigned long long *s_key = reinterpret_cast<unsigned long long *>(ring);
    const bool single = p.n_tok == 1;                  // one token: every CTA for itself, no barrier
    for (int t = single ? 0 : blockIdx.x; t < p.n_tok; t += gridDim.x) {
        const bool nan = __syncthreads_or(token_keys(p.part + (size_t)t * p.E, p.slices, (size_t)p.n_tok * p.E, p.E, s_key));
        if (warp == 0) topk_warp(s_key, p.E, p.k, nan, single ? sh.idx : p.idx + (size_t)t * p.k, single ? sh.w : p.w + (size_t)t * p.k, lane);
        __syncthreads();
    }
    // which tokens chose an expert: a 128-bit mask each
    uint32_t(*s_mask)[4] = reinterpret_cast<uint32_t(*)[4]>(ring + 16384);
    uint16_t *s_first = reinterpret_cast<uint16_t *>(ring + 16384 + MAX_E * 16), *s_idx = s_first + MAX_E;
    if (!single)
        for (int i = tid; i < p.E * 4; i += TC_THREADS) (&s_mask[0][0])[i] = 0u;
    if (tid == 0 && !sh.dead && !single) {
        red_release_gpu(p.bars);
        if (!grid_wait(p.bars, gridDim.x)) { sh.dead = 1; atomicCAS(&g_few_error, 0, ERR_GRID); }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    const bool dead = sh.dead != 0;
    // ---- routed experts in ascending order, their rows of h in token order (the same in every CTA) -------------------------------
    if (single) {                                      // the winners' ranks, without masks
        if (tid < p.k) {
            const int e = sh.idx[tid];
            int r = 0;
            for (int j = 0; j < p.k; ++j) r += sh.idx[j] < e;
            sh.expert[r] = (uint16_t)e;
            sh.first[r] = sh.group[r] = sh.row[tid] = (uint16_t)r;
            sh.token[r] = 0;
        }
        if (tid == 0) {
            sh.first[p.k] = sh.group[p.k] = (uint16_t)p.k;             // the shared expert's group, if there is one
            sh.n_routed = p.k;
            sh.n_groups = p.k + p.shared;
        }
    } else {
        if (!dead)
            for (int i = tid; i < choices; i += TC_THREADS) {
                const int e = __ldcg(p.idx + i), t = i / p.k;
                s_idx[i] = (uint16_t)e;
                atomicOr(&s_mask[e][t >> 5], 1u << (t & 31));
            }
        __syncthreads();
        {   // a thread owns `per` neighbouring experts; prefix sums of (experts, groups) and rows over the block
            const int per = (p.E + TC_THREADS - 1) / TC_THREADS, e0 = min(tid * per, p.E), e1 = min(e0 + per, p.E);
            auto tokens = [&](int e) { return __popc(s_mask[e][0]) + __popc(s_mask[e][1]) + __popc(s_mask[e][2]) + __popc(s_mask[e][3]); };
            uint32_t cnt = 0, rows = 0;                    // experts | groups << 16
            for (int e = e0; e < e1; ++e) {
                const int n = tokens(e);
                cnt += (n > 0 ? 0x10001u : 0u) + (n > GROUP ? 0x10000u : 0u);
                rows += n;
            }
            uint32_t ci = cnt, ri = rows;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, o), ru = __shfl_up_sync(0xffffffffu, ri, o);
                if (lane >= o) { ci += cu; ri += ru; }
            }
            if (lane == 31) { sh.scan[warp] = ci; sh.scan[8 + warp] = ri; }
            __syncthreads();
            for (int v = 0; v < warp; ++v) { ci += sh.scan[v]; ri += sh.scan[8 + v]; }
            uint32_t c = ci - cnt, r = ri - rows;
            for (int e = e0; e < e1; ++e) {
                const int n = tokens(e);
                if (n == 0) continue;
                const uint32_t a = c & 0xffffu, g = c >> 16;
                sh.expert[a] = (uint16_t)e;
                sh.first[a] = s_first[e] = (uint16_t)r;
                sh.group[g] = (uint16_t)a;
                if (n > GROUP) sh.group[g + 1] = (uint16_t)(a | 0x8000);
                c += 0x10001u + (n > GROUP ? 0x10000u : 0u);
                r += n;
            }
            if (tid == TC_THREADS - 1) {
                int n_grp = ci >> 16;
                sh.n_routed = ci & 0xffffu;
                sh.first[sh.n_routed] = (uint16_t)ri;
                if (p.shared) {
                    sh.group[n_grp++] = (uint16_t)sh.n_routed;
                    if (p.n_tok > GROUP) sh.group[n_grp++] = (uint16_t)(sh.n_routed | 0x8000);
                }
                sh.n_groups = n_grp;
            }
        }
        __syncthreads();
        if (!dead)
            for (int i = tid; i < choices; i += TC_THREADS) {
                const int e = s_idx[i], t = i / p.k;
                int r = s_first[e];
                for (int q = 0; q < t >> 5; ++q) r += __popc(s_mask[e][q]);
                r += __popc(s_mask[e][t >> 5] & ((1u << (t & 31)) - 1u));
                sh.row[i] = (uint16_t)r;
                sh.token[r] = (uint8_t)t;
            }
    }
    fence_proxy_async_all();                           // the copies write where the masks were
    __syncthreads();
    const unsigned routed = sh.n_routed;
    const Items it1(max((routed + p.shared) * p.ft, 1u), p.kc1, p.split_cap), it2(max(sh.n_groups * p.nt, 1), p.fs, p.split_cap);
    const int f_steps = p.f / 64;
    // rows of h of routed expert a (a == routed: the shared expert), and of group g
    auto rows_of = [&](unsigned a, int &row0) {
        row0 = a < routed ? (int)sh.first[a] : choices;
        return (a < routed ? (int)sh.first[a + 1] : choices + p.n_tok) - row0;
    };
    // stage 1 begins with the shared expert: with several tokens its tiles take longest
    auto expert_of = [&](unsigned i) { return !p.shared ? i : (i == 0 ? routed : i - 1); };
    auto group_of = [&](unsigned g, unsigned &a, int &row0) {
        a = sh.group[g] & 0x7fff;
        const int skip = sh.group[g] >> 15 ? GROUP : 0, n = rows_of(a, row0) - skip;
        row0 += skip;
        return min(n, GROUP);
    };

    if (warp == 0) {
        // ================================ producer ================================
        const bool elected = elect_one();
        if (lane == 0) { prefetch_tmap(&tmX); prefetch_tmap(&tmW1); prefetch_tmap(&tmW3); prefetch_tmap(&tmW2); prefetch_tmap(&tmH); }
        bool ok = !dead;                               // the same in every lane: the lanes exchange values below
        int s = 0, use = 0, n_items = 0;
        // the next item is asked for while the current one is loaded; the counter's first answer is item gridDim.x
        auto ask = [&](int stage, unsigned taken) { return lane == 0 ? taken + atomicAdd(p.next + stage - 1, 1u) : 0u; };
        auto announce = [&](unsigned item) {
            if (lane == 0) {
                sh.queue[n_items % QUEUE] = item;
                mbar_arrive(QUEUED(n_items % QUEUE));
            }
            ++n_items;
        };
        unsigned ans = 0;
        for (unsigned item = blockIdx.x; ok && item < it1.total; item = __shfl_sync(0xffffffffu, ans, 0)) {
            ans = ask(1, gridDim.x);
            announce(item);
            const unsigned i = item % p.ft, q = item / p.ft, ks = q % it1.split, a = expert_of(q / it1.split);
            const bool own = a >= routed;
            const CUtensorMap *m1 = own ? &tmS1 : &tmW1, *m3 = own ? &tmS3 : &tmW3;
            const int row0 = own ? 0 : (int)sh.expert[a] * p.d;
            for (unsigned kc = it1.begin(ks); kc < it1.begin(ks + 1) && ok; ++kc) {
                if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(EMPTY(s), (use - 1) & 1));
                if (ok && elected) {
                    const uint32_t dst = smem_u32(ring + s * STAGE);
                    mbar_arrive_expect_tx(FULL(s), A_BYTES + NP * 128);
                    tma_load_3d(dst, m1, 0, row0 + (int)kc * 64, (int)i * 2, FULL(s));
                    tma_load_3d(dst + A_BYTES / 2, m3, 0, row0 + (int)kc * 64, (int)i * 2, FULL(s));
                    tma_load_2d(dst + A_BYTES, &tmX, (int)kc * 64, 0, FULL(s));
                }
                if (++s == STAGES) { s = 0; ++use; }
            }
        }
        announce(NO_ITEM);
        // stage 2: weights of the first units ahead of the barrier, their rows of h behind it
        auto weights = [&](unsigned a, unsigned j, unsigned c2, int n16, int slot) {
            const bool own = a >= routed;
            const int row0 = (own ? 0 : (int)sh.expert[a] * p.f) + (int)c2 * 128, nk = min(2, f_steps - 2 * (int)c2);
            const uint32_t dst = smem_u32(ring + slot * STAGE);
            mbar_arrive_expect_tx(FULL(slot), nk * (A_BYTES / 2 + n16 * 2048));
            for (int c = 0; c < nk; ++c)
                tma_load_3d(dst + c * (A_BYTES / 2), own ? &tmS2 : &tmW2, 0, row0 + c * 64, (int)j * 2, FULL(slot));
        };
        auto acts = [&](int row0, unsigned c2, int n16, int slot) {
            const uint32_t dst = smem_u32(ring + slot * STAGE) + A_BYTES;
            const int nk = min(2, f_steps - 2 * (int)c2);
            for (int c = 0; c < nk; ++c)
                for (int r = 0; r < n16; ++r)
                    tma_load_2d(dst + (c * n16 + r) * 2048, &tmH, (int)c2 * 128 + c * 64, row0 + 16 * r, FULL(slot));
        };
        int n_ahead = 0;
        bool open = false;                             // the barrier has been passed
        auto pass = [&]() {
            if (!grid_wait(p.bars + (it1.split > 1 ? 3 : 1), gridDim.x)) { ok = false; if (lane == 0 && !dead) atomicCAS(&g_few_error, 0, ERR_GRID); }
            ok = __all_sync(0xffffffffu, ok);
            fence_proxy_async_all();                   // h was written with ordinary stores
            if (ok && elected)
                for (int i = 0; i < n_ahead; ++i) {
                    const uint32_t v = sh.ahead[i];    // the i-th unit ahead: group | step << 12 | ring slot << 28
                    unsigned a;
                    int row0;
                    const int n = group_of(v & 0xfff, a, row0);
                    acts(row0, (v >> 12) & 0xffff, (n + 15) >> 4, v >> 28);
                }
            open = true;
        };
        // the first items go by CTA number, so that each CTA knows which weights to have brought into L2: about 6 units beyond
        // the ring's (29 MB in all; 16 were 1 to 2 us slower), a quarter of the work at most
        const unsigned units = max(it2.per / it2.split, 1u);
        const unsigned fixed = max(min(it2.total / (4 * gridDim.x), (STAGES + 6 + units - 1) / units), 1u);
        unsigned round = 0;
        auto prefetch = [&](unsigned item, unsigned skip) {
            const unsigned j = item % p.nt, q = item / p.nt, g = q / it2.split, ks = q - g * it2.split;
            unsigned a;
            int row0;
            group_of(g, a, row0);
            const bool own = a >= routed;
            for (unsigned c2 = it2.begin(ks) + skip; c2 < it2.begin(ks + 1); ++c2) {
                const int row = (own ? 0 : (int)sh.expert[a] * p.f) + (int)c2 * 128, nk = min(2, f_steps - 2 * (int)c2);
                for (int c = 0; c < nk; ++c) tma_prefetch_3d(own ? &tmS2 : &tmW2, 0, row + c * 64, (int)j * 2);
            }
        };
        for (unsigned item = blockIdx.x; ok && item < it2.total;) {
            const bool by_number = ++round < fixed;
            if (!by_number) ans = ask(2, fixed * gridDim.x);
            announce(item);
            const unsigned j = item % p.nt, q = item / p.nt, g = q / it2.split, ks = q - g * it2.split;
            unsigned a;
            int row0;
            const int n16 = (group_of(g, a, row0) + 15) >> 4;
            for (unsigned c2 = it2.begin(ks); c2 < it2.begin(ks + 1) && ok; ++c2) {
                if (!open && n_ahead == STAGES) {
                    if (elected) {
                        prefetch(item, c2 - it2.begin(ks));
                        for (unsigned r = round; r < fixed && blockIdx.x + r * gridDim.x < it2.total; ++r) prefetch(blockIdx.x + r * gridDim.x, 0);
                    }
                    __syncwarp();
                    pass();
                }
                if (ok && use > 0) ok = __all_sync(0xffffffffu, mbar_wait(EMPTY(s), (use - 1) & 1));
                if (ok && elected) {
                    weights(a, j, c2, n16, s);
                    if (open) acts(row0, c2, n16, s);
                    else sh.ahead[n_ahead] = g | (c2 << 12) | ((uint32_t)s << 28);
                }
                if (!open) ++n_ahead;
                if (++s == STAGES) { s = 0; ++use; }
            }
            item = by_number ? blockIdx.x + round * gridDim.x : __shfl_sync(0xffffffffu, ans, 0);
        }
        if (ok && !open) pass();
        announce(NO_ITEM);
        if (!ok && !dead && lane == 0) atomicCAS(&g_few_error, 0, ERR_PRODUCER);
        __syncwarp();
    } else if (warp == 1) {
        // ================================ MMA issuer ================================
        const bool elected = elect_one();
        bool ok = !dead;
        int s = 0, n_done = 0, n_items = 0;
        uint32_t ph = 0;
#pragma unroll 1
        for (int stage = 1; stage <= 2; ++stage) {
            for (;;) {
                ok = ok && mbar_wait(QUEUED(n_items % QUEUE), (n_items / QUEUE) & 1);
                if (!__all_sync(0xffffffffu, ok)) break;
                const unsigned item = *reinterpret_cast<volatile uint32_t *>(&sh.queue[n_items % QUEUE]);
                ++n_items;
                if (item == NO_ITEM) break;
                unsigned lo, hi;
                int n16 = NP / 16;
                if (stage == 1) {
                    const unsigned ks = item / p.ft % it1.split;
                    lo = it1.begin(ks); hi = it1.begin(ks + 1);
                } else {
                    const unsigned q = item / p.nt, g = q / it2.split, ks = q - g * it2.split;
                    unsigned a;
                    int row0;
                    n16 = (group_of(g, a, row0) + 15) >> 4;
                    lo = it2.begin(ks); hi = it2.begin(ks + 1);
                }
                const uint32_t idesc = make_idesc_bf16(128, 16 * n16, 1, 0);
                const int acc = n_done & 1;
                const uint32_t d0 = tmem + acc * 2 * NP;
                if (n_done >= 2) {
                    ok = mbar_wait(ACC_EMPTY(acc), ((n_done >> 1) - 1) & 1);
                    tc_fence_after_sync();
                }
                for (unsigned kc = lo; kc < hi; ++kc) {
                    ok = ok && mbar_wait(FULL(s), ph);
                    tc_fence_after_sync();
                    if (elected && ok) {
                        const uint32_t a = smem_u32(ring + s * STAGE), b = a + A_BYTES;
                        if (stage == 1) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint64_t db = make_smem_desc(b + k * 32, 16, 1024, kLayoutSw128);
                                mma_bf16_ss(d0, make_smem_desc(a + k * 2048, 8192, 1024, kLayoutSw128), db, idesc, kc != lo || k != 0);
                                mma_bf16_ss(d0 + NP, make_smem_desc(a + A_BYTES / 2 + k * 2048, 8192, 1024, kLayoutSw128), db, idesc, kc != lo || k != 0);
                            }
                        } else {
                            const int steps = min(2, f_steps - 2 * (int)kc);
                            for (int c = 0; c < steps; ++c)
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    mma_bf16_ss(d0, make_smem_desc(a + c * (A_BYTES / 2) + k * 2048, 8192, 1024, kLayoutSw128),
                                                make_smem_desc(b + c * n16 * 2048 + k * 32, 16, 1024, kLayoutSw128), idesc, kc != lo || c != 0 || k != 0);
                        }
                        mma_commit(EMPTY(s));
                        if (kc == hi - 1) mma_commit(ACC_FULL(acc));
                    }
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
                ++n_done;
            }
        }
        if (!ok && !dead && lane == 0) atomicCAS(&g_few_error, 0, ERR_MMA);
        __syncwarp();
    } else {
        // ================================ epilogue ================================
        const int L = (warp & 3) * 32 + lane;          // TMEM lane = weight column of the tile
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const size_t ld1 = (size_t)p.ft * 128, slab1 = (size_t)p.rows * 2 * ld1, slab2 = (size_t)p.rows * p.d;
        bool ok = !dead;
        int n_done = 0, n_items = 0;
#pragma unroll 1
        for (int stage = 1; stage <= 2; ++stage) {
            for (;;) {
                // every thread takes the same way through the named barriers, time-out or not
                ok = ok && mbar_wait(QUEUED(n_items % QUEUE), (n_items / QUEUE) & 1);
                named_bar_sync(1, 128);
                if (!ok) sh.last = -1;
                named_bar_sync(1, 128);
                if (sh.last == -1) { ok = false; break; }
                const unsigned item = *reinterpret_cast<volatile uint32_t *>(&sh.queue[n_items % QUEUE]);
                ++n_items;
                if (item == NO_ITEM) break;
                const int acc = n_done & 1;
                const uint32_t d0 = tmem + lane_base + acc * 2 * NP;
                const bool landed = __all_sync(0xffffffffu, mbar_wait(ACC_FULL(acc), (n_done >> 1) & 1));
                ok = ok && landed;
                tc_fence_after_sync();
                ++n_done;
                if (stage == 2) {
                    const unsigned j = item % p.nt, q = item / p.nt, g = q / it2.split, ks = q - g * it2.split;
                    unsigned a;
                    int row0;
                    const int n = group_of(g, a, row0), col = (int)j * 128 + L;
                    float *y = p.pieces + ks * slab2 + (size_t)row0 * p.d + col;
                    for (int c = 0; c < n && landed; c += 16) {
                        uint32_t v[16];
                        tmem_ld16(d0 + c, v);
                        tmem_wait_ld();
                        if (col < p.d)
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (c + i < n) y[(size_t)(c + i) * p.d] = __uint_as_float(v[i]);
                    }
                    tc_fence_before_sync();
                    mbar_arrive(ACC_EMPTY(acc));
                    continue;
                }
                const unsigned i1 = item % p.ft, q = item / p.ft, ks = q % it1.split, a = expert_of(q / it1.split);
                int row0;
                const int n = rows_of(a, row0), col = (int)i1 * 128 + L;
                float *piece = p.pieces + (size_t)row0 * 2 * ld1 + col;          // of split 0
                for (int r0 = 0; r0 < n && landed; r0 += 8) {
                    uint32_t v1[8], v3[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const int rr = min(r0 + r, n - 1), t = a < routed ? sh.token[row0 + rr] : rr;
                        tmem_ld1(d0 + t, v1[r]);
                        tmem_ld1(d0 + NP + t, v3[r]);
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        if (r0 + r >= n) break;
                        const float x1 = __uint_as_float(v1[r]), x3 = __uint_as_float(v3[r]);
                        if (it1.split > 1) {
                            float *o = piece + ks * slab1 + (size_t)(r0 + r) * 2 * ld1;
                            o[0] = x1;
                            o[ld1] = x3;
                        } else if (col < p.f) p.h[(size_t)(row0 + r0 + r) * p.f + col] = __float2bfloat16_rn(silu(x1) * x3);
                    }
                }
                tc_fence_before_sync();
                mbar_arrive(ACC_EMPTY(acc));
            }
            // h is read by bulk copies, the pieces and y by ordinary loads
            auto arrive = [&](int bar) {
                if (stage == 1) fence_proxy_async_all();
                named_bar_sync(1, 128);
                if (L == 0 && !dead) red_release_gpu(p.bars + bar);
            };
            arrive(stage);
            if (stage == 1 && it1.split > 1) {
                // tiles cut along their reduction: all CTAs sum the pieces, in order, and write h
                if (L == 0 && !dead && !grid_wait(p.bars + 1, gridDim.x)) atomicCAS(&g_few_error, 0, ERR_GRID);
                named_bar_sync(1, 128);
                // LAT (few rows of h): one column a thread and all its pieces in flight; otherwise four columns a thread.  Two
                // instantiations, because the first launch after other work waits for its instructions.
                const unsigned elems = dead ? 0u : (unsigned)p.rows * (unsigned)p.f, threads = gridDim.x * 128;
                if constexpr (LAT) {
                    for (unsigned u = blockIdx.x * 128 + L; u < elems; u += threads) {
                        const unsigned r = u / p.f, c = u - r * p.f;
                        const float *o = p.pieces + (size_t)r * 2 * ld1 + c;
                        float v1[16], v3[16], x1 = 0.f, x3 = 0.f;
#pragma unroll
                        for (unsigned z = 0; z < 16; ++z) {
                            v1[z] = z < it1.split ? __ldcg(o + z * slab1) : 0.f;
                            v3[z] = z < it1.split ? __ldcg(o + z * slab1 + ld1) : 0.f;
                        }
#pragma unroll
                        for (unsigned z = 0; z < 16; ++z) { x1 += v1[z]; x3 += v3[z]; }
                        p.h[u] = __float2bfloat16_rn(silu(x1) * x3);
                    }
                } else {
                    // two groups of four columns at a time, `threads` groups apart, four pieces of both in flight
                    for (unsigned u0 = (blockIdx.x * 128 + L) * 4; u0 < elems; u0 += threads * 8) {
                        float x1[2][4] = {}, x3[2][4] = {};
                        const float *o[2];
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const unsigned u = min(u0 + g * threads * 4, elems - 4), r = u / p.f, c = u - r * p.f;
                            o[g] = p.pieces + (size_t)r * 2 * ld1 + c;
                        }
                        for (unsigned z0 = 0; z0 < it1.split; z0 += 4) {
                            float4 v1[2][4], v3[2][4];
#pragma unroll
                            for (int g = 0; g < 2; ++g)
#pragma unroll
                                for (unsigned z = 0; z < 4; ++z) {
                                    const bool in = z0 + z < it1.split;
                                    const float *q = o[g] + (z0 + z) * slab1;
                                    v1[g][z] = in ? __ldcg(reinterpret_cast<const float4 *>(q)) : make_float4(0.f, 0.f, 0.f, 0.f);
                                    v3[g][z] = in ? __ldcg(reinterpret_cast<const float4 *>(q + ld1)) : make_float4(0.f, 0.f, 0.f, 0.f);
                                }
#pragma unroll
                            for (int g = 0; g < 2; ++g)
#pragma unroll
                                for (unsigned z = 0; z < 4; ++z) {
                                    x1[g][0] += v1[g][z].x; x1[g][1] += v1[g][z].y; x1[g][2] += v1[g][z].z; x1[g][3] += v1[g][z].w;
                                    x3[g][0] += v3[g][z].x; x3[g][1] += v3[g][z].y; x3[g][2] += v3[g][z].z; x3[g][3] += v3[g][z].w;
                                }
                        }
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const unsigned u = u0 + g * threads * 4;
                            if (u >= elems) break;
                            const __nv_bfloat162 lo = __floats2bfloat162_rn(silu(x1[g][0]) * x3[g][0], silu(x1[g][1]) * x3[g][1]),
                                                 hi = __floats2bfloat162_rn(silu(x1[g][2]) * x3[g][2], silu(x1[g][3]) * x3[g][3]);
                            *reinterpret_cast<uint2 *>(p.h + u) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                        }
                    }
                }
                arrive(3);
            }
        }
        if (!ok && !dead) atomicCAS(&g_few_error, 0, ERR_EPILOGUE);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) { tc_fence_after_sync(); tmem_dealloc(tmem, C::COLS); }
    // ---- stage 3: the weighted sum ------------------------------------------------------------------------------------------------
    if (tid == 0 && !dead && !grid_wait(p.bars + 2, gridDim.x)) atomicCAS(&g_few_error, 0, ERR_GRID);
    __syncthreads();
    if (dead) return;
    const size_t slab = (size_t)p.rows * p.d;
    const int n = p.k + p.shared;
    const long long threads = (long long)gridDim.x * TC_THREADS, me = (long long)blockIdx.x * TC_THREADS + tid;
    // V columns a thread, Z pieces each of nine choices (eight and the shared expert) in flight
    auto weighted_sum = [&](auto v_, auto z_) {
        constexpr int V = decltype(v_)::value, Z = decltype(z_)::value, J = 9;
        const int per_row = p.d / V;
        for (long long u = me; u < (long long)p.n_tok * per_row; u += threads) {
            const int t = (int)(u / per_row), c = (int)(u - (long long)t * per_row) * V;
            float sum[V] = {};
            for (int j0 = 0; j0 < n; j0 += J) {
                float y[J][V] = {}, g[J];
                for (unsigned z0 = 0; z0 < it2.split; z0 += Z) {
                    float v[J][Z][V];
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const bool in = j0 + j < n, own = j0 + j >= p.k;
                        const size_t row = !in ? 0 : own ? choices + t : sh.row[t * p.k + j0 + j];
                        const float *src = p.pieces + row * p.d + c;
                        if (z0 == 0) g[j] = !in || own ? 1.f : single ? sh.w[j0 + j] : __ldcg(p.w + (size_t)t * p.k + j0 + j);
#pragma unroll
                        for (unsigned z = 0; z < Z; ++z) {
                            const bool ld = in && z0 + z < it2.split;
                            if constexpr (V == 4) {
                                const float4 q = ld ? __ldcg(reinterpret_cast<const float4 *>(src + (z0 + z) * slab)) : make_float4(0.f, 0.f, 0.f, 0.f);
                                v[j][z][0] = q.x; v[j][z][1] = q.y; v[j][z][2] = q.z; v[j][z][3] = q.w;
                            } else v[j][z][0] = ld ? __ldcg(src + (z0 + z) * slab) : 0.f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int z = 0; z < Z; ++z)
#pragma unroll
                            for (int i = 0; i < V; ++i) y[j][i] += v[j][z][i];
                }
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (j0 + j < n)
#pragma unroll
                        for (int i = 0; i < V; ++i) sum[i] = fmaf(g[j], y[j][i], sum[i]);
            }
            __nv_bfloat16 *o = p.out + (size_t)t * p.d + c;
            if constexpr (V == 4) {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(sum[0], sum[1]), hi = __floats2bfloat162_rn(sum[2], sum[3]);
                *reinterpret_cast<uint2 *>(o) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
            } else *o = __float2bfloat16_rn(sum[0]);
        }
    };
    if constexpr (LAT) weighted_sum(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    else weighted_sum(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
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
    int rows, split_cap, grid;
};
static TcLayout tc_layout(int n_tok, int d, int f, int E, int k, int shared) {
    TcLayout L{};
    const int ft = (f + 127) / 128;
    L.grid = sm_count();
    L.rows = n_tok * (k + shared);
    // pieces cost 8 bytes per row and weight column and item; many rows come with many tiles, which need no cutting
    L.split_cap = 4608 / L.rows < 1 ? 1 : (4608 / L.rows > 16 ? 16 : 4608 / L.rows);
    const size_t wide = (size_t)2 * ft * 128 > (size_t)d ? (size_t)2 * ft * 128 : (size_t)d;
    size_t o = 0;
    L.part = o;     o += up256((size_t)gate_slices(n_tok, d, E) * n_tok * E * sizeof(double));
    L.idx = o;      o += up256((size_t)n_tok * k * 4);
    L.w = o;        o += up256((size_t)n_tok * k * 4);
    L.counters = o; o += up256(N_COUNTERS * 4);
    L.h = o;        o += up256((size_t)L.rows * f * 2);
    L.pieces = o;   o += up256((size_t)L.split_cap * L.rows * wide * 4);       // stage 1's are dead when stage 2's y are written
    L.total = o;
    return L;
}

static bool tc_supported(int d, int f, int E, int dtype) {
    return dtype == FDMLA_BF16 && d % 64 == 0 && f % 64 == 0 && (long long)E * d < (1LL << 31) && (long long)E * f < (1LL << 31) &&
           f <= (1 << 18) && (long long)(E + 1) * ((f + 127) / 128) * 16 < (1LL << 31) && (long long)(E + 66) * ((d + 127) / 128) * 16 < (1LL << 31);
}
static bool tc_aligned(const Args &a) {
    return ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.W1) | reinterpret_cast<uintptr_t>(a.W3) |
             reinterpret_cast<uintptr_t>(a.W2) | reinterpret_cast<uintptr_t>(a.S1) | reinterpret_cast<uintptr_t>(a.S3) |
             reinterpret_cast<uintptr_t>(a.S2)) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;
}

template <int NP, bool LAT>
static int launch_layer(const TcProblem &p, const Args &a, int grid, cudaStream_t s) {
    CUtensorMap tmX, tmH, tm[6];
    if (!make_tensor_map_bf16(&tmX, a.x, a.n_tok, a.d, NP) ||
        !make_tensor_map_bf16(&tmH, p.h, p.rows, a.f, 16)) return FDMLA_ERR_CUDA;
    const void *base[6] = {a.W1, a.W3, a.W2, a.S1, a.S3, a.S2};
    for (int i = 0; i < 6; ++i) {
        if (i >= 3 && !a.shared) { tm[i] = tm[i - 3]; continue; }
        const long long rows = (i % 3 == 2 ? a.f : a.d) * (long long)(i < 3 ? a.E : 1);
        if (!make_tensor_map_bf16_chunked(&tm[i], base[i], rows, i % 3 == 2 ? a.d : a.f, 64, 2)) return FDMLA_ERR_CUDA;
    }
    if (!allow_smem<layer_kernel<NP, LAT>>(Cfg<NP>::SMEM)) return FDMLA_ERR_CUDA;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = Cfg<NP>::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeCooperative;
    at[0].val.cooperative = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;     // set up while the gate kernel runs
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, layer_kernel<NP, LAT>, p, tmX, tmH, tm[0], tm[1], tm[2], tm[3], tm[4], tm[5]) != cudaSuccess) {
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
    p.bars = counters; p.next = counters + 4;
    p.rows = L.rows; p.split_cap = L.split_cap;
    p.h = reinterpret_cast<__nv_bfloat16 *>(ws + L.h);
    p.pieces = reinterpret_cast<float *>(ws + L.pieces);
    p.out = static_cast<__nv_bfloat16 *>(a.out);
    if (launch_gate<__nv_bfloat16>(a.x, a.Wg, part, counters, N_COUNTERS, a.n_tok, a.d, a.E, p.slices, s) != FDMLA_OK) return FDMLA_ERR_CUDA;
    // one column a thread in the sums of pieces while that is at most two rounds over the grid
    if (a.n_tok <= 16)
        return (long long)p.rows * a.f <= 256LL * L.grid ? launch_layer<16, true>(p, a, L.grid, s) : launch_layer<16, false>(p, a, L.grid, s);
    if (a.n_tok <= 32) return launch_layer<32, false>(p, a, L.grid, s);
    if (a.n_tok <= 64) return launch_layer<64, false>(p, a, L.grid, s);
    return launch_layer<128, false>(p, a, L.grid, s);
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
bool few_set_error(int code) { return cudaMemcpyToSymbol(few::g_few_error, &code, sizeof(int)) == cudaSuccess; }

}  // namespace fdmla
