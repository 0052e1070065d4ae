// Attention weight per cached row on the tensor cores (included by cache_weights.cu): bf16, d a multiple of 64 up to 576, pages
// a multiple of 64 rows.
//
// D = K Q^T with the keys as the M side: a thread of the epilogue owns one key and sums 2^(s - m) / l over the columns of its
// accumulator row in registers - no reduction between threads, no atomics between tiles.  Tiles are 256 keys x up to 256 query
// rows, computed by a pair of CTAs (cta_group::2): each CTA holds the accumulator rows of its own 128 keys, brings those keys
// and HALF of the query rows, so that 128 query rows x 576 take 74 KB instead of 147 and the ring beside them is deep enough to
// cover the latency of HBM (four slots of one CTA alone would hold 64 KB in flight).
//   ROWS = false  at most 256 query rows per sequence (a decode step): they stay in shared memory while the keys of the
//                 sequence stream past; a pair takes a contiguous run of tiles, at a change of sequence the queries are
//                 exchanged chunk by chunk as the last MMAs release them (all keys ahead of all queries cost 5 us a change).
//                 Bound by reading the rows once.
//   ROWS = true   more query rows (a prompt, a window of queries): a tile's keys stay and the query rows stream, 256 at a time (an
//                 MMA costs about 60 cycles to issue: with 128 the issue, not the MMA, bounds), the sums staying in registers; tiles are dealt out round robin and, when there are
//                 few, cut along the query rows into `splits` whose partial sums a second kernel adds in order.  Bound by the
//                 MMAs, 2 * 256 * 256 * d operations per step.
// Either way one operand is resident in chunks of 64 columns (RFULL / REMPTY per chunk) and the other one passes through the ring
// (FULL / EMPTY per slot, in chunks of 64 columns too).
//
// Warp 0 issues the copies, warp 1 (of the leader) the MMAs, warps 2-5 read the accumulators.  Waits are bounded (codes 51-53).
//
// Measured, replayed from a CUDA graph with the copy of weights in front: 128 sequences of 4096 keys, 128 heads 108 us (604 MB of
// rows at 6.6 TB/s inside the kernel); 32 queries of 128 heads over 5000 and 16384 keys 86 us (1.2 PFLOP/s, 66 % of the tensor
// cycles, 59 to 73 % by SM; a chunk of 64 columns takes 320 to 340 cycles where its MMAs need 256, with L2 at 18 % of its rate).
#pragma once

#include <atomic>

namespace fdmla {

bool make_tensor_map_bf16(CUtensorMap *m, const void *base, long long rows, int cols, int box_rows);

namespace cw {

constexpr int TC_THREADS = 192, KEYS = 256, QROWS = 256, MAX_CHUNKS = 9, MAX_SLOTS = 12;
constexpr int KEY_CHUNK = 128 * 128;                 // one CTA's 128 keys x 64 columns
enum { ERR_PRODUCER = 51, ERR_MMA = 52, ERR_EPILOGUE = 53 };
__device__ int g_acc_error = 0;

struct TcShared {                                    // in front of the operands
    uint64_t bars[2 * MAX_SLOTS + 2 * MAX_CHUNKS + 4];
    uint32_t tmem;
    int dead, b0, tile0, n_tiles, scan[TC_THREADS / 32];
    alignas(16) float2 ml[2][QROWS];                 // m log2(e) and 1 / l of the tile's query rows
    int last[2][QROWS];                              // last key each of them sees
    alignas(16) int left_out[2][4];                  // per epilogue warp: some of its rows see nothing (l <= 0)
};

struct TcProblem {
    AccProblem a;
    int chunks, n_cols;                              // d / 64; query rows of an accumulator (N of the MMA)
    int slots, slot_bytes, res_bytes;                // ring slots and their size; resident operand per chunk
    int splits, row_tiles;
    float *partial;                                  // [splits][B][max_pages page_size] when splits > 1
};

// One step of the resident operand's life: sequence b, resident operand set `item`, and the tiles that stream past it.
template <bool ROWS>
struct Walker {
    const TcProblem *q;
    int b, tile, left;                               // ROWS = false: next tile of the run, tiles left in it
    long long item, base;                            // ROWS = true: next item; items of the sequences before b
    int n, t0, count;                                // of the located piece: keys of b, first key, streaming steps
    int r_lo;                                        // ROWS = true: first row tile
    int split;
    __device__ __forceinline__ Walker(const TcProblem &p_, const TcShared &sh, int unit)
        : q(&p_), b(ROWS ? 0 : sh.b0), tile(sh.tile0), left(sh.n_tiles), item(unit), base(0), n(0), t0(0), count(0), r_lo(0), split(0) {}
    __device__ __forceinline__ bool next(int units) {
        const TcProblem &p = *q;
        if (ROWS) {
            for (; b < p.a.B; ++b) {
                n = p.a.pg.length(b);
                const long long mine = (long long)((n + KEYS - 1) / KEYS) * p.splits;
                if (item < base + mine) {
                    const int r = (int)(item - base), tl = r / p.splits;
                    split = r - tl * p.splits;
                    t0 = tl * KEYS;
                    r_lo = (int)((long long)p.row_tiles * split / p.splits);
                    count = (int)((long long)p.row_tiles * (split + 1) / p.splits) - r_lo;
                    item += units;
                    return true;
                }
                base += mine;
            }
            return false;
        }
        if (left == 0) return false;
        for (;; ++b, tile = 0) {
            n = p.a.pg.length(b);
            const int nt = (n + KEYS - 1) / KEYS;
            if (tile >= nt) continue;
            t0 = tile * KEYS;
            count = min(nt - tile, left);
            left -= count;
            tile += count;
            return true;
        }
    }
    // does row tile r see any key of the piece
    __device__ __forceinline__ bool sees(int r) const {
        const TcProblem &p = *q;
        if (!p.a.causal) return true;
        const int q0 = r * QROWS % p.a.Sq, q1 = min(q0 + min(QROWS, p.a.R - r * QROWS), p.a.Sq) - 1;
        const bool wraps = q0 + min(QROWS, p.a.R - r * QROWS) > p.a.Sq;
        return (wraps ? p.a.Sq - 1 : q1) + n - p.a.Sq >= t0;
    }
};

// 2^x to two units in the last place, 0 for results below the normal numbers
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool ROWS>
__global__ void __launch_bounds__(TC_THREADS, 1)
accumulate_kernel(const TcProblem p, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK) {
    using namespace ptx;
    extern __shared__ uint8_t smem_raw[];
    TcShared &sh = *reinterpret_cast<TcShared *>(smem_raw);
    uint8_t *res = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + sizeof(TcShared) + 1023) & ~uintptr_t(1023));
    uint8_t *ring = res + p.chunks * p.res_bytes;
    const uint32_t bar0 = smem_u32(sh.bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (MAX_SLOTS + s); };
    auto RFULL = [&](int c) { return bar0 + 8u * (2 * MAX_SLOTS + c); };
    auto REMPTY = [&](int c) { return bar0 + 8u * (2 * MAX_SLOTS + MAX_CHUNKS + c); };
    auto ACC_FULL = [&](int a) { return bar0 + 8u * (2 * MAX_SLOTS + 2 * MAX_CHUNKS + a); };
    auto ACC_EMPTY = [&](int a) { return bar0 + 8u * (2 * MAX_SLOTS + 2 * MAX_CHUNKS + 2 + a); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cluster_ctarank();
    const int unit = blockIdx.x >> 1, units = gridDim.x >> 1;
    const AccProblem &a = p.a;

    if (tid == 0) {
        sh.dead = *reinterpret_cast<volatile int *>(&g_acc_error) != 0;           // an earlier launch gave up a wait: do nothing
        for (int s = 0; s < MAX_SLOTS; ++s) { mbar_init(FULL(s), 1); mbar_init(EMPTY(s), 1); }
        for (int c = 0; c < MAX_CHUNKS; ++c) { mbar_init(RFULL(c), 1); mbar_init(REMPTY(c), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(ACC_FULL(i), 1); mbar_init(ACC_EMPTY(i), 2); }
        fence_mbar_init();
    }
    if (warp == 1) { tmem_alloc_2cta(smem_u32(&sh.tmem), 2 * QROWS); tmem_relinquish_2cta(); }
    if (!ROWS) {
        // this pair's run of tiles: every thread counts the tiles of a share of the sequences, the one whose share holds the
        // run's first tile finds it
        const int per = (a.B + TC_THREADS - 1) / TC_THREADS, lo = min(tid * per, a.B), hi = min(lo + per, a.B);
        int mine = 0;
        for (int b = lo; b < hi; ++b) mine += (a.pg.length(b) + KEYS - 1) / KEYS;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        if (lane == 31) sh.scan[warp] = incl;
        __syncthreads();
        int total = 0;
        for (int w = 0; w < TC_THREADS / 32; ++w) { if (w < warp) incl += sh.scan[w]; total += sh.scan[w]; }
        const int first = (int)((long long)total * unit / units), end = (int)((long long)total * (unit + 1) / units);
        if (tid == 0) { sh.n_tiles = end - first; sh.b0 = 0; sh.tile0 = 0; }
        __syncthreads();
        if (end > first && first >= incl - mine && first < incl) {
            int before = incl - mine, b = lo;
            for (;; ++b) {
                const int nt = (a.pg.length(b) + KEYS - 1) / KEYS;
                if (first < before + nt) break;
                before += nt;
            }
            sh.b0 = b;
            sh.tile0 = first - before;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();                                                          // the peer's barriers exist
    tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    const bool dead = ld_shared_cluster_u32(map_to_cta(smem_u32(&sh.dead), 0)) != 0;     // both CTAs take the leader's reading

    if (warp == 0) {
        // ================================ producer ================================
        const bool elected = elect_one();
        if (lane == 0) { prefetch_tmap(&tmQ); prefetch_tmap(&tmK); }
        const uint32_t full_lead = map_to_cta(FULL(0), 0), rfull_lead = map_to_cta(RFULL(0), 0);
        bool ok = !dead;
        int s = 0, use = 0, n_res = 0;
        // page of the 64 keys number `lane & 3` of a tile; only looked at (row_of) a tile later, so that nobody waits for the load
        auto page_of = [&](int b, int t0, int n) {
            const int t = min(t0 + 64 * (lane & 3), n - 1);
            return __ldg(a.pg.table + (size_t)b * a.pg.max_pages + t / a.pg.page_size);
        };
        // row in the pool of the tile's 64 keys number i; a bad page reads page 0
        auto row_of = [&](int page, int t0, int n, int i) {
            int pg = __shfl_sync(0xffffffffu, page, i);
            const int t = t0 + 64 * i;
            if (pg < 0 || pg >= a.pg.num_pages) {
                if (t < n) g_cache_error = ERR_PAGE;
                pg = 0;
            }
            return pg * a.pg.page_size + t % a.pg.page_size;
        };
        // this CTA's two blocks of 64 keys, columns 64 c .. + 63
        auto load_keys = [&](int r0, int r1, int halves, int c, uint32_t dst, uint32_t bar) {
            if (2 * rank < halves) tma_load_2d_pair(dst, &tmK, c * 64, r0, bar);
            if (2 * rank + 1 < halves) tma_load_2d_pair(dst + KEY_CHUNK / 2, &tmK, c * 64, r1, bar);
        };
        const int half_cols = p.n_cols / 2;
        auto visible = [&](const Walker<ROWS> &v) {
            if (!ROWS) return true;
            for (int i = 0; i < v.count; ++i)
                if (v.sees(v.r_lo + i)) return true;
            return false;
        };
        Walker<ROWS> w(p, sh, unit);
        bool more = w.next(units);
        // Each lane waits for itself, so a wait that gives up may do so in some lanes only: they agree here, before the branch, since
        // the lanes vote and exchange page ids inside.
        while ((ok = __all_sync(0xffffffffu, ok)) && more) {
            Walker<ROWS> after = w;                    // the set behind this one: its resident operand is brought into L2 meanwhile
            more = after.next(units);
            if (visible(w) && ok) {
                const int b = w.b;
                int page = page_of(b, w.t0, w.n), r0 = 0, r1 = 0;
                if (ROWS) { r0 = row_of(page, w.t0, w.n, 2 * rank); r1 = row_of(page, w.t0, w.n, 2 * rank + 1); }
                const int halves0 = min(4, (w.n - w.t0 + 63) / 64);
                int page_after = 0;
                if (ROWS && more) page_after = page_of(after.b, after.t0, after.n);
                bool first = true;
                for (int i = 0; i < w.count && ok; ++i) {
                    int halves = 0, q_row = 0;
                    if (ROWS) {
                        if (!w.sees(w.r_lo + i)) continue;
                        q_row = b * a.R + (w.r_lo + i) * QROWS + rank * half_cols;
                    } else {
                        const int t0 = w.t0 + i * KEYS;
                        r0 = row_of(page, t0, w.n, 2 * rank);
                        r1 = row_of(page, t0, w.n, 2 * rank + 1);
                        halves = min(4, (w.n - t0 + 63) / 64);
                        if (i + 1 < w.count) page = page_of(b, t0 + KEYS, w.n);          // the next tile's, ahead of time
                    }
                    for (int c = 0; c < p.chunks && ok; ++c) {
                        // chunk c of both operands is freed by the same MMAs of the previous set, and the first MMAs need chunk 0 of both
                        if (first) {
                            if (n_res > 0) ok = mbar_wait(REMPTY(c), (n_res - 1) & 1);
                            if (ok && elected) {
                                const uint32_t dst = smem_u32(res + c * p.res_bytes), bar = rfull_lead + 8u * c;
                                if (rank == 0) mbar_arrive_expect_tx(RFULL(c), ROWS ? halves0 * (KEY_CHUNK / 2) : p.n_cols * 128);
                                if (ROWS) load_keys(r0, r1, halves0, c, dst, bar);
                                else tma_load_2d_pair(dst, &tmQ, c * 64, b * a.R + rank * half_cols, bar);
                            }
                        }
                        if (use > 0) ok = ok && mbar_wait(EMPTY(s), (use - 1) & 1);
                        if (ok && elected) {
                            const uint32_t dst = smem_u32(ring + s * p.slot_bytes), bar = full_lead + 8u * s;
                            if (ROWS) {
                                if (rank == 0) mbar_arrive_expect_tx(FULL(s), p.n_cols * 128);
                                tma_load_2d_pair(dst, &tmQ, c * 64, q_row, bar);
                            } else {
                                if (rank == 0) mbar_arrive_expect_tx(FULL(s), halves * (KEY_CHUNK / 2));
                                load_keys(r0, r1, halves, c, dst, bar);
                            }
                        }
                        if (++s == p.slots) { s = 0; ++use; }
                    }
                    if (!ROWS || first) ok = __all_sync(0xffffffffu, ok);        // the lanes exchange page ids below
                    if (first && more) {
                        int n0 = 0, n1 = 0;
                        if (ROWS) { n0 = row_of(page_after, after.t0, after.n, 2 * rank); n1 = row_of(page_after, after.t0, after.n, 2 * rank + 1); }
                        if (elected)
                            for (int c = 0; c < p.chunks; ++c) {
                                if (ROWS) {
                                    tma_prefetch_2d(&tmK, c * 64, n0);
                                    tma_prefetch_2d(&tmK, c * 64, n1);
                                } else if (after.b != b) tma_prefetch_2d(&tmQ, c * 64, after.b * a.R + rank * half_cols);
                            }
                        __syncwarp();
                    }
                    first = false;
                }
                ++n_res;
            }
            w = after;
        }
        if (!ok && !dead && lane == 0) atomicCAS(&g_acc_error, 0, ERR_PRODUCER);
        __syncwarp();
    } else if (warp == 1) {
        // ================================ MMA issuer (the leader's) ================================
        const bool elected = elect_one();
        const uint32_t idesc = make_idesc_bf16(KEYS, p.n_cols, 0, 0);
        bool ok = !dead;
        int s = 0, n_done = 0, n_res = 0;
        uint32_t ph = 0;
        Walker<ROWS> w(p, sh, unit);
        while (rank == 0 && w.next(units)) {
            if (!__all_sync(0xffffffffu, ok)) break;
            int last = -1, first = -1;                                           // first and last step that runs
            for (int i = 0; i < w.count; ++i)
                if (!ROWS || w.sees(w.r_lo + i)) { last = i; if (first < 0) first = i; }
            if (last < 0) continue;
            for (int i = first; i <= last; ++i) {
                if (ROWS && !w.sees(w.r_lo + i)) continue;
                const int acc = n_done & 1;
                if (n_done >= 2) {
                    ok = ok && mbar_wait_cluster(ACC_EMPTY(acc), ((n_done >> 1) - 1) & 1);
                    tc_fence_after_sync();
                }
                for (int c = 0; c < p.chunks; ++c) {
                    if (i == first) ok = ok && mbar_wait(RFULL(c), n_res & 1);
                    ok = ok && mbar_wait(FULL(s), ph);
                    tc_fence_after_sync();
                    if (elected && ok) {
                        const uint32_t rc = smem_u32(res + c * p.res_bytes), sc = smem_u32(ring + s * p.slot_bytes);
                        const uint32_t keys = ROWS ? rc : sc, q = ROWS ? sc : rc;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_bf16_ss_2cta(tmem + acc * QROWS, make_smem_desc(keys + k * 32, 16, 1024, kLayoutSw128),
                                             make_smem_desc(q + k * 32, 16, 1024, kLayoutSw128), idesc, (c | k) != 0);
                        mma_commit_2cta(EMPTY(s), 3);
                        if (i == last) mma_commit_2cta(REMPTY(c), 3);
                        if (c == p.chunks - 1) mma_commit_2cta(ACC_FULL(acc), 3);
                    }
                    if (++s == p.slots) { s = 0; ph ^= 1; }
                }
                ++n_done;
            }
            ++n_res;
        }
        if (!ok && !dead && lane == 0) atomicCAS(&g_acc_error, 0, ERR_MMA);
        __syncwarp();
    } else {
        // ================================ epilogue ================================
        const int L = (warp & 3) * 32 + lane;                                    // accumulator row = key of this CTA
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t acc_empty_lead = map_to_cta(ACC_EMPTY(0), 0);
        bool ok = !dead;
        int n_done = 0;
        // thread L fetches m and l of rows L and L + 128 of the tile of query rows that starts at r0 (nobody waits for the loads
        // here) ...
        struct Stats { float m[2], l[2]; };
        auto fetch = [&](int b, int r0, Stats &st) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const size_t r = (size_t)b * a.R + min(r0 + L + 128 * i, a.R - 1);
                st.m[i] = __ldg(a.m + r);
                st.l[i] = __ldg(a.l + r);
            }
        };
        // ... and keeps, in shared memory, m log2(e), 1 / l and the last key the row sees.  A row that sees nothing gets (inf, 0):
        // every exponential of a finite score is 0.  Its scores need not be finite (a padded batch), so a tile with such a row is
        // summed with the comparison that leaves terms out instead of multiplying them by 0.
        auto keep = [&](int buf, int n, int r0, const Stats &st) {
            bool out = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = L + 128 * i, r = r0 + c;
                const bool seen = r < a.R && !(st.l[i] <= 0.f);
                sh.ml[buf][c] = seen ? make_float2(st.m[i] * 1.4426950408889634f, 1.f / st.l[i]) : make_float2(CUDART_INF_F, 0.f);
                sh.last[buf][c] = !seen ? -1 : (a.causal ? r % a.Sq + n - a.Sq : n - 1);
                out |= r < a.R && !seen;
            }
            out = __any_sync(0xffffffffu, out);
            if (lane == 0) sh.left_out[buf][warp & 3] = out;
        };
        auto some_left_out = [&](int buf) {
            const int4 o = *reinterpret_cast<const int4 *>(sh.left_out[buf]);
            return (o.x | o.y | o.z | o.w) != 0;
        };
        // sum over the columns 0 .. cols - 1 of an accumulator
        auto sum_tile = [&](int acc, int buf, int cols, int t, bool masked) {
            const uint32_t d0 = tmem + lane_base + acc * QROWS;
            float g0 = 0.f, g1 = 0.f;
#pragma unroll 1
            for (int c = 0; c < cols; c += 32) {
                uint32_t v[32];
                tmem_ld32(d0 + c, v);
                tmem_wait_ld();
                if (!masked && c + 32 <= cols) {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float4 q = *reinterpret_cast<const float4 *>(&sh.ml[buf][c + j]);
                        g0 = fmaf(ex2(fmaf(__uint_as_float(v[j]), a.scale_log2, -q.x)), q.y, g0);
                        g1 = fmaf(ex2(fmaf(__uint_as_float(v[j + 1]), a.scale_log2, -q.z)), q.w, g1);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float2 q = sh.ml[buf][c + j];
                        const float e = ex2(fmaf(__uint_as_float(v[j]), a.scale_log2, -q.x)) * q.y;
                        if (c + j < cols && t <= sh.last[buf][c + j]) g0 += e;
                    }
                }
            }
            return g0 + g1;
        };
        auto release = [&](int acc) {
            tc_fence_before_sync();
            named_bar_sync(1, 128);
            if (L == 0) mbar_arrive_cluster_relaxed(acc_empty_lead + 8u * acc);
        };
        auto add = [&](long long row, float g) {
            if (row >= 0) atomicAdd(a.weights + row, g);       // one addition per key; atomic in case sequences share a page
        };
        int buf = 0;
        Walker<ROWS> w(p, sh, unit);
        while (!dead && w.next(units)) {
            const int b = w.b, n = w.n;
            if (!ROWS) {
                Stats ml;
                fetch(b, 0, ml);
                buf ^= 1;
                keep(buf, n, 0, ml);
                named_bar_sync(1, 128);
                const bool some_out = some_left_out(buf);
                for (int i = 0; i < w.count; ++i) {
                    const int acc = n_done & 1, t = w.t0 + i * KEYS + rank * 128 + L;
                    const long long row = t < n ? a.pg.row(b, t) : -1;           // under the tile's copies and MMAs
                    ok = __all_sync(0xffffffffu, ok && mbar_wait(ACC_FULL(acc), (n_done >> 1) & 1));
                    tc_fence_after_sync();
                    ++n_done;
                    float g = 0.f;
                    if (ok) g = sum_tile(acc, buf, a.R, t, some_out || (a.causal && w.t0 + (i + 1) * KEYS > n - a.Sq + 1));
                    release(acc);
                    if (ok) add(row, g);
                }
            } else {
                Stats ml;
                int i = 0;
                auto skip = [&]() { while (i < w.count && !w.sees(w.r_lo + i)) ++i; };
                skip();
                if (i < w.count) fetch(b, (w.r_lo + i) * QROWS, ml);
                const int t = w.t0 + rank * 128 + L;
                float g = 0.f;
                while (i < w.count) {
                    const int r = w.r_lo + i, acc = n_done & 1;
                    buf ^= 1;                                                    // the other buffer's readers passed a barrier since
                    keep(buf, n, r * QROWS, ml);
                    named_bar_sync(1, 128);
                    ++i;
                    skip();
                    if (i < w.count) fetch(b, (w.r_lo + i) * QROWS, ml);         // under this tile's arithmetic
                    ok = __all_sync(0xffffffffu, ok && mbar_wait(ACC_FULL(acc), (n_done >> 1) & 1));
                    tc_fence_after_sync();
                    ++n_done;
                    if (ok) g += sum_tile(acc, buf, min(QROWS, a.R - r * QROWS), t,
                                          some_left_out(buf) || (a.causal && w.t0 + KEYS > n - a.Sq + 1));
                    release(acc);
                }
                if (!ok || t >= n) continue;
                if (p.splits == 1) add(a.pg.row(b, t), g);
                else p.partial[((size_t)w.split * a.B + b) * ((size_t)a.pg.max_pages * a.pg.page_size) + t] = g;
            }
        }
        if (!ok && !dead) atomicCAS(&g_acc_error, 0, ERR_EPILOGUE);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();                                        // neither CTA leaves while the pair can still touch its memory
    if (warp == 1) { tc_fence_after_sync(); tmem_dealloc_2cta(tmem, 2 * QROWS); }
}

// weights += the splits' partial sums, in order.  After a time-out (of the launch in front or an earlier one) the partial sums were
// not all written: nothing is added.
__global__ void __launch_bounds__(256) add_partials_kernel(const float *__restrict__ partial, float *__restrict__ weights, const Pages pg,
                                                           int B, int splits) {
    const int b = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
    const size_t cap = (size_t)pg.max_pages * pg.page_size;
    if (t >= pg.length(b) || *reinterpret_cast<volatile int *>(&g_acc_error) != 0) return;
    float g = 0.f;
    for (int s = 0; s < splits; ++s) g += partial[((size_t)s * B + b) * cap + t];
    const long long row = pg.row(b, t);
    if (row >= 0) atomicAdd(weights + row, g);
}

static bool accumulate_tc_supported(int B, long long R, int d, int page_size, int max_pages, int num_pages, int dtype) {
    if (((long long)page_size * max_pages / KEYS + 1) * B > 2147483647LL) return false;              // tiles are counted in 32 bits
    return dtype == FDMLA_BF16 && d % 64 == 0 && d <= 64 * MAX_CHUNKS && page_size % 64 == 0 && num_pages > 0 &&
           (long long)B * R + QROWS <= 2147483647LL;
}

// CTA pairs resident at once, one CTA per SM (cached per device); 0 if clusters of two cannot be launched
template <bool ROWS>
static int resident_pairs() {
    static std::atomic<int> cached[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    n = cached[dev].load(std::memory_order_relaxed);
    if (n != 0) return n > 0 ? n : 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * (kNumSMs / 2));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = kMaxSmemPerBlock;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(accumulate_kernel<ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmemPerBlock) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, accumulate_kernel<ROWS>, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = -1;
    }
    cached[dev].store(n, std::memory_order_relaxed);
    return n > 0 ? n : 0;
}

// Splits of the query rows: six items per pair if every sequence were as long as the page table allows.
static int row_splits(int B, long long R, long long cap) {
    const long long tiles = (cap + KEYS - 1) / KEYS * B, row_tiles = (R + QROWS - 1) / QROWS;
    if (row_tiles <= 1 || tiles <= 0) return 1;
    long long s = (6 * (kNumSMs / 2) + tiles - 1) / tiles;
    if (s > row_tiles) s = row_tiles;
    return (int)(s > 64 ? 64 : s);
}

template <bool ROWS>
static int launch_accumulate(TcProblem &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, cudaStream_t s) {
    constexpr int fixed = (int)sizeof(TcShared) + 1024;
    p.res_bytes = ROWS ? KEY_CHUNK : p.n_cols / 2 * 128;
    p.slot_bytes = ROWS ? p.n_cols / 2 * 128 : KEY_CHUNK;
    const int room = kMaxSmemPerBlock - fixed - p.chunks * p.res_bytes;
    p.slots = room / p.slot_bytes < MAX_SLOTS ? room / p.slot_bytes : MAX_SLOTS;
    const int smem = fixed + p.chunks * p.res_bytes + p.slots * p.slot_bytes;
    const int pairs = resident_pairs<ROWS>();
    if (pairs <= 0) return FDMLA_ERR_CUDA;
    const AccProblem &a = p.a;
    const long long tiles = ((long long)a.pg.max_pages * a.pg.page_size + KEYS - 1) / KEYS * a.B * p.splits;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, accumulate_kernel<ROWS>, p, tmQ, tmK) != cudaSuccess) { cudaGetLastError(); return FDMLA_ERR_CUDA; }
    if (p.splits > 1) {
        const dim3 grid((unsigned)(((long long)a.pg.max_pages * a.pg.page_size + 255) / 256), a.B);
        add_partials_kernel<<<grid, 256, 0, s>>>(p.partial, a.weights, a.pg, a.B, p.splits);
    }
    return check_launch();
}

static int run_accumulate_tc(const AccProblem &a, void *workspace, cudaStream_t s) {
    TcProblem p{};
    p.a = a;
    p.chunks = a.d / 64;
    p.row_tiles = (a.R + QROWS - 1) / QROWS;
    const bool rows = p.row_tiles > 1;
    p.n_cols = rows ? QROWS : (a.R + 31) / 32 * 32;                  // an M = 256 MMA takes N in steps of 32
    p.splits = row_splits(a.B, a.R, (long long)a.pg.max_pages * a.pg.page_size);
    p.partial = static_cast<float *>(workspace);
    CUtensorMap tmQ, tmK;
    if (!make_tensor_map_bf16(&tmQ, a.Q, (long long)a.B * a.R, a.d, p.n_cols / 2) ||
        !make_tensor_map_bf16(&tmK, a.pool, (long long)a.pg.num_pages * a.pg.page_size, a.d, 64)) return FDMLA_ERR_CUDA;
    return rows ? launch_accumulate<true>(p, tmQ, tmK, s) : launch_accumulate<false>(p, tmQ, tmK, s);
}

}  // namespace cw
}  // namespace fdmla
