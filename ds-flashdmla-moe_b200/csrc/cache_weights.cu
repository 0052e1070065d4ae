// A latent cache that may not grow: the attention weight every cached row has received, and the eviction of the rows that
// received least ("consume K_lat/V_lat from the KV-cache", README.md:15 of the reference, is all it says about the cache).
//
// Beside the pool [num_pages, page_size, d] stand weights [num_pages, page_size] fp32 and positions [num_pages, page_size]
// int32, addressed through the same page table:
//   accumulate:  weights[row of key t] += sum over the query rows r that see t of exp(scale q_r . k_t - m_r) / l_r
//                with the m, l that the attention of the same step returned
//   evict:       of a sequence with more than `keep` rows the newest stay (position >= next - recent), then the heaviest,
//                ties: the lower row.  Survivors in front of row `keep` do not move, the others fill the evicted rows'
//                places, both in ascending order, so as few rows as possible are copied and no copy reads what another
//                writes.  The attention does not depend on the order of the rows (their rotary part holds the position).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"
#include "ptx.cuh"

namespace fdmla {
namespace cw {

constexpr int ERR_PAGE = 4;                      // the code the attention kernels use for a bad page id or length
__device__ int g_cache_error = 0;

struct Pages {
    const int32_t *table;                        // [B, max_pages]
    const int32_t *seqlens;                      // [B]
    int page_size, max_pages, num_pages;
    __device__ __forceinline__ int length(int b) const {
        const int n = seqlens[b], cap = max_pages * page_size;
        if (n < 0 || n > cap) { g_cache_error = ERR_PAGE; return n < 0 ? 0 : cap; }
        return n;
    }
    // physical row of logical row t of sequence b, or -1
    __device__ __forceinline__ long long row(int b, int t) const {
        const int lp = t / page_size, pg = table[(size_t)b * max_pages + lp];
        if (pg < 0 || pg >= num_pages) { g_cache_error = ERR_PAGE; return -1; }
        return (long long)pg * page_size + (t - lp * page_size);
    }
};

struct AccProblem {
    const void *Q, *pool;                        // [B, R, d] with R = H Sq rows (row r is query r mod Sq), [num_pages, page_size, d]
    const float *m, *l;                          // [B, R]
    float *weights;                              // [num_pages, page_size]
    Pages pg;
    int B, R, Sq, d, causal;
    float scale_log2;                            // softmax scale times log2(e)
};

// ---- accumulate on CUDA cores: any type and width ---------------------------------------------------------------------------
// Block: 32 keys of one sequence (a lane owns a key, its row in shared memory) x all query rows, four rows per warp at a time.
// Bound by shared memory and the broadcast loads of the queries, five loads to four multiply-adds: 12.6 TFLOP/s in bf16 at
// 128 sequences of 4096 keys and 128 heads (6.15 ms).
constexpr int ACC_WARPS = 8, ACC_ROWS = 4;

template <typename T>
__global__ void __launch_bounds__(ACC_WARPS * 32) accumulate_simt_kernel(const AccProblem p) {
    extern __shared__ float s_k[];               // [32][d + 1], then [ACC_WARPS][32]
    const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = p.pg.length(b), t0 = blockIdx.x * 32, t = t0 + lane, ld = p.d + 1;
    if (t0 >= n) return;
    for (int j = warp; j < 32; j += ACC_WARPS) {
        const long long row = t0 + j < n ? p.pg.row(b, t0 + j) : -1;
        const T *src = static_cast<const T *>(p.pool) + row * p.d;
        for (int i = lane; i < p.d; i += 32) s_k[j * ld + i] = row >= 0 ? to_f32(src[i]) : 0.f;
    }
    __syncthreads();
    float got = 0.f;
    for (int r0 = warp * ACC_ROWS; r0 < p.R; r0 += ACC_WARPS * ACC_ROWS) {
        float s[ACC_ROWS] = {};
        const T *q[ACC_ROWS];
#pragma unroll
        for (int j = 0; j < ACC_ROWS; ++j)
            q[j] = static_cast<const T *>(p.Q) + ((size_t)b * p.R + (r0 + j < p.R ? r0 + j : r0)) * p.d;
        for (int i = 0; i < p.d; ++i) {
            const float k = s_k[lane * ld + i];
#pragma unroll
            for (int j = 0; j < ACC_ROWS; ++j) s[j] = fmaf(to_f32(q[j][i]), k, s[j]);
        }
#pragma unroll
        for (int j = 0; j < ACC_ROWS; ++j) {
            const int r = r0 + j;
            if (r >= p.R) break;
            const float l = p.l[(size_t)b * p.R + r], m = p.m[(size_t)b * p.R + r];
            const int last = p.causal ? r % p.Sq + n - p.Sq : n - 1;
            if (l <= 0.f || t > last) continue;            // a row without a visible key gives nothing
            got += exp2f(fmaf(s[j], p.scale_log2, -m * 1.4426950408889634f)) / l;
        }
    }
    __syncthreads();
    s_k[warp * 32 + lane] = got;
    __syncthreads();
    if (warp == 0 && t < n) {
        float sum = 0.f;
        for (int w = 0; w < ACC_WARPS; ++w) sum += s_k[w * 32 + lane];
        const long long row = p.pg.row(b, t);
        if (row >= 0) atomicAdd(p.weights + row, sum);     // one addition per key; atomic in case sequences share a page
    }
}

// ---- new rows: no weight yet, positions counted on ---------------------------------------------------------------------------
__global__ void __launch_bounds__(128) stamp_kernel(float *__restrict__ weights, int32_t *__restrict__ positions,
                                                    const int32_t *__restrict__ table, const int32_t *__restrict__ start,
                                                    const int32_t *__restrict__ first, int n_tokens, int page_size, int max_pages,
                                                    int num_pages) {
    const int b = blockIdx.y, t = blockIdx.x * 128 + threadIdx.x;
    if (t >= n_tokens) return;
    const long long pos = (long long)start[b] + t, lp = pos / page_size;
    if (pos < 0 || lp >= max_pages) return;
    const int pg = table[(size_t)b * max_pages + lp];
    if (pg < 0 || pg >= num_pages) { g_cache_error = ERR_PAGE; return; }
    const size_t row = (size_t)pg * page_size + (size_t)(pos - lp * page_size);
    weights[row] = 0.f;
    positions[row] = first[b] + t;
}

// ---- evict, part 1: which rows stay ------------------------------------------------------------------------------------------
// One cluster per sequence; CTA r holds the sort keys of its contiguous share of the rows in shared memory, read once.  The
// keep-th largest key comes from three rounds of 11-, 11- and 10-bit histograms summed over the cluster; the ranks of equal
// keys, evicted rows and moving rows from counts per warp (a warp owns a contiguous share of its CTA's rows).  A barrier of 16
// CTAs costs about 1 us, so there are five: a histogram of its own for every round (nobody waits before clearing one), the
// counts of equal keys from the last round's, evicted and moving rows counted together.  Reading all 2048 bins of 16 CTAs took
// 6 us a round; now every CTA reads their 64 sums of 32 bins, then the 32 bins of the one that matters: 131072 rows 40 -> 23 us.
// Bound by latency: 14 us for 128 sequences of 4096 rows (one CTA each: keys 3, rounds 3, ranks and lists 6).
constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32, BINS = 2048, MAX_CLUSTER = 16;
constexpr int MAX_SEG = 49152;                   // rows per CTA: 192 KB of keys

struct SelectProblem {
    const float *weights;
    const int32_t *positions;
    Pages pg;
    const int32_t *next;                         // [B] position of the next row to come
    int32_t *kept;                               // [B, keep]: the row that row j held before, -1 past the end
    int32_t *new_lens;                           // [B]
    int32_t *movers, *holes;                     // [B, cap] scratch each: rows that move and evicted rows they replace, in order
    int keep, recent, seg, cap;
};

__device__ __forceinline__ uint32_t sort_key(float w) {
    if (isnan(w)) return 0u;                     // below everything
    const uint32_t u = __float_as_uint(w + 0.f); // -0 counts as 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void cluster_barrier(int cs) {
    if (cs > 1) ptx::cluster_sync_all();
    else __syncthreads();
}

struct SelShared {
    uint32_t hist[3][BINS], coarse[3][BINS / 32];
    uint32_t part[MAX_CLUSTER][BINS / 32];
    uint32_t warp_n[3][SEL_WARPS + 1];           // per warp: equal keys, evicted rows, moving rows; then their prefix sums
    uint32_t cta_n[3];                           // of the whole CTA, read by the others
    uint32_t base[3];                            // of the CTAs before this one
    uint32_t total[3];                           // of the whole cluster
    uint32_t scan[SEL_WARPS], prefix, remaining, group;
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {              // inclusive, over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += u;
    }
    return v;
}
// count `c` per warp (in sh.warp_n[c]) -> exclusive prefix sums over the CTA's warps, and the CTA's total
__device__ __forceinline__ void warp_ranks(SelShared &sh, int c) {
    const int lane = threadIdx.x & 31;
    const uint32_t v = sh.warp_n[c][lane];
    const uint32_t incl = warp_scan(v);
    sh.warp_n[c][lane] = incl - v;
    if (lane == 31) sh.cta_n[c] = incl;
}
// by one warp: sum of *word over the first n CTAs of the cluster
__device__ __forceinline__ uint32_t sum_ctas(const uint32_t *word, int n) {
    const int lane = threadIdx.x & 31;
    uint32_t v = 0;
    if (lane < n) v = ptx::ld_shared_cluster_u32(ptx::map_to_cta(ptx::smem_u32(word), lane));
    return __reduce_add_sync(0xffffffffu, v);
}

__global__ void __launch_bounds__(SEL_THREADS, 1) select_kernel(const SelectProblem p, const int cs) {
    extern __shared__ uint32_t s_key[];
    __shared__ SelShared sh;
    ptx::launch_dependents();
    const int rank = cs > 1 ? (int)ptx::cluster_ctarank() : 0, b = blockIdx.x / cs;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = p.pg.length(b);
    int32_t *kept = p.kept + (size_t)b * p.keep;
    const int K = n < p.keep ? n : p.keep;
    for (int j = rank * SEL_THREADS + tid; j < p.keep; j += cs * SEL_THREADS) kept[j] = j < K ? j : -1;
    if (n <= p.keep) {                           // the whole cluster leaves: nothing goes
        if (rank == 0 && tid == 0) p.new_lens[b] = n;
        return;
    }

    const int lo = rank * p.seg < n ? rank * p.seg : n, hi = lo + p.seg < n ? lo + p.seg : n, rows = hi - lo;
    const int newest = p.next[b] - p.recent;
    // four rows a thread at a time: first their pages, then positions and weights, so that three latencies serve four rows
    const int32_t *table = p.pg.table + (size_t)b * p.pg.max_pages;
    for (int i0 = tid; i0 < rows; i0 += 4 * SEL_THREADS) {
        int pg[4], in_page[4], pos[4];
        float wt[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = lo + min(i0 + j * SEL_THREADS, rows - 1), lp = t / p.pg.page_size;
            pg[j] = __ldg(table + lp);
            in_page[j] = t - lp * p.pg.page_size;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (pg[j] < 0 || pg[j] >= p.pg.num_pages) { g_cache_error = ERR_PAGE; pg[j] = -1; }
            const size_t row = (size_t)max(pg[j], 0) * p.pg.page_size + in_page[j];
            pos[j] = pg[j] >= 0 ? __ldcg(p.positions + row) : 0;
            wt[j] = pg[j] >= 0 ? __ldcg(p.weights + row) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * SEL_THREADS;
            if (i < rows) s_key[i] = pg[j] < 0 ? 0u : (pos[j] >= newest ? 0xffffffffu : sort_key(wt[j]));
        }
    }
    if (tid == 0) { sh.prefix = 0u; sh.remaining = (uint32_t)K; }
    for (int i = tid; i < 3 * BINS; i += SEL_THREADS) (&sh.hist[0][0])[i] = 0u;

    // the K-th largest key, from the top digit down
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : (round == 1 ? 10 : 0), bits = round == 2 ? 10 : 11, bins = 1 << bits;
        uint32_t *hist = sh.hist[round];
        __syncthreads();
        const uint32_t prefix = sh.prefix, want = sh.remaining;
        for (int i = tid; i < rows; i += SEL_THREADS) {
            const uint32_t key = s_key[i];
            if (round == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
        if (cs == 1) {
            __syncthreads();
            // thread i owns two bins, from the top; the digit is where the running count reaches what is still to be taken
            const int hi_bin = bins - 1 - 2 * tid;
            const uint32_t c0 = hi_bin >= 1 ? hist[hi_bin] : 0u, c1 = hi_bin >= 1 ? hist[hi_bin - 1] : 0u;
            uint32_t incl = warp_scan(c0 + c1);
            if (lane == 31) sh.scan[warp] = incl;
            __syncthreads();
            incl += __reduce_add_sync(0xffffffffu, lane < warp ? sh.scan[lane] : 0u);
            const uint32_t before = incl - c0 - c1;
            if (before < want && want <= incl) {     // exactly one thread
                const bool first = before + c0 >= want;
                sh.prefix = (prefix << bits) | (uint32_t)(first ? hi_bin : hi_bin - 1);
                sh.remaining = want - before - (first ? 0u : c0);
            }
            continue;
        }
        // sums of 32 bins
        __syncthreads();
        const int groups = bins / 32;
        for (int g = warp; g < groups; g += SEL_WARPS) {
            const uint32_t n = __reduce_add_sync(0xffffffffu, hist[g * 32 + lane]);
            if (lane == 0) sh.coarse[round][g] = n;
        }
        cluster_barrier(cs);                     // every CTA's histogram stands
        {   // a thread per CTA and group
            const int r = tid >> 6, g = tid & 63;
            sh.part[r][g] = r < cs && g < groups ? ptx::ld_shared_cluster_u32(ptx::map_to_cta(ptx::smem_u32(&sh.coarse[round][g]), r)) : 0u;
        }
        __syncthreads();
        if (warp == 0) {                         // lane i owns the groups 63 - 2 i and 62 - 2 i
            uint32_t c0 = 0, c1 = 0;
            for (int r = 0; r < cs; ++r) { c0 += sh.part[r][63 - 2 * lane]; c1 += sh.part[r][62 - 2 * lane]; }
            const uint32_t incl = warp_scan(c0 + c1), before = incl - c0 - c1;
            if (before < want && want <= incl) {
                const bool first = before + c0 >= want;
                sh.group = 63 - 2 * lane - (first ? 0 : 1);
                sh.remaining = want - before - (first ? 0u : c0);
            }
        }
        __syncthreads();
        const uint32_t group = sh.group;
        if (tid < 32 * MAX_CLUSTER) {            // a thread per CTA and bin of the group
            const int r = tid >> 5;
            sh.part[r][lane] = r < cs ? ptx::ld_shared_cluster_u32(ptx::map_to_cta(ptx::smem_u32(&hist[group * 32 + lane]), r)) : 0u;
        }
        __syncthreads();
        if (warp == 0) {                         // lane i owns bin 31 - i of the group
            uint32_t c = 0;
            for (int r = 0; r < cs; ++r) c += sh.part[r][31 - lane];
            const uint32_t left = sh.remaining, incl = warp_scan(c);
            __syncwarp();
            if (incl - c < left && left <= incl) {
                sh.prefix = (prefix << bits) | (group * 32 + 31 - lane);
                sh.remaining = left - (incl - c);
            }
        }
    }
    __syncthreads();
    const uint32_t T = sh.prefix, take = sh.remaining;       // of the keys equal to T the first `take` rows stay

    // a warp owns rows [wlo, whi) of the CTA
    const int per = ((rows + SEL_WARPS - 1) / SEL_WARPS + 31) & ~31;
    const int wlo = warp * per < rows ? warp * per : rows, whi = wlo + per < rows ? wlo + per : rows;
    uint32_t cnt = 0;
    for (int i = wlo + lane; i < whi; i += 32) cnt += s_key[i] == T;
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) sh.warp_n[0][warp] = cnt;
    __syncthreads();
    if (warp == 0) warp_ranks(sh, 0);
    if (warp == 1) {                             // a CTA's keys equal to T: its count in the last round's histogram
        const uint32_t n = sum_ctas(&sh.hist[2][T & 1023u], rank);
        if (lane == 0) sh.base[0] = n;
    }
    __syncthreads();
    const uint32_t eq0 = sh.base[0] + sh.warp_n[0][warp];
    const uint32_t below = (1u << lane) - 1u;
    int32_t *movers = p.movers + (size_t)b * p.cap, *holes_at = p.holes + (size_t)b * p.cap;
    for (int pass = 0; pass < 2; ++pass) {       // 0: count, 1: list
        uint32_t eq = eq0;
        uint32_t holes = 0, moves = 0;
        if (pass > 0) { holes = sh.base[1] + sh.warp_n[1][warp]; moves = sh.base[2] + sh.warp_n[2][warp]; }
        for (int i0 = wlo; i0 < whi; i0 += 32) {
            const int i = i0 + lane, t = lo + i;
            const bool live = i < whi;
            const uint32_t key = live ? s_key[i] : 0u;
            const uint32_t eqs = __ballot_sync(0xffffffffu, live && key == T);
            const bool stays = live && (key > T || (key == T && eq + __popc(eqs & below) < take));
            const uint32_t hole = __ballot_sync(0xffffffffu, live && t < K && !stays);
            const uint32_t move = __ballot_sync(0xffffffffu, live && t >= K && stays);
            if (pass == 1 && ((move >> lane) & 1u)) movers[moves + __popc(move & below)] = t;
            if (pass == 1 && ((hole >> lane) & 1u)) holes_at[holes + __popc(hole & below)] = t;
            eq += __popc(eqs);
            holes += __popc(hole);
            moves += __popc(move);
        }
        if (pass == 0) {
            if (lane == 0) { sh.warp_n[1][warp] = holes; sh.warp_n[2][warp] = moves; }
            __syncthreads();
            if (warp < 2) warp_ranks(sh, 1 + warp);
            cluster_barrier(cs);
            if (warp < 2) {
                const uint32_t n = sum_ctas(&sh.cta_n[1 + warp], rank), all = sum_ctas(&sh.cta_n[1 + warp], cs);
                if (lane == 0) { sh.base[1 + warp] = n; sh.total[1 + warp] = all; }
            }
            __syncthreads();
        }
    }
    __threadfence();
    cluster_barrier(cs);                         // the lists stand; nobody leaves while its counts are read
    for (uint32_t r = rank * SEL_THREADS + tid; r < sh.total[1]; r += cs * SEL_THREADS) kept[__ldcg(holes_at + r)] = __ldcg(movers + r);
    if (rank == 0 && tid == 0) p.new_lens[b] = K;            // last: it may be the array the lengths were read from
}

// ---- evict, part 2: the copies -----------------------------------------------------------------------------------------------
// A warp takes `span` places (up to 32, fewer when there are few), reads what goes there (kept) and copies the rows that change
// place (5.8 TB/s read and written at 135 000 rows of 1152 bytes), two at a time with three vectors of each in flight per lane (a row of 1152 bytes is 72 vectors of 16; four rows at a
// time take more registers and were 5 % slower).  Rows are read and written once: streaming loads and stores.
template <typename V>
__global__ void __launch_bounds__(256) move_kernel(uint8_t *__restrict__ pool, float *__restrict__ weights,
                                                   int32_t *__restrict__ positions, const int32_t *kept, const Pages pg, int B, int keep,
                                                   int row_bytes, int span) {
    ptx::wait_for_primary();                     // kept is the select kernel's
    const int lane = threadIdx.x & 31;
    const int groups = (keep + span - 1) / span;
    const long long warps = (long long)gridDim.x * 8;
    const int vecs = row_bytes / (int)sizeof(V);
    for (long long g = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); g < (long long)B * groups; g += warps) {
        const int b = (int)(g / groups), j = (int)(g - (long long)b * groups) * span + lane;
        const int src = lane < span && j < keep ? __ldcg(kept + (size_t)b * keep + j) : -1;
        long long from = -1, to = -1;
        if (src >= 0 && src != j) {
            from = pg.row(b, src);
            to = pg.row(b, j);
        }
        const bool moves = from >= 0 && to >= 0;
        uint32_t todo = __ballot_sync(0xffffffffu, moves);
        while (todo) {
            const V *f[2];
            V *d[2];
            int n = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int a = todo ? __ffs(todo) - 1 : 0;
                const long long fr = __shfl_sync(0xffffffffu, from, a), tt = __shfl_sync(0xffffffffu, to, a);
                if (todo) { f[i] = reinterpret_cast<const V *>(pool + fr * row_bytes); d[i] = reinterpret_cast<V *>(pool + tt * row_bytes); ++n; }
                else { f[i] = f[0]; d[i] = d[0]; }
                todo &= todo - 1;
            }
            for (int v0 = lane; v0 < vecs; v0 += 96) {
                V x[2][3];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        if (i < n && v0 + 32 * q < vecs) x[i][q] = __ldcs(f[i] + v0 + 32 * q);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        if (i < n && v0 + 32 * q < vecs) __stcs(d[i] + v0 + 32 * q, x[i][q]);
            }
        }
        if (moves) {
            weights[to] = weights[from];
            positions[to] = positions[from];
        }
    }
}

}  // namespace cw

}  // namespace fdmla

#include "cache_weights_tc.cuh"

namespace fdmla {

int cache_error_flag(int reset) {
    int page = 0, wait = 0;
    if (cudaMemcpyFromSymbol(&page, cw::g_cache_error, sizeof(int)) != cudaSuccess ||
        cudaMemcpyFromSymbol(&wait, cw::g_acc_error, sizeof(int)) != cudaSuccess) return -1;
    if (reset && (page | wait)) {
        const int zero = 0;
        if (cudaMemcpyToSymbol(cw::g_cache_error, &zero, sizeof(int)) != cudaSuccess ||
            cudaMemcpyToSymbol(cw::g_acc_error, &zero, sizeof(int)) != cudaSuccess) return -1;
    }
    return wait ? wait : page;
}
bool cache_set_error(int code) { return cudaMemcpyToSymbol(cw::g_acc_error, &code, sizeof(int)) == cudaSuccess; }

}  // namespace fdmla

using namespace fdmla;

static bool pages_ok(int B, int page_size, int max_pages, int num_pages) {
    return B <= 65535 && (long long)page_size * max_pages <= 2147483647LL && (long long)page_size * num_pages <= 2147483647LL;
}

extern "C" size_t fdmla_cache_accumulate_workspace_bytes(int B, int H, int Sq, int d_qk, int page_size, int max_pages, int dtype) {
    if (B <= 0 || H <= 0 || Sq <= 0 || d_qk <= 0 || page_size <= 0 || max_pages <= 0) return 0;
    if (!cw::accumulate_tc_supported(B, (long long)H * Sq, d_qk, page_size, max_pages, 1, dtype)) return 0;
    const long long cap = (long long)page_size * max_pages;
    const int splits = cw::row_splits(B, (long long)H * Sq, cap);
    return splits > 1 ? (size_t)splits * B * cap * sizeof(float) : 0;
}

extern "C" int fdmla_cache_accumulate(const void *Q, const void *kv_pool, const int32_t *page_table, const int32_t *seqlens,
                                      const float *m, const float *l, float *weights, void *workspace, size_t workspace_bytes,
                                      int B, int H, int Sq, int d_qk, int page_size, int max_pages, int num_pages, float scale,
                                      int causal, int dtype, void *stream) {
    if (B < 0 || H < 0 || Sq < 0 || d_qk <= 0 || page_size <= 0 || max_pages < 0 || num_pages < 0) return FDMLA_ERR_INVALID;
    if (dtype != FDMLA_F32 && dtype != FDMLA_BF16) return FDMLA_ERR_INVALID;
    if (B == 0 || H == 0 || Sq == 0 || max_pages == 0) return FDMLA_OK;
    if (!Q || !kv_pool || !page_table || !seqlens || !m || !l || !weights) return FDMLA_ERR_INVALID;
    if (!pages_ok(B, page_size, max_pages, num_pages) || (long long)H * Sq > 2147483647LL) return FDMLA_ERR_UNSUPPORTED;
    if (workspace_bytes < fdmla_cache_accumulate_workspace_bytes(B, H, Sq, d_qk, page_size, max_pages, dtype)) return FDMLA_ERR_WORKSPACE;
    if (workspace_bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255))) return FDMLA_ERR_WORKSPACE;
    cw::AccProblem p{};
    p.Q = Q; p.pool = kv_pool; p.m = m; p.l = l; p.weights = weights;
    p.pg = cw::Pages{page_table, seqlens, page_size, max_pages, num_pages};
    p.B = B; p.R = H * Sq; p.Sq = Sq; p.d = d_qk; p.causal = causal ? 1 : 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    cudaStream_t s = (cudaStream_t)stream;
    const bool tc = cw::accumulate_tc_supported(B, p.R, d_qk, page_size, max_pages, num_pages, dtype) &&
                    ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(kv_pool)) & 15) == 0;
    if (fdmla_get_backend() == FDMLA_BACKEND_TENSOR && !tc) return FDMLA_ERR_UNSUPPORTED;
    if (tc && tensor_kernels_allowed()) {
        note_kernel("tcgen05");
        return cw::run_accumulate_tc(p, workspace, s);
    }
    note_kernel("portable");
    // the keys' rows, then the warps' sums in the same place (more than the rows for d < 7)
    const long long rows = 32LL * (d_qk + 1) * 4, sums = cw::ACC_WARPS * 32 * 4, smem = rows > sums ? rows : sums;
    if (smem > kMaxSmemPerBlock) return FDMLA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(((long long)max_pages * page_size + 31) / 32), B);
    if (!(dtype == FDMLA_F32 ? allow_smem<cw::accumulate_simt_kernel<float>>(kMaxSmemPerBlock)
                             : allow_smem<cw::accumulate_simt_kernel<__nv_bfloat16>>(kMaxSmemPerBlock))) return FDMLA_ERR_CUDA;
    if (dtype == FDMLA_F32) cw::accumulate_simt_kernel<float><<<grid, cw::ACC_WARPS * 32, (size_t)smem, s>>>(p);
    else cw::accumulate_simt_kernel<__nv_bfloat16><<<grid, cw::ACC_WARPS * 32, (size_t)smem, s>>>(p);
    return check_launch();
}

extern "C" int fdmla_cache_stamp(float *weights, int32_t *positions, const int32_t *page_table, const int32_t *start_pos,
                                 const int32_t *first_position, int B, int n_tokens, int page_size, int max_pages, int num_pages,
                                 void *stream) {
    if (B < 0 || n_tokens < 0 || page_size <= 0 || max_pages < 0 || num_pages < 0) return FDMLA_ERR_INVALID;
    if (B == 0 || n_tokens == 0) return FDMLA_OK;
    if (!weights || !positions || !page_table || !start_pos || !first_position) return FDMLA_ERR_INVALID;
    if (!pages_ok(B, page_size, max_pages, num_pages)) return FDMLA_ERR_UNSUPPORTED;
    cw::stamp_kernel<<<dim3((n_tokens + 127) / 128, B), 128, 0, (cudaStream_t)stream>>>(weights, positions, page_table, start_pos,
                                                                                       first_position, n_tokens, page_size, max_pages, num_pages);
    return check_launch();
}

extern "C" size_t fdmla_cache_evict_workspace_bytes(int B, int keep, int page_size, int max_pages) {
    if (B <= 0 || keep <= 0 || page_size <= 0 || max_pages <= 0) return 0;
    const long long cap = (long long)page_size * max_pages, movers = keep < cap ? keep : cap;
    return (size_t)2 * B * movers * sizeof(int32_t);
}

extern "C" int fdmla_cache_evict(void *kv_pool, float *weights, int32_t *positions, const int32_t *page_table,
                                 const int32_t *seqlens, const int32_t *next_position, int32_t *kept, int32_t *new_seqlens,
                                 void *workspace, size_t workspace_bytes, int B, int keep, int recent, int d_qk, int page_size,
                                 int max_pages, int num_pages, int dtype, void *stream) {
    if (B < 0 || keep <= 0 || recent < 0 || recent > keep || d_qk <= 0 || page_size <= 0 || max_pages < 0 || num_pages < 0) return FDMLA_ERR_INVALID;
    if (dtype != FDMLA_F32 && dtype != FDMLA_BF16) return FDMLA_ERR_INVALID;
    if (B == 0) return FDMLA_OK;
    if (!kv_pool || !weights || !positions || !page_table || !seqlens || !next_position || !kept || !new_seqlens) return FDMLA_ERR_INVALID;
    if (!pages_ok(B, page_size, max_pages, num_pages) || keep > (1 << 30)) return FDMLA_ERR_UNSUPPORTED;
    cudaStream_t s = (cudaStream_t)stream;
    const int cap = page_size * max_pages;
    if (cap > cw::MAX_CLUSTER * (cw::MAX_SEG - 32)) return FDMLA_ERR_UNSUPPORTED;
    // CTAs per sequence: enough for every SM as long as a CTA keeps a few thousand rows, and room for the keys of the longest
    int cs = 1;
    while (cs < cw::MAX_CLUSTER && ((cap + cs - 1) / cs > cw::MAX_SEG - 32 || ((long long)B * cs * 2 <= kNumSMs && cap / cs > 4096))) cs *= 2;
    const int seg = (((cap + cs - 1) / cs) + 31) & ~31;                       // at most MAX_SEG
    if (max_pages > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || workspace_bytes < fdmla_cache_evict_workspace_bytes(B, keep, page_size, max_pages))) return FDMLA_ERR_WORKSPACE;
    cw::SelectProblem p{};
    p.weights = weights; p.positions = positions;
    p.pg = cw::Pages{page_table, seqlens, page_size, max_pages, num_pages};
    p.next = next_position; p.kept = kept; p.new_lens = new_seqlens; p.movers = static_cast<int32_t *>(workspace);
    p.keep = keep; p.recent = recent; p.seg = seg; p.cap = keep < cap ? keep : cap;
    p.holes = p.movers + (size_t)B * p.cap;
    const size_t smem = (size_t)seg * 4;
    if (!allow_smem<cw::select_kernel>(cw::MAX_SEG * 4)) return FDMLA_ERR_CUDA;
    if (cs > 8 && cudaFuncSetAttribute(cw::select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return FDMLA_ERR_CUDA;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)B * cs);
    cfg.blockDim = dim3(cw::SEL_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cs; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, cw::select_kernel, p, cs) != cudaSuccess) { cudaGetLastError(); return FDMLA_ERR_CUDA; }
    if (cap <= keep) return check_launch();                   // no sequence can be over its bound
    const int row_bytes = d_qk * (dtype == FDMLA_F32 ? 4 : 2);
    // a warp per `span` places: few rows are spread over the SMs
    int span = 32;
    while (span > 4 && (long long)B * ((keep + span - 1) / span) < 4LL * 8 * kNumSMs) span /= 2;
    const long long warps = (long long)B * ((keep + span - 1) / span);
    const unsigned blocks = (unsigned)(warps > 8LL * 8 * kNumSMs ? 8 * kNumSMs : (warps + 7) / 8);
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;       // set up while the select kernel runs
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t mv{};
    mv.gridDim = dim3(blocks);
    mv.blockDim = dim3(256);
    mv.stream = s;
    mv.attrs = &pdl;
    mv.numAttrs = 1;
    uint8_t *pool = static_cast<uint8_t *>(kv_pool);
    const int32_t *k = kept;
    cudaError_t e;
    if (row_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(kv_pool) & 15) == 0)
        e = cudaLaunchKernelEx(&mv, cw::move_kernel<uint4>, pool, weights, positions, k, p.pg, B, keep, row_bytes, span);
    else if (row_bytes % 4 == 0 && (reinterpret_cast<uintptr_t>(kv_pool) & 3) == 0)
        e = cudaLaunchKernelEx(&mv, cw::move_kernel<unsigned int>, pool, weights, positions, k, p.pg, B, keep, row_bytes, span);
    else
        e = cudaLaunchKernelEx(&mv, cw::move_kernel<unsigned short>, pool, weights, positions, k, p.pg, B, keep, row_bytes, span);
    if (e != cudaSuccess) { cudaGetLastError(); return FDMLA_ERR_CUDA; }
    return check_launch();
}
