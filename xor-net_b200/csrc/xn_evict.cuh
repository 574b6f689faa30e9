// Eviction from a stream by accumulated attention weight: which positions stay, and their rows'
// move to the front.
//
// Per layer and KV head, of `len` positions: the last `recent` stay, and of the others the
// m = keep - recent with the largest account; of equal accounts the lowest position first; a NaN
// counts as lower than any number.  The kept positions keep their order.
#pragma once
#include "xn_common.cuh"
#include "xn_read.cuh"

namespace xn {

struct EvictDev {
    const int* pages;          // the stream's page table on the device
    int layer0, n_layers;      // layers [layer0, layer0 + n_layers)
    int acc_len;               // positions behind it have an account of zero (the same in all these layers)
    int len, keep, recent;
    int head0;                 // first (layer, KV head) row of this request among the launch's rows
    int copy;                  // 1: the rows go to k_out / v_out and the stream stays as it is;
                               // 0: they move to its front; 2: all of them stay where they are
    int* kept_ws;              // [n_layers][num_kv_heads][keep]
    int* kept;                 // the caller's copy, or nullptr
    float* k_out;
    float* v_out;
    float* w_out;              // the kept positions' accounts for the caller, or nullptr
};

// A launch's requests, as a kernel parameter.
constexpr int kEvictEntries = 24;
struct EvictTable {
    int n;
    int pad;
    EvictDev e[kEvictEntries];
};

namespace ev {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kCountMax = 512;     // candidates that are ranked by counting
constexpr int kMaxRun = 32;        // candidates of a thread whose keys are kept on chip

// Floats in the order of unsigned integers; NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (!(x == x)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* smem, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(smem)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t peer_ld(const void* smem, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_addr(smem, rank)) : "memory");
    return v;
}

__device__ __forceinline__ uint4 peer_ld4u(const void* smem, uint32_t rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(peer_addr(smem, rank))
                 : "memory");
    return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// The float behind a key; false where a key stands for several (NaNs, zeros).
__device__ __forceinline__ bool key_value(uint32_t k, float& x) {
    x = __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
    return k != 0u && k != 0x80000000u;
}

// Exclusive prefix of v over the block in thread order, and the block's total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* scratch, uint32_t& total) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) scratch[w] = inc;
    __syncthreads();
    const uint32_t mine = scratch[lane];   // 32 warps
    uint32_t winc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, winc, o);
        if (lane >= o) winc += up;
    }
    total = __shfl_sync(0xffffffffu, winc, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, winc - mine, w);
    __syncthreads();
    return before + inc - v;
}

}  // namespace ev

// One cluster of 1, 2, 4 or 8 blocks per (layer, KV head).  Thread t of block r owns the `run`
// candidates from (r * 1024 + t) * run on -- run is a power of two up to 32, so they share a page --
// and keeps their keys in its own row of shared memory: the account is read from memory once, 16
// bytes per load, and thread order is position order.  Radix selection: the threshold key is found
// 11, 11 and 10 bits at a time from histograms that the blocks read from one another (fewer steps when
// a bin is kept whole); then one scan of the (above, equal) counts gives every thread the place of its
// first kept position, ties included, and it writes its run.  Bound by the latency of these steps and
// by fetching instructions that run once, so the loops are rolled.  Measured: 64 rows of 8192 candidates
// 16 us, of which a pass takes 3500 to 5000 cycles (histogram 1700, the peers' bins 2400, scan 900); 8 rows
// of 131072 candidates 28 us; 5 of 268 (counted) with the copy 8.5 us.  (The peers' bins by way of sums over
// 32 of them, read by one warp: 900 cycles less per pass with eight blocks, 1300 more with one or two.)
// Streams too long for that (run = 0) read their keys again in every pass.
__global__ void __launch_bounds__(ev::kThreads, 1)
evict_select_kernel(const __grid_constant__ EvictTable tab, const float* __restrict__ pool, long long pool_pages,
                    int num_kv_heads, int cluster, int run_or_0) {
    using namespace ev;
    pdl_launch_dependents();
    extern __shared__ __align__(16) uint32_t keys_s[];   // [1024][run + 1]
    __shared__ __align__(16) uint32_t hist[2][kBins];   // by pass parity: peers may still read the other one
    __shared__ uint32_t scratch[32];
    __shared__ uint32_t counts[2];                  // this block's candidates above / at the threshold
    __shared__ uint32_t found[3];
    const int row = int(blockIdx.x) / cluster;
    const uint32_t rank = cluster_rank();
    int rq = 0;
    while (rq + 1 < tab.n && row >= tab.e[rq + 1].head0) ++rq;
    const EvictDev& r = tab.e[rq];
    const int local = row - r.head0;
    const int l = r.layer0 + local / num_kv_heads, h = local % num_kv_heads;
    const int tid = threadIdx.x, lane = tid & 31;
    const int n_cand = r.len - r.recent;
    const int m = r.keep - r.recent;                // candidates to keep, 0 <= m <= n_cand
    // positions [lo, hi) are this thread's
    const int run = run_or_0 ? run_or_0 : (((n_cand + cluster * kThreads - 1) / (cluster * kThreads)) + 3) / 4 * 4;
    const int lo = int(min((long long)(int(rank) * kThreads + tid) * run, (long long)n_cand)), hi = min(n_cand, lo + run);
    const int* pages = r.pages;
    const int valid = r.acc_len;
    const float* base = pool + (size_t(l) * size_t(pool_pages) * num_kv_heads + h) * kPageTokens;
    const int page_step = num_kv_heads * kPageTokens;
    auto load = [&](int j) -> float {
        return j < valid ? base[(long long)pages[j / kPageTokens] * page_step + j % kPageTokens] : 0.f;
    };
    uint32_t* mine = keys_s + tid * (run + 1);
    pdl_wait();
    int* kept = r.kept_ws + size_t(local) * r.keep;
    int* kept_user = r.kept ? r.kept + size_t(local) * r.keep : nullptr;
    float* w_user = r.w_out ? r.w_out + size_t(local) * r.keep : nullptr;
    auto emit = [&](uint32_t at, int j, uint32_t key) {
        kept[at] = j;
        if (kept_user) kept_user[at] = j;
        float x;
        if (w_user) w_user[at] = key_value(key, x) ? x : load(j);
    };
    if (n_cand <= kCountMax) {   // (one block then)
        // Few candidates: thread j counts those that go before candidate j -- a third of the radix passes'
        // time at 300 of them, as much at 1000.
        if (rank != 0) return;   // (a cluster that another row's length asked for)
        const uint32_t k = tid < n_cand ? order_key(load(tid)) : 0u;
        if (tid < kCountMax) keys_s[tid] = k;
        __syncthreads();
        int before = 0;
        if (tid < n_cand) {
            int j = 0;
#pragma unroll 2
            for (; j + 4 <= tid; j += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(&keys_s[j]);
                before += (x.x >= k) + (x.y >= k) + (x.z >= k) + (x.w >= k);
            }
            for (; j < tid; ++j) before += keys_s[j] >= k;
            for (; j < n_cand && (j & 3); ++j) before += keys_s[j] > k;
#pragma unroll 2
            for (; j < n_cand; j += 4) {   // (keys behind the last candidate are 0: above nothing)
                const uint4 x = *reinterpret_cast<const uint4*>(&keys_s[j]);
                before += (x.x > k) + (x.y > k) + (x.z > k) + (x.w > k);
            }
        }
        const bool stays = tid < n_cand && before < m;
        uint32_t total;
        const uint32_t at = block_scan(stays ? 1u : 0u, scratch, total);
        if (stays) emit(at, tid, k);
        for (int i = tid; i < r.recent; i += kThreads) emit(uint32_t(m + i), n_cand + i, 0u);
        return;
    }
    if (run_or_0) {
        const float* at = base;
        if (lo < min(valid, n_cand)) at += (long long)pages[lo / kPageTokens] * page_step + lo % kPageTokens;
#pragma unroll 1
        for (int i = 0; i < run; i += 4) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (lo + i < min(valid, n_cand)) x = *reinterpret_cast<const float4*>(at + i);
            mine[i] = order_key(x.x);
            mine[i + 1] = order_key(lo + i + 1 < valid ? x.y : 0.f);
            mine[i + 2] = order_key(lo + i + 2 < valid ? x.z : 0.f);
            mine[i + 3] = order_key(lo + i + 3 < valid ? x.w : 0.f);
        }
    }
    auto key_at = [&](int i) -> uint32_t { return run_or_0 ? mine[i] : order_key(load(lo + i)); };

    uint32_t prefix = 0, mask = 0, left = uint32_t(m);   // the threshold is the left-th largest with this prefix
    const bool all = m == n_cand, none = m == 0;
    bool whole_bin = false;
    if (!all && !none) {
#pragma unroll 1
        for (int pass = 0; pass < 3 && !whole_bin; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
            const uint32_t bins = pass < 2 ? 2048u : 1024u;
            uint32_t* hs = hist[pass & 1];
            hs[tid] = 0;
            hs[tid + kThreads] = 0;
            __syncthreads();
#pragma unroll 2
            for (int i = 0; i < run; ++i) {
                const uint32_t k = lo + i < hi ? key_at(i) : 0u;
                const bool in = lo + i < hi && (k & mask) == prefix;
                if (pass > 0 && !__any_sync(0xffffffffu, in)) continue;
                const uint32_t bin = in ? (k >> shift) & (bins - 1) : kBins;
                // equal accounts are common (positions never looked at): a warp that agrees adds once
                const bool same = __all_sync(0xffffffffu, bin == __shfl_sync(0xffffffffu, bin, 0));
                if (in && (!same || lane == 0)) atomicAdd(&hs[bin], same ? 32u : 1u);
            }
            // the bin, counted from the top, that holds the left-th largest: the first threads sum four bins
            // each over the cluster, the highest on the lowest threads
            const int top = int(bins) - 4 - tid * 4;
            uint4 c = make_uint4(0u, 0u, 0u, 0u);
            if (cluster > 1) cluster_sync_all();
            else __syncthreads();
            if (top >= 0) {
                if (cluster > 1) {
                    uint4 x[kMaxCluster];
#pragma unroll
                    for (int p = 0; p < kMaxCluster; ++p) x[p] = p < cluster ? peer_ld4u(&hs[top], uint32_t(p)) : c;
#pragma unroll
                    for (int p = 0; p < kMaxCluster; ++p) {
                        c.x += x[p].x;
                        c.y += x[p].y;
                        c.z += x[p].z;
                        c.w += x[p].w;
                    }
                } else {
                    c = *reinterpret_cast<const uint4*>(&hs[top]);
                }
            }
            uint32_t total;
            const uint32_t sum = (c.x + c.y) + (c.z + c.w);
            const uint32_t before = block_scan(sum, scratch, total);
            if (before < left && left <= before + sum) {     // exactly one thread
                uint32_t rest = left - before, bin = uint32_t(top) + 3, n = c.w;
                if (rest > n) { rest -= n; --bin; n = c.z; if (rest > n) { rest -= n; --bin; n = c.y; if (rest > n) { rest -= n; --bin; n = c.x; } } }
                found[0] = bin;
                found[1] = rest;
                found[2] = rest == n;                        // the whole bin stays: no need to look into it
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= (bins - 1) << shift;
            left = found[1];
            whole_bin = found[2] != 0;
            __syncthreads();
        }
    }
    // what a key is: 2 kept, 1 tied at the threshold (the first `left` of those stay), 0 out
    auto kind = [&](uint32_t k) -> int {
        if (all) return 2;
        if (none) return 0;
        const uint32_t t = k & mask;
        return t > prefix ? 2 : (t == prefix ? (whole_bin ? 2 : 1) : 0);
    };
    uint32_t gt = 0, eq = 0;
#pragma unroll 1
    for (int i = 0; i < hi - lo; ++i) {
        const int x = kind(key_at(i));
        gt += x == 2;
        eq += x == 1;
    }
    uint32_t gt_all, eq_all, gt_at, eq_at;
    if (run_or_0) {            // at most 1024 * 32 of either: both in one scan
        uint32_t both;
        const uint32_t at = block_scan(gt | eq << 16, scratch, both);
        gt_at = at & 0xffffu;
        eq_at = at >> 16;
        gt_all = both & 0xffffu;
        eq_all = both >> 16;
    } else {
        gt_at = block_scan(gt, scratch, gt_all);
        eq_at = block_scan(eq, scratch, eq_all);
    }
    uint32_t gt_before = 0, eq_before = 0;
    if (cluster > 1) {
        if (tid == 0) {
            counts[0] = gt_all;
            counts[1] = eq_all;
        }
        cluster_sync_all();
        if (lane < int(rank)) {
            gt_before = peer_ld(&counts[0], uint32_t(lane));
            eq_before = peer_ld(&counts[1], uint32_t(lane));
        }
#pragma unroll
        for (int o = 1; o < kMaxCluster; o <<= 1) {
            gt_before += __shfl_xor_sync(0xffffffffu, gt_before, o);
            eq_before += __shfl_xor_sync(0xffffffffu, eq_before, o);
        }
        gt_before = __shfl_sync(0xffffffffu, gt_before, 0);
        eq_before = __shfl_sync(0xffffffffu, eq_before, 0);
        cluster_arrive();      // no block leaves while another still reads its counts (or histograms): waited for below
    }
    // of the tied ones the first `left` (in position order over the whole row) stay
    uint32_t er = eq_before + eq_at;
    uint32_t at = gt_before + gt_at + min(er, left);
    if (gt + eq > 0)
#pragma unroll 1
        for (int i = 0; i < hi - lo; ++i) {
            const uint32_t k = key_at(i);
            const int x = kind(k);
            if (x == 2 || (x == 1 && er < left)) emit(at++, lo + i, k);
            er += x == 1;
        }
    // the last `recent` positions, shared out over the cluster
#pragma unroll 1
    for (int i = int(rank) * kThreads + tid; i < r.recent; i += cluster * kThreads) emit(uint32_t(m + i), n_cand + i, 0u);
    if (cluster > 1) cluster_wait();
}

// What the row kernels move: f32 rows (row_words = 4 * nv floats, K and V pools) or u8 blocks.
struct EvictPools {
    float* k;
    float* v;
    uint8_t* u8;
    float* account;
    long long pool_pages;
    int num_kv_heads, head_dim, nv, dq;
};

// The kept rows into the caller's dense arrays; the stream stays.  One warp moves kRows rows at a
// time, K and V together, all their loads in flight before the first store: 16 bytes per lane and
// row.  Bound by memory: each kept row is read and written once; 131072 rows of 128 floats, K and V: 42 us,
// 6.4 TB/s.
template <int ROWS>
__global__ void __launch_bounds__(256)
evict_copy_kernel(const __grid_constant__ EvictTable tab, EvictPools p) {
    pdl_wait();
    int rq = 0;
    while (rq + 1 < tab.n && int(blockIdx.x) >= tab.e[rq + 1].head0) ++rq;
    const EvictDev& r = tab.e[rq];
    if (r.copy != 1) return;
    const int local = int(blockIdx.x) - r.head0;
    const int l = r.layer0 + local / p.num_kv_heads, h = local % p.num_kv_heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int* pages = r.pages;
    const int* kept = r.kept_ws + size_t(local) * r.keep;
    const size_t lbase = size_t(l) * size_t(p.pool_pages);
    const int D = p.head_dim;
    const bool vec = (D & 3) == 0 && ((reinterpret_cast<uintptr_t>(r.k_out) | reinterpret_cast<uintptr_t>(r.v_out)) & 15) == 0;
    for (int i0 = (int(blockIdx.y) * 8 + warp) * ROWS; i0 < r.keep; i0 += int(gridDim.y) * 8 * ROWS) {
        const int n = min(ROWS, r.keep - i0);
        size_t src[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int j = kept[min(i0 + i, r.keep - 1)];
            const size_t blk = (lbase + size_t(pages[j / kPageTokens])) * p.num_kv_heads + h;
            src[i] = p.u8 ? blk * (size_t(kPageTokens) * (2 * size_t(p.dq) + 8)) + size_t(j % kPageTokens) * p.dq
                          : (blk * kPageTokens + size_t(j % kPageTokens)) * size_t(p.nv) * 4;
            if (p.u8) src[i] = (src[i] << 6) | size_t(j % kPageTokens);   // the scales are found from the row's place
        }
        float* kd = r.k_out + (size_t(local) * r.keep + i0) * D;
        float* vd = r.v_out + (size_t(local) * r.keep + i0) * D;
        if (p.u8) {
            for (int i = 0; i < n; ++i) {
                const int tk = int(src[i] & 63);
                const uint8_t* krow = p.u8 + (src[i] >> 6);
                const uint8_t* blk = krow - size_t(tk) * p.dq;
                const float* sc = reinterpret_cast<const float*>(blk + 2 * size_t(kPageTokens) * p.dq);
                const uint8_t* vrow = krow + size_t(kPageTokens) * p.dq;
                for (int d = lane; d < D; d += 32) {
                    kd[size_t(i) * D + d] = (float(krow[d]) - 128.0f) * sc[tk];
                    vd[size_t(i) * D + d] = (float(vrow[d]) - 128.0f) * sc[kPageTokens + tk];
                }
            }
            continue;
        }
        for (int c = lane * 4; c < D; c += 128) {
            float4 a[ROWS], b[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                a[i] = __ldcs(reinterpret_cast<const float4*>(p.k + src[i] + c));
                b[i] = __ldcs(reinterpret_cast<const float4*>(p.v + src[i] + c));
            }
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                if (i >= n) break;
                float* ko = kd + size_t(i) * D + c;
                float* vo = vd + size_t(i) * D + c;
                if (vec) {
                    __stcs(reinterpret_cast<float4*>(ko), a[i]);
                    __stcs(reinterpret_cast<float4*>(vo), b[i]);
                } else {
                    const float ka[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, va[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
                    for (int e = 0; e < 4; ++e)
                        if (c + e < D) {
                            ko[e] = ka[e];
                            vo[e] = va[e];
                        }
                }
            }
        }
    }
}

// The kept rows to the front of the same stream.  Row i comes from kept[i] >= i, so blocks of rows
// taken in ascending order never overwrite a row that is still to be read -- provided one block of
// threads walks them in order and every load of a step is done before its first store.  The loads
// of the next step are issued before the stores of this one (they read positions behind them).
// One block per (layer, KV head, K or V, slice of 128 bytes of a row); the account moves with the
// slice of K that holds a row's first bytes.  `unit` is 16 bytes for f32 rows and, for u8 rows,
// 4 bytes (their scales move with the first slice of K and of V).  Bound by that chain: a step is a
// kept position, its page, its row and a barrier, one step ahead.  131072 positions cut to 16384, 8 heads
// of 128: 355 us with the selection (copied out 70); 8192 to 2048 50 us.
constexpr int kMoveThreads = 512;
constexpr int kMoveSlice = 128;    // bytes of a row per block
__global__ void __launch_bounds__(kMoveThreads)
evict_move_kernel(const __grid_constant__ EvictTable tab, EvictPools p) {
    pdl_wait();
    int rq = 0;
    while (rq + 1 < tab.n && int(blockIdx.x) >= tab.e[rq + 1].head0) ++rq;
    const EvictDev& r = tab.e[rq];
    if (r.copy) return;
    const int row = int(blockIdx.x);
    const int local = row - r.head0;
    const int l = r.layer0 + local / p.num_kv_heads, h = local % p.num_kv_heads;
    const bool is_v = blockIdx.y & 1;
    const int slice = int(blockIdx.y) >> 1;
    const int row_bytes = p.u8 ? p.dq : p.nv * 16;
    const int off = slice * kMoveSlice;
    const int bytes = min(kMoveSlice, row_bytes - off);
    const int* pages = r.pages;
    const int* kept = r.kept_ws + size_t(local) * r.keep;
    const int valid = r.acc_len;
    const size_t lbase = size_t(l) * size_t(p.pool_pages);
    unsigned char* base;
    size_t blk_bytes;
    if (p.u8) {
        blk_bytes = size_t(kPageTokens) * (2 * size_t(p.dq) + 8);
        base = p.u8 + (is_v ? size_t(kPageTokens) * p.dq : 0);
    } else {
        blk_bytes = size_t(kPageTokens) * row_bytes;
        base = reinterpret_cast<unsigned char*>(is_v ? p.v : p.k);
    }
    auto block_at = [&](int j) { return ((lbase + size_t(pages[j / kPageTokens])) * p.num_kv_heads + h) * blk_bytes; };
    const int unit = p.u8 ? 4 : 16;
    const int tpr = bytes / unit;                       // threads per row
    const int rows = kMoveThreads / tpr;                // rows per step
    const int sub = int(threadIdx.x) % tpr, i_in = int(threadIdx.x) / tpr;
    const bool on = i_in < rows;
    const bool first = slice == 0 && sub == 0;
    // u8: scales of this half (K or V); f32 and u8: the account, moved by the K half
    struct Row { uint4 a; float scale, w; };
    auto read = [&](int i) -> Row {
        Row x = {};
        if (!on || i >= r.keep) return x;
        const int j = kept[i];
        const size_t b = block_at(j);
        const unsigned char* s = base + b + size_t(j % kPageTokens) * row_bytes + off + size_t(sub) * unit;
        if (p.u8) {
            x.a.x = *reinterpret_cast<const uint32_t*>(s);
            if (first)
                x.scale = reinterpret_cast<const float*>(p.u8 + b + 2 * size_t(kPageTokens) * p.dq)[(is_v ? kPageTokens : 0) + j % kPageTokens];
        } else {
            x.a = *reinterpret_cast<const uint4*>(s);
        }
        if (first && !is_v && p.account)
            x.w = j < valid ? p.account[account_offset(pages, p.pool_pages, l, p.num_kv_heads, h, j)] : 0.f;
        return x;
    };
    auto write = [&](int i, const Row& x) {
        if (!on || i >= r.keep) return;
        const size_t b = block_at(i);
        unsigned char* d = base + b + size_t(i % kPageTokens) * row_bytes + off + size_t(sub) * unit;
        if (p.u8) {
            *reinterpret_cast<uint32_t*>(d) = x.a.x;
            if (first)
                reinterpret_cast<float*>(p.u8 + b + 2 * size_t(kPageTokens) * p.dq)[(is_v ? kPageTokens : 0) + i % kPageTokens] = x.scale;
        } else {
            *reinterpret_cast<uint4*>(d) = x.a;
        }
        if (first && !is_v && p.account)
            p.account[account_offset(pages, p.pool_pages, l, p.num_kv_heads, h, i)] = x.w;
    };
    Row cur = read(i_in);
    __syncthreads();
    for (int i0 = 0; i0 < r.keep; i0 += rows) {
        Row next = {};
        if (i0 + rows < r.keep) next = read(i0 + rows + i_in);
        write(i0 + i_in, cur);
        cur = next;
        __syncthreads();
    }
}

}  // namespace xn
