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
constexpr int kMaxRun = 32;        // candidates a thread can hold

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

// One cluster of 1, 2, 4 or 8 blocks per (layer, KV head).  Thread t of block r owns the RUN
// candidates from (r * 1024 + t) * RUN on, a quarter of a page or so, and keeps their keys in
// registers (RUN > 0): the account is read from memory once, 16 bytes per load, and thread order is
// position order.  Radix selection: the threshold key is found 11, 11 and 10 bits at a time from
// shared-memory histograms that the blocks read from one another; then one scan of the (above,
// equal) counts gives every thread the place of its first kept position, ties included, and it
// writes its run.  Bound by the latency of these steps, about 2 microseconds each, not by bandwidth:
// [8 heads x 131072 positions: 12 us against 93 us for a loop over the slice in shared memory with a
// ballot and four barriers per 512 positions.]
// RUN = 0: streams too long for that; the keys are read again in every pass.
template <int RUN>
__global__ void __launch_bounds__(ev::kThreads, 1)
evict_select_kernel(const __grid_constant__ EvictTable tab, const float* __restrict__ pool, long long pool_pages,
                    int num_kv_heads, int cluster) {
    using namespace ev;
    pdl_launch_dependents();
    __shared__ uint32_t hist[2][kBins];             // by pass parity: peers may still read the other one
    __shared__ uint32_t scratch[32];
    __shared__ uint32_t counts[2];                  // this block's candidates above / at the threshold
    __shared__ uint32_t found[2];
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
    // positions [lo, hi) are this thread's; without RUN a run that covers the stream
    const int run = RUN > 0 ? RUN : (((n_cand + cluster * kThreads - 1) / (cluster * kThreads)) + 3) / 4 * 4;
    const long long lo_ll = (long long)(int(rank) * kThreads + tid) * run;
    const int lo = int(lo_ll < n_cand ? lo_ll : n_cand), hi = min(n_cand, lo + run);
    const int* pages = r.pages;
    const int valid = r.acc_len;
    const size_t base = (size_t(l) * size_t(pool_pages)) * num_kv_heads * kPageTokens + size_t(h) * kPageTokens;
    const size_t pstep = size_t(num_kv_heads) * kPageTokens;
    auto load = [&](int j) -> float {
        return j < valid ? pool[base + size_t(pages[j / kPageTokens]) * pstep + size_t(j % kPageTokens)] : 0.f;
    };
    // four positions from a multiple of four on: they never leave a page
    auto load4 = [&](int j) -> float4 {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < valid && j < n_cand) {
            x = *reinterpret_cast<const float4*>(pool + base + size_t(pages[j / kPageTokens]) * pstep + size_t(j % kPageTokens));
            if (j + 1 >= valid) x.y = 0.f;
            if (j + 2 >= valid) x.z = 0.f;
            if (j + 3 >= valid) x.w = 0.f;
        }
        return x;
    };
    constexpr int R = RUN > 0 ? RUN : 4;
    uint32_t keys[R];
    pdl_wait();
    if (RUN > 0) {
        float4 x[R / 4];
#pragma unroll
        for (int i = 0; i < R / 4; ++i) x[i] = load4(lo + 4 * i);
#pragma unroll
        for (int i = 0; i < R / 4; ++i) {
            keys[4 * i] = order_key(x[i].x);
            keys[4 * i + 1] = order_key(x[i].y);
            keys[4 * i + 2] = order_key(x[i].z);
            keys[4 * i + 3] = order_key(x[i].w);
        }
    }
    // f(j, key) for every candidate of the thread in order, all lanes of a warp together
    auto each = [&](auto&& f) {
        if (RUN > 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) f(lo + i, keys[i], lo + i < hi);
        } else {
            for (int i = 0; i < run; ++i) {
                const int j = lo + i;
                const bool in = j < hi;
                f(j, in ? order_key(load(j)) : 0u, in);
            }
        }
    };

    uint32_t prefix = 0, mask = 0, left = uint32_t(m);   // the threshold is the left-th largest with this prefix
    const bool all = m == n_cand, none = m == 0;
    if (!all && !none) {
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10;
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
            const uint32_t bins = 1u << bits;
            uint32_t* hs = hist[pass & 1];
            hs[tid] = 0;
            hs[tid + kThreads] = 0;
            __syncthreads();
            each([&](int, uint32_t k, bool in_run) {
                const bool in = in_run && (k & mask) == prefix;
                const uint32_t bin = (k >> shift) & (bins - 1);
                // equal accounts are common (positions never looked at): a warp that agrees adds once
                const uint32_t act = __ballot_sync(0xffffffffu, in);
                if (act == 0) return;
                const int lead = __ffs(act) - 1;
                const uint32_t b0 = __shfl_sync(0xffffffffu, bin, lead);
                if (__all_sync(0xffffffffu, !in || bin == b0)) {
                    if (lane == lead) atomicAdd(&hs[b0], uint32_t(__popc(act)));
                } else if (in) {
                    atomicAdd(&hs[bin], 1u);
                }
            });
            // the bin, counted from the top, that holds the left-th largest: a thread sums two bins (one
            // in the last pass) over the cluster, the highest on the lowest threads
            const int per = int(bins) / kThreads;
            const int top = int(bins) - 1 - tid * per;
            uint32_t a = 0, b = 0;
            if (cluster > 1) {
                cluster_sync_all();
#pragma unroll
                for (int p = 0; p < kMaxCluster; ++p)
                    if (p < cluster) {
                        a += peer_ld(&hs[top], uint32_t(p));
                        if (per == 2) b += peer_ld(&hs[top - 1], uint32_t(p));
                    }
            } else {
                __syncthreads();
                a = hs[top];
                if (per == 2) b = hs[top - 1];
            }
            uint32_t total;
            const uint32_t before = block_scan(a + b, scratch, total);
            if (before < left && left <= before + a + b) {   // exactly one thread
                const bool first = left <= before + a;
                found[0] = uint32_t(first ? top : top - 1);
                found[1] = left - before - (first ? 0u : a);
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= (bins - 1) << shift;
            left = found[1];
            __syncthreads();
        }
    }
    // m == 0 keeps no candidate, m == n_cand keeps all
    uint32_t gt = 0, eq = 0;
    if (all) gt = uint32_t(hi - lo);
    else if (!none)
        each([&](int, uint32_t k, bool in) {
            gt += in && k > prefix;
            eq += in && k == prefix;
        });
    uint32_t gt_all, eq_all;
    const uint32_t gt_at = block_scan(gt, scratch, gt_all);
    const uint32_t eq_at = block_scan(eq, scratch, eq_all);
    uint32_t gt_before = 0, eq_before = 0;
    if (cluster > 1) {
        if (tid == 0) {
            counts[0] = gt_all;
            counts[1] = eq_all;
        }
        __syncthreads();
        cluster_sync_all();
        for (uint32_t p = 0; p < rank; ++p) {
            gt_before += peer_ld(&counts[0], p);
            eq_before += peer_ld(&counts[1], p);
        }
        cluster_sync_all();   // no block leaves while another still reads its counts (or histograms)
    }
    int* kept = r.kept_ws + size_t(local) * r.keep;
    int* kept_user = r.kept ? r.kept + size_t(local) * r.keep : nullptr;
    float* w_user = r.w_out ? r.w_out + size_t(local) * r.keep : nullptr;
    auto emit = [&](uint32_t at, int j) {
        kept[at] = j;
        if (kept_user) kept_user[at] = j;
        if (w_user) w_user[at] = load(j);
    };
    if (!none) {
        // of the equal ones the first `left` (in position order over the whole row) stay
        uint32_t er = eq_before + eq_at;
        uint32_t at = gt_before + gt_at + min(er, left);
        each([&](int j, uint32_t k, bool in) {
            const bool is_eq = !all && in && k == prefix;
            if (in && (all || k > prefix || (is_eq && er < left))) emit(at++, j);
            er += is_eq;
        });
    }
    // the last `recent` positions, shared out over the cluster
    for (int i = int(rank) * kThreads + tid; i < r.recent; i += cluster * kThreads) emit(uint32_t(m + i), n_cand + i);
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
// row.  Bound by memory: each kept row is read and written once.
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
// 4 bytes (their scales move with the first slice of K and of V).
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
