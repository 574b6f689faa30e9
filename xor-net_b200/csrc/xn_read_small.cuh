// The latency-bound read: few streams, short prefixes, few rows, f32 cache, head_dim <= 128.
//
// One cluster of 1, 2, 4 or 8 blocks per (request, KV head); block c owns a contiguous share of the
// positions.  Two dependent loads (page ids, then the rows, straight into registers) stand before the
// arithmetic; the scores stay in shared memory; every block sends its softmax state and its share of
// the output columns to the block that writes them, through distributed shared memory, and one
// cluster barrier later all is there -- also what turns the scores into attention weights, when they
// are wanted.  One launch, no partial records, no counters in global memory.  What it is made of is
// latencies of 300 to 1200 cycles, about 6000 cycles in all, so loads are issued together and
// nothing is read remotely.  (A version whose blocks pulled their peers' states, with a barrier
// before and behind, took 13000 cycles.)  197 positions, 20/5 heads of 128, one row: 6.7 us; 1025 with
// an account: 12.0 us (the split-KV kernel and the account's launch: 17).
#pragma once
#include "xn_decode.cuh"
#include "xn_evict.cuh"
#include "xn_read.cuh"

namespace xn {
namespace rs {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kHeads = 4;             // heads per pass over the rows
constexpr int kMaxTokens = 256;       // positions of one block
constexpr int kMaxRows = 32;          // one after the other; their weights are one running sum
constexpr int kKeys = 4;              // pairs of keys that a warp has in flight
constexpr int kAhead = 8;             // rows of V that a warp has in flight

__device__ __forceinline__ void peer_st(const void* smem, uint32_t rank, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(ev::peer_addr(smem, rank)), "f"(v) : "memory");
}
__device__ __forceinline__ void peer_st4(const void* smem, uint32_t rank, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(ev::peer_addr(smem, rank)), "f"(v.x), "f"(v.y),
                 "f"(v.z), "f"(v.w)
                 : "memory");
}

}  // namespace rs

__global__ void __launch_bounds__(rs::kThreads, 1)
read_small_kernel(const __grid_constant__ ReadTable tab, const float* __restrict__ k_pool,
                  const float* __restrict__ v_pool, float* __restrict__ acct_pool, long long pool_pages,
                  int num_kv_heads, int head_dim, int nv, float scale, int cluster, int want) {
    using namespace rs;
    __shared__ __align__(16) float sc[kHeads][kMaxTokens];        // scores, then weights relative to this block's maximum
    __shared__ __align__(16) float red[kWarps][kHeads][128];
    // what the cluster's blocks send here, by pass parity: their sums of this block's columns (chunk
    // c / cluster of head hh from block p), their maxima and sums
    __shared__ __align__(16) float4 part[2][ev::kMaxCluster * kHeads * (32 / ev::kMaxCluster)];
    __shared__ float ml[2][ev::kMaxCluster][kHeads][2];
    __shared__ float own[kHeads][2], share_w[kHeads][ev::kMaxCluster];
    __shared__ float acc_s[kMaxTokens];
    pdl_launch_dependents();
    if (cluster > 1) ev::cluster_arrive();   // waited for before the first remote store: the peers must have started
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const int sub = lane & 15, grp = lane >> 4;                   // sixteen lanes share a key
    const int rank = int(ev::cluster_rank());
    const int unit = int(blockIdx.x) / cluster;
    ReadEntry e = tab.e[unit / num_kv_heads];
    // every field is a constant-cache miss: all of them now, together
    asm volatile("" : "+l"(e.q), "+l"(e.out), "+l"(e.pages), "+l"(e.user), "+l"(e.user_hs), "+l"(e.q_hs), "+l"(e.q_ts), "+l"(e.o_hs),
                 "+l"(e.o_ts), "+r"(e.rows), "+r"(e.kv_len), "+r"(e.layer), "+r"(e.old_from), "+r"(e.old_len), "+r"(e.store));
    const int h = unit % num_kv_heads;
    const int share = (e.kv_len + cluster - 1) / cluster;
    const int t0 = min(e.kv_len, share * rank);
    const int nt = min(e.kv_len, t0 + share) - t0;
    const int dp = nv * 4;
    // this head's rows of page 0; a page further is `page_step` floats on
    const size_t head_off = (size_t(e.layer) * size_t(pool_pages) * num_kv_heads + h) * size_t(kPageTokens * dp);
    const float* k_head = k_pool + head_off;
    const float* v_head = v_pool + head_off;
    const int page_step = num_kv_heads * kPageTokens * dp;        // < 2^31: the caller admits at most 148 or so heads
    auto row_off = [&](int tok, int page) { return (long long)page * page_step + ((t0 + tok) % kPageTokens) * dp; };
    if (want)
        for (int i = tid; i < nt; i += kThreads) acc_s[i] = 0.f;
    const int chunks = 32 / cluster;      // column groups of four that a block writes
    const bool vec = (head_dim & 3) == 0 && ((reinterpret_cast<uintptr_t>(e.q) | uintptr_t(e.q_hs * 4) | uintptr_t(e.q_ts * 4)) & 15) == 0;
    // page ids of the first step's keys and values (the table is written between kernels only)
    auto page_of = [&](int tok) { return e.pages[(t0 + min(tok, nt - 1)) / kPageTokens]; };
    int kpage[kKeys], vpage[kAhead];
    if (nt > 0) {
#pragma unroll
        for (int u = 0; u < kKeys; ++u) kpage[u] = page_of(w * 2 + u * kWarps * 2 + grp);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) vpage[i] = page_of(w + kWarps * i);
    }
    pdl_wait();                           // rows, queries and accounts may come from the kernel before this one

    int pass = 0;
#pragma unroll 1
    for (int t = 0; t < e.rows; ++t)
#pragma unroll 1
        for (int sb = 0; sb < tab.subs; ++sb, ++pass) {
            const int head0 = h * tab.group + sb * tab.gt;
            const int nheads = min(tab.gt, tab.group - sb * tab.gt);
            const int par = pass & 1;
            const float* qrow = e.q + size_t(head0) * e.q_hs + size_t(t) * e.q_ts;
            float4 q[kHeads][2], kk[kKeys][2], va[kAhead];
#pragma unroll
            for (int hh = 0; hh < kHeads; ++hh)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int idx = j * 16 + sub;
                    q[hh][j] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (vec && hh < nheads && idx < nv) q[hh][j] = *reinterpret_cast<const float4*>(qrow + size_t(hh) * e.q_hs + idx * 4);
                }
            auto load_k = [&](int base) {
#pragma unroll
                for (int u = 0; u < kKeys; ++u) {
                    kk[u][0] = kk[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (base + u * kWarps * 2 >= nt) continue;    // (the same for the whole warp)
                    const int key = base + u * kWarps * 2 + grp;
                    const float* row = k_head + row_off(key, kpage[u]) + sub * 4;
                    if (key < nt && sub < nv) kk[u][0] = *reinterpret_cast<const float4*>(row);
                    if (key < nt && 16 + sub < nv) kk[u][1] = *reinterpret_cast<const float4*>(row + 64);
                }
            };
            auto load_v = [&](int tok0) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int tok = tok0 + kWarps * i;
                    if (tok >= nt) break;
                    va[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (lane < nv) va[i] = *reinterpret_cast<const float4*>(v_head + row_off(tok, vpage[i]) + lane * 4);
                }
            };
            if (nt > 0) {
                if (pass > 0 && nt > kWarps * kAhead) {   // the loops below have moved on
#pragma unroll
                    for (int u = 0; u < kKeys; ++u) kpage[u] = page_of(w * 2 + u * kWarps * 2 + grp);
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) vpage[i] = page_of(w + kWarps * i);
                }
                load_k(w * 2);
                load_v(w);
            }
            if (!vec)
#pragma unroll 1
                for (int hh = 0; hh < nheads; ++hh)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = (j * 16 + sub) * 4;
                        if (d >= head_dim) continue;
                        const float* r = qrow + size_t(hh) * e.q_hs + d;
                        float4 x = make_float4(r[0], 0.f, 0.f, 0.f);
                        if (d + 1 < head_dim) x.y = r[1];
                        if (d + 2 < head_dim) x.z = r[2];
                        if (d + 3 < head_dim) x.w = r[3];
#pragma unroll
                        for (int k = 0; k < kHeads; ++k)
                            if (k == hh) q[k][j] = x;
                    }
            // ---- scores: sixteen lanes per key, two keys per warp instruction, kKeys of those in flight
#pragma unroll 1
            for (int base = w * 2; base < nt; base += kWarps * 2 * kKeys) {
                if (base != w * 2) {
#pragma unroll
                    for (int u = 0; u < kKeys; ++u) kpage[u] = page_of(base + u * kWarps * 2 + grp);
                    load_k(base);
                }
#pragma unroll
                for (int u = 0; u < kKeys; ++u) {
                    if (base + u * kWarps * 2 >= nt) break;
                    const int key = base + u * kWarps * 2 + grp;
                    float part_dot[kHeads];
#pragma unroll
                    for (int hh = 0; hh < kHeads; ++hh) {
                        float2 p2 = make_float2(0.f, 0.f);
#pragma unroll
                        for (int j = 0; j < 2; ++j) dot4_acc(p2, q[hh][j], kk[u][j]);
                        part_dot[hh] = p2.x + p2.y;
                    }
                    const float dot = group_reduce<kHeads, 16>(part_dot, sub);
                    if (sub < kHeads && key < nt) sc[owned_head<kHeads>(sub)][key] = dot * scale;
                }
            }
            __syncthreads();
            // ---- this block's softmax: one warp per head
            if (w < kHeads) {
                float m = -INFINITY;
                for (int i = lane; i < nt; i += 32) m = fmaxf(m, sc[w][i]);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float ms = m == -INFINITY ? 0.f : m;
                float l = 0.f;
#pragma unroll 1
                for (int i = lane; i < nt; i += 32) {
                    const float p = expf(sc[w][i] - ms);
                    sc[w][i] = p;
                    l += p;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                if (lane == 0) {
                    own[w][0] = m;
                    own[w][1] = l;
                }
            }
            if (cluster > 1 && pass == 0) ev::cluster_wait();
            __syncthreads();
            if (tid < cluster * kHeads) {   // the softmax state to every block, this one included
                const int p = tid / kHeads, hh = tid % kHeads;
                peer_st(&ml[par][rank][hh][0], uint32_t(p), own[hh][0]);
                peer_st(&ml[par][rank][hh][1], uint32_t(p), own[hh][1]);
            }
            // ---- weighted V rows: a lane holds four columns
            float4 acc[kHeads];
#pragma unroll
            for (int hh = 0; hh < kHeads; ++hh) acc[hh] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int tok0 = w; tok0 < nt; tok0 += kWarps * kAhead) {
                if (tok0 != w) {
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) vpage[i] = page_of(tok0 + kWarps * i);
                    load_v(tok0);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int tok = tok0 + kWarps * i;
                    if (tok >= nt) break;
#pragma unroll
                    for (int hh = 0; hh < kHeads; ++hh) fma4_scalar(acc[hh], sc[hh][tok], va[i]);
                }
            }
#pragma unroll
            for (int hh = 0; hh < kHeads; ++hh) *reinterpret_cast<float4*>(&red[w][hh][lane * 4]) = acc[hh];
            __syncthreads();
            if (tid < kHeads * 32) {
                const int hh = tid >> 5, ch = tid & 31;
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int ww = 0; ww < kWarps; ++ww) {
                    const float4 x = *reinterpret_cast<const float4*>(&red[ww][hh][ch * 4]);
                    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
                }
                // to the block that writes these columns
                const int to = ch / chunks, at = (rank * kHeads + hh) * chunks + ch % chunks;
                if (cluster > 1) peer_st4(&part[par][at], uint32_t(to), s);
                else part[par][at] = s;
            }
            if (cluster > 1) {
                ev::cluster_arrive();
                ev::cluster_wait();
            } else {
                __syncthreads();
            }
            // ---- the blocks' states have met: lane (hh, p) of the first warp weighs block p's share
            if (w == 0) {
                const int hh = lane / ev::kMaxCluster, p = lane % ev::kMaxCluster;
                const float mp = p < cluster ? ml[par][p][hh][0] : -INFINITY, lp = p < cluster ? ml[par][p][hh][1] : 0.f;
                float M = mp;
#pragma unroll
                for (int o = 1; o < ev::kMaxCluster; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
                const float wgt = mp == -INFINITY ? 0.f : expf(mp - M);
                float L = lp * wgt;
#pragma unroll
                for (int o = 1; o < ev::kMaxCluster; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
                share_w[hh][p] = wgt / L;   // (what turns that block's weights into the row's)
            }
            __syncthreads();
            if (tid < kHeads * chunks) {
                const int hh = tid / chunks, c = tid % chunks;
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int p = 0; p < ev::kMaxCluster; ++p) {
                    if (p >= cluster) break;
                    const float wgt = share_w[hh][p];
                    const float4 x = part[par][(p * kHeads + hh) * chunks + c];
                    s.x = fmaf(wgt, x.x, s.x);
                    s.y = fmaf(wgt, x.y, s.y);
                    s.z = fmaf(wgt, x.z, s.z);
                    s.w = fmaf(wgt, x.w, s.w);
                }
                const int d = (rank * chunks + c) * 4;
                if (hh < nheads && d < head_dim) {
                    float* row = e.out + (long long)(head0 + hh) * e.o_hs + (long long)t * e.o_ts + d;
                    if (d + 3 < head_dim && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
                        *reinterpret_cast<float4*>(row) = s;
                    } else {
                        row[0] = s.x;
                        if (d + 1 < head_dim) row[1] = s.y;
                        if (d + 2 < head_dim) row[2] = s.z;
                        if (d + 3 < head_dim) row[3] = s.w;
                    }
                }
            }
            if (want)
                for (int i = tid; i < nt; i += kThreads) {
                    float s = acc_s[i];
#pragma unroll
                    for (int hh = 0; hh < kHeads; ++hh)
                        if (hh < nheads) s = fmaf(sc[hh][i], share_w[hh][rank], s);
                    acc_s[i] = s;
                }
            __syncthreads();   // (the next pass writes new scores)
        }
    if (want) {
        const AccountDev a = {e.user, e.user_hs, e.old_from, e.old_len, e.store, e.kv_len, 0, e.layer};
        for (int i = tid; i < nt; i += kThreads)
            account_store(a, e.pages, acct_pool, pool_pages, num_kv_heads, h, t0 + i, acc_s[i]);
    }
}

}  // namespace xn
