// A read of some query rows (a few to about 48 per KV head with the heads of its group) over an f32 cache:
// few enough that the read of K and V should bound it, too many for the split-KV kernel, which goes over
// the cache once per row and four heads.
//
// Bulk tensor copies bring 64-token tiles of K and V as they are (f32) into a ring of shared-memory
// stages; eight warps do the arithmetic with warp-level MMAs (m16n8k16, f16 in, f32 accumulators)
// on operands split into two f16 values as in xn_read_tc.cuh -- three products, 22 bits -- but
// converted here, in registers, so that nothing is written back and read again: a conversion pass of
// its own moves twice the bytes of the whole read.  (The tcgen05 MMAs want their operands in shared
// memory or tensor memory in f16, i.e. that pass.  Two forms of the tcgen05 kernel whose own warps
// converted each tile took 90 to 110 us where this one takes 40 to 60: every converted element goes
// through a chain of load, maximum over the rows that share a scale, split and store, and with 4 or 8
// warps per SM that chain's latency, 2000 cycles per 8 KB, is what one waits for.)
//
//   S = Q K^T   warp w owns positions [8 w, 8 w + 8) of the tile, all rows: it converts them once, with a
//               scale of their own;
//   softmax     row maxima through shared memory; P as hi and lo to shared memory;
//   O += P V    warp w owns columns [32 (w & 3), +32) and positions [32 (w >> 2), +32): again every
//               element is converted once.  A tile's O starts from zero in the MMA accumulator and is
//               added to the running one in f32, which undoes the sub-block's scale.
//
// Positions far below the largest of those that share their scale (2^-16: their bits would go) have their
// scores, and their share of O, computed in f32.
//
// The order of the contraction index, and of the output columns among the MMA's, is free: both are
// chosen so that every shared-memory access is a conflict-free 16-byte one of the 128-byte-swizzled
// tile.  Work is cut as in the table form of the split-KV kernel: block b of G takes an equal share of
// the tiles of all (request, KV head, row tile) units; the block that delivers a cut unit's last
// partial record combines them.
//
// Measured: 6000 cycles per 64-token tile for up to 16 rows (8500 instructions over the eight warps; two
// warps per scheduler wait for one another's latencies), i.e. 3.1 TB/s; 20 requests of 500-1500
// positions, 20/5 heads of 128, 4 rows each (16 per KV head): 48 us, the split-KV kernel 64, the
// tensor-core passes 80.
#pragma once
#include <cuda.h>

#include "xn_read_tc.cuh"

namespace xn {
namespace rm {

constexpr int kThreads = 288;             // eight warps and the copy warp
constexpr int kTileBytes = 32768;         // 64 positions of 128 f32 columns: K, and as much for V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kSub = 8192;                // a column block: 64 rows of 128 bytes
__host__ __device__ constexpr int stages(int mt) { return mt <= 2 ? 3 : 2; }
__host__ __device__ constexpr int rows(int mt) { return 16 * mt; }
__host__ __device__ constexpr size_t smem_bytes(int mt) {
    // stages | Q hi, lo (later the O of the upper position half) | P hi, lo | maxima, sums by warp | row factors, maxima | barriers
    return size_t(stages(mt)) * kStageBytes + size_t(rows(mt)) * 512 + size_t(rows(mt)) * 256 + size_t(rows(mt)) * 32 +
           size_t(rows(mt)) * 2 * 4 + 512;
}
__host__ __device__ constexpr size_t part_floats(int mt, int dp) { return size_t(rows(mt)) * (size_t(dp) + 2); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (magnitudes: their bits order as they do)
__device__ __forceinline__ float warp_max(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }
__device__ __forceinline__ float finite_max4(const float4& x) {   // infinities and NaNs do not set a scale
    float m = 0.f;
    m = fabsf(x.x) < INFINITY ? fmaxf(m, fabsf(x.x)) : m;
    m = fabsf(x.y) < INFINITY ? fmaxf(m, fabsf(x.y)) : m;
    m = fabsf(x.z) < INFINITY ? fmaxf(m, fabsf(x.z)) : m;
    m = fabsf(x.w) < INFINITY ? fmaxf(m, fabsf(x.w)) : m;
    return m;
}
// a split whose lo half is 0 behind an infinite or NaN hi
__device__ __forceinline__ void split2_safe(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __float22half2_rn(x);
    const float2 back = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float a = x.x - back.x, b = x.y - back.y;
    lo = rt::pack2(a == a ? a : 0.f, b == b ? b : 0.f);
}

}  // namespace rm

template <int MT>
__global__ void __launch_bounds__(rm::kThreads, 1)
read_mid_kernel(const __grid_constant__ ReadTable tab, const __grid_constant__ CUtensorMap k_map,
                const __grid_constant__ CUtensorMap v_map, float* __restrict__ partials, int* __restrict__ sync,
                long long pool_pages, int num_kv_heads, int head_dim, int nv, float scale_log2, int want,
                int* __restrict__ status) {
    using namespace rm;
    constexpr int R = 16 * MT;            // packed rows of a unit
    constexpr int ST = stages(MT);
    constexpr unsigned kFull = 0xffffffffu;
    constexpr float kLn2 = 0.6931471805599453f;
    constexpr float kPScale = rt::kPScale;
    extern __shared__ __align__(1024) unsigned char mid_smem[];
    unsigned char* q_s = mid_smem + size_t(ST) * kStageBytes;          // [hi | lo][R][256 bytes]
    unsigned char* p_s = q_s + size_t(R) * 512;                        // [hi | lo][R][128 bytes]
    float* xm = reinterpret_cast<float*>(p_s + size_t(R) * 256);       // [R][8]
    float* cq_s = xm + R * 8;                                          // [R] row factors
    float* m_s = cq_s + R;                                             // [R] maxima
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(m_s + R);
    uint64_t* empty_bar = full_bar + ST;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + ST);
    volatile int* last_flag = abort_flag + 1;
    volatile int* dead_flag = abort_flag + 2;   // [2], by tile parity

    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    if (smem_u32(mid_smem) & 1023u) {     // (the swizzled tiles need it; never seen otherwise)
        if (tid == 0) report_status(status, kDevBadIndex);
        return;
    }
    const int n_kb = (head_dim + 31) / 32;
    const long long T = tab.n_tiles, G = tab.n_blocks, blk = blockIdx.x;
    const long long t_lo = T * blk / G, t_hi = T * (blk + 1) / G;
    auto block_of = [&](long long tile) { return int(((tile + 1) * G - 1) / T); };
    if (tid == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 8);
        }
        *abort_flag = 0;
        dead_flag[0] = dead_flag[1] = 0;
        mbar_fence_init();
    }
    __syncthreads();
    pdl_wait();

    if (w == 8) {
        // =============================== copies ===============================
        if (lane == 0) {
            bool ok = true;
            int fill = 0, rq = 0, issued = 0;
            for (long long cur = t_lo; cur < t_hi && ok; ++cur, ++fill) {
                while (rq + 1 < tab.n && cur >= tab.e[rq + 1].tile0) ++rq;
                const ReadEntry& e = tab.e[rq];
                const long long in = cur - e.tile0;
                const int unit = int(in / e.n_tiles), tile = int(in % e.n_tiles);
                const int h = unit / e.n_rt;
                const int s = fill % ST;
                const int page = e.pages[tile];
                if (fill >= ST && !mbar_spin_bounded(&empty_bar[s], uint32_t((fill / ST - 1) & 1))) {
                    report_status(status, kDevWaitEmpty);
                    ok = false;
                    break;
                }
                if (!XN_PAGE_OK(page, pool_pages)) {
                    report_status(status, kDevBadIndex);
                    ok = false;
                    break;
                }
                const int row = int(((long long)e.layer * pool_pages + page) * num_kv_heads + h) * kPageTokens;
                unsigned char* at = mid_smem + size_t(s) * kStageBytes;
                mbar_arrive_expect_tx(&full_bar[s], uint32_t(2 * n_kb) * kSub);
                ++issued;
                for (int kb = 0; kb < n_kb; ++kb) pf::tma_load_2d(at + kb * kSub, &k_map, kb * 32, row, &full_bar[s]);
                for (int kb = 0; kb < n_kb; ++kb) pf::tma_load_2d(at + kTileBytes + kb * kSub, &v_map, kb * 32, row, &full_bar[s]);
                if (*abort_flag) break;
            }
            if (!ok) *abort_flag = 1;
            if (*abort_flag)   // nobody may be waiting for them any more: no copy outlives the block
                for (int f = max(0, issued - ST); f < issued; ++f) mbar_spin_bounded(&full_bar[f % ST], uint32_t((f / ST) & 1));
        }
        return;
    }

    // =============================== arithmetic ===============================
    auto barrier = [&]() { named_bar_sync(1, 256); };
    const int g = lane >> 2, t4 = lane & 3;
    const int cbw = w & 3, kh = w >> 2;   // O: column block and position half of this warp
    const bool my_cols = cbw < n_kb;
    const int dp = nv * 4;
    int fill = 0, rq = 0;
    for (long long cur = t_lo; cur < t_hi;) {
        while (rq + 1 < tab.n && cur >= tab.e[rq + 1].tile0) ++rq;
        const ReadEntry& e = tab.e[rq];
        const long long unit_l = (cur - e.tile0) / e.n_tiles;
        const int unit = int(unit_l);
        const long long unit0 = e.tile0 + unit_l * e.n_tiles;
        const int tile_begin = int(cur - unit0), tile_end = int(min((long long)e.n_tiles, t_hi - unit0));
        const int h = unit / e.n_rt, row0 = (unit % e.n_rt) * R;
        const int b0 = block_of(unit0), b1 = block_of(unit0 + e.n_tiles - 1);
        const int n_packed = e.rows * tab.group;
        cur = unit0 + tile_end;

        // ---- query rows: scaled by row, split, in the contraction order of the K fragments: step ks takes
        // the 16-byte chunks 2 t + (ks & 1) of column block ks / 2, lane t of a fragment one of them
        {
            const bool vec = (head_dim & 3) == 0 && ((reinterpret_cast<uintptr_t>(e.q) | uintptr_t(e.q_hs * 4) | uintptr_t(e.q_ts * 4)) & 15) == 0;
            float4 x[2 * MT];
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {
                const int p = row0 + w * 2 * MT + i, d = lane * 4;
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p < n_packed && d < head_dim) {
                    const float* row = e.q + (long long)(h * tab.group + p % tab.group) * e.q_hs + (long long)(p / tab.group) * e.q_ts + d;
                    if (vec) {
                        x[i] = *reinterpret_cast<const float4*>(row);
                    } else {
                        x[i].x = row[0];
                        if (d + 1 < head_dim) x[i].y = row[1];
                        if (d + 2 < head_dim) x[i].z = row[2];
                        if (d + 3 < head_dim) x[i].w = row[3];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {
                const int rr = w * 2 * MT + i;
                float up, down;
                rt::scale_of(warp_max(finite_max4(x[i])), up, down);
                uint32_t hi0, lo0, hi1, lo1;
                split2_safe(make_float2(x[i].x * up, x[i].y * up), hi0, lo0);
                split2_safe(make_float2(x[i].z * up, x[i].w * up), hi1, lo1);
                // chunk `lane`: column block lane / 8, chunk c = lane % 8 of it -> step, fragment lane
                const int c = lane & 7, ks = (lane >> 3) * 2 + (c & 1), t = c >> 1;
                const int x7 = rr & 7;
                unsigned char* row = q_s + size_t(rr) * 256;
                *reinterpret_cast<uint32_t*>(row + (((ks * 2) ^ x7) << 4) + t * 4) = hi0;
                *reinterpret_cast<uint32_t*>(row + (((ks * 2 + 1) ^ x7) << 4) + t * 4) = hi1;
                row += size_t(R) * 256;
                *reinterpret_cast<uint32_t*>(row + (((ks * 2) ^ x7) << 4) + t * 4) = lo0;
                *reinterpret_cast<uint32_t*>(row + (((ks * 2 + 1) ^ x7) << 4) + t * 4) = lo1;
                if (lane == 0) cq_s[rr] = down * scale_log2;
            }
        }
        barrier();
        float cq[MT][2], m_run[MT][2], l_run[MT][2];
        int limit[MT][2];                 // positions below it are visible to the row
        float4 o[MT][2][2];               // [m tile][row g, g + 8][columns 8 t.., 8 t + 4..] of the column block
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int rr = mt * 16 + hf * 8 + g, p = row0 + rr;
                cq[mt][hf] = cq_s[rr];
                limit[mt][hf] = p >= n_packed ? 0 : (e.causal ? e.kv_len - e.rows + p / tab.group + 1 : e.kv_len);
                m_run[mt][hf] = -INFINITY;
                l_run[mt][hf] = 0.f;
                o[mt][hf][0] = o[mt][hf][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        const int limit_first = e.causal ? e.kv_len - e.rows + row0 / tab.group + 1 : e.kv_len;   // the tile's first row's

        for (int tile = tile_begin; tile < tile_end; ++tile, ++fill) {
            const int s = fill % ST, tok0 = tile * kPageTokens;
            const int ntok = min(kPageTokens, e.kv_len - tok0);
            const unsigned char* ks_s = mid_smem + size_t(s) * kStageBytes;
            const unsigned char* vs_s = ks_s + kTileBytes;
            if (!warp_spin_bounded(&full_bar[s], uint32_t((fill / ST) & 1), lane)) {
                if (lane == 0) { report_status(status, kDevWaitFull); dead_flag[fill & 1] = 1; *abort_flag = 1; }
            }
            // ---- K fragments of this warp's eight positions, their own scale
            float sc[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) sc[mt][0] = sc[mt][1] = sc[mt][2] = sc[mt][3] = 0.f;
            float fk;
            unsigned bad_k;               // lanes whose part of K the MMAs do not take (an infinity, a NaN, values far
                                          // below their neighbours'): four bits per position
            {
                const int key = w * 8 + g;
                float4 kx[8];
                float mx = 0.f;
                bool ok = true;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    kx[ks] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if ((ks >> 1) < n_kb && key < ntok)
                        kx[ks] = *reinterpret_cast<const float4*>(ks_s + (ks >> 1) * kSub + key * 128 + (((2 * t4 + (ks & 1)) ^ g) << 4));
                    mx = fmaxf(mx, rt::max4(kx[ks]));
                    ok = ok && rt::finite4(kx[ks]);
                }
                bad_k = __ballot_sync(kFull, !ok);
                ok = bad_k == 0u;
                if (!ok) {
                    mx = 0.f;
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) mx = fmaxf(mx, finite_max4(kx[ks]));
                }
                const float largest = warp_max(mx);
                if (__any_sync(kFull, mx > 0.f && mx < largest * rt::kRowSpread)) {
                    // positions far below the largest of the eight would lose bits to its scale: their scores
                    // in f32 as well (seldom)
                    float row = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
                    row = fmaxf(row, __shfl_xor_sync(kFull, row, 2));
                    const bool small = row > 0.f && row < largest * rt::kRowSpread;
                    bad_k |= __ballot_sync(kFull, small);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        if (small) kx[ks] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                float up;
                rt::scale_of(largest, up, fk);
                const float2 up2 = make_float2(up, up);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    if ((ks >> 1) >= n_kb) break;
                    const float2 a = __fmul2_rn(make_float2(kx[ks].x, kx[ks].y), up2), b = __fmul2_rn(make_float2(kx[ks].z, kx[ks].w), up2);
                    uint32_t bh0, bl0, bh1, bl1;
                    if (ok) {
                        rt::split2(a, bh0, bl0);
                        rt::split2(b, bh1, bl1);
                    } else {
                        split2_safe(a, bh0, bl0);
                        split2_safe(b, bh1, bl1);
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const int rr = mt * 16 + (lane & 15);
                        const uint32_t at = smem_u32(q_s) + uint32_t(rr) * 256 + uint32_t(((ks * 2 + (lane >> 4)) ^ (rr & 7)) << 4);
                        uint32_t ah[4], al[4];
                        ldsm4(al, at + R * 256);
                        ldsm4(ah, at);
                        mma(sc[mt], al, bh0, bh1);
                        mma(sc[mt], ah, bl0, bl1);
                        mma(sc[mt], ah, bh0, bh1);
                    }
                }
            }
            // ---- scores in log2 units, masked; row maxima
            const int key0 = tok0 + w * 8 + 2 * t4;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float cm = cq[mt][hf] * fk;
                    float a = sc[mt][2 * hf] * cm, b = sc[mt][2 * hf + 1] * cm;
                    if (bad_k) {   // those positions' scores in f32 (a split product of an infinity is not one)
                        const int p = row0 + mt * 16 + hf * 8 + g;
#pragma unroll 1
                        for (int u = 0; u < 2; ++u) {
                            const int key = 2 * t4 + u;
                            if (((bad_k >> (4 * key)) & 15u) == 0u || p >= n_packed) continue;
                            const float* qr = e.q + (long long)(h * tab.group + p % tab.group) * e.q_hs + (long long)(p / tab.group) * e.q_ts;
                            float dot = 0.f;
#pragma unroll 1
                            for (int d = 0; d < head_dim; ++d)
                                dot = fmaf(qr[d], *reinterpret_cast<const float*>(ks_s + (d >> 5) * kSub + (w * 8 + key) * 128 +
                                                                                 ((((d >> 2) & 7) ^ key) << 4) + (d & 3) * 4), dot);
                            (u ? b : a) = dot * scale_log2;
                        }
                    }
                    if (tok0 + kPageTokens > limit_first) {
                        if (key0 >= limit[mt][hf]) a = -INFINITY;
                        if (key0 + 1 >= limit[mt][hf]) b = -INFINITY;
                    }
                    sc[mt][2 * hf] = a;
                    sc[mt][2 * hf + 1] = b;
                    float m = fmaxf(a, b);
                    m = fmaxf(m, __shfl_xor_sync(kFull, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(kFull, m, 2));
                    if (t4 == 0) xm[(mt * 16 + hf * 8 + g) * 8 + w] = m;
                }
            if (want) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const int p = row0 + mt * 16 + hf * 8 + g;
                        if (p >= n_packed) continue;
                        float* row = e.scores + (long long)(h * tab.group + p % tab.group) * e.sc_hs + (long long)(p / tab.group) * e.sc_ts + key0;
                        // (rows of scores are padded to four floats: a pair never leaves its row's storage)
                        if (key0 < e.kv_len) *reinterpret_cast<float2*>(row) = make_float2(sc[mt][2 * hf] * kLn2, sc[mt][2 * hf + 1] * kLn2);
                    }
            }
            barrier();
            if (dead_flag[fill & 1]) break;   // the same for all: set before the barrier, the other parity is the next tile's
            // ---- weights
            float alpha[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int rr = mt * 16 + hf * 8 + g;
                    const float4 a = *reinterpret_cast<const float4*>(xm + rr * 8), b = *reinterpret_cast<const float4*>(xm + rr * 8 + 4);
                    const float m_new = fmaxf(m_run[mt][hf], fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w))));
                    const float ms = m_new == -INFINITY ? 0.f : m_new;
                    alpha[mt][hf] = m_new == m_run[mt][hf] ? 1.f : pf::ex2(m_run[mt][hf] - m_new);
                    m_run[mt][hf] = m_new;
                    const float pa = pf::ex2(sc[mt][2 * hf] - ms), pb = pf::ex2(sc[mt][2 * hf + 1] - ms);
                    l_run[mt][hf] = fmaf(l_run[mt][hf], alpha[mt][hf], pa + pb);
                    uint32_t hi, lo;
                    rt::split2(make_float2(pa * kPScale, pb * kPScale), hi, lo);
                    unsigned char* at = p_s + size_t(rr) * 128 + ((w ^ (rr & 7)) << 4) + t4 * 4;
                    *reinterpret_cast<uint32_t*>(at) = hi;
                    *reinterpret_cast<uint32_t*>(at + size_t(R) * 128) = lo;
                }
            barrier();
            // ---- O += P V over this warp's 32 positions and 32 columns
            if (my_cols) {
                float4 vx[2][4];
                float mx = 0.f;
                unsigned least = ~0u;   // the smallest magnitude of any lane's four columns that are not all zeros, as bits minus one
                bool ok = true;
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = kh * 32 + st * 16 + 2 * t4 + (r & 1) + 8 * (r >> 1);
                        vx[st][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (key < ntok) vx[st][r] = *reinterpret_cast<const float4*>(vs_s + cbw * kSub + key * 128 + ((g ^ (key & 7)) << 4));
                        const float q = rt::max4(vx[st][r]);
                        mx = fmaxf(mx, q);
                        least = __viaddmin_u32(__float_as_uint(q), ~0u, least);
                        ok = ok && rt::finite4(vx[st][r]);
                    }
                ok = __all_sync(kFull, ok);
                if (!ok) {   // infinities and NaNs: left out here, added below for the rows that see them
                    mx = 0.f;
                    least = ~0u;
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float4& x = vx[st][r];
                            x.x = fabsf(x.x) < INFINITY ? x.x : 0.f;
                            x.y = fabsf(x.y) < INFINITY ? x.y : 0.f;
                            x.z = fabsf(x.z) < INFINITY ? x.z : 0.f;
                            x.w = fabsf(x.w) < INFINITY ? x.w : 0.f;
                            const float q = rt::max4(x);
                            mx = fmaxf(mx, q);
                            least = __viaddmin_u32(__float_as_uint(q), ~0u, least);
                        }
                }
                const float largest = warp_max(mx);
                unsigned small = 0u;   // of the 32 positions, those whose 32 columns are far below the largest: added below too
                if (__any_sync(kFull, least < __float_as_uint(largest * rt::kRowSpread))) {
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float q = rt::max4(vx[st][r]);
                            q = fmaxf(q, __shfl_xor_sync(kFull, q, 4));
                            q = fmaxf(q, __shfl_xor_sync(kFull, q, 8));
                            q = fmaxf(q, __shfl_xor_sync(kFull, q, 16));
                            if (!(q > 0.f && q < largest * rt::kRowSpread)) continue;
                            small |= 1u << (st * 16 + 2 * t4 + (r & 1) + 8 * (r >> 1));
                            vx[st][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                    small = __reduce_or_sync(kFull, small);
                }
                float up, fv;
                rt::scale_of(largest, up, fv);
                const float f = fv * (1.0f / kPScale);
                const float2 up2 = make_float2(up, up);
                // columns i of the lane's four go to the MMA's column tile i
                uint32_t bh[2][4][2], bl[2][4][2];
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float4 a = vx[st][2 * q], b = vx[st][2 * q + 1];
                        rt::split2(__fmul2_rn(make_float2(a.x, b.x), up2), bh[st][0][q], bl[st][0][q]);
                        rt::split2(__fmul2_rn(make_float2(a.y, b.y), up2), bh[st][1][q], bl[st][1][q]);
                        rt::split2(__fmul2_rn(make_float2(a.z, b.z), up2), bh[st][2][q], bl[st][2][q]);
                        rt::split2(__fmul2_rn(make_float2(a.w, b.w), up2), bh[st][3][q], bl[st][3][q]);
                    }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float c[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
                    const int rr = mt * 16 + (lane & 15);
                    uint32_t ah[2][4], al[2][4];
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        const uint32_t at = smem_u32(p_s) + uint32_t(rr) * 128 + uint32_t(((kh * 4 + st * 2 + (lane >> 4)) ^ (rr & 7)) << 4);
                        ldsm4(ah[st], at);
                        ldsm4(al[st], at + R * 128);
                    }
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma(c[i], al[st], bh[st][i][0], bh[st][i][1]);
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma(c[i], ah[st], bl[st][i][0], bl[st][i][1]);
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma(c[i], ah[st], bh[st][i][0], bh[st][i][1]);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const float al_ = alpha[mt][hf];
                        float4& x = o[mt][hf][0];
                        float4& y = o[mt][hf][1];
                        x = make_float4(fmaf(c[0][2 * hf], f, x.x * al_), fmaf(c[1][2 * hf], f, x.y * al_),
                                        fmaf(c[2][2 * hf], f, x.z * al_), fmaf(c[3][2 * hf], f, x.w * al_));
                        y = make_float4(fmaf(c[0][2 * hf + 1], f, y.x * al_), fmaf(c[1][2 * hf + 1], f, y.y * al_),
                                        fmaf(c[2][2 * hf + 1], f, y.z * al_), fmaf(c[3][2 * hf + 1], f, y.w * al_));
                    }
                }
                if (!ok || small != 0u) {
#pragma unroll 1
                    for (int k = 0; k < 32; ++k) {
                        const int key = kh * 32 + k;
                        if (key >= ntok) break;
                        float v[8];
                        bool any = false;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {   // the lane's columns 8 t .. 8 t + 7
                            v[i] = *reinterpret_cast<const float*>(vs_s + cbw * kSub + key * 128 + (((2 * t4 + (i >> 2)) ^ (key & 7)) << 4) + (i & 3) * 4);
                            if (fabsf(v[i]) < INFINITY && !(small >> k & 1u)) v[i] = 0.f;
                            else any = true;
                        }
                        if (!any) continue;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int hf = 0; hf < 2; ++hf) {
                                if (tok0 + key >= limit[mt][hf]) continue;
                                const int row = mt * 16 + hf * 8 + g;
                                const unsigned char* at = p_s + size_t(row) * 128 + (((key >> 3) ^ (row & 7)) << 4) + (key & 7) * 2;
                                const float pw = (__half2float(*reinterpret_cast<const __half*>(at)) +
                                                  __half2float(*reinterpret_cast<const __half*>(at + size_t(R) * 128))) * (1.0f / kPScale);
                                float4& x = o[mt][hf][0];
                                float4& y = o[mt][hf][1];
                                // (finite columns got 0 here; 0 * weight adds nothing to them unless the weight itself is no number)
                                x.x = fmaf(pw, v[0], x.x); x.y = fmaf(pw, v[1], x.y); x.z = fmaf(pw, v[2], x.z); x.w = fmaf(pw, v[3], x.w);
                                y.x = fmaf(pw, v[4], y.x); y.y = fmaf(pw, v[5], y.y); y.z = fmaf(pw, v[6], y.z); y.w = fmaf(pw, v[7], y.w);
                            }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[s]);
        }
        if (dead_flag[0] | dead_flag[1]) break;

        // ---- the unit's (or this block's part's) rows: sums over lanes and warps, O over the position halves
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                float l = l_run[mt][hf];
                l += __shfl_xor_sync(kFull, l, 1);
                l += __shfl_xor_sync(kFull, l, 2);
                const int rr = mt * 16 + hf * 8 + g;
                if (t4 == 0) {
                    xm[rr * 8 + w] = l;          // (the last tile's maxima have been read behind its second barrier)
                    if (w == 0) m_s[rr] = m_run[mt][hf];
                }
            }
        float4* o_s = reinterpret_cast<float4*>(q_s);   // [R][32 chunks], chunk c of row r at c ^ (r & 7): the query rows are done
        barrier();
        if (kh == 1 && my_cols) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int rr = mt * 16 + hf * 8 + g, ch = cbw * 8 + 2 * t4 + q;
                        o_s[rr * 32 + (ch ^ (rr & 7))] = o[mt][hf][q];
                    }
        }
        barrier();
        const bool whole = b1 == b0;
        const int slot = int(blk) == b0 ? 2 * int(blk) + 1 : 2 * int(blk);
        float* rec = partials + size_t(slot) * part_floats(MT, dp);
        if (kh == 0) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int rr = mt * 16 + hf * 8 + g, p = row0 + rr;
                    const float4 a = *reinterpret_cast<const float4*>(xm + rr * 8), b = *reinterpret_cast<const float4*>(xm + rr * 8 + 4);
                    const float l = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
                    if (p >= n_packed) continue;
                    const float inv = whole ? (limit[mt][hf] <= 0 ? 0.f : 1.0f / l) : 1.0f;   // (scores of -inf throughout: NaN)
                    const int head = h * tab.group + p % tab.group, t = p / tab.group;
                    if (cbw == 0 && t4 == 0) {
                        if (!whole) {
                            rec[size_t(R) * dp + rr] = m_s[rr];
                            rec[size_t(R) * dp + R + rr] = l;
                        } else if (want) {
                            e.lse[(long long)head * e.lse_hs + t] = limit[mt][hf] <= 0 ? INFINITY : (m_s[rr] + log2f(l)) * kLn2;
                        }
                    }
                    if (!my_cols) continue;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int ch = cbw * 8 + 2 * t4 + q, d = ch * 4;
                        if (d >= head_dim) continue;
                        const float4 y = o_s[rr * 32 + (ch ^ (rr & 7))], x = o[mt][hf][q];
                        const float4 v = make_float4((x.x + y.x) * inv, (x.y + y.y) * inv, (x.z + y.z) * inv, (x.w + y.w) * inv);
                        if (!whole) {
                            *reinterpret_cast<float4*>(rec + size_t(rr) * dp + d) = v;
                        } else {
                            float* row = e.out + (long long)head * e.o_hs + (long long)t * e.o_ts + d;
                            if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {   // (head_dim is a multiple of 4)
                                *reinterpret_cast<float4*>(row) = v;
                            } else {
                                row[0] = v.x; row[1] = v.y; row[2] = v.z; row[3] = v.w;
                            }
                        }
                    }
                }
        }
        barrier();   // partial records are written (and the exchange areas are free again)
        if (whole) continue;
        if (tid == 0) {
            __threadfence();
            const int old = atomicAdd(&sync[kSyncMerge0 + b0], 1);
            const int last = old == b1 - b0;
            if (last) {
                sync[kSyncMerge0 + b0] = 0;   // re-armed for the next launch
                __threadfence();
            }
            *last_flag = last;
        }
        barrier();
        if (!*last_flag) continue;
        const int count = b1 - b0 + 1;
        auto part_at = [&](int i) { return partials + size_t(2 * b0 + 1 + 2 * i - (i > 0 ? 1 : 0)) * part_floats(MT, dp); };
        for (int idx = tid; idx < R * nv; idx += 256) {
            const int rr = idx / nv, ch = idx % nv, p = row0 + rr;
            if (p >= n_packed) continue;
            float m = -INFINITY;
            for (int i = 0; i < count; ++i) m = fmaxf(m, __ldcg(part_at(i) + size_t(R) * dp + rr));
            float l = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < count; ++i) {
                const float* q = part_at(i);
                const float mi = __ldcg(q + size_t(R) * dp + rr);
                const float wgt = mi == -INFINITY ? 0.f : pf::ex2(mi - m);
                l = fmaf(__ldcg(q + size_t(R) * dp + R + rr), wgt, l);
                const float4 y = __ldcg(reinterpret_cast<const float4*>(q + size_t(rr) * dp) + ch);
                x.x = fmaf(wgt, y.x, x.x);
                x.y = fmaf(wgt, y.y, x.y);
                x.z = fmaf(wgt, y.z, x.z);
                x.w = fmaf(wgt, y.w, x.w);
            }
            const int head = h * tab.group + p % tab.group, t = p / tab.group;
            const bool sees = !e.causal || e.kv_len - e.rows + t >= 0;
            const float inv = sees ? 1.0f / l : 0.f;
            float* row = e.out + (long long)head * e.o_hs + (long long)t * e.o_ts + ch * 4;
            row[0] = x.x * inv; row[1] = x.y * inv; row[2] = x.z * inv; row[3] = x.w * inv;
            if (want && ch == 0) e.lse[(long long)head * e.lse_hs + t] = sees ? (m + log2f(l)) * kLn2 : INFINITY;
        }
    }
}

}  // namespace xn
