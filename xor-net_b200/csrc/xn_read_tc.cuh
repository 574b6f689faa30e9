// Attention of many query rows over a cached prefix on the 5th-generation tensor cores (tcgen05),
// with f32-grade results: the read that does not append (cross attention), its causal form, and
// the account of attention weight of its rows.  sm_100a only.
//
//     S = Q K^T / sqrt(D),  P = softmax(S),  O = P V,  a[j] = sum over rows and group heads of P[.][j]
//
// Arithmetic.  Every f32 operand x is scaled by a power of two (per query row, per 64-token page of
// K and of V, so that the largest magnitude lies in [2^13, 2^14)) and split into two f16 values,
// x = hi + lo with hi = f16(x) and lo = f16(x - hi): 22 significand bits, and an absolute floor of
// 2^-39 of the page's (or row's) largest value for elements far below it.  A page's rows that are far
// larger or smaller than its median row are kept out of its scale and multiplied in f32, so that the
// floor is never above 2^-23 of a row's own largest element.  A product takes three MMAs, lo*hi +
// hi*lo + hi*hi, with f32 accumulators; the lo*lo term (2^-22 relative) is left out.  kind::f16 runs
// at twice the rate of kind::tf32, whose hi/lo split has as many bits, and its operands are half as
// large.  P is split the same way, scaled by 2^14: a weight has a floor of 2^-39 of its query row's
// largest.  Sums over more than 128 positions are not left to the tensor cores' accumulator: every
// 128-position tile of O starts from zero there and is added up in f32 registers; so are the softmax
// sums.
//
// Passes: (1) page_images_kernel writes K, V and Q once as hi/lo images in the shared-memory layout
// (128-byte swizzle) that the MMAs read, so that no later block converts anything; (2)
// read_tc_kernel, one block per (KV head, 128 packed query rows, range of pages), packed row =
// row * group + head of the group, so that the heads of a group share every K and V tile; (3)
// read_merge_kernel when a range was split; (4) account_tc_kernel for the attention weights.
#pragma once
#include <cuda_fp16.h>

#include "xn_common.cuh"
#include "xn_evict.cuh"
#include "xn_prefill_tf32.cuh"
#include "xn_read.cuh"

namespace xn {

// One request of a launch.
struct TcReq {
    const float* q;
    float* out;
    long long q_hs, q_ts, o_hs, o_ts;
    int rows;
    int kv_len;
    int causal;        // row t sees positions up to kv_len - rows + t; else all
    int page_off;
    int layer;
    int n_pages;       // pages of the prefix
    int n_qt;          // 128-row tiles of packed query rows per KV head
    long long img0;    // page image (page, head) = img0 + page * num_kv_heads + head
    long long qimg0;   // query image (head, tile) = qimg0 + head * n_qt + tile
    AccountDev acct;   // the account kernel's destination
};

// A block of read_tc_kernel: 128 packed rows of one KV head over pages [page_begin, page_end).
struct TcItem {
    int req, head, qt;
    int page_begin, page_end;
    int part;          // partial record, or -1: the block writes the output itself
};
// A row tile that was split over several items: its partial records are consecutive.
struct TcMerge {
    int req, head, qt;
    int part_begin, part_count;
    int pad;
};
// A block of account_tc_kernel: 128 positions of one KV head.
struct TcKeyTile {
    int req, head, tile, qt_begin;
};

// What the softmax needs to know about a page's K [0] and V [1]: factors that undo the scaling (of a V
// image that is all zeros: kZeroFactor), and the rows that hold an infinity or a NaN or are far larger or
// smaller than the page's others (their images are zero; they are added on the side, in f32).  any_bad: bit
// 0 there are such rows, bit 1 there are large ones among them.
struct __align__(16) PageMeta {
    float f[2];
    unsigned any_bad[2];
    unsigned long long bad[2];
};

// Where the cache rows are, for the rare exact path and the image kernel.
struct CacheView {
    const float* k;
    const float* v;
    const uint8_t* u8;
    long long pool_pages;
    int num_kv_heads, head_dim, nv, dq;
};

namespace rt {

constexpr int kBM = 128;
constexpr int kPage = 64;
constexpr int kSub = kPage * 128;        // one column block (64 halves) of one page
constexpr int kRowsSub = kBM * 128;      // one column block of 128 rows
constexpr float kPScale = 16384.0f;      // 2^14: P is split at this scale
constexpr float kRowSpread = 0x1p-16f;   // rows of a page that share a scale lie within this of one another
constexpr float kApart = 0x1p-10f;       // pages whose V factors are further apart than this do not share a sum
constexpr float kZeroFactor = 0x1p-100f; // (factors of other pages are 2^-73 and more: scale_of)
constexpr int kThreads = 320;            // copy warp, MMA warp, two softmax warpgroups
constexpr int kVStages = 3;
constexpr int kQBytes = 4 * kRowsSub;    // 64 KB: hi and lo, two column blocks
constexpr int kKBytes = 4 * kRowsSub;
constexpr int kVBytes = 4 * kSub;        // 32 KB
constexpr int kSmemData = kQBytes + kKBytes + kVStages * kVBytes;
constexpr int kSmemBytes = kSmemData + 3 * 1024;   // 227 KB, all there is: the block's window starts 1024-byte aligned
static_assert(kSmemBytes <= 232448, "shared memory of a block");
constexpr int kTmemS = 0;                // 2 x 128 columns
constexpr int kTmemO = 256;              // P_hi V_hi, then P_hi V_lo + P_lo V_hi: up to 128 columns each
constexpr int kSoftWarps = 8;

constexpr int kAcctStages = 3;           // 64 KB each: one K tile or 128 query rows
constexpr int kAcctSmemData = kAcctStages * kKBytes;
constexpr int kAcctSmemBytes = kAcctSmemData + 1024 + 4096;

__host__ __device__ inline int blocks_of(int head_dim) { return head_dim > 64 ? 2 : 1; }
__host__ __device__ inline size_t page_image_bytes(int head_dim) { return size_t(4) * blocks_of(head_dim) * kSub; }
__host__ __device__ inline size_t q_image_bytes(int head_dim) { return size_t(2) * blocks_of(head_dim) * kRowsSub; }
// a partial record: O [128][dp], then m [128], l [128]
__host__ __device__ inline size_t part_floats(int dp) { return size_t(kBM) * dp + 2 * kBM; }

// Instruction descriptor, kind::f16 with f16 operands and f32 accumulators.
__host__ __device__ constexpr uint32_t make_idesc16(int m, int n, int b_mn_major) {
    return (1u << 4) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void mma16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

// Power of two that brings a largest magnitude m into [2^13, 2^14), and its inverse.  Magnitudes
// below 2^-60 stay smaller than that, so that the product of two inverse factors never vanishes
// (masked scores are -inf times that product); nothing but zeros: as for 1.
__device__ __forceinline__ void scale_of(float m, float& up, float& down) {
    int e = int((__float_as_uint(m) >> 23) & 255u) - 127;
    e = m == 0.f ? 0 : max(e, -60);
    up = __uint_as_float(uint32_t(127 + 13 - e) << 23);
    down = __uint_as_float(uint32_t(127 - 13 + e) << 23);
}

// the larger of m and |x|, or NaN
__device__ __forceinline__ float max_nan(float m, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}

__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(taddr) : "memory");
    return r;
}

__device__ __forceinline__ void tmem_st1(uint32_t taddr, uint32_t v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(taddr), "r"(v) : "memory");
}

__device__ __forceinline__ bool finite4(const float4& x) {
    // x - x is 0 for finite x and NaN otherwise
    return (x.x - x.x) + (x.y - x.y) + (x.z - x.z) + (x.w - x.w) == 0.f;
}
__device__ __forceinline__ float max4(const float4& x) {
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// (hi, lo) f16 pairs of two f32 values
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __float22half2_rn(x);
    const float2 back = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    const float2 rest = __fadd2_rn(x, make_float2(-back.x, -back.y));
    lo = pack2(rest.x, rest.y);
}

// One arrival per warp: every lane's tensor-memory work is complete (wait::ld / wait::st) and ordered
// before it.
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
    pf::fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// Four scaled values of a lane (columns 4 * lane ..) into the hi and lo images of a row: column block
// lane / 16, 16-byte chunk (lane % 16) / 2 at chunk position chunk ^ (row & 7).
__device__ __forceinline__ void store_row_image(unsigned char* hi_img, unsigned char* lo_img, size_t block_stride,
                                                int row, int lane, int nb, float4 x, bool safe) {
    if ((lane >> 4) >= nb) return;
    uint2 hi, lo;
    split2(make_float2(x.x, x.y), hi.x, lo.x);
    split2(make_float2(x.z, x.w), hi.y, lo.y);
    if (!safe) lo = make_uint2(0u, 0u);   // a query row with an infinity: inf - inf must not become NaN
    const size_t at = size_t(lane >> 4) * block_stride + size_t(row) * 128 +
                      size_t((((lane & 15) >> 1) ^ (row & 7)) * 16 + (lane & 1) * 8);
    *reinterpret_cast<uint2*>(hi_img + at) = hi;
    *reinterpret_cast<uint2*>(lo_img + at) = lo;
}

// Four columns (4 * lane ..) of token tk of a cache block, zeros past the row's end.
__device__ __forceinline__ float4 cache_row4(const CacheView& c, size_t blk, int tk, int lane, bool v) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c.u8) {
        const uint8_t* b = c.u8 + blk * (size_t(kPage) * (2 * size_t(c.dq) + 8));
        if (lane * 4 < c.dq) {
            const float s = reinterpret_cast<const float*>(b + 2 * size_t(kPage) * c.dq)[(v ? kPage : 0) + tk];
            const uchar4 u = *reinterpret_cast<const uchar4*>(b + size_t((v ? kPage : 0) + tk) * c.dq + lane * 4);
            // (bytes past head_dim hold 128, but 0 * s is NaN for an infinite scale)
            if (lane * 4 + 0 < c.head_dim) x.x = (float(u.x) - 128.0f) * s;
            if (lane * 4 + 1 < c.head_dim) x.y = (float(u.y) - 128.0f) * s;
            if (lane * 4 + 2 < c.head_dim) x.z = (float(u.z) - 128.0f) * s;
            if (lane * 4 + 3 < c.head_dim) x.w = (float(u.w) - 128.0f) * s;
        }
    } else if (lane < c.nv) {   // rows are padded with zeros to whole float4
        x = *reinterpret_cast<const float4*>((v ? c.v : c.k) + (blk * kPage + tk) * size_t(c.nv) * 4 + size_t(lane) * 4);
    }
    return x;
}

// Four columns of a packed query row (row p of a KV head's group), zeros past the end.
__device__ __forceinline__ float4 query_row4(const TcReq& r, int head, int group, int p, int lane, int D, bool vec) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    const int d = lane * 4;
    if (p >= r.rows * group || d >= D) return x;
    const float* row = r.q + (long long)(head * group + p % group) * r.q_hs + (long long)(p / group) * r.q_ts + d;
    if (vec) return *reinterpret_cast<const float4*>(row);
    x.x = row[0];
    if (d + 1 < D) x.y = row[1];
    if (d + 2 < D) x.z = row[2];
    if (d + 3 < D) x.w = row[3];
    return x;
}
__device__ __forceinline__ bool query_vec(const TcReq& r, int D) {
    return (D & 3) == 0 && ((reinterpret_cast<uintptr_t>(r.q) | uintptr_t(r.q_hs * 4) | uintptr_t(r.q_ts * 4)) & 15) == 0;
}

// q . k of one query row and one cached row in f32, for the positions whose K is not in the images: k is
// the row's floats, or with u8 its bytes, of scale s.  (Not inlined: in line it takes registers from the
// loops around it, 447 us becomes 453 for 1024 rows over 8192 positions, 32/8 heads.)
__device__ __noinline__ float dot_row(const void* __restrict__ k, float s, bool u8, const float* __restrict__ q, bool vec, int D) {
    float dot = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
        float4 x, y;
        if (u8) {   // (bytes and floats behind head_dim are not looked at: 0 * s is NaN for an infinite scale)
            const uchar4 b = *reinterpret_cast<const uchar4*>(static_cast<const uint8_t*>(k) + d);
            x = make_float4((float(b.x) - 128.0f) * s, (float(b.y) - 128.0f) * s, (float(b.z) - 128.0f) * s, (float(b.w) - 128.0f) * s);
        } else {
            x = *reinterpret_cast<const float4*>(static_cast<const float*>(k) + d);
        }
        if (vec) {
            y = *reinterpret_cast<const float4*>(q + d);
        } else {
            y = make_float4(q[d], 0.f, 0.f, 0.f);
            if (d + 1 < D) y.y = q[d + 1]; else x.y = 0.f;
            if (d + 2 < D) y.z = q[d + 2]; else x.z = 0.f;
            if (d + 3 < D) y.w = q[d + 3]; else x.w = 0.f;
        }
        dot = fmaf(y.x, x.x, dot);
        dot = fmaf(y.y, x.y, dot);
        dot = fmaf(y.z, x.z, dot);
        dot = fmaf(y.w, x.w, dot);
    }
    return dot;
}
__device__ __forceinline__ float exact_dot(const CacheView& c, const int* pages, int layer, int head, int key, const float* q,
                                           bool vec, int D) {
    const size_t blk = (size_t(layer) * size_t(c.pool_pages) + size_t(pages[key / kPage])) * c.num_kv_heads + head;
    const int tk = key % kPage;
    if (!c.u8) return dot_row(c.k + (blk * kPage + tk) * size_t(c.nv) * 4, 0.f, false, q, vec, D);
    const uint8_t* b = c.u8 + blk * (size_t(kPage) * (2 * size_t(c.dq) + 8));
    return dot_row(b + size_t(tk) * c.dq, reinterpret_cast<const float*>(b + 2 * size_t(kPage) * c.dq)[tk], true, q, vec, D);
}

// One element of a cached row, whatever the format (rare paths only).
__device__ __forceinline__ float cache_elem(const CacheView& c, const int* pages, int layer, int head, int key, int d, bool v) {
    const size_t blk = (size_t(layer) * size_t(c.pool_pages) + size_t(pages[key / kPage])) * c.num_kv_heads + head;
    const int tk = key % kPage;
    if (c.u8) {
        const uint8_t* b = c.u8 + blk * (size_t(kPage) * (2 * size_t(c.dq) + 8));
        const float sc = reinterpret_cast<const float*>(b + 2 * size_t(kPage) * c.dq)[(v ? kPage : 0) + tk];
        return (float(b[size_t((v ? kPage : 0) + tk) * c.dq + d]) - 128.0f) * sc;
    }
    return (v ? c.v : c.k)[(blk * kPage + tk) * size_t(c.nv) * 4 + d];
}

}  // namespace rt

// Pass 1.  Blocks [0, 2 n_pages): K or V of one page of one KV head each; the rest: half a 128-row query
// tile each.  A warp handles eight rows, 4 columns per lane.  Bound by memory: 4 bytes read and 4
// written per element; blocks are small so that several per SM overlap one's loads with another's
// stores.
__global__ void __launch_bounds__(256, 4)
page_images_kernel(const TcReq* __restrict__ reqs, int n_reqs, long long n_pages,
                   const int* __restrict__ page_ids, CacheView c, unsigned char* __restrict__ images,
                   PageMeta* __restrict__ meta, unsigned char* __restrict__ q_images,
                   float2* __restrict__ row_meta, float scale_log2, int group, int* __restrict__ status) {
    using namespace rt;
    pdl_launch_dependents();
    __shared__ __align__(16) float s_max[8];
    __shared__ unsigned s_least[8];
    __shared__ __align__(8) unsigned char s_bad[8];
    __shared__ float s_row[kPage], s_median;
    constexpr unsigned kFull = 0xffffffffu;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = c.head_dim, nb = blocks_of(D);
    const bool is_q = (long long)blockIdx.x >= 2 * n_pages;
    const long long id = (is_q ? (long long)blockIdx.x - 2 * n_pages : (long long)blockIdx.x) >> 1;
    const int part = blockIdx.x & 1;      // K or V; half of the query tile
    pdl_wait();
    int rq = -1;                          // the last request that begins at or before id
    for (int i = 0; i < n_reqs; i += 32)
        rq += __popc(__ballot_sync(kFull, i + lane < n_reqs && id >= (is_q ? reqs[min(i + lane, n_reqs - 1)].qimg0
                                                                              : reqs[min(i + lane, n_reqs - 1)].img0)));
    const TcReq& r = reqs[rq];
    float4 x[8];
    if (!is_q) {
        const long long local = id - r.img0;
        const int page = int(local / c.num_kv_heads), h = int(local % c.num_kv_heads);
        const int page_id = page_ids[r.page_off + page];
        const bool page_ok = XN_PAGE_OK(page_id, c.pool_pages);
        if (!page_ok && threadIdx.x == 0) report_status(status, kDevBadIndex);
        const int ntok = page_ok ? min(kPage, r.kv_len - page * kPage) : 0;
        const size_t blk = (size_t(r.layer) * size_t(c.pool_pages) + size_t(page_id)) * c.num_kv_heads + h;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tk = warp * 8 + i;
            x[i] = tk < ntok ? cache_row4(c, blk, tk, lane, part != 0) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        // the largest magnitude, and the smallest of any lane's four columns that are not all zeros (as bits
        // minus one, so that zeros count as the largest)
        unsigned least = ~0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = max_nan(max_nan(max_nan(fabsf(x[i].x), x[i].y), x[i].z), x[i].w);
            m = max_nan(m, q);
            least = min(least, __float_as_uint(q) - 1u);
        }
        unsigned bits = __reduce_max_sync(kFull, __float_as_uint(m)), bad = 0;   // as bits: finite < infinity < NaN
        if (bits >= 0x7f800000u) {
            m = 0.f;
            least = ~0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!__all_sync(kFull, finite4(x[i]))) {
                    bad |= 1u << i;
                    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                m = fmaxf(m, max4(x[i]));
                least = min(least, __float_as_uint(max4(x[i])) - 1u);
            }
            bits = __reduce_max_sync(kFull, __float_as_uint(m));
        }
        least = __reduce_min_sync(kFull, least);
        if (lane == 0) {
            s_max[warp] = __uint_as_float(bits);
            s_least[warp] = least;
            s_bad[warp] = (unsigned char)bad;
        }
        __syncthreads();
        unsigned large = 0u;
        float page_max = fmaxf(max4(*reinterpret_cast<const float4*>(s_max)), max4(*reinterpret_cast<const float4*>(s_max + 4)));
#pragma unroll
        for (int i = 0; i < 8; ++i) least = min(least, s_least[i]);
        if (least != ~0u && __uint_as_float(least + 1u) < page_max * kRowSpread) {
            // Rows that share a scale have an absolute floor of 2^-39 of its largest element, which is a
            // matter of f32 only while their own largest ones lie within 2^16 of one another.  Rows further
            // than 2^8 from the median row's (zeros aside) leave the image and are added on the side, like
            // rows with an infinity.  (Seldom: the whole block comes here or nobody does.)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned row = __reduce_max_sync(kFull, __float_as_uint(max4(x[i])));
                if (lane == 0) s_row[warp * 8 + i] = __uint_as_float(row);
            }
            __syncthreads();
            if (threadIdx.x < kPage) {
                const float mine = s_row[threadIdx.x];
                int before = 0, all = 0;
                for (int i = 0; i < kPage; ++i) {
                    const float v = s_row[i];
                    all += v > 0.f;
                    before += v > 0.f && (v < mine || (v == mine && i < int(threadIdx.x)));
                }
                if (mine > 0.f && before == all / 2) s_median = mine;
            }
            __syncthreads();
            const float lo = s_median * 0x1p-8f, hi = s_median * 0x1p8f;
            large = page_max > hi ? 2u : 0u;
            page_max = 0.f;
            for (int i = 0; i < kPage; ++i)
                if (s_row[i] >= lo && s_row[i] <= hi) page_max = fmaxf(page_max, s_row[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float row = s_row[warp * 8 + i];
                if (row == 0.f || (row >= lo && row <= hi)) continue;
                bad |= 1u << i;
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (lane == 0) s_bad[warp] = (unsigned char)bad;
            __syncthreads();
        }
        const bool empty = page_max == 0.f;
        float up, down;
        scale_of(page_max, up, down);
        if (threadIdx.x == 0) {
            const unsigned long long rows = *reinterpret_cast<const unsigned long long*>(s_bad);
            PageMeta& pm = meta[id];
            // (a V page of zeros takes no part in the choice of its neighbour's scale; K's factor undoes scores)
            pm.f[part] = part && empty ? kZeroFactor : down;
            pm.any_bad[part] = (rows != 0 ? 1u : 0u) | large;
            pm.bad[part] = rows;
        }
        unsigned char* hi = images + size_t(id) * page_image_bytes(D) + size_t(part) * 2 * nb * kSub;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            store_row_image(hi, hi + size_t(nb) * kSub, kSub, warp * 8 + i, lane, nb,
                            make_float4(x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up), true);
    } else {
        const int local = int(id - r.qimg0);
        const int h = local / r.n_qt, qt = local % r.n_qt;
        const bool vec = query_vec(r, D);
        unsigned char* img = q_images + size_t(id) * q_image_bytes(D);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = query_row4(r, h, group, qt * kBM + part * 64 + warp * 8 + i, lane, D, vec);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int rr = part * 64 + warp * 8 + i;
            const float m = max_nan(max_nan(max_nan(max_nan(0.f, x[i].x), x[i].y), x[i].z), x[i].w);
            const unsigned bits = __reduce_max_sync(kFull, __float_as_uint(m));
            const bool ok = bits < 0x7f800000u;
            float up, down;
            scale_of(ok ? __uint_as_float(bits) : 1.f, up, down);
            store_row_image(img, img + size_t(nb) * kRowsSub, kRowsSub, rr, lane, nb,
                            make_float4(x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up), ok);
            // y: the log-sum-exp of the row, written by the attention kernel; rows past the end
            // (and rows that see nothing) keep +inf, which gives them no weight anywhere
            if (lane == 0) row_meta[size_t(id) * kBM + rr] = make_float2(down * scale_log2, INFINITY);
        }
    }
}

// Pass 2.  Shared memory: Q images 64 KB | K tile (two pages) 64 KB | three V pages of 32 KB.  Tensor
// memory: two S / P buffers of 128 columns, one O tile of 2 x 128.  What the MMAs cost decides the
// forms: one with A in tensor memory takes about 115 cycles for N = 128 and hardly more for N = 256
// (64 would be the arithmetic's time), so S = Q K^T reads both operands from shared memory and
// P_hi meets [V_hi | V_lo] as one N = 256 operand.  (With Q in tensor memory and three N = 128
// products: 5900 cycles per tile of 128 positions, all of them MMA time.)  K has one buffer, whose
// lo half is used first and refilled while the hi half is still read.  Roles (320 threads): warp 0
// copies images (1-D bulk copies), warp 1 issues the MMAs -- the S of tile j + 1 before the O of
// tile j, so that the softmax of a tile runs beside them -- and warps 2..9 are two softmax
// warpgroups: thread r of each owns packed row r; warpgroup w takes page w of every tile and columns
// [64 w, 64 w + 64) of O.  S is read from tensor memory, P goes back over it as hi (32 columns) and
// lo (32 columns).  Measured: 5000-5200 cycles per tile, 3070 of them MMA time; the rest is the way of
// its 128 KB of images into the SM (25 bytes per cycle and SM, 7 TB/s over all).  Before the first tile
// come 6000-9000 cycles of launch, Q and K latency, behind the last one 8000 of PV, sums and output.
// Every wait is bounded; on expiry the kernel records a status code, drains and returns.
__global__ void __launch_bounds__(rt::kThreads, 1)
read_tc_kernel(const TcReq* __restrict__ reqs, const TcItem* __restrict__ items, const int* __restrict__ page_ids,
               CacheView c, const unsigned char* __restrict__ images, const PageMeta* __restrict__ meta,
               const unsigned char* __restrict__ q_images, float2* __restrict__ row_meta,
               float* __restrict__ partials, float scale_log2, int group, int want_lse, int* __restrict__ status) {
    using namespace rt;
    using pf::fence_after_sync;
    using pf::fence_before_sync;
    using pf::mma_commit;
    using pf::smem_desc;
    using pf::tmem_ld32;
    using pf::tmem_st32;
    using pf::tmem_wait_ld;
    using pf::tmem_wait_st;
    extern __shared__ __align__(1024) unsigned char read_smem[];
    unsigned char* smem = read_smem;
    if (smem_u32(smem) & 1023u) {   // (the swizzled images need it; never seen otherwise)
        if (threadIdx.x == 0) report_status(status, kDevBadIndex);
        return;
    }
    unsigned char* q_s = smem;
    unsigned char* k_s = q_s + kQBytes;
    unsigned char* v_s = k_s + kKBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemData);
    uint64_t* q_full = bars + 0;
    uint64_t* k_full = bars + 1;               // [2]: lo, hi
    uint64_t* k_empty = k_full + 2;            // [2]
    uint64_t* v_full = k_empty + 2;            // [3]
    uint64_t* v_empty = v_full + kVStages;     // [3]
    uint64_t* s_full = v_empty + kVStages;     // [2]
    uint64_t* p_full = s_full + 2;             // [2]
    uint64_t* o_full = p_full + 2;
    uint64_t* o_empty = o_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
    // by tile parity: a fast warp of the next tile must not be seen by a slow one of this tile
    volatile int* sm_dead = abort_flag + 1;              // [2]
    float* xchg = reinterpret_cast<float*>(bars + 32);   // [2 tiles][2 warpgroups][128 rows]

    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const TcItem it = items[blockIdx.x];
    const TcReq& r = reqs[it.req];
    const int D = c.head_dim, nb = blocks_of(D);
    const int n_pages = it.page_end - it.page_begin;
    const int n_tiles = (n_pages + 1) / 2;
    const int k_steps = (D + 15) / 16;
    const int n_pv = (D + 15) / 16 * 16;
    const long long qid = r.qimg0 + (long long)it.head * r.n_qt + it.qt;
    const long long img0 = r.img0 + (long long)it.page_begin * c.num_kv_heads + it.head;

    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(o_full, 1);
        mbar_init(o_empty, kSoftWarps);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
        }
        for (int s = 0; s < kVStages; ++s) {
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], kSoftWarps);
        }
        *abort_flag = 0;
        sm_dead[0] = sm_dead[1] = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();   // the images come from the kernel before this one

    if (warp == 0) {
        // =============================== image copies ===============================
        if (lane == 0) {
            const size_t img_bytes = page_image_bytes(D);
            const size_t step = size_t(c.num_kv_heads) * img_bytes;   // next page of the same head
            const unsigned char* base = images + size_t(img0) * img_bytes;
            mbar_arrive_expect_tx(q_full, uint32_t(q_image_bytes(D)));
            bulk_g2s(q_s, q_images + size_t(qid) * q_image_bytes(D), uint32_t(q_image_bytes(D)), q_full);
            int k_tiles[2] = {0, 0}, v_pages = 0;          // asked for so far
            auto load_k = [&](int j, int part) -> bool {   // part 0: lo, 1: hi
                if (j > 0 && !mbar_spin_bounded(&k_empty[part], uint32_t((j - 1) & 1))) return false;
                const int np = min(2, n_pages - 2 * j), b0 = part ? 0 : nb;
                mbar_arrive_expect_tx(&k_full[part], uint32_t(np * nb) * kSub);
                ++k_tiles[part];
                for (int p = 0; p < np; ++p)
                    for (int b = b0; b < b0 + nb; ++b)
                        bulk_g2s(k_s + size_t(b) * kRowsSub + size_t(p) * kSub,
                                 base + size_t(2 * j + p) * step + size_t(b) * kSub, kSub, &k_full[part]);
                return true;
            };
            auto load_v = [&](int pg) -> bool {
                const int st = pg % kVStages;
                if (pg >= kVStages && !mbar_spin_bounded(&v_empty[st], uint32_t((pg / kVStages - 1) & 1))) return false;
                const uint32_t bytes = uint32_t(2 * nb) * kSub;
                mbar_arrive_expect_tx(&v_full[st], bytes);
                ++v_pages;
                bulk_g2s(v_s + size_t(st) * kVBytes, base + size_t(pg) * step + size_t(2 * nb) * kSub, bytes, &v_full[st]);
                return true;
            };
            bool ok = load_k(0, 0) && load_k(0, 1);
            for (int j = 0; j < n_tiles && ok; ++j) {
                if (j + 1 < n_tiles) ok = load_k(j + 1, 0) && load_k(j + 1, 1);
                for (int p = 2 * j; p < min(2 * j + 2, n_pages) && ok; ++p) ok = load_v(p);
                if (*abort_flag) break;
            }
            if (!ok) { report_status(status, kDevWaitEmpty); *abort_flag = 1; }
            if (*abort_flag) {   // nobody may be waiting for them any more: no copy outlives the block
                mbar_spin_bounded(q_full, 0);
                for (int part = 0; part < 2; ++part)
                    if (k_tiles[part]) mbar_spin_bounded(&k_full[part], uint32_t((k_tiles[part] - 1) & 1));
                for (int pg = max(0, v_pages - kVStages); pg < v_pages; ++pg)
                    mbar_spin_bounded(&v_full[pg % kVStages], uint32_t((pg / kVStages) & 1));
            }
        }
    } else if (warp == 1) {
        // =============================== MMA issuer ===============================
        if (lane == 0) {
            const uint32_t id_qk = make_idesc16(kBM, kBM, 0);
            const uint32_t id_pv = make_idesc16(kBM, nb * 64, 1);        // P_lo V_hi
            const uint32_t id_pv2 = make_idesc16(kBM, nb * 128, 1);      // P_hi [V_hi | V_lo]
            const uint64_t qd = smem_desc(smem_u32(q_s), 0, 1024, pf::kLayoutSw128);
            const uint64_t kd = smem_desc(smem_u32(k_s), 0, 1024, pf::kLayoutSw128);
            const uint64_t vd0 = smem_desc(smem_u32(v_s), kSub, 1024, pf::kLayoutSw128);
            const uint64_t lo_rows = uint64_t(nb) * kRowsSub >> 4;   // hi image -> lo image, 128 rows
            bool ok = mbar_spin_bounded(q_full, 0);
            if (!ok) { report_status(status, kDevWaitFull); *abort_flag = 1; }
            int v_st = 0, v_ph = 0;
            auto issue_qk = [&](int j) -> bool {
                if (!mbar_spin_bounded(&k_full[0], uint32_t(j & 1))) return false;
                fence_after_sync();
                const uint32_t d = tmem + kTmemS + (j & 1) * 128;
                auto term = [&](uint64_t a0, uint64_t b0, uint32_t acc) {
                    if (k_steps == 8) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint64_t o = uint64_t(ks >> 2) * (kRowsSub >> 4) + uint64_t(ks & 3) * 2;
                            mma16_ss(d, a0 + o, b0 + o, id_qk, ks > 0 ? 1u : acc);
                        }
                    } else {
                        for (int ks = 0; ks < k_steps; ++ks) {
                            const uint64_t o = uint64_t(ks >> 2) * (kRowsSub >> 4) + uint64_t(ks & 3) * 2;
                            mma16_ss(d, a0 + o, b0 + o, id_qk, ks > 0 ? 1u : acc);
                        }
                    }
                };
                // the small products first: they meet a small accumulator
                term(qd, kd + lo_rows, 0u);
                mma_commit(&k_empty[0]);
                if (!mbar_spin_bounded(&k_full[1], uint32_t(j & 1))) return false;
                fence_after_sync();
                term(qd + lo_rows, kd, 1u);
                term(qd, kd, 1u);
                mma_commit(&k_empty[1]);
                mma_commit(&s_full[j & 1]);
                return true;
            };
            auto issue_pv = [&](int j) -> bool {
                if (!mbar_spin_bounded(&p_full[j & 1], uint32_t((j >> 1) & 1))) return false;
                if (j >= 1 && !mbar_spin_bounded(o_empty, uint32_t((j - 1) & 1))) return false;
                const int np = min(2, n_pages - 2 * j);
                const uint32_t d = tmem + kTmemO;
                for (int p = 0; p < np; ++p) {
                    if (!mbar_spin_bounded(&v_full[v_st], uint32_t(v_ph))) return false;
                    fence_after_sync();
                    const uint64_t vd = vd0 + uint64_t(v_st) * (kVBytes >> 4);
                    const uint32_t pa = tmem + kTmemS + (j & 1) * 128 + p * 64;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) mma16_ts(d, pa + ks * 8, vd + ks * 128, id_pv2, (p > 0 || ks > 0) ? 1u : 0u);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) mma16_ts(d + nb * 64, pa + 32 + ks * 8, vd + ks * 128, id_pv, 1u);
                    mma_commit(&v_empty[v_st]);
                    if (++v_st == kVStages) { v_st = 0; v_ph ^= 1; }
                }
                mma_commit(o_full);
                return true;
            };
            for (int j = 0; j < n_tiles && ok; ++j) {
                if (!issue_qk(j)) { ok = false; break; }
                if (j >= 1 && !issue_pv(j - 1)) { ok = false; break; }
            }
            if (ok && !issue_pv(n_tiles - 1)) ok = false;
            if (!ok) { report_status(status, kDevWaitMma); *abort_flag = 1; }
        }
    } else {
        // =============================== softmax + epilogue ===============================
        constexpr unsigned kFull = 0xffffffffu;
        const int wg = (warp - 2) >> 2;
        const int quarter = warp & 3;
        const int rr = quarter * 32 + lane;               // row of the tile
        const uint32_t lane_base = uint32_t(quarter * 32) << 16;
        const int pr = it.qt * kBM + rr;                  // packed row
        const int n_packed = r.rows * group;
        const int t = pr / group;
        const int col0 = wg * 64;
        // positions below `limit` are visible
        const int limit = pr >= n_packed ? 0 : (r.causal ? r.kv_len - r.rows + t + 1 : r.kv_len);
        const int limit_first = r.causal ? r.kv_len - r.rows + (it.qt * kBM) / group + 1 : r.kv_len;
        const int* pages = page_ids + r.page_off;
        auto wg_barrier = [&]() { named_bar_sync(1, 256); };
        const float cq = __ldcg(&row_meta[size_t(qid) * kBM + rr]).x;
        const bool my_cols = col0 < n_pv;                 // head_dim <= 64: the second half has none

        float2 o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = make_float2(0.f, 0.f);
        float m_ref = -INFINITY, l_sum = 0.f;
        float alpha_prev = 1.f, f_prev = 0.f;             // pending accumulation of tile j - 1
        bool dead = false;
        auto scale_o = [&](float alpha) {                 // the maximum seldom moves after the first tiles
            if (!__any_sync(kFull, alpha != 1.f)) return;
            const float2 a2 = make_float2(alpha, alpha);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __fmul2_rn(o[i], a2);
        };
        // O = O * alpha + (tile j of tensor memory) * f
        auto add_tile = [&](int j, float alpha, float f) -> bool {
            scale_o(alpha);
            if (!warp_spin_bounded(o_full, uint32_t(j & 1), lane)) return false;
            fence_after_sync();
            if (my_cols) {
                const float2 f2 = make_float2(f, f);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t a[32];
                    tmem_ld32(tmem + kTmemO + nb * 64 + lane_base + col0 + hf * 32, a);   // the small products
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[hf * 16 + i] = __ffma2_rn(make_float2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), f2, o[hf * 16 + i]);
                    tmem_ld32(tmem + kTmemO + lane_base + col0 + hf * 32, a);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[hf * 16 + i] = __ffma2_rn(make_float2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), f2, o[hf * 16 + i]);
                }
            }
            warp_arrive(o_empty, lane);
            return true;
        };
        const PageMeta* pm = meta + img0;
        for (int j = 0; j < n_tiles; ++j) {
            const int sb = j & 1;
            const bool two = 2 * j + 1 < n_pages;
            const bool have = wg == 0 || two;
            // both pages' factors (uniform over the block)
            const PageMeta* pm0 = pm + size_t(2 * j) * c.num_kv_heads;
            const PageMeta* pm1 = two ? pm0 + c.num_kv_heads : pm0;
            const uint4 a0 = *reinterpret_cast<const uint4*>(pm0), a1 = *reinterpret_cast<const uint4*>(pm1);   // f[2], any_bad[2]
            const float fv0 = __uint_as_float(a0.y), fv1 = __uint_as_float(a1.y);
            const float cm = cq * __uint_as_float(wg ? a1.x : a0.x);
            // The products of both pages' V images go to one accumulator, so P of the page with the smaller
            // factor is scaled down by their ratio.  Up to 2^10 that leaves weights a resolution of 2^-29 of
            // the largest; a page further below keeps its P and is added on the side, row by row in f32.
            // (Below at all, where large rows are added on the side: they need the P.)
            const float fv = fmaxf(fv0, fv1), fv_low = fminf(fv0, fv1);
            const float apart_below = ((a0.w | a1.w) & 2u) ? 1.f : kApart;
            const bool bad_k = a0.z | a1.z;
            const bool bad_v = (a0.w | a1.w) != 0u || (fv_low < fv * kApart && fv_low != kZeroFactor);
            if (!warp_spin_bounded(&s_full[sb], uint32_t((j >> 1) & 1), lane)) dead = true;
            if (lane == 0 && dead) { sm_dead[sb] = 1; *abort_flag = 1; }
            fence_after_sync();
            const uint32_t s_addr = tmem + kTmemS + lane_base + sb * 128 + col0;
            const int key0 = (it.page_begin + 2 * j + wg) * kPage;
            const bool some_masked = key0 + kPage > limit_first;
            float mx = -INFINITY;
            if (!dead && have) {
                if (bad_k) {
                    // rows of K that are not in the image: their scores one by one, in f32, put where the
                    // MMA left zeros
                    unsigned long long b = (wg ? pm1 : pm0)->bad[0];
                    while (b) {
                        const int cidx = __ffsll((long long)b) - 1;
                        b &= b - 1;
                        float dot = 0.f;
                        if (pr < n_packed)
                            dot = exact_dot(c, pages, r.layer, it.head, key0 + cidx,
                                            r.q + size_t(it.head * group + pr % group) * r.q_hs + size_t(t) * r.q_ts, query_vec(r, D), D);
                        __syncwarp();
                        tmem_st1(s_addr + cidx, __float_as_uint(dot * scale_log2 / cm));
                    }
                }
                // the scores are read twice, 32 at a time: all 64 beside O's 64 registers would spill
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t x[32];
                    tmem_ld32(s_addr + hf * 32, x);
                    tmem_wait_ld();
                    if (some_masked) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (key0 + hf * 32 + i >= limit) x[i] = 0xff800000u;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(x[i]));
                }
                mx *= cm;
            }
            float* xc = xchg + sb * 256;
            xc[wg * 128 + rr] = mx;
            wg_barrier();
            dead = __any_sync(kFull, sm_dead[sb] != 0);
            if (dead) break;   // taken by all eight warps: the flag was set before the barrier
            mx = fmaxf(mx, xc[(wg ^ 1) * 128 + rr]);
            const float m_new = fmaxf(m_ref, mx);
            const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
            float alpha = m_new == m_ref ? 1.f : pf::ex2(m_ref - m_new);
            m_ref = m_new;
            l_sum *= alpha;
            if (have) {
                float pscale = (wg ? fv1 : fv0) / fv;   // powers of two: exact
                pscale = pscale < apart_below ? kPScale : kPScale * pscale;
                float2 ps = make_float2(0.f, 0.f);
                const float2 cm2 = make_float2(cm, cm), nm2 = make_float2(neg_m, neg_m), sc2 = make_float2(pscale, pscale);
                uint32_t hi[32], lo[32];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t x[32];
                    tmem_ld32(s_addr + hf * 32, x);
                    tmem_wait_ld();
                    if (some_masked) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (key0 + hf * 32 + i >= limit) x[i] = 0xff800000u;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 p = __ffma2_rn(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), cm2, nm2);
                        p.x = pf::ex2(p.x);
                        p.y = pf::ex2(p.y);
                        ps = __fadd2_rn(ps, p);
                        split2(__fmul2_rn(p, sc2), hi[hf * 16 + i], lo[hf * 16 + i]);
                    }
                }
                l_sum += ps.x + ps.y;
                tmem_st32(s_addr, hi);
                tmem_st32(s_addr + 32, lo);
                tmem_wait_st();
            }
            if (bad_v) {
                // rows of V that are not in the image, or all of a page that is set apart (uniform over the
                // block): bring O up to date, then add p * v for the rows that see them; P of both pages is
                // read back from tensor memory
                if (j > 0) {
                    if (!add_tile(j - 1, alpha_prev, f_prev)) { report_status(status, kDevWaitMma); *abort_flag = 1; }
                }
                scale_o(alpha);
                alpha = 1.f;
                fence_before_sync();
                wg_barrier();
                fence_after_sync();
                for (int p = 0; p < 2; ++p) {
                    const float fp = p ? fv1 : fv0;
                    const bool apart = fp < fv * apart_below, side = apart && fp != kZeroFactor;
                    unsigned long long b = p == 0 ? pm0->bad[1] : (two ? pm1->bad[1] : 0ull);
                    if (side) {
                        const int ntok = r.kv_len - (it.page_begin + 2 * j + p) * kPage;
                        b = ntok >= kPage ? ~0ull : (1ull << ntok) - 1;
                    }
                    const float unscale = apart ? 1.0f / kPScale : fv / (kPScale * fp);
                    while (b) {
                        const int cidx = __ffsll((long long)b) - 1;
                        b &= b - 1;
                        uint32_t hw = tmem_ld1(tmem + kTmemS + lane_base + sb * 128 + p * 64 + cidx / 2);
                        uint32_t lw = tmem_ld1(tmem + kTmemS + lane_base + sb * 128 + p * 64 + 32 + cidx / 2);
                        const float2 h2 = __half22float2(*reinterpret_cast<__half2*>(&hw));
                        const float2 l2 = __half22float2(*reinterpret_cast<__half2*>(&lw));
                        const float pv = ((cidx & 1) ? h2.y + l2.y : h2.x + l2.x) * unscale;
                        const int key = (it.page_begin + 2 * j + p) * kPage + cidx;
                        // the row of V through the exchange area of the tile before (nobody reads that now)
                        float* vrow = xchg + (sb ^ 1) * 256;
                        const int e = tid - 64;
                        if (e < 128) vrow[e] = e < D ? cache_elem(c, pages, r.layer, it.head, key, e, true) : 0.f;
                        wg_barrier();
                        if (key < limit) {   // (a weight of zero times an infinity is a NaN, as in a plain sum)
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                o[i].x = fmaf(pv, vrow[col0 + 2 * i], o[i].x);
                                o[i].y = fmaf(pv, vrow[col0 + 2 * i + 1], o[i].y);
                            }
                        }
                        wg_barrier();
                    }
                }
                fence_before_sync();
                wg_barrier();
                if ((wg ? fv1 : fv0) < fv * apart_below) {   // nothing of that page is left for the MMAs
                    fence_after_sync();
#pragma unroll 1
                    for (int i = 0; i < 64; ++i) tmem_st1(s_addr + i, 0u);
                }
            } else if (j > 0) {
                warp_arrive(&p_full[sb], lane);
                if (!add_tile(j - 1, alpha_prev, f_prev)) { report_status(status, kDevWaitMma); *abort_flag = 1; }
                alpha_prev = alpha;
                f_prev = fv * (1.0f / kPScale);
                continue;
            }
            alpha_prev = alpha;
            f_prev = fv * (1.0f / kPScale);
            warp_arrive(&p_full[sb], lane);
        }
        if (dead && lane == 0) report_status(status, kDevWaitFull);
        if (!dead) {
            if (!add_tile(n_tiles - 1, alpha_prev, f_prev)) { report_status(status, kDevWaitMma); *abort_flag = 1; }
            // (the exchange area of the tile before the last one: every thread has read the last one's
            // only behind the barrier below)
            float* xc = xchg + (n_tiles & 1) * 256;
            xc[wg * 128 + rr] = l_sum;
            wg_barrier();
            const float l_tot = l_sum + xc[(wg ^ 1) * 128 + rr];
            const bool whole = it.part < 0;
            const float inv = whole ? (limit <= 0 ? 0.f : 1.0f / l_tot) : 1.0f;   // (scores of -inf throughout: NaN)
            if (wg == 0) {
                if (!whole) {
                    float* rec = partials + size_t(it.part) * part_floats(c.nv * 4) + size_t(kBM) * c.nv * 4;
                    rec[rr] = m_ref;
                    rec[kBM + rr] = l_tot;
                } else if (want_lse && limit > 0) {
                    row_meta[size_t(qid) * kBM + rr].y = m_ref + log2f(l_tot);
                }
            }
            // through shared memory (the K tile is idle) so that whole rows leave in one instruction
            float4* tile = reinterpret_cast<float4*>(k_s);   // [128 rows][32 chunks]
            if (my_cols) {
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const int chunk = (col0 >> 2) + (i >> 1);
                    tile[rr * 32 + (chunk ^ (rr & 31))] = make_float4(o[i].x * inv, o[i].y * inv, o[i + 1].x * inv, o[i + 1].y * inv);
                }
            }
            wg_barrier();
            // 16 rows per warp; lane i knows where row i goes
            const int w8 = warp - 2;
            const int my_p = it.qt * kBM + w8 * 16 + (lane & 15);
            const bool vec = (D & 3) == 0 && ((reinterpret_cast<uintptr_t>(r.out) | uintptr_t(r.o_hs * 4) | uintptr_t(r.o_ts * 4)) & 15) == 0;
            const long long my_off = whole ? (long long)(it.head * group + my_p % group) * r.o_hs + (long long)(my_p / group) * r.o_ts
                                           : (long long)(w8 * 16 + (lane & 15)) * c.nv * 4;
            float* dst = whole ? r.out : partials + size_t(it.part) * part_floats(c.nv * 4);
            const int n_rows = min(16, n_packed - it.qt * kBM - w8 * 16);
#pragma unroll 4
            for (int i = 0; i < 16; ++i) {
                float* row = dst + __shfl_sync(kFull, my_off, i) + lane * 4;
                if (i >= n_rows || lane >= c.nv) continue;
                const float4 x = tile[(w8 * 16 + i) * 32 + (lane ^ ((w8 * 16 + i) & 31))];
                if (vec || !whole) {
                    *reinterpret_cast<float4*>(row) = x;
                } else {
                    row[0] = x.x;
                    if (lane * 4 + 1 < D) row[1] = x.y;
                    if (lane * 4 + 2 < D) row[2] = x.z;
                    if (lane * 4 + 3 < D) row[3] = x.w;
                }
            }
        }
    }

    fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Pass 3.  The partial records of a split row tile, combined with their log-sum-exp weights: one warp
// per row, the tile's rows over blockIdx.y.
__global__ void __launch_bounds__(256)
read_merge_kernel(const TcReq* __restrict__ reqs, const TcMerge* __restrict__ merges,
                  const float* __restrict__ partials, float2* __restrict__ row_meta, int group, int head_dim,
                  int nv, int want_lse) {
    using namespace rt;
    pdl_launch_dependents();
    const TcMerge mg = merges[blockIdx.x];
    const TcReq& r = reqs[mg.req];
    const int lane = threadIdx.x & 31;
    const int i = int(blockIdx.y) * 8 + int(threadIdx.x >> 5);
    const int p = mg.qt * kBM + i;
    if (p >= r.rows * group) return;
    pdl_wait();
    const size_t stride = part_floats(nv * 4);
    const float* rec = partials + size_t(mg.part_begin) * stride;
    const float* ml = rec + size_t(kBM) * nv * 4;
    float m = -INFINITY;
    for (int k = 0; k < mg.part_count; ++k) m = fmaxf(m, ml[size_t(k) * stride + i]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < mg.part_count; ++k) {
        const float mk = ml[size_t(k) * stride + i];
        const float w = mk == -INFINITY ? 0.f : pf::ex2(mk - m);
        l = fmaf(ml[size_t(k) * stride + kBM + i], w, l);
        if (lane < nv) {
            const float4 x = *reinterpret_cast<const float4*>(rec + size_t(k) * stride + size_t(i) * nv * 4 + lane * 4);
            o.x = fmaf(w, x.x, o.x);
            o.y = fmaf(w, x.y, o.y);
            o.z = fmaf(w, x.z, o.z);
            o.w = fmaf(w, x.w, o.w);
        }
    }
    const bool sees = !r.causal || r.kv_len - r.rows + p / group >= 0;
    const float inv = sees ? 1.0f / l : 0.f;
    float* row = r.out + size_t(mg.head * group + p % group) * r.o_hs + size_t(p / group) * r.o_ts;
    const int d = lane * 4;
    if (d + 0 < head_dim) row[d + 0] = o.x * inv;
    if (d + 1 < head_dim) row[d + 1] = o.y * inv;
    if (d + 2 < head_dim) row[d + 2] = o.z * inv;
    if (d + 3 < head_dim) row[d + 3] = o.w * inv;
    if (want_lse && lane == 0 && sees)
        row_meta[size_t(r.qimg0 + (long long)mg.head * r.n_qt + mg.qt) * kBM + i].y = m + log2f(l);
}

// The three image slots of account_tc_kernel: one holds the K tile, the query images alternate between
// the other two; the next K tile takes the one of those that falls free first.
struct AcctSlots {
    int k = 0, q0 = 1, q1 = 2;
    __device__ int q(int j) const { return j & 1 ? q1 : q0; }
    __device__ void next(int n_q) {
        const int free = n_q & 1 ? q1 : q0, last = n_q & 1 ? q0 : q1;
        q1 = k;
        q0 = last;
        k = free;
    }
};

// Pass 4.  The account: S^T = K Q^T for 128 positions of one KV head against every tile of 128 packed
// query rows that sees them, p = 2^(s - lse), summed over the rows in f32.  Positions are the rows of
// the accumulator, so a thread owns a position and the sum needs no exchange and no atomics (its
// order is fixed).  Half the MMAs of the attention itself.  Roles as above.  Blocks are resident and
// take their share of the key tiles, the next K tile arriving in the third image slot during the sums
// of this one (2 requests x 64 rows over 4097-6001 positions, 8 heads: 27 us; with a block per tile,
// loads and sums in turn, 42).  With few positions and many rows the row tiles are dealt out to a
// cluster of blocks, whose first block adds up the sums through the others' shared memory.  Bound by
// the images' way into the SM: 64 KB per 128 x 128 scores, 2600 cycles beside 1540 of MMA time.
__global__ void __launch_bounds__(rt::kThreads, 1)
account_tc_kernel(const TcReq* __restrict__ reqs, const TcKeyTile* __restrict__ tiles, int n_tiles, const int* __restrict__ page_ids,
                  CacheView c, const unsigned char* __restrict__ images, const PageMeta* __restrict__ meta,
                  const unsigned char* __restrict__ q_images, const float2* __restrict__ row_meta,
                  float* __restrict__ pool, float scale_log2, int group, int cluster, int* __restrict__ status) {
    using namespace rt;
    using pf::fence_after_sync;
    using pf::fence_before_sync;
    using pf::mma_commit;
    using pf::smem_desc;
    using pf::tmem_ld32;
    using pf::tmem_wait_ld;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    float2* rm_s = reinterpret_cast<float2*>(smem + kAcctSmemData);   // [2][128]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kAcctSmemData + 2 * kBM * 8);
    uint64_t* full = bars + 0;       // [3], of the ring of images
    uint64_t* empty = bars + 3;      // [3]
    uint64_t* s_full = bars + 6;     // [2]
    uint64_t* s_empty = bars + 8;    // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 10);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
    float* xchg = reinterpret_cast<float*>(bars + 16);        // [2][128]

    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = int(ev::cluster_rank());
    const int D = c.head_dim, nb = blocks_of(D);
    const int k_steps = (D + 15) / 16;
    const int stride = int(gridDim.x) / cluster, first = int(blockIdx.x) / cluster;
    // the block's tiles, heaviest first, every other round from the light end
    auto tile_at = [&](int round) { return round * stride + ((round & 1) ? stride - 1 - first : first); };
    const int n_rounds = (n_tiles + stride - 1) / stride;
    const TcKeyTile kt0 = tiles[first];   // (plan data: there before the kernel before this one ends)
    auto key_tile = [&](int round) { return round == 0 ? kt0 : tiles[tile_at(round)]; };
    auto row_tiles = [&](const TcKeyTile& kt) {   // row tiles rank, rank + cluster, ...
        const int n = reqs[kt.req].n_qt - kt.qt_begin;
        return n > rank ? (n - rank - 1) / cluster + 1 : 0;
    };
    auto image0 = [&](const TcKeyTile& kt) { return reqs[kt.req].img0 + (long long)(2 * kt.tile) * c.num_kv_heads + kt.head; };
    if (tid == 0) {
        for (int s = 0; s < kAcctStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_empty[s], kSoftWarps);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(256u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            const size_t img_bytes = page_image_bytes(D);
            const uint32_t q_bytes = uint32_t(q_image_bytes(D));
            bool ok = true;
            int js = 0;                     // query images so far
            unsigned used = 0, odd = 0;     // per slot: used before; parity of its uses
            AcctSlots sl;
            auto take = [&](int s, uint32_t bytes) -> bool {
                if ((used >> s & 1u) && !mbar_spin_bounded(&empty[s], (odd >> s & 1u) ^ 1u)) return false;
                mbar_arrive_expect_tx(&full[s], bytes);
                used |= 1u << s;
                odd ^= 1u << s;
                return true;
            };
            for (int round = 0; round < n_rounds && ok; ++round) {
                if (tile_at(round) >= n_tiles) continue;
                const TcKeyTile kt = key_tile(round);
                const TcReq& r = reqs[kt.req];
                const int np = min(2, r.n_pages - 2 * kt.tile), n_q = row_tiles(kt);
                const long long qid0 = r.qimg0 + (long long)kt.head * r.n_qt + kt.qt_begin + rank;
                const int ks = sl.k;
                if (!take(ks, uint32_t(np * 2 * nb) * kSub)) { ok = false; break; }
                for (int p = 0; p < np; ++p)
                    for (int b = 0; b < 2 * nb; ++b)
                        bulk_g2s(smem + size_t(ks) * kKBytes + size_t(b) * kRowsSub + size_t(p) * kSub,
                                 images + (size_t(image0(kt)) + size_t(p) * c.num_kv_heads) * img_bytes + size_t(b) * kSub, kSub, &full[ks]);
                for (int j = 0; j < n_q; ++j, ++js) {
                    // (the row factors of two query images before have been read)
                    if (js >= 2 && !mbar_spin_bounded(&s_empty[js & 1], uint32_t(((js >> 1) - 1) & 1))) { ok = false; break; }
                    const int qs = sl.q(j);
                    if (!take(qs, q_bytes + kBM * 8)) { ok = false; break; }
                    bulk_g2s(smem + size_t(qs) * kKBytes, q_images + size_t(qid0 + j * cluster) * q_bytes, q_bytes, &full[qs]);
                    bulk_g2s(rm_s + (js & 1) * kBM, row_meta + size_t(qid0 + j * cluster) * kBM, kBM * 8, &full[qs]);
                }
                sl.next(n_q);
                if (*abort_flag) break;
            }
            if (!ok) { report_status(status, kDevWaitEmpty); *abort_flag = 1; }
            if (*abort_flag)     // (as above)
                for (int s = 0; s < kAcctStages; ++s)
                    if (used >> s & 1u) mbar_spin_bounded(&full[s], (odd >> s & 1u) ^ 1u);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = make_idesc16(kBM, kBM, 0);
            const uint64_t d0 = smem_desc(smem_u32(smem), 0, 1024, pf::kLayoutSw128);
            const uint64_t lo_rows = uint64_t(nb) * kRowsSub >> 4;
            bool ok = true;
            int js = 0;
            unsigned odd = 0;
            AcctSlots sl;
            auto filled = [&](int s) -> bool {
                const bool there = mbar_spin_bounded(&full[s], odd >> s & 1u);
                odd ^= 1u << s;
                return there;
            };
            for (int round = 0; round < n_rounds && ok; ++round) {
                if (tile_at(round) >= n_tiles) continue;
                const int n_q = row_tiles(key_tile(round));
                const int k_slot = sl.k;
                if (!filled(k_slot)) { ok = false; break; }
                for (int j = 0; j < n_q; ++j, ++js) {
                    const int s = js & 1, q_slot = sl.q(j);
                    if (!filled(q_slot) || (js >= 2 && !mbar_spin_bounded(&s_empty[s], uint32_t(((js >> 1) - 1) & 1)))) { ok = false; break; }
                    fence_after_sync();
                    const uint64_t kd = d0 + uint64_t(k_slot) * (kKBytes >> 4), qd = d0 + uint64_t(q_slot) * (kKBytes >> 4);
                    const uint32_t d = tmem + s * 128;
#pragma unroll
                    for (int term = 0; term < 3; ++term) {
                        const uint64_t a0 = kd + (term == 0 ? lo_rows : 0), b0 = qd + (term == 1 ? lo_rows : 0);
                        for (int ks = 0; ks < k_steps; ++ks) {
                            const uint64_t o = uint64_t(ks >> 2) * (kRowsSub >> 4) + uint64_t(ks & 3) * 2;
                            mma16_ss(d, a0 + o, b0 + o, idesc, (term > 0 || ks > 0) ? 1u : 0u);
                        }
                    }
                    mma_commit(&empty[q_slot]);
                    mma_commit(&s_full[s]);
                }
                mma_commit(&empty[k_slot]);
                sl.next(n_q);
            }
            if (!ok) { report_status(status, kDevWaitMma); *abort_flag = 1; }
        }
    } else {
        const int wg = (warp - 2) >> 2;
        const int quarter = warp & 3;
        const int rr = quarter * 32 + lane;
        const uint32_t lane_base = uint32_t(quarter * 32) << 16;
        bool dead = false;
        int js = 0, tp = 0;
        for (int round = 0; round < n_rounds; ++round) {
            if (tile_at(round) >= n_tiles) continue;
            const TcKeyTile kt = key_tile(round);
            const TcReq& r = reqs[kt.req];
            const int n_q = row_tiles(kt);
            const int key = kt.tile * kBM + rr;
            const bool in = key < r.kv_len;
            const int* pages = page_ids + r.page_off;
            const PageMeta& pm = meta[image0(kt) + (rr >= kPage && 2 * kt.tile + 1 < r.n_pages ? c.num_kv_heads : 0)];
            const float fk = pm.f[0];
            const bool bad = in && ((pm.bad[0] >> (rr & 63)) & 1);
            const unsigned bad_lanes = __ballot_sync(0xffffffffu, bad);
            // packed rows from `first_row` on see the position
            const int first_row = r.causal ? max(0, (key - (r.kv_len - r.rows)) * group) : 0;
            float sum = 0.f;
            for (int j = 0; j < n_q && !dead; ++j, ++js) {
                const int s = js & 1;
                if (!warp_spin_bounded(&s_full[s], uint32_t((js >> 1) & 1), lane)) { dead = true; break; }
                fence_after_sync();
                const int row0 = (kt.qt_begin + rank + j * cluster) * kBM + wg * 64;
                const float2* rm = rm_s + s * kBM + wg * 64;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t x[32];
                    tmem_ld32(tmem + lane_base + s * 128 + wg * 64 + hf * 32, x);
                    tmem_wait_ld();
                    const int from = first_row - (row0 + hf * 32);   // columns before this one do not count
                    float s0 = 0.f, s1 = 0.f;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float4 f = *reinterpret_cast<const float4*>(rm + hf * 32 + i);
                        const float a = pf::ex2(fmaf(__uint_as_float(x[i]) * fk, f.x, -f.y));
                        const float b = pf::ex2(fmaf(__uint_as_float(x[i + 1]) * fk, f.z, -f.w));
                        s0 += i >= from ? a : 0.f;
                        s1 += i + 1 >= from ? b : 0.f;
                    }
                    if (!bad) sum += s0 + s1;
                    // positions whose K is not in the image: a lane per query row
                    for (unsigned left = bad_lanes; left != 0u; left &= left - 1) {
                        const int src = __ffs(int(left)) - 1, p = row0 + hf * 32 + lane;
                        const int from_row = __shfl_sync(0xffffffffu, first_row, src);
                        float w = 0.f;
                        if (p >= from_row && p < r.rows * group)
                            w = pf::ex2(exact_dot(c, pages, r.layer, kt.head, key - lane + src,
                                                  r.q + size_t(kt.head * group + p % group) * r.q_hs + size_t(p / group) * r.q_ts,
                                                  query_vec(r, D), D) * scale_log2 - rm[hf * 32 + lane].y);
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
                        if (lane == src) sum += w;
                    }
                }
                warp_arrive(&s_empty[s], lane);
            }
            // the two halves of the rows (a warp that gave up waiting still comes to every barrier)
            float* xc = xchg + tp * kBM;
            if (wg == 1) xc[rr] = sum;
            named_bar_sync(1, 256);
            if (wg == 0) {
                sum += xc[rr];
                if (cluster > 1) xc[rr] = sum;   // (one tile per block then)
                else if (in && !dead) account_store(r.acct, page_ids, pool, c.pool_pages, c.num_kv_heads, kt.head, key, sum);
            }
            tp ^= 1;
        }
        if (dead && lane == 0) { report_status(status, kDevWaitFull); *abort_flag = 1; }
    }
    __syncwarp();

    fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
    }
    if (cluster > 1) {
        __syncwarp();
        ev::cluster_sync_all();
        const TcKeyTile kt = kt0;
        const TcReq& r = reqs[kt.req];
        const int key = kt.tile * kBM + tid;
        if (rank == 0 && tid < kBM && key < r.kv_len) {
            float sum = xchg[tid];
            for (int p = 1; p < cluster; ++p) sum += __uint_as_float(ev::peer_ld(&xchg[tid], uint32_t(p)));
            account_store(r.acct, page_ids, pool, c.pool_pages, c.num_kv_heads, kt.head, key, sum);
        }
        __syncwarp();
        ev::cluster_sync_all();   // no block leaves while its sums are read
    }
}

}  // namespace xn
