// Small kernels of the reads that do not append: rows that see nothing, and the account of
// attention weight of a read of few rows.
//
// The account of one KV head and position j is  a[j] = sum over the rows t and the heads of the
// group of  p[t][j] = exp(s[t][j] - lse[t]),  in f32.  It lives beside the cache pages (one float
// per KV head and position, paged like K and V), so that it moves with them.
#pragma once
#include "xn_common.cuh"

namespace xn {

// Where the account of one read goes.
struct AccountDev {
    float* user;           // caller's [num_kv_heads][user_hs] copy of the result, or nullptr
    long long user_hs;
    int old_from;          // what the new weights are added to: kAcct*
    int old_len;           // ... of the positions before this one (the others start at zero)
    int store;             // write the result into the paged account
    int kv_len;
    int page_off, layer;
};
enum : int { kAcctZero = 0, kAcctPool = 1, kAcctUser = 2 };

__device__ __forceinline__ size_t account_offset(const int* pages, long long pool_pages, int layer,
                                                 int num_kv_heads, int kv_head, int slot) {
    return ((size_t(layer) * size_t(pool_pages) + size_t(pages[slot / kPageTokens])) * num_kv_heads + kv_head) *
               kPageTokens + size_t(slot % kPageTokens);
}

__device__ __forceinline__ void account_store(const AccountDev& a, const int* page_ids, float* pool,
                                              long long pool_pages, int num_kv_heads, int kv_head, int key,
                                              float sum) {
    float* cell = nullptr;
    if (a.store || (a.old_from == kAcctPool && key < a.old_len))
        cell = pool + account_offset(page_ids + a.page_off, pool_pages, a.layer, num_kv_heads, kv_head, key);
    float* user = a.user ? a.user + size_t(kv_head) * size_t(a.user_hs) + key : nullptr;
    if (key < a.old_len) {
        if (a.old_from == kAcctPool) sum += *cell;
        else if (a.old_from == kAcctUser) sum += *user;
    }
    if (a.store) *cell = sum;
    if (user) *user = sum;
}

// One row block of a request in a launch of the kernel below.
struct FewAccount {
    AccountDev a;
    const float* scores;   // [num_heads][rows][sc_ts]
    const float* lse;      // [num_heads][rows]
    long long sc_hs, sc_ts, lse_hs;
    int rows;
    int row_limit0;        // positions the first row sees; row t sees row_limit0 + t * row_step
    int row_step;          // 1 causal, 0 otherwise
};

// (32 rows at a time: thousands of like weights added to one running sum round the same way every time --
// 16 000 of 1/79 were off by 1.6e-4, in blocks 3.5e-6)
__device__ __forceinline__ float account_sum(const FewAccount& r, int h, int group, int key) {
    float sum = 0.f;
    for (int t0 = 0; t0 < r.rows; t0 += 32) {
        float block = 0.f;
        for (int t = t0; t < min(r.rows, t0 + 32); ++t) {
            if (key >= r.row_limit0 + t * r.row_step) continue;
#pragma unroll 4
            for (int g = 0; g < group; ++g) {
                const size_t head = size_t(h) * group + g;
                const float s = r.scores[head * r.sc_hs + size_t(t) * r.sc_ts + key];
                block += expf(s - r.lse[head * r.lse_hs + t]);
            }
        }
        sum += block;
    }
    return sum;
}

// One thread per cached position, blockIdx.y = KV head, blockIdx.z = request: 4 (G rows + 1..2)
// bytes per position, read coalesced along the positions; a few per cent of what the attention
// kernel before it reads.  The sum's order is fixed (blocks of rows, rows, heads): the same bits every time.
__global__ void __launch_bounds__(256)
account_few_kernel(const FewAccount* __restrict__ reqs, const int* __restrict__ page_ids,
                   float* __restrict__ pool, long long pool_pages, int num_kv_heads, int group) {
    pdl_launch_dependents();
    const FewAccount r = reqs[blockIdx.z];
    const int key = int(blockIdx.x) * 256 + int(threadIdx.x);
    if (key >= r.a.kv_len) return;
    pdl_wait();            // scores and log-sum-exps come from the kernel before this one
    account_store(r.a, page_ids, pool, pool_pages, num_kv_heads, blockIdx.y, key, account_sum(r, blockIdx.y, group, key));
}

// The same for a read that came as a ReadTable.
__global__ void __launch_bounds__(256)
account_table_kernel(const __grid_constant__ ReadTable tab, float* __restrict__ pool, long long pool_pages, int num_kv_heads) {
    pdl_launch_dependents();
    const ReadEntry& e = tab.e[blockIdx.z];
    const int key = int(blockIdx.x) * 256 + int(threadIdx.x);
    if (key >= e.kv_len) return;
    const FewAccount r = {{e.user, e.user_hs, e.old_from, e.old_len, e.store, e.kv_len, 0, e.layer},
                          e.scores, e.lse, e.sc_hs, e.sc_ts, e.lse_hs, e.rows,
                          e.causal ? e.kv_len - e.rows + 1 : e.kv_len, e.causal};
    pdl_wait();
    account_store(r.a, e.pages, pool, pool_pages, num_kv_heads, blockIdx.y, key, account_sum(r, blockIdx.y, tab.group, key));
}

// Rows that see no position: zeros.
__global__ void __launch_bounds__(256)
zero_rows_kernel(float* __restrict__ out, long long o_hs, long long o_ts, int num_heads, int rows, int head_dim) {
    const long long total = (long long)num_heads * rows * head_dim;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const int d = int(e % head_dim);
        const long long row = e / head_dim;
        out[size_t(row / rows) * o_hs + size_t(row % rows) * o_ts + d] = 0.f;
    }
}

// The paged account of positions [t0, t0 + n): to or from a dense [num_kv_heads][n] array.
__global__ void __launch_bounds__(256)
account_copy_kernel(const int* __restrict__ pages, float* __restrict__ pool, long long pool_pages, int layer,
                    int num_kv_heads, int t0, int n, int valid, float* __restrict__ out,
                    const float* __restrict__ in) {
    const int i = int(blockIdx.x) * 256 + int(threadIdx.x), h = blockIdx.y;
    if (i >= n) return;
    float* cell = pool + account_offset(pages, pool_pages, layer, num_kv_heads, h, t0 + i);
    if (in) *cell = in[size_t(h) * n + i];
    if (out) out[size_t(h) * n + i] = t0 + i < valid ? *cell : 0.f;
}

// Positions [t0, t0 + n) of the paged account to zero (positions that had none so far).
__global__ void __launch_bounds__(256)
account_zero_kernel(const int* __restrict__ pages, float* __restrict__ pool, long long pool_pages, int layer,
                    int num_kv_heads, int t0, int n) {
    const int i = int(blockIdx.x) * 256 + int(threadIdx.x), h = blockIdx.y;
    if (i < n) pool[account_offset(pages, pool_pages, layer, num_kv_heads, h, t0 + i)] = 0.f;
}

}  // namespace xn
