// Host side of the reads that do not append, of the account of attention weight and of eviction:
// argument checks, planning, launches.  Included by xn_attn.cu inside its unnamed namespace, after
// the submission code whose buffers and plan slots it shares; every function runs under the
// context's lock.
#pragma once

// The caller's current device, put back on the way out.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before != device) cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Plan slots are reused once their launches are done, staging is grown, events are waited for: none
// of it can be recorded into a graph and replayed.
int32_t refuse_capture(xn_ctx* c) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    XN_CUDA(c, cudaStreamIsCapturing(c->stream, &st));
    if (st != cudaStreamCaptureStatusNone)
        return fail(c, XN_ERR_ARG, "this call cannot be captured into a CUDA graph");
    return XN_OK;
}

int32_t ensure_account_pool(xn_ctx* c) {
    if (c->acct_pool) return XN_OK;
    const size_t n = size_t(c->pool_pages) * c->num_layers * c->num_kv_heads * kPageTokens;
    XN_CUDA(c, guarded_malloc(c, reinterpret_cast<void**>(&c->acct_pool), n * 4, "account"));
    XN_CUDA(c, cudaMemsetAsync(c->acct_pool, 0, n * 4, c->stream));
    return XN_OK;
}

int64_t layer_len(const xn_stream* s, int layer) { return std::min(s->hw[size_t(layer)], s->cap); }

// The launches behind a plan are recorded so that its slot is not reused before they are done.
int32_t finish_slot(xn_ctx* c, PlanSlot* slot) {
    XN_CUDA(c, cudaGetLastError());
    XN_CUDA(c, cudaEventRecord(slot->ev, c->stream));
    slot->used = true;
    return XN_OK;
}

int32_t upload_slot(xn_ctx* c, PlanSlot* slot, size_t bytes) {
    XN_CUDA(c, cudaMemcpyAsync(slot->dev, slot->host, bytes, cudaMemcpyHostToDevice, c->copy_stream));
    XN_CUDA(c, cudaEventRecord(slot->up_ev, c->copy_stream));
    XN_CUDA(c, cudaStreamWaitEvent(c->stream, slot->up_ev, 0));
    c->stats.h2d_bytes += bytes;
    return XN_OK;
}

// A plan under construction: arrays placed one behind the other, copied to a slot at the end.
struct PlanBuf {
    std::vector<unsigned char> data;
    template <class T>
    size_t put(const std::vector<T>& v) {
        const size_t at = align_up(data.size(), 16);
        data.resize(at + v.size() * sizeof(T));
        if (!v.empty()) memcpy(data.data() + at, v.data(), v.size() * sizeof(T));
        return at;
    }
};

int32_t commit_plan(xn_ctx* c, const PlanBuf& b, PlanSlot** out) {
    const size_t bytes = std::max<size_t>(16, align_up(b.data.size(), 16));
    int32_t rc = acquire_slot(c, bytes, out);
    if (rc != XN_OK) return rc;
    if (!b.data.empty()) memcpy((*out)->host, b.data.data(), b.data.size());
    return upload_slot(c, *out, bytes);
}

// A launch that may start while its predecessor drains (the kernel waits before it reads or writes
// what the predecessor touches).
template <class... KArgs, class... Args>
cudaError_t launch_pdl(xn_ctx* c, void (*fn)(KArgs...), dim3 grid, int threads, size_t smem, bool pdl,
                       unsigned cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = c->stream;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (pdl && !c->profile) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim = {cluster, 1, 1};
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    c->stats.kernel_launches += 1;
    return cudaLaunchKernelEx(&cfg, fn, static_cast<KArgs>(args)...);
}

// ---- rows into a stream -----------------------------------------------------------------------

int32_t kv_write_locked(xn_ctx* c, xn_stream* s, int32_t layer, int64_t t0, int64_t n, const float* k,
                        const float* v, uint32_t flags) {
    if (!stream_ok(c, s)) return fail(c, XN_ERR_HANDLE, "stream handle is not live");
    if (flags & ~uint32_t(XN_REQ_DEVICE_PTRS | XN_REQ_SEQ_MAJOR | XN_REQ_ROPE))
        return fail(c, XN_ERR_ARG, "xn_kv_write: unknown flags 0x%x", flags);
    if (layer < 0 || layer >= c->num_layers || t0 < 0 || n < 0 || n > s->cap || t0 > s->cap - n)
        return fail(c, XN_ERR_ARG, "slot range outside the stream's capacity");
    if (n == 0) return XN_OK;
    if (!k || !v) return fail(c, XN_ERR_ARG, "null tensor pointer");
    if (t0 + n > (int64_t(1) << 30)) return fail(c, XN_ERR_CAPACITY, "position %lld too large", (long long)(t0 + n));
    const int64_t shift = s->shift[size_t(layer)];
    if (flags & XN_REQ_ROPE) {
        if (!c->cos_d) return fail(c, XN_ERR_NO_TABLES, "context was created without RoPE tables");
        if (t0 + shift + n > c->max_pos)
            return fail(c, XN_ERR_CAPACITY, "position %lld beyond the RoPE table (%d rows)", (long long)(t0 + shift + n), c->max_pos);
    }
    if (s->hw[size_t(layer)] > s->cap)
        return fail(c, XN_ERR_CAPACITY, "xn_kv_write: the stream has folded around its capacity");
    int32_t rc = refuse_capture(c);
    if (rc != XN_OK) return rc;
    const int Hkv = c->num_kv_heads, D = c->head_dim;
    const size_t floats = size_t(Hkv) * size_t(n) * D;
    const bool host = !(flags & XN_REQ_DEVICE_PTRS);
    StreamRollback undo(c);
    undo.note(s, layer);
    if ((rc = ensure_pages(c, s, t0 + n)) != XN_OK) return rc;
    if (host) {
        if ((rc = grow_io(c, align_up(floats * 4, 16) * 2)) != XN_OK) return rc;
        memcpy(c->io_host, k, floats * 4);
        memcpy(c->io_host + align_up(floats * 4, 16), v, floats * 4);
    }
    ReqDev d = {};
    d.k = host ? reinterpret_cast<const float*>(c->io_dev) : k;
    d.v = host ? reinterpret_cast<const float*>(c->io_dev + align_up(floats * 4, 16)) : v;
    const bool sm = flags & XN_REQ_SEQ_MAJOR;
    d.kv_hs = sm ? D : (long long)n * D;
    d.kv_ts = sm ? (long long)Hkv * D : D;
    d.layer = layer;
    d.seq_len = int(n);
    d.index_pos = int(t0);
    d.rope_off = int(shift);
    d.cap = int(std::min<int64_t>(s->cap, int64_t(1) << 30));
    d.n_pages = int(s->pages.size());
    d.flags = (flags & XN_REQ_ROPE) ? 1u : 0u;   // (with no query heads below: only K rotates, nothing moves q)
    PlanBuf b;
    const size_t o_req = b.put(std::vector<ReqDev>{d});
    const size_t o_page = b.put(s->pages);
    PlanSlot* slot = nullptr;
    if ((rc = commit_plan(c, b, &slot)) != XN_OK) return rc;
    const int* pages_d = reinterpret_cast<const int*>(slot->dev + o_page);
    if (host) {
        XN_CUDA(c, cudaMemcpyAsync(c->io_dev, c->io_host, align_up(floats * 4, 16) * 2, cudaMemcpyHostToDevice, c->stream));
        c->stats.h2d_bytes += floats * 8;
    }
    undo.commit();
    int64_t& hw = s->hw[size_t(layer)];
    if (t0 > hw) {   // positions that were skipped read as zeros
        const int64_t gap = t0 - hw;
        if (c->kv_u8)
            kv8::slots_fill_u8_kernel<<<int(std::min<long long>((gap * Hkv + 7) / 8, 4096)), 256, 0, c->stream>>>(
                pages_d, c->pool8, c->pool_pages, layer, Hkv, D, c->dq, hw, gap, 0, 0ull);
        else
            slots_fill_kernel<<<int(std::min<long long>((gap * Hkv * D + 255) / 256, 4096)), 256, 0, c->stream>>>(
                pages_d, c->k_pool, c->v_pool, c->pool_pages, layer, Hkv, D, c->nv, hw, gap, 0, 0ull);
        c->stats.kernel_launches += 1;
    }
    hw = std::max(hw, t0 + n);
    forget_account(s, layer, t0, t0 + n);
    const long long rows = n * 2 * Hkv;
    const ReqDev* req_d = reinterpret_cast<const ReqDev*>(slot->dev + o_req);
    if (c->kv_u8) {
        kv8::rope_append_u8_kernel<<<dim3(unsigned(std::min<long long>((rows + 7) / 8, 4096))), 256, 0, c->stream>>>(
            req_d, pages_d, c->pool8, c->cos_d, c->sin_d, c->pool_pages, 0, Hkv, D, c->dq);
    } else {
        auto append = (D % 8 != 0 && D % 4 == 0 && D <= 128) ? rope_append_kernel<true> : rope_append_kernel<false>;
        append<<<dim3(unsigned(std::min<long long>((rows + 63) / 64, 4096))), 256, 0, c->stream>>>(
            req_d, pages_d, c->k_pool, c->v_pool, c->cos_d, c->sin_d, c->pool_pages, 0, Hkv, D, c->nv);
    }
    c->stats.kernel_launches += 1;
    if ((rc = finish_slot(c, slot)) != XN_OK) return rc;
    if (host) XN_CUDA(c, cudaStreamSynchronize(c->stream));
    return XN_OK;
}

// ---- the account of positions [t0, t0 + n), out or in ------------------------------------------

int32_t account_copy_locked(xn_ctx* c, xn_stream* s, int32_t layer, int64_t t0, int64_t n, float* out,
                            const float* in, uint32_t flags) {
    if (!stream_ok(c, s)) return fail(c, XN_ERR_HANDLE, "stream handle is not live");
    if (flags & ~uint32_t(XN_REQ_DEVICE_PTRS)) return fail(c, XN_ERR_ARG, "unknown flags 0x%x", flags);
    if (layer < 0 || layer >= c->num_layers) return fail(c, XN_ERR_ARG, "layer %d outside 0..%d", layer, c->num_layers - 1);
    const int64_t len = layer_len(s, layer);
    if (t0 < 0 || n < 0 || t0 > len || n > len - t0)
        return fail(c, XN_ERR_ARG, "positions [%lld, %lld) outside the layer's %lld", (long long)t0, (long long)(t0 + n), (long long)len);
    if (n == 0) return XN_OK;
    if (!out && !in) return fail(c, XN_ERR_ARG, "null tensor pointer");
    if (in && s->hw[size_t(layer)] > s->cap)
        return fail(c, XN_ERR_CAPACITY, "the account of a stream that has folded around its capacity");
    int32_t rc = refuse_capture(c);
    if (rc != XN_OK) return rc;
    if ((rc = ensure_account_pool(c)) != XN_OK) return rc;
    const bool host = !(flags & XN_REQ_DEVICE_PTRS);
    const size_t bytes = size_t(n) * c->num_kv_heads * 4;
    if (host) {
        if ((rc = grow_io(c, bytes)) != XN_OK) return rc;
        if (in) {
            memcpy(c->io_host, in, bytes);
            XN_CUDA(c, cudaMemcpyAsync(c->io_dev, c->io_host, bytes, cudaMemcpyHostToDevice, c->stream));
            c->stats.h2d_bytes += bytes;
        }
    }
    PlanBuf b;
    b.put(s->pages);
    PlanSlot* slot = nullptr;
    if ((rc = commit_plan(c, b, &slot)) != XN_OK) return rc;
    const int* pages_d = reinterpret_cast<const int*>(slot->dev);
    int64_t& valid = s->acc_len[size_t(layer)];
    if (in && valid < t0) {
        account_zero_kernel<<<dim3(unsigned((t0 - valid + 255) / 256), unsigned(c->num_kv_heads)), 256, 0, c->stream>>>(
            pages_d, c->acct_pool, c->pool_pages, layer, c->num_kv_heads, int(valid), int(t0 - valid));
        c->stats.kernel_launches += 1;
    }
    account_copy_kernel<<<dim3(unsigned((n + 255) / 256), unsigned(c->num_kv_heads)), 256, 0, c->stream>>>(
        pages_d, c->acct_pool, c->pool_pages, layer, c->num_kv_heads, int(t0), int(n), int(valid),
        out ? (host ? reinterpret_cast<float*>(c->io_dev) : out) : nullptr,
        in ? (host ? reinterpret_cast<const float*>(c->io_dev) : in) : nullptr);
    c->stats.kernel_launches += 1;
    if ((rc = finish_slot(c, slot)) != XN_OK) return rc;
    if (in) valid = t0 + n;
    if (host) {
        if (out) XN_CUDA(c, cudaMemcpyAsync(c->io_host, c->io_dev, bytes, cudaMemcpyDeviceToHost, c->stream));
        XN_CUDA(c, cudaStreamSynchronize(c->stream));
        if (out) {
            memcpy(out, c->io_host, bytes);
            c->stats.d2h_bytes += bytes;
        }
    }
    return XN_OK;
}

// ---- reads -------------------------------------------------------------------------------------

// A row block of one request, with device addresses.
struct ReadSub {
    int req;
    xn_stream* stream;
    int layer, rows;
    int kv;                 // positions the last row (or, without the causal rule, every row) sees
    bool causal;
    const float* q;
    float* out;
    long long q_hs, q_ts, o_hs, o_ts;
    bool want;              // attention weights are wanted
    AccountDev acct;        // page_off and layer filled in at the launch
};

int32_t validate_read(xn_ctx* c, const xn_read_req& r) {
    if (!stream_ok(c, r.stream)) return fail(c, XN_ERR_HANDLE, "stream handle is not live");
    if (r.layer < 0 || r.layer >= c->num_layers)
        return fail(c, XN_ERR_ARG, "layer %d outside 0..%d", r.layer, c->num_layers - 1);
    if (r.flags & ~uint32_t(XN_REQ_DEVICE_PTRS | XN_REQ_SEQ_MAJOR | XN_READ_CAUSAL | XN_READ_ACCOUNT | XN_READ_ACCOUNT_SET))
        return fail(c, XN_ERR_ARG, "xn_cross_attention: unknown flags 0x%x", r.flags);
    const int64_t len = layer_len(r.stream, r.layer);
    if (r.rows < 0 || r.kv_len < -1) return fail(c, XN_ERR_ARG, "negative rows or kv_len");
    if (r.kv_len > len)
        return fail(c, XN_ERR_ARG, "kv_len %lld: layer %d holds %lld positions", (long long)r.kv_len, r.layer, (long long)len);
    if (len > (int64_t(1) << 30)) return fail(c, XN_ERR_CAPACITY, "%lld positions are too many", (long long)len);
    if (r.rows > 0 && (!r.q || !r.out)) return fail(c, XN_ERR_ARG, "null tensor pointer");
    if ((long long)r.rows * c->group > (1ll << 30)) return fail(c, XN_ERR_CAPACITY, "%d rows are too many", r.rows);
    const int64_t kv = r.kv_len < 0 ? len : r.kv_len;
    if (r.weights && (r.weights_stride < 0 || (r.weights_stride != 0 && r.weights_stride < kv)))
        return fail(c, XN_ERR_ARG, "weights_stride %lld is less than kv_len %lld", (long long)r.weights_stride, (long long)kv);
    const bool account = r.flags & (XN_READ_ACCOUNT | XN_READ_ACCOUNT_SET);
    if ((account || (r.flags & XN_READ_CAUSAL)) && r.stream->hw[size_t(r.layer)] > r.stream->cap)
        return fail(c, XN_ERR_CAPACITY, "the stream has folded around its capacity: neither a causal read nor an account");
    if ((account || r.weights) && c->kv_u8 && c->head_dim > 128)
        return fail(c, XN_ERR_SHAPE, "attention weights of the u8 cache format need head_dim <= 128");
    return XN_OK;
}

CacheView cache_view(const xn_ctx* c) {
    return {c->k_pool, c->v_pool, c->pool8, c->pool_pages, c->num_kv_heads, c->head_dim, c->nv, c->dq};
}

using MidFn = void (*)(const ReadTable, const CUtensorMap, const CUtensorMap, float*, int*, long long, int, int, int, float, int, int*);
MidFn pick_mid(int mt) {
    return mt == 1 ? read_mid_kernel<1> : mt == 2 ? read_mid_kernel<2> : mt == 3 ? read_mid_kernel<3> : read_mid_kernel<4>;
}

int32_t ready_read_kernels(xn_ctx* c) {
    if (c->read_funcs_ready) return XN_OK;
    if (!c->kv_u8) {
        const SplitKernels k = pick_splits(c->nv_class, c->gt, c->nv_exact);
        XN_CUDA(c, cudaFuncSetAttribute(reinterpret_cast<const void*>(k.scores.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, int(k.scores.smem)));
        for (int mt = 1; mt <= 4 && c->tf32_ok; ++mt)
            XN_CUDA(c, cudaFuncSetAttribute(reinterpret_cast<const void*>(pick_mid(mt)), cudaFuncAttributeMaxDynamicSharedMemorySize, int(rm::smem_bytes(mt))));
        for (const ReadKernel& r : k.read)
            XN_CUDA(c, cudaFuncSetAttribute(reinterpret_cast<const void*>(r.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, int(r.smem)));
    }
    XN_CUDA(c, cudaFuncSetAttribute(reinterpret_cast<const void*>(read_tc_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, rt::kSmemBytes));
    XN_CUDA(c, cudaFuncSetAttribute(reinterpret_cast<const void*>(account_tc_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, rt::kAcctSmemBytes));
    XN_CUDA(c, cudaFuncSetAttribute(reinterpret_cast<const void*>(evict_select_kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    int(ev::kThreads * (ev::kMaxRun + 1) * 4)));
    c->read_funcs_ready = true;
    return XN_OK;
}

// The stream's page table on the device: all of it, whatever part the caller reads, so that a stream
// that occurs several times in a call has one address there (no page comes or goes during a read).
int32_t device_pages(xn_ctx* c, xn_stream* s, const int** out) {
    const size_t n = s->pages.size();
    if (n > s->pages_d_cap) {
        XN_CUDA(c, cudaStreamSynchronize(c->stream));   // launches in flight may still read the old one
        XN_CUDA(c, guarded_free(c, s->pages_d));
        s->pages_d = nullptr;
        s->pages_d_cap = s->pages_d_valid = 0;
        const size_t want = align_up(n + n / 2, 64);
        XN_CUDA(c, guarded_malloc(c, reinterpret_cast<void**>(&s->pages_d), want * 4, "page table"));
        s->pages_d_cap = want;
    }
    if (n > s->pages_d_valid) {
        // pageable memory: the call returns when the entries have been taken
        XN_CUDA(c, cudaMemcpyAsync(s->pages_d + s->pages_d_valid, s->pages.data() + s->pages_d_valid, (n - s->pages_d_valid) * 4,
                                   cudaMemcpyHostToDevice, c->stream));
        s->pages_d_valid = n;
    }
    *out = s->pages_d;
    return XN_OK;
}

// f32 cache, up to kReadEntries requests per launch, described by the launch parameter alone.  mt = 0:
// few rows that all see the same prefix (the small kernel, or the split-KV kernel over a table); else the
// mid kernel with mt * 16 packed rows per unit.
int32_t launch_read_table(xn_ctx* c, const ReadSub* subs, int n, bool want, int mt) {
    const int Hq = c->num_heads, Hkv = c->num_kv_heads;
    ReadTable& t = c->read_table;
    t.n = n;
    t.subs = c->subs;
    t.gt = c->gt;
    t.group = c->group;
    t.n_tiles = 0;
    int32_t rc;
    size_t floats = 0;
    int max_kv = 0, max_rows = 0;
    for (int i = 0; i < n; ++i) {
        const ReadSub& s = subs[i];
        ReadEntry& e = t.e[i];
        e.q = s.q; e.q_hs = s.q_hs; e.q_ts = s.q_ts;
        e.out = s.out; e.o_hs = s.o_hs; e.o_ts = s.o_ts;
        if ((rc = device_pages(c, s.stream, &e.pages)) != XN_OK) return rc;
        e.rows = s.rows; e.kv_len = s.kv; e.layer = s.layer;
        const int tile = mt ? kPageTokens : c->tile_tokens;
        e.n_tiles = (s.kv + tile - 1) / tile;
        e.causal = s.causal && s.rows > 1 ? 1 : 0;
        e.n_rt = mt ? (s.rows * c->group + 16 * mt - 1) / (16 * mt) : 1;
        e.tile0 = t.n_tiles;
        t.n_tiles += (long long)e.n_tiles * Hkv * (mt ? e.n_rt : c->subs * s.rows);
        max_kv = std::max(max_kv, s.kv);
        max_rows = std::max(max_rows, s.rows);
        if (!want) continue;
        e.user = s.acct.user; e.user_hs = s.acct.user_hs;
        e.old_from = s.acct.old_from; e.old_len = s.acct.old_len; e.store = s.acct.store;
        e.sc_ts = (long long)align_up(size_t(s.kv), 4);
        e.sc_hs = e.sc_ts * s.rows;
        e.lse_hs = s.rows;
        floats += size_t(e.sc_hs) * Hq + align_up(size_t(s.rows) * Hq, 4);
    }
    // Small calls: a cluster per (request, KV head), of as many blocks (of 32 positions or more) as there
    // are SMs for, if a block's share of the positions is then small.
    // (20 query heads over 5, one row: at 1025 positions 14.2 us beside 17.1 with an account and 11.0 beside
    // 10.8 without; at 2000, 15.5 beside 17.5 and 15.1 beside 14.1 -- the split-KV kernel adds a launch for
    // the account, and reads faster once every block has a few tiles)
    const int small_max = want ? rs::kMaxTokens : rs::kMaxTokens / 2;
    if (mt == 0 && c->head_dim <= 128 && max_rows <= rs::kMaxRows && n * Hkv <= c->sm_count) {
        int cluster = 1;
        while (cluster < ev::kMaxCluster && n * Hkv * cluster * 2 <= c->sm_count && max_kv > cluster * 32) cluster *= 2;
        if ((max_kv + cluster - 1) / cluster <= small_max) {
            if (c->profile && (rc = profile_begin(c, 0)) != XN_OK) return rc;
            XN_CUDA(c, launch_pdl(c, read_small_kernel, dim3(unsigned(n * Hkv * cluster)), rs::kThreads, 0, true, unsigned(cluster), t,
                                  c->k_pool, c->v_pool, c->acct_pool, c->pool_pages, Hkv, c->head_dim, c->nv, c->scale, cluster,
                                  want ? 1 : 0));
            if (c->profile && (rc = profile_end(c)) != XN_OK) return rc;
            c->stats.decode_launches += 1;
            return XN_OK;
        }
    }
    if (want) {
        if ((rc = grow_device(c, &c->read_ws, &c->read_ws_cap, floats)) != XN_OK) return rc;
        float* at = c->read_ws;
        for (int i = 0; i < n; ++i) {
            ReadEntry& e = t.e[i];
            e.scores = at;
            at += size_t(e.sc_hs) * Hq;
            e.lse = at;
            at += align_up(size_t(e.rows) * Hq, 4);
        }
    }
    t.n_blocks = int(std::min<long long>(t.n_tiles, mt ? c->sm_count : c->decode_ctas));
    static_assert(kSyncHeaderWords == kSyncMerge0, "layout of the synchronisation array");
    if (size_t(t.n_blocks) + kSyncMerge0 > c->sync_cap)
        return fail(c, XN_ERR_CAPACITY, "internal: %d blocks exceed the arrival counters", t.n_blocks);
    const size_t part = mt ? rm::part_floats(mt, c->nv * 4) : c->gt * part_stride_floats(c->nv);
    if ((rc = grow_device(c, &c->partials, &c->partials_cap, size_t(2 * t.n_blocks) * part)) != XN_OK) return rc;
    if (c->profile && (rc = profile_begin(c, 0)) != XN_OK) return rc;
    if (mt) {
        XN_CUDA(c, launch_pdl(c, pick_mid(mt), dim3(unsigned(t.n_blocks)), rm::kThreads, rm::smem_bytes(mt), true, 0, t, c->k_map,
                              c->v_map_rows, c->partials, c->sync_d, c->pool_pages, Hkv, c->head_dim, c->nv,
                              c->scale * 1.4426950408889634f, want ? 1 : 0, c->status_d));
    } else {
        const ReadKernel k = pick_splits(c->nv_class, c->gt, c->nv_exact).read[want ? 1 : 0];
        XN_CUDA(c, launch_pdl(c, k.fn, dim3(unsigned(t.n_blocks)), k.threads, k.smem, true, 0, t, c->k_pool, c->v_pool, c->partials,
                              c->sync_d, c->pool_pages, Hkv, c->head_dim, c->nv, c->scale, c->status_d));
    }
    if (c->profile && (rc = profile_end(c)) != XN_OK) return rc;
    c->stats.decode_launches += 1;
    if (want)
        XN_CUDA(c, launch_pdl(c, account_table_kernel, dim3(unsigned((max_kv + 255) / 256), unsigned(Hkv), unsigned(n)), 256, 0, true, 0,
                              t, c->acct_pool, c->pool_pages, Hkv));
    return XN_OK;
}

// Few rows: the split-KV kernel of the decode path over the prefix, one unit per (KV head, head
// subgroup, row); with weights, its variant that also leaves the scores, and the account kernel.
int32_t launch_read_few(xn_ctx* c, const std::vector<ReadSub>& subs, bool want) {
    const int Hq = c->num_heads, Hkv = c->num_kv_heads;
    std::vector<ReqDev> rd(subs.size());
    std::vector<int32_t> page_ids, kv_lens;
    std::vector<UnitDev> units;
    std::vector<FewAccount> acct;
    size_t sc_floats = 0, lse_floats = 0;
    long long key_rows = 0;
    int max_kv = 0;
    for (size_t i = 0; i < subs.size(); ++i) {
        const ReadSub& s = subs[i];
        ReqDev& d = rd[i];
        d = {};
        d.q = s.q; d.q_hs = s.q_hs; d.q_ts = s.q_ts;
        d.out = s.out; d.o_hs = s.o_hs; d.o_ts = s.o_ts;
        d.page_off = int(page_ids.size());
        // (a row block of a longer request keeps the account of all its positions)
        d.n_pages = (std::max(s.kv, want ? s.acct.kv_len : 0) + kPageTokens - 1) / kPageTokens;
        page_ids.insert(page_ids.end(), s.stream->pages.begin(), s.stream->pages.begin() + d.n_pages);
        d.layer = s.layer; d.seq_len = s.rows;
        d.cap = int(std::min<int64_t>(s.stream->cap, int64_t(1) << 30));
        if (want) {
            d.sc_ts = (long long)align_up(size_t(s.kv), 4);
            d.sc_hs = d.sc_ts * s.rows;
            d.lse_hs = s.rows;
            d.scores = reinterpret_cast<float*>(sc_floats);   // offsets until the buffer is there
            d.lse = reinterpret_cast<float*>(lse_floats);
            sc_floats += size_t(d.sc_hs) * Hq;
            lse_floats += align_up(size_t(s.rows) * Hq, 4);
            max_kv = std::max(max_kv, s.acct.kv_len);
        }
        for (int h = 0; h < Hkv; ++h)
            for (int sb = 0; sb < c->subs; ++sb)
                for (int t = 0; t < s.rows; ++t) {
                    UnitDev u = {};
                    u.kv_len = s.causal ? s.kv - s.rows + t + 1 : s.kv;
                    if (u.kv_len <= 0) continue;   // zeroed by the caller
                    u.req = int(i); u.kv_head = h;
                    u.head0 = h * c->group + sb * c->gt;
                    u.nheads = std::min(c->gt, c->group - sb * c->gt);
                    u.t_q = t;
                    u.part_begin = -1; u.part_count = 1; u.merge_slot = -1;
                    units.push_back(u);
                    kv_lens.push_back(u.kv_len);
                    key_rows += u.kv_len;
                }
    }
    if ((long long)units.size() > kMaxUnits)
        return fail(c, XN_ERR_CAPACITY, "%zu attention rows in one submission exceed the limit %lld", units.size(), kMaxUnits);
    int32_t rc;
    if (want) {
        if ((rc = grow_device(c, &c->read_ws, &c->read_ws_cap, sc_floats + lse_floats)) != XN_OK) return rc;
        for (size_t i = 0; i < subs.size(); ++i) {
            ReqDev& d = rd[i];
            d.scores = c->read_ws + reinterpret_cast<uintptr_t>(d.scores);
            d.lse = c->read_ws + sc_floats + reinterpret_cast<uintptr_t>(d.lse);
            FewAccount a = {};
            a.a = subs[i].acct;
            a.a.page_off = d.page_off;
            a.a.layer = subs[i].layer;
            a.scores = d.scores; a.lse = d.lse;
            a.sc_hs = d.sc_hs; a.sc_ts = d.sc_ts; a.lse_hs = d.lse_hs;
            a.rows = subs[i].rows;
            a.row_limit0 = subs[i].causal ? subs[i].kv - subs[i].rows + 1 : subs[i].kv;
            a.row_step = subs[i].causal ? 1 : 0;
            acct.push_back(a);
        }
    }
    SplitPlan sp = plan_split(kv_lens.data(), int(units.size()), c->tile_tokens, c->decode_chunks);
    int n_cut = 0;
    for (size_t u = 0; u < units.size(); ++u) {
        units[u].part_begin = sp.unit_part_begin[u];
        units[u].part_count = sp.unit_part_count[u];
        units[u].merge_slot = sp.unit_part_count[u] > 1 ? n_cut++ : -1;
    }
    if (size_t(n_cut) + 2 > c->sync_cap)
        return fail(c, XN_ERR_CAPACITY, "internal: %d cut units exceed the arrival counters", n_cut);
    if ((rc = grow_device(c, &c->partials, &c->partials_cap,
                          size_t(sp.n_parts) * c->gt *
                              (c->kv_u8 ? kv8::part_stride(c->dq) : part_stride_floats(c->nv)))) != XN_OK)
        return rc;
    PlanBuf b;
    const size_t o_req = b.put(rd), o_unit = b.put(units), o_item = b.put(sp.items), o_cta = b.put(sp.cta_item_begin),
                 o_page = b.put(page_ids), o_acct = b.put(acct);
    PlanSlot* slot = nullptr;
    if ((rc = commit_plan(c, b, &slot)) != XN_OK) return rc;
    const ReqDev* reqs_d = reinterpret_cast<const ReqDev*>(slot->dev + o_req);
    const UnitDev* units_d = reinterpret_cast<const UnitDev*>(slot->dev + o_unit);
    const ItemDev* items_d = reinterpret_cast<const ItemDev*>(slot->dev + o_item);
    const int* cta_d = reinterpret_cast<const int*>(slot->dev + o_cta);
    const int* pages_d = reinterpret_cast<const int*>(slot->dev + o_page);
    if (sp.ctas > 0) {
        if (c->profile && (rc = profile_begin(c, 0)) != XN_OK) return rc;
        if (c->kv_u8) {
            const bool mma = c->kv8_mma && key_rows >= c->kv8_mma_min_rows;
            const Split8Fn fn = mma ? pick_split8_mma(c->dq, c->gt) : pick_split8(c->dq, c->gt, c->kv8_epl);
            const size_t sm = mma ? kv8m::smem_bytes(c->gt, c->dq) : kv8::smem_bytes(c->gt, c->kv8_epl);
            fn<<<std::min(sp.ctas, c->decode_ctas), kv8::kThreads, sm, c->stream>>>(
                reqs_d, units_d, items_d, cta_d, sp.ctas, pages_d, c->pool8, c->partials, c->sync_d, c->pool_pages,
                Hkv, c->head_dim, c->scale * 1.4426950408889634f, c->cos_d, c->sin_d, c->status_d);
        } else {
            const SplitKernels ks = pick_splits(c->nv_class, c->gt, c->nv_exact);
            const SplitKernel& k = want ? ks.scores : ks.decode;
            c->pcache.table.n = 0;
            k.fn<<<std::min(sp.ctas, c->decode_ctas), k.threads, k.smem, c->stream>>>(
                reqs_d, units_d, items_d, cta_d, sp.ctas, pages_d, c->k_pool, c->v_pool, c->partials, c->sync_d,
                c->pool_pages, Hkv, c->head_dim, c->nv, c->scale, c->cos_d, c->sin_d, c->status_d, c->pcache.table);
        }
        XN_CUDA(c, cudaGetLastError());
        if (c->profile && (rc = profile_end(c)) != XN_OK) return rc;
        c->stats.kernel_launches += 1;
        c->stats.decode_launches += 1;
    }
    // (blockIdx.z carries the request: at most 65535 of them per launch)
    for (size_t z0 = 0; z0 < acct.size(); z0 += 65535) {
        const unsigned nz = unsigned(std::min<size_t>(65535, acct.size() - z0));
        XN_CUDA(c, launch_pdl(c, account_few_kernel, dim3(unsigned((max_kv + 255) / 256), unsigned(Hkv), nz), 256, 0,
                              sp.ctas > 0 && z0 == 0, 0, reinterpret_cast<const FewAccount*>(slot->dev + o_acct) + z0, pages_d,
                              c->acct_pool, c->pool_pages, Hkv, c->group));
    }
    return finish_slot(c, slot);
}

// How the row tiles of a launch are cut along the cache: with fewer tiles than SMs, or a last round
// of blocks that leaves most SMs idle, tiles are split into ranges of pages whose partial results
// are merged.  Every candidate piece size is rated by dealing its pieces out to the SMs, longest first
// and every other round from the end, which is nearly what the hardware does.  In units of one
// 128-position tile (2.7 us): a block costs kReadBlockCost beside its tiles, a split one kReadSplitCost
// more, and the merge its launch and two transfers of 64 KB per piece.  (Against a rating by rounds of
// blocks times their mean load: 4 x 37 rows over 130-1501 positions, 32 heads: 12.6 units for 15.0;
// 1024 rows over 8192 positions, 32/8 heads: 135 without a merge for 140 and a merge of 1024 pieces.)
constexpr double kReadBlockCost = 3.6, kReadSplitCost = 0.4, kReadMergeCost = 1.1, kReadPieceCost = 0.007;
int read_piece_tiles(const std::vector<int>& tiles, int sms) {
    int longest = 1;
    for (int t : tiles) longest = std::max(longest, t);
    std::vector<int> whole(size_t(longest) + 1), parts(size_t(longest) + 1);
    std::vector<double> load(static_cast<size_t>(sms));
    int best = longest;
    double best_cost = -1;
    for (int piece = longest;; piece = std::max(1, piece * 7 / 8)) {
        std::fill(whole.begin(), whole.end(), 0);
        std::fill(parts.begin(), parts.end(), 0);
        long long n_parts = 0;
        for (int t : tiles) {
            const int n = (t + piece - 1) / piece;
            if (n == 1) {
                ++whole[size_t(t)];
                continue;
            }
            n_parts += n;   // t % n pieces of t / n + 1 tiles, the others of t / n
            parts[size_t(t / n)] += n - t % n;
            if (t % n) parts[size_t(t / n + 1)] += t % n;
        }
        std::fill(load.begin(), load.end(), 0.0);
        long long at = 0;
        for (int t = longest; t >= 0; --t)
            for (int k = 0; k < whole[size_t(t)] + parts[size_t(t)]; ++k, ++at) {
                const long long lane = at % sms;
                load[size_t((at / sms) & 1 ? sms - 1 - lane : lane)] += t + kReadBlockCost + (k < parts[size_t(t)] ? kReadSplitCost : 0);
            }
        const double cost = *std::max_element(load.begin(), load.end()) + (n_parts ? kReadMergeCost + kReadPieceCost * double(n_parts) : 0);
        if (best_cost < 0 || cost < best_cost * 0.99) { best_cost = cost; best = piece; }
        if (piece <= 2) break;
    }
    return best;
}

// Many rows: the tensor-core passes of xn_read_tc.cuh.
int32_t launch_read_tc(xn_ctx* c, const std::vector<ReadSub>& subs) {
    const int Hkv = c->num_kv_heads, D = c->head_dim, G = c->group;
    std::vector<TcReq> reqs(subs.size());
    std::vector<int32_t> page_ids;
    struct Row { int req, head, qt, tiles, pages; };
    std::vector<Row> rows;
    std::vector<TcKeyTile> key_tiles;
    long long n_img = 0, n_qimg = 0;
    bool want = false;
    for (size_t i = 0; i < subs.size(); ++i) {
        const ReadSub& s = subs[i];
        TcReq& r = reqs[i];
        r = {};
        r.q = s.q; r.out = s.out;
        r.q_hs = s.q_hs; r.q_ts = s.q_ts; r.o_hs = s.o_hs; r.o_ts = s.o_ts;
        r.rows = s.rows; r.kv_len = s.kv; r.causal = s.causal ? 1 : 0;
        r.page_off = int(page_ids.size());
        r.layer = s.layer;
        r.n_pages = (s.kv + kPageTokens - 1) / kPageTokens;
        r.n_qt = int(((long long)s.rows * G + rt::kBM - 1) / rt::kBM);
        page_ids.insert(page_ids.end(), s.stream->pages.begin(), s.stream->pages.begin() + r.n_pages);
        r.img0 = n_img;
        r.qimg0 = n_qimg;
        n_img += (long long)r.n_pages * Hkv;
        n_qimg += (long long)r.n_qt * Hkv;
        r.acct = s.acct;
        r.acct.page_off = r.page_off;
        r.acct.layer = s.layer;
        for (int qt = r.n_qt - 1; qt >= 0; --qt) {
            const int last_t = std::min((qt + 1) * rt::kBM - 1, s.rows * G - 1) / G;
            const int limit = std::max(1, s.causal ? s.kv - s.rows + last_t + 1 : s.kv);
            const int pages = (limit + kPageTokens - 1) / kPageTokens;
            for (int h = 0; h < Hkv; ++h) rows.push_back({int(i), h, qt, (pages + 1) / 2, pages});
        }
        if (s.want) {
            want = true;
            for (int tile = 0; tile < (r.n_pages + 1) / 2; ++tile) {
                int qt0 = 0;
                if (s.causal) qt0 = int(std::max<long long>(0, (long long)(tile * rt::kBM - (s.kv - s.rows)) * G / rt::kBM));
                for (int h = 0; h < Hkv; ++h) key_tiles.push_back({int(i), h, tile, qt0});
            }
        }
    }
    std::stable_sort(rows.begin(), rows.end(), [](const Row& a, const Row& b) { return a.tiles > b.tiles; });
    std::stable_sort(key_tiles.begin(), key_tiles.end(), [&](const TcKeyTile& a, const TcKeyTile& b) {
        return reqs[size_t(a.req)].n_qt - a.qt_begin > reqs[size_t(b.req)].n_qt - b.qt_begin;
    });
    std::vector<int> weights;
    weights.reserve(rows.size());
    for (const Row& r : rows) weights.push_back(r.tiles);
    const int piece = read_piece_tiles(weights, c->sm_count);
    std::vector<TcItem> items;
    std::vector<TcMerge> merges;
    int n_parts = 0;
    for (const Row& r : rows) {
        const int n = (r.tiles + piece - 1) / piece;
        if (n > 1) merges.push_back({r.req, r.head, r.qt, n_parts, n, 0});
        for (int k = 0; k < n; ++k) {
            const int lo = int((long long)r.tiles * k / n) * 2, hi = std::min(r.pages, int((long long)r.tiles * (k + 1) / n) * 2);
            items.push_back({r.req, r.head, r.qt, lo, hi, n > 1 ? n_parts++ : -1});
        }
    }
    std::stable_sort(items.begin(), items.end(), [](const TcItem& a, const TcItem& b) {
        return a.page_end - a.page_begin > b.page_end - b.page_begin;
    });
    if (2 * (n_img + n_qimg) > (1ll << 31) - 1)
        return fail(c, XN_ERR_CAPACITY, "%lld pages and row tiles in one submission are too many", n_img + n_qimg);

    // workspace: page images | query images | page factors | row factors | partial records
    const size_t img_b = size_t(n_img) * rt::page_image_bytes(D), q_b = size_t(n_qimg) * rt::q_image_bytes(D);
    const size_t meta_b = align_up(size_t(n_img) * sizeof(PageMeta), 256), row_b = size_t(n_qimg) * rt::kBM * sizeof(float2);
    const size_t part_b = size_t(n_parts) * rt::part_floats(c->nv * 4) * 4;
    int32_t rc = grow_device(c, &c->read_ws, &c->read_ws_cap, (img_b + q_b + meta_b + row_b + part_b) / 4 + 64);
    if (rc != XN_OK) return rc;
    unsigned char* ws = reinterpret_cast<unsigned char*>(c->read_ws);
    unsigned char* img = ws;
    unsigned char* qimg = img + img_b;
    PageMeta* meta = reinterpret_cast<PageMeta*>(qimg + q_b);
    float2* row_meta = reinterpret_cast<float2*>(qimg + q_b + meta_b);
    float* parts = reinterpret_cast<float*>(qimg + q_b + meta_b + row_b);
    PlanBuf b;
    const size_t o_req = b.put(reqs), o_item = b.put(items), o_merge = b.put(merges), o_key = b.put(key_tiles),
                 o_page = b.put(page_ids);
    PlanSlot* slot = nullptr;
    if ((rc = commit_plan(c, b, &slot)) != XN_OK) return rc;
    const TcReq* reqs_d = reinterpret_cast<const TcReq*>(slot->dev + o_req);
    const int* pages_d = reinterpret_cast<const int*>(slot->dev + o_page);
    const CacheView view = cache_view(c);
    const float scale_log2 = c->scale * 1.4426950408889634f;
    if (c->profile && (rc = profile_begin(c, 1)) != XN_OK) return rc;
    XN_CUDA(c, launch_pdl(c, page_images_kernel, dim3(unsigned(2 * (n_img + n_qimg))), 256, 0, true, 0, reqs_d, int(subs.size()), n_img,
                          pages_d, view, img, meta, qimg, row_meta, scale_log2, G, c->status_d));
    XN_CUDA(c, launch_pdl(c, read_tc_kernel, dim3(unsigned(items.size())), rt::kThreads, size_t(rt::kSmemBytes), true, 0, reqs_d,
                          reinterpret_cast<const TcItem*>(slot->dev + o_item), pages_d, view, img, meta, qimg, row_meta,
                          parts, scale_log2, G, want ? 1 : 0, c->status_d));
    if (!merges.empty())
        XN_CUDA(c, launch_pdl(c, read_merge_kernel, dim3(unsigned(merges.size()), rt::kBM / 8), 256, 0, true, 0, reqs_d,
                              reinterpret_cast<const TcMerge*>(slot->dev + o_merge), parts, row_meta, G, D, c->nv, want ? 1 : 0));
    // a cluster of blocks per key tile while a quarter of the SMs would have nothing to do, and each block is
    // left two row tiles (prompts of 600 over 8 heads 50 us, 4 of 300 over 2 heads 68, one of 2000 over 2 heads
    // 130, one of 2048 over 5 heads 156; doubling until there are two rounds of blocks 61, 81, 122 and 153;
    // only up to half the SMs 56, 64, 130 and 207)
    int cluster = 1, most_qt = 0;
    for (const TcReq& r : reqs) most_qt = std::max(most_qt, r.n_qt);
    while (cluster < ev::kMaxCluster && (long long)key_tiles.size() * cluster * 4 < 3 * c->sm_count && most_qt >= 4 * cluster) cluster *= 2;
    if (want) {
        const int blocks = cluster > 1 ? int(key_tiles.size()) * cluster : std::min<int>(int(key_tiles.size()), c->sm_count);
        XN_CUDA(c, launch_pdl(c, account_tc_kernel, dim3(unsigned(blocks)), rt::kThreads, size_t(rt::kAcctSmemBytes), true,
                              unsigned(cluster), reqs_d, reinterpret_cast<const TcKeyTile*>(slot->dev + o_key), int(key_tiles.size()),
                              pages_d, view, img, meta, qimg, row_meta, c->acct_pool, scale_log2, G, cluster, c->status_d));
    }
    if (c->profile && (rc = profile_end(c)) != XN_OK) return rc;
    c->stats.prefill_launches += 1;
    return finish_slot(c, slot);
}

// Which kernels take the requests of a call that have more than a row or two but no more than 128 packed
// ones (rows x heads of a group).  Measured
// over 1 to 20 requests of 300-2500 positions, head counts 20/5, 32/32 and 16/2 and head sizes 64, 100 and
// 128, the times follow, in us, with P thousands of (position, KV head) pairs:
//   split-KV, per row   10 + 0.12 u P           u: passes over the cache, rows x ceil(group / 4)
//   mid kernel          10 + {0.33, 0.46, 0.6, 0.85} P + (4.5 + 0.27 blocks / units) mt   for mt tiles of 16 rows
//   tensor-core passes  20 + 0.55 P             (0.28 P up to head size 64)
// and the account adds about 5 + 2 rows, 6 + 1.5 rows and 5 + 0.17 P to them.
// e.g. 20 requests x 8 rows, 32/32 heads of 100, 1000 positions: 520 / 212 / 366; 1 x 8 rows, 20/5 of 128,
// 2000 positions: 19 / 39 / 25; 20 x 12 rows, 20/5 of 128, 1000 positions: 161 / 87 / 81.
// Over the u8 format, which the mid kernel does not read: 30 + 0.05 u P, and 20 + 0.75 P (0.45 P up to
// head size 64); e.g. 20 x 8 rows, 20/5 of 128, 1000 positions: 71 / 89, x 20 rows: 141 / 90.
enum ReadPath { kPathAuto = 0, kPathFew, kPathMid, kPathTc };
struct ReadEstimate {
    double pairs = 0, few = 0, mid = 0;
    long long units = 0;
    int mt = 0, rows = 0;
    bool want = false;
    void add(const xn_ctx* c, const ReadSub& s) {
        const double p = double(s.kv) * c->num_kv_heads * 1e-3;
        const int m = int((std::min<long long>((long long)s.rows * c->group, 128) + 15) / 16), rt = (m + 3) / 4;
        static const double rate[5] = {0, 0.33, 0.46, 0.6, 0.85};
        pairs += p;
        few += 0.12 * p * s.rows * c->subs;
        mid += rate[std::min(m, 4)] * rt * p;
        mt = std::max(mt, std::min(m, 4));
        units += (long long)c->num_kv_heads * rt;
        want = want || s.want;
        rows = std::max(rows, s.rows);
    }
    ReadPath best(const xn_ctx* c) const {
        if (units == 0) return kPathFew;
        const double f = 10 + few + (want ? 5 + 2 * rows : 0);
        const double m = 10 + mid + (4.5 + 0.27 * c->sm_count / double(units)) * mt + (want ? 6 + 1.5 * rows : 0);
        const double t = 20 + (c->head_dim > 64 ? 0.55 : 0.28) * pairs + (want ? 5 + 0.17 * pairs : 0);
        if (c->kv_u8) return 30 + few * (0.05 / 0.12) <= 20 + (c->head_dim > 64 ? 0.75 : 0.45) * pairs ? kPathFew : kPathTc;
        if (!c->tf32_ok) return f <= t ? kPathFew : kPathTc;   // (the mid kernel reads by tensor map)
        return f <= std::min(m, t) ? kPathFew : (m <= t ? kPathMid : kPathTc);
    }
};

// Bytes of images, and of scores, that one launch may need at most; more goes out in several.
constexpr size_t kReadImageBudget = size_t(4) << 30;
constexpr size_t kReadScoreBudget = size_t(512) << 20;

int32_t read_locked(xn_ctx* c, int32_t n, const xn_read_req* reqs) {
    if (n < 0 || (n > 0 && !reqs)) return fail(c, XN_ERR_ARG, "bad request array");
    if (n == 0) return XN_OK;
    const int Hq = c->num_heads, Hkv = c->num_kv_heads, D = c->head_dim;
    const bool host = !(reqs[0].flags & XN_REQ_DEVICE_PTRS);
    int32_t rc;
    bool any_account = false;
    std::vector<std::pair<xn_stream*, int>> accounted;
    for (int i = 0; i < n; ++i) {
        const xn_read_req& r = reqs[i];
        if ((rc = validate_read(c, r)) != XN_OK) return rc;
        if (host == bool(r.flags & XN_REQ_DEVICE_PTRS))
            return fail(c, XN_ERR_ARG, "host and device requests cannot be mixed in one batch");
        if (r.flags & (XN_READ_ACCOUNT | XN_READ_ACCOUNT_SET)) {
            any_account = true;
            accounted.push_back({r.stream, r.layer});
        }
    }
    std::sort(accounted.begin(), accounted.end());
    if (std::adjacent_find(accounted.begin(), accounted.end()) != accounted.end())
        return fail(c, XN_ERR_ARG, "two requests of one call keep the same account");
    if ((rc = refuse_capture(c)) != XN_OK) return rc;
    if ((rc = ready_read_kernels(c)) != XN_OK) return rc;
    if (any_account && (rc = ensure_account_pool(c)) != XN_OK) return rc;

    // host pointers: [q of all | out of all | weights of all] through the staging buffers
    size_t io_in = 0, io_out = 0;
    std::vector<size_t> w_off;
    if (host) {
        for (int i = 0; i < n; ++i) {
            const size_t qb = align_up(size_t(Hq) * reqs[i].rows * D * 4, 16);
            io_in += qb;
            io_out += qb;
            const int64_t kv = reqs[i].kv_len < 0 ? layer_len(reqs[i].stream, reqs[i].layer) : reqs[i].kv_len;
            if (reqs[i].weights) io_out += align_up(size_t(Hkv) * kv * 4, 16);
        }
        if ((rc = grow_io(c, io_in + io_out)) != XN_OK) return rc;
    }
    size_t in_at = 0, out_at = io_in;
    // [1]: with weights.  table: few rows that all see the whole prefix; few: the others, and the u8 format;
    // mid: the mid kernel's; between: to be dealt out by the estimates
    std::vector<ReadSub> table[2], mid[2], few[2], tc, between;
    ReadEstimate estimate;
    struct Zero { float* out; long long o_hs, o_ts; int rows; };
    std::vector<Zero> zeros;
    for (int i = 0; i < n; ++i) {
        const xn_read_req& r = reqs[i];
        const int64_t kv = r.kv_len < 0 ? layer_len(r.stream, r.layer) : r.kv_len;
        ReadSub s = {};
        s.req = i;
        s.stream = r.stream;
        s.layer = r.layer;
        s.rows = r.rows;
        s.kv = int(kv);
        s.causal = r.flags & XN_READ_CAUSAL;
        s.q = r.q;
        s.out = r.out;
        float* w = r.weights;
        int64_t w_hs = r.weights_stride ? r.weights_stride : kv;
        const size_t qb = size_t(Hq) * r.rows * D * 4;
        if (host) {
            if (qb) memcpy(c->io_host + in_at, r.q, qb);
            s.q = reinterpret_cast<const float*>(c->io_dev + in_at);
            s.out = reinterpret_cast<float*>(c->io_dev + out_at);
            in_at += align_up(qb, 16);
            out_at += align_up(qb, 16);
            if (w) {
                w = reinterpret_cast<float*>(c->io_dev + out_at);
                w_hs = kv;
                out_at += align_up(size_t(Hkv) * kv * 4, 16);
            }
        }
        const bool sm = r.flags & XN_REQ_SEQ_MAJOR;
        s.q_hs = s.o_hs = sm ? D : (long long)r.rows * D;
        s.q_ts = s.o_ts = sm ? (long long)Hq * D : D;
        const bool store = r.flags & (XN_READ_ACCOUNT | XN_READ_ACCOUNT_SET);
        s.want = kv > 0 && (store || w);
        s.acct.user = w;
        s.acct.user_hs = w_hs;
        s.acct.store = store ? 1 : 0;
        s.acct.old_from = (store && !(r.flags & XN_READ_ACCOUNT_SET)) ? kAcctPool : kAcctZero;
        s.acct.old_len = s.acct.old_from == kAcctPool ? int(std::min(kv, r.stream->acc_len[size_t(r.layer)])) : 0;
        s.acct.kv_len = int(kv);
        if (r.rows == 0 && !s.want) continue;
        if (kv == 0) {
            if (r.rows > 0) zeros.push_back({s.out, s.o_hs, s.o_ts, r.rows});
            continue;
        }
        const long long packed = (long long)r.rows * c->group;
        if (D <= 128 && r.rows > 0 && (c->kv_u8 && s.want)) tc.push_back(s);   // (the only ones for those)
        else if (D > 128 || r.rows == 0 || (c->read_path == kPathAuto && (long long)r.rows * c->subs <= 2)) few[0].push_back(s);
        else if (c->read_path == kPathAuto && packed > rt::kBM) tc.push_back(s);
        else {
            estimate.add(c, s);
            between.push_back(s);
        }
    }
    const ReadPath path = c->read_path != kPathAuto ? ReadPath(c->read_path) : estimate.best(c);
    (path == kPathTc ? tc : few[0]).insert((path == kPathTc ? tc : few[0]).end(), between.begin(), between.end());
    std::vector<ReadSub> rest;
    rest.swap(few[0]);
    for (const ReadSub& s : rest) {
        const bool fits = !s.want || align_up(size_t(s.kv), 4) * Hq * size_t(s.rows) <= kReadScoreBudget / 4;
        const bool plain_rows = s.rows > 0 && !c->kv_u8 && fits;
        if (plain_rows && path == kPathMid && D <= 128 && c->tf32_ok && (c->read_path == kPathMid || (long long)s.rows * c->subs > 2)) {
            mid[s.want ? 1 : 0].push_back(s);
            continue;
        }
        if (s.causal && s.rows > s.kv) zeros.push_back({s.out, s.o_hs, s.o_ts, int(s.rows - s.kv)});
        if (plain_rows && (!s.causal || s.rows == 1)) table[s.want ? 1 : 0].push_back(s);
        else few[s.want ? 1 : 0].push_back(s);
    }
    if (host && io_in) {
        XN_CUDA(c, cudaMemcpyAsync(c->io_dev, c->io_host, io_in, cudaMemcpyHostToDevice, c->stream));
        c->stats.h2d_bytes += io_in;
    }
    for (const Zero& z : zeros) {
        const long long total = (long long)Hq * z.rows * D;
        zero_rows_kernel<<<unsigned(std::min<long long>((total + 255) / 256, 4096)), 256, 0, c->stream>>>(
            z.out, z.o_hs, z.o_ts, Hq, z.rows, D);
        c->stats.kernel_launches += 1;
    }
    for (size_t i = 0; i < tc.size();) {
        size_t bytes = 0, j = i;
        for (; j < tc.size(); ++j) {
            const size_t b = size_t((tc[j].kv + kPageTokens - 1) / kPageTokens) * Hkv * rt::page_image_bytes(D) +
                             (size_t(tc[j].rows) * c->group / rt::kBM + 1) * Hkv * rt::q_image_bytes(D);
            if (j > i && bytes + b > kReadImageBudget) break;
            bytes += b;
        }
        if ((rc = launch_read_tc(c, std::vector<ReadSub>(tc.begin() + long(i), tc.begin() + long(j)))) != XN_OK) return rc;
        i = j;
    }
    for (int w = 0; w < 4; ++w) {
        const std::vector<ReadSub>& list = w < 2 ? table[w] : mid[w - 2];
        const bool want = w & 1;
        for (size_t i = 0; i < list.size();) {
            // (a launch's scores fit the budget, or it is one request)
            size_t j = i, floats = 0;
            long long most = 1;
            for (; j < list.size() && j - i < size_t(kReadEntries); ++j) {
                const size_t f = want ? align_up(size_t(list[j].kv), 4) * Hq * size_t(list[j].rows) : 0;
                if (j > i && floats + f > kReadScoreBudget / 4) break;
                floats += f;
                most = std::max(most, (long long)list[j].rows * c->group);
            }
            const int mt = w < 2 ? 0 : int(std::min<long long>(4, (most + 15) / 16));
            if ((rc = launch_read_table(c, list.data() + i, int(j - i), want, mt)) != XN_OK) return rc;
            i = j;
        }
    }
    // the other few rows, in portions of a quarter of the units that a launch takes; with weights, whose scores fit, a request of
    // too many rows (long prompts of head_dim > 128) in several row blocks whose weights add up
    if (!few[0].empty()) {
        std::vector<ReadSub> part;
        long long units = 0;
        for (const ReadSub& s : few[0]) {
            const long long per_row = (long long)Hkv * c->subs;
            for (int t0 = 0; t0 < s.rows;) {
                const int take = int(std::min<long long>(s.rows - t0, std::max(1ll, (kMaxUnits / 4 - units) / per_row)));
                ReadSub x = s;
                x.q += (long long)t0 * s.q_ts;
                x.out += (long long)t0 * s.o_ts;
                x.rows = take;
                if (s.causal) x.kv = std::max(0, s.kv - s.rows + t0 + take);
                if (x.kv > 0) {
                    part.push_back(x);
                    units += take * per_row;
                }
                t0 += take;
                if (units >= kMaxUnits / 4) {
                    if ((rc = launch_read_few(c, part, false)) != XN_OK) return rc;
                    part.clear();
                    units = 0;
                }
            }
        }
        if (!part.empty() && (rc = launch_read_few(c, part, false)) != XN_OK) return rc;
    }
    std::vector<ReadSub> part;
    size_t floats = 0;
    long long units = 0;
    const long long per_row = (long long)Hkv * c->subs, most_units = kMaxUnits / 4;
    auto flush = [&]() -> int32_t {
        if (part.empty()) return XN_OK;
        const int32_t e = launch_read_few(c, part, true);
        part.clear();
        floats = 0;
        units = 0;
        return e;
    };
    for (const ReadSub& s : few[1]) {
        const size_t row = align_up(size_t(s.kv), 4) * Hq;
        const int most = int(std::max<long long>(1, std::min<long long>((long long)(kReadScoreBudget / 4 / row), most_units / per_row)));
        if (s.rows <= most) {
            if ((floats + row * s.rows > kReadScoreBudget / 4 || units + s.rows * per_row > most_units) && (rc = flush()) != XN_OK)
                return rc;
            part.push_back(s);
            floats += row * s.rows;
            units += s.rows * per_row;
            continue;
        }
        if ((rc = flush()) != XN_OK) return rc;
        for (int t0 = 0; t0 < s.rows; t0 += most) {
            ReadSub x = s;
            x.rows = std::min(most, s.rows - t0);
            x.q += (long long)t0 * s.q_ts;
            x.out += (long long)t0 * s.o_ts;
            // the block's own rule: row t of it sees the positions up to limit0 + t
            if (s.causal) x.kv = s.kv - s.rows + t0 + x.rows;
            const bool firstb = t0 == 0;
            if (!firstb) {
                x.acct.old_from = s.acct.store ? kAcctPool : kAcctUser;
                x.acct.old_len = s.kv;
            }
            // (acct.kv_len stays the whole prefix, so that positions the block does not see are written too)
            if (x.kv <= 0) x.kv = 0;
            part.push_back(x);
            if ((rc = flush()) != XN_OK) return rc;
        }
    }
    if ((rc = flush()) != XN_OK) return rc;
    for (int i = 0; i < n; ++i) {
        const xn_read_req& r = reqs[i];
        if (!(r.flags & (XN_READ_ACCOUNT | XN_READ_ACCOUNT_SET))) continue;
        const int64_t kv = r.kv_len < 0 ? layer_len(r.stream, r.layer) : r.kv_len;
        int64_t& valid = r.stream->acc_len[size_t(r.layer)];
        valid = (r.flags & XN_READ_ACCOUNT_SET) ? kv : std::max(valid, kv);
    }
    c->stats.batches += 1;
    c->stats.calls += uint64_t(n);
    if (host) {
        if (io_out) XN_CUDA(c, cudaMemcpyAsync(c->io_host + io_in, c->io_dev + io_in, io_out, cudaMemcpyDeviceToHost, c->stream));
        c->stats.d2h_bytes += io_out;
        XN_CUDA(c, cudaStreamSynchronize(c->stream));
        if ((rc = check_device_status(c)) != XN_OK) return rc;
        size_t at = io_in;
        for (int i = 0; i < n; ++i) {
            const xn_read_req& r = reqs[i];
            const size_t qb = size_t(Hq) * r.rows * D * 4;
            if (qb) memcpy(r.out, c->io_host + at, qb);
            at += align_up(qb, 16);
            if (!r.weights) continue;
            const int64_t kv = r.kv_len < 0 ? layer_len(r.stream, r.layer) : r.kv_len;
            const int64_t w_hs = r.weights_stride ? r.weights_stride : kv;
            for (int h = 0; h < Hkv; ++h)
                if (kv) memcpy(r.weights + size_t(h) * w_hs, c->io_host + at + size_t(h) * kv * 4, size_t(kv) * 4);
            at += align_up(size_t(Hkv) * kv * 4, 16);
        }
    }
    return XN_OK;
}

// ---- eviction ------------------------------------------------------------------------------------

int32_t evict_locked(xn_ctx* c, int32_t n, const xn_evict_req* reqs) {
    if (n < 0 || (n > 0 && !reqs)) return fail(c, XN_ERR_ARG, "bad request array");
    if (n == 0) return XN_OK;
    const int Hkv = c->num_kv_heads, D = c->head_dim;
    const bool host = !(reqs[0].flags & XN_REQ_DEVICE_PTRS);
    int32_t rc;
    std::unordered_set<xn_stream*> seen;
    struct One { int l0, nl; int64_t len, kept; bool copy, move; };
    std::vector<One> ones(static_cast<size_t>(n));
    for (int i = 0; i < n; ++i) {
        const xn_evict_req& r = reqs[i];
        if (!stream_ok(c, r.stream)) return fail(c, XN_ERR_HANDLE, "stream handle is not live");
        if (r.flags & ~uint32_t(XN_REQ_DEVICE_PTRS | XN_EVICT_COPY)) return fail(c, XN_ERR_ARG, "xn_kv_evict: unknown flags 0x%x", r.flags);
        if (host == bool(r.flags & XN_REQ_DEVICE_PTRS))
            return fail(c, XN_ERR_ARG, "host and device requests cannot be mixed in one batch");
        if (r.layer < -1 || r.layer >= c->num_layers) return fail(c, XN_ERR_ARG, "layer %d outside -1..%d", r.layer, c->num_layers - 1);
        if (r.keep < 1 || r.recent < 0 || r.recent > r.keep)
            return fail(c, XN_ERR_ARG, "keep %lld, recent %lld: 1 <= keep and 0 <= recent <= keep are wanted", (long long)r.keep, (long long)r.recent);
        if (!seen.insert(r.stream).second) return fail(c, XN_ERR_ARG, "a stream occurs twice in one call");
        One& o = ones[size_t(i)];
        o.copy = r.flags & XN_EVICT_COPY;
        if (o.copy ? (!r.k_out || !r.v_out) : (r.k_out || r.v_out))
            return fail(c, XN_ERR_ARG, "k_out and v_out belong to XN_EVICT_COPY, and to it alone");
        o.l0 = r.layer < 0 ? 0 : r.layer;
        o.nl = r.layer < 0 ? c->num_layers : 1;
        o.len = layer_len(r.stream, o.l0);
        for (int l = o.l0; l < o.l0 + o.nl; ++l) {
            if (r.stream->hw[size_t(l)] > r.stream->cap)
                return fail(c, XN_ERR_CAPACITY, "the stream has folded around its capacity: its order is lost");
            if (layer_len(r.stream, l) != o.len)
                return fail(c, XN_ERR_ARG, "layers %d and %d hold %lld and %lld positions: evict them one by one", o.l0, l,
                            (long long)o.len, (long long)layer_len(r.stream, l));
        }
        if (o.len > (int64_t(1) << 30)) return fail(c, XN_ERR_CAPACITY, "%lld positions are too many", (long long)o.len);
        o.kept = std::min(r.keep, o.len);
        o.move = !o.copy && o.kept < o.len;
    }
    if ((rc = refuse_capture(c)) != XN_OK) return rc;
    if ((rc = ready_read_kernels(c)) != XN_OK) return rc;

    // host pointers: outputs one behind the other in the staging buffer
    size_t io = 0;
    if (host) {
        for (int i = 0; i < n; ++i) {
            const size_t rows = size_t(ones[size_t(i)].nl) * Hkv * size_t(ones[size_t(i)].kept);
            if (reqs[i].kept) io += align_up(rows * 4, 16);
            if (reqs[i].weights_out) io += align_up(rows * 4, 16);
            if (ones[size_t(i)].copy) io += 2 * align_up(rows * D * 4, 16);
        }
        if (io && (rc = grow_io(c, io)) != XN_OK) return rc;
    }
    // Entries of layers with one account length each; a launch takes up to kEvictEntries of them.
    std::vector<EvictDev> ev;
    size_t kept_ws = 0, at = 0;
    for (int i = 0; i < n; ++i) {
        const One& o = ones[size_t(i)];
        if (o.len == 0) continue;
        const xn_evict_req& r = reqs[i];
        EvictDev e = {};
        e.len = int(o.len);
        e.keep = int(o.kept);
        e.recent = int(std::min(r.recent, o.kept));
        e.copy = o.copy ? 1 : (o.move ? 0 : 2);
        const size_t per_layer = size_t(Hkv) * size_t(o.kept), rows = per_layer * o.nl;
        if (host) {
            auto take = [&](size_t bytes) { unsigned char* p = c->io_dev + at; at += align_up(bytes, 16); return p; };
            if (r.kept) e.kept = reinterpret_cast<int*>(take(rows * 4));
            if (r.weights_out) e.w_out = reinterpret_cast<float*>(take(rows * 4));
            if (o.copy) {
                e.k_out = reinterpret_cast<float*>(take(rows * D * 4));
                e.v_out = reinterpret_cast<float*>(take(rows * D * 4));
            }
        } else {
            e.kept = r.kept;
            e.w_out = r.weights_out;
            e.k_out = r.k_out;
            e.v_out = r.v_out;
        }
        if (!o.copy && !o.move && !e.kept && !e.w_out) continue;   // nothing to do, nothing to report
        if ((rc = device_pages(c, r.stream, &e.pages)) != XN_OK) return rc;
        for (int l = o.l0; l < o.l0 + o.nl;) {
            int m = l + 1;
            while (m < o.l0 + o.nl && r.stream->acc_len[size_t(m)] == r.stream->acc_len[size_t(l)]) ++m;
            EvictDev x = e;
            x.layer0 = l;
            x.n_layers = m - l;
            x.acc_len = int(std::min(r.stream->acc_len[size_t(l)], o.len));
            const size_t skip = size_t(l - o.l0) * per_layer;
            if (x.kept) x.kept += skip;
            if (x.w_out) x.w_out += skip;
            if (x.k_out) x.k_out += skip * D;
            if (x.v_out) x.v_out += skip * D;
            x.kept_ws = reinterpret_cast<int*>(kept_ws);   // an offset until the buffer is there
            kept_ws += size_t(x.n_layers) * per_layer;
            ev.push_back(x);
            l = m;
        }
    }
    if (ev.empty()) return XN_OK;
    if ((rc = grow_device(c, &c->read_ws, &c->read_ws_cap, kept_ws)) != XN_OK) return rc;
    const EvictPools pools = {c->k_pool, c->v_pool, c->pool8, c->acct_pool, c->pool_pages, Hkv, D, c->nv, c->dq};
    for (size_t i0 = 0; i0 < ev.size(); i0 += kEvictEntries) {
        EvictTable tab;
        tab.n = int(std::min<size_t>(kEvictEntries, ev.size() - i0));
        int head0 = 0, longest = 1, keep_most = 1;
        bool any_copy = false, any_move = false;
        for (int i = 0; i < tab.n; ++i) {
            EvictDev& e = tab.e[i];
            e = ev[i0 + size_t(i)];
            e.kept_ws = reinterpret_cast<int*>(c->read_ws) + reinterpret_cast<uintptr_t>(e.kept_ws);
            e.head0 = head0;
            head0 += e.n_layers * Hkv;
            longest = std::max(longest, e.len - e.recent);
            keep_most = std::max(keep_most, e.keep);
            any_copy |= e.copy == 1;
            any_move |= e.copy == 0;
        }
        // blocks per (layer, head): 4096 candidates each (a run of 4 per thread) up to 8 blocks, longer
        // runs beyond that
        int cluster = 1, run = 4;
        while (cluster < ev::kMaxCluster && longest > cluster * ev::kThreads * run) cluster *= 2;
        while (run <= ev::kMaxRun && longest > cluster * ev::kThreads * run) run *= 2;
        if (run > ev::kMaxRun) run = 0;
        XN_CUDA(c, launch_pdl(c, evict_select_kernel, dim3(unsigned(head0 * cluster)), ev::kThreads, size_t(ev::kThreads) * (run + 1) * 4,
                              true, unsigned(cluster), tab, c->acct_pool, c->pool_pages, Hkv, cluster, run));
        if (any_copy)
            XN_CUDA(c, launch_pdl(c, evict_copy_kernel<4>, dim3(unsigned(head0), unsigned(std::min((keep_most + 31) / 32, 65535))), 256, 0,
                                  true, 0, tab, pools));
        if (any_move) {
            const int row_bytes = c->kv_u8 ? c->dq : c->nv * 16;
            const unsigned slices = unsigned((row_bytes + kMoveSlice - 1) / kMoveSlice);
            XN_CUDA(c, launch_pdl(c, evict_move_kernel, dim3(unsigned(head0), 2 * slices), kMoveThreads, 0, true, 0, tab, pools));
        }
    }
    // the streams shrink: lengths, accounts, and the pages that no layer needs any more (their next
    // owner's launches come behind these on the context's stream)
    for (int i = 0; i < n; ++i) {
        const One& o = ones[size_t(i)];
        if (!o.move) continue;
        xn_stream* s = reqs[i].stream;
        for (int l = o.l0; l < o.l0 + o.nl; ++l) {
            s->hw[size_t(l)] = o.kept;
            s->acc_len[size_t(l)] = s->acc_len[size_t(l)] > 0 ? o.kept : 0;
            s->shift[size_t(l)] += o.len - o.kept;
        }
        int64_t most = 0;
        for (int l = 0; l < c->num_layers; ++l) most = std::max(most, layer_len(s, l));
        while (int64_t(s->pages.size()) > (most + kPageTokens - 1) / kPageTokens) {
            c->free_pages.push_back(s->pages.back());
            s->pages.pop_back();
        }
        s->pages_d_valid = std::min(s->pages_d_valid, s->pages.size());
        c->pcache.valid = false;   // the kept plan may name this stream's pages and length
    }
    if (host) {
        if (io) XN_CUDA(c, cudaMemcpyAsync(c->io_host, c->io_dev, io, cudaMemcpyDeviceToHost, c->stream));
        XN_CUDA(c, cudaStreamSynchronize(c->stream));
        c->stats.d2h_bytes += io;
        size_t p = 0;
        for (int i = 0; i < n; ++i) {
            const One& o = ones[size_t(i)];
            if (o.len == 0) continue;
            const size_t rows = size_t(o.nl) * Hkv * size_t(o.kept);
            auto give = [&](void* to, size_t bytes) { memcpy(to, c->io_host + p, bytes); p += align_up(bytes, 16); };
            if (reqs[i].kept) give(reqs[i].kept, rows * 4);
            if (reqs[i].weights_out) give(reqs[i].weights_out, rows * 4);
            if (o.copy) {
                give(reqs[i].k_out, rows * D * 4);
                give(reqs[i].v_out, rows * D * 4);
            }
        }
    }
    return XN_OK;
}
