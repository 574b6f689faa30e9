"""Reads that do not append (cross attention), the account of attention weight, eviction: against
plain implementations in 64 bits.

Tolerances.  Inputs are N(0, 1), so a score q.k / sqrt(D) is of order 1.  On the tensor-core path
an operand keeps 22 significand bits (relative error 2^-23 each) and the lo * lo term (2^-22) is
dropped: independent errors of at most 4 * 2^-23 per product give a score error of rms
4 * 2^-23 * |q| |k| / D ~ 5e-7; the 24 accumulation steps add at most 24 * 2^-24 ~ 1.4e-6 of the
score.  exp, the sum and the second product add 2^-22 each.  In all below 4e-6 relative to the
result's norm; the f32 path is closer.  A single output (up to ~4) may be off by four times that."""
import os

import numpy as np
import pytest

import oracle as xo
import xor_net_b200 as xn
from gpu_util import errs

pytestmark = pytest.mark.gpu

REL, ABS = 4e-6, 2e-5


def near(got, want, what="", rel=REL, abs_tol=ABS):
    a, r = errs(got, want)
    assert np.all(np.isfinite(np.asarray(got))) and r <= rel and a <= abs_tol, f"{what}: max abs {a:.3e}, rel {r:.3e}"


def plain(q, k, v, causal=False):
    """q [Hq, R, D], k, v [Hkv, n, D] -> out [Hq, R, D], weights summed per KV head [Hkv, n], in f64."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    Hq, R, D = q.shape
    Hkv, n, _ = k.shape
    G = Hq // Hkv
    out, w = np.zeros((Hq, R, D)), np.zeros((Hkv, n))
    for h in range(Hq):
        for t in range(R):
            m = max(0, n - R + t + 1) if causal else n
            if m == 0:
                continue
            s = k[h // G, :m] @ q[h, t] / np.sqrt(D)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h, t] = p @ v[h // G, :m]
            w[h // G, :m] += p
    return out, w


def context(monkeypatch, path, *args, **kw):
    """path: "few", "mid" and "tc" force the f32 kernels, the warp-MMA one and the tcgen05 passes (where the
    shape allows them), "auto" leaves the choice."""
    if path != "auto":
        monkeypatch.setenv("XORNET_ATTN_READ_PATH", path)
    return xn.Context(*args, **kw)


def rows(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def filled(ctx, rng, n, layer=0, cap=None):
    st = ctx.new_stream(cap or max(n, 1))
    k, v = rows(rng, ctx.num_kv_heads, n, ctx.head_dim), rows(rng, ctx.num_kv_heads, n, ctx.head_dim)
    if n:
        st.write(layer, 0, k, v)
    return st, k, v


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("Hq,Hkv,D", [(20, 5, 128), (4, 4, 64), (6, 2, 100), (5, 1, 33), (8, 2, 8), (16, 2, 80), (3, 1, 1)])
def test_write_and_read_shapes(monkeypatch, path, Hq, Hkv, D):
    rng = np.random.default_rng(D + Hq)
    ctx = context(monkeypatch, path, 2, Hq, Hkv, D, pool_pages=64, shuffle_seed=5)
    for n, R in [(1, 1), (1, 3), (63, 2), (64, 1), (65, 7), (127, 33), (129, 1), (200, 130), (300, 5)]:
        st, k, v = filled(ctx, rng, n, layer=1)
        assert np.array_equal(st.read_range(1, 0, n)[0], k) and np.array_equal(st.read_range(1, 0, n)[1], v)
        q = rows(rng, Hq, R, D)
        (out,), (w,) = ctx.cross_attention([st], 1, [q], weights=True)
        want, want_w = plain(q, k, v)
        near(out, want, f"n={n} R={R}")
        near(w, want_w, f"weights n={n} R={R}", abs_tol=ABS * max(1, R * Hq // Hkv))
        (out2,) = ctx.cross_attention([st], 1, [q])
        near(out2, want, f"without weights n={n} R={R}")
        # a shorter prefix; the rest of the stream is not seen
        m = max(1, n // 2)
        (out,) = ctx.cross_attention([st], 1, [q], kv_lens=[m])
        near(out, plain(q, k[:, :m], v[:, :m])[0], f"prefix {m} of {n}")
        st.destroy()
    ctx.close()


@pytest.mark.parametrize("D", [129, 200, 256])
def test_long_rows_of_the_cache(D):
    rng = np.random.default_rng(D)
    ctx = xn.Context(1, 4, 2, D, pool_pages=16)
    st, k, v = filled(ctx, rng, 150)
    q = rows(rng, 4, 40, D)
    (out,), (w,) = ctx.cross_attention([st], 0, [q], weights=True, causal=True)
    want, want_w = plain(q, k, v, causal=True)
    near(out, want)
    near(w, want_w, abs_tol=40 * 2 * ABS)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("n,R", [(1, 1), (64, 64), (70, 3), (129, 129), (200, 40), (40, 90), (1, 130), (300, 257)])
def test_causal_rows_and_rows_that_see_nothing(monkeypatch, path, n, R):
    rng = np.random.default_rng(n * 1000 + R)
    ctx = context(monkeypatch, path, 1, 6, 2, 64, pool_pages=16)
    st, k, v = filled(ctx, rng, n)
    q = rows(rng, 6, R, 64)
    (out,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True)
    want, want_w = plain(q, k, v, causal=True)
    near(out, want)
    near(w, want_w, abs_tol=ABS * R)
    if R > n:
        assert np.array_equal(out[:, : R - n], np.zeros_like(out[:, : R - n]))
    (out,) = ctx.cross_attention([st], 0, [q], causal=True)
    near(out, want)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
def test_batches_share_streams_mix_lengths_and_leave_neighbours_alone(monkeypatch, path):
    import torch

    rng = np.random.default_rng(3)
    Hq, Hkv, D = 8, 2, 64
    ctx = context(monkeypatch, path, 2, Hq, Hkv, D, pool_pages=64, shuffle_seed=11)
    a, ka, va = filled(ctx, rng, 500, layer=0)
    b, kb, vb = filled(ctx, rng, 77, layer=1)
    c = ctx.new_stream(10)   # holds nothing
    cases = [(a, 0, ka, va, 1, 500), (a, 0, ka, va, 5, 65), (b, 1, kb, vb, 33, 77), (c, 0, ka, va, 4, 0), (b, 1, kb, vb, 0, 77),
             (a, 0, ka, va, 140, 300), (a, 0, ka, va, 2, 0)]
    for seq_major in (False, True):
        entries, outs, keep = [], [], []
        for st, layer, k, v, R, n in cases:
            q = rows(rng, Hq, R, D)
            src = q.transpose(1, 0, 2) if seq_major else q
            # odd alignment: every tensor starts one float into its buffer, between guard values
            buf = torch.full((q.size + 2,), 7.0, device="cuda")
            buf[1:-1] = torch.from_numpy(np.ascontiguousarray(src)).reshape(-1)
            out = torch.full((q.size + 2,), 9.0, device="cuda")
            w = torch.full((Hkv * 600 + 1,), 3.0, device="cuda")
            entries.append((st, layer, R, n, buf[1:].data_ptr(), out[1:].data_ptr(), w[1:].data_ptr(), 600))
            outs.append((q, k, v, R, n, out, w))
            keep.append(buf)
        torch.cuda.synchronize()
        flags = xn.REQ_DEVICE_PTRS | (xn.REQ_SEQ_MAJOR if seq_major else 0)
        ctx.submit_reads(ctx.make_read_batch(entries, flags))
        ctx.synchronize()
        for q, k, v, R, n, out, w in outs:
            got = out.cpu().numpy()
            assert got[0] == 9.0 and got[-1] == 9.0
            got = got[1:-1].reshape((R, Hq, D) if seq_major else (Hq, R, D))
            got = got.transpose(1, 0, 2) if seq_major else got
            wn = w.cpu().numpy()
            want, want_w = plain(q, k[:, :n], v[:, :n])
            if R:
                near(got, want, f"R={R} n={n}") if n else np.testing.assert_array_equal(got, 0.0)
            for h in range(Hkv):
                row = wn[1 + h * 600: 1 + h * 600 + 600]
                assert np.all(row[n:] == 3.0)
                if n and R:
                    near(row[:n], want_w[h], abs_tol=ABS * R * 4)
                elif n:
                    assert np.array_equal(row[:n], np.zeros(n, np.float32))
            assert wn[0] == 3.0
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("lens", [(100, 5000), (5000, 100), (4096, 4097), (4097, 4096)])
def test_one_stream_with_a_short_and_a_long_prefix_in_one_call(monkeypatch, path, lens):
    """The prefixes lie on both sides of 64 pages, where the stream's page table on the device grows; the
    streams between and behind would take the place of a table that went away.  In another layer and in
    the second round (tables there already) as well."""
    rng = np.random.default_rng(lens[0])
    Hq, Hkv, D, n = 4, 2, 64, 5000
    for R, weights in [(1, False), (1, True), (9, False), (9, True)]:
        ctx = context(monkeypatch, path, 2, Hq, Hkv, D, pool_pages=90, shuffle_seed=5)
        st, k, v = filled(ctx, rng, n)
        k1, v1 = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D)
        st.write(1, 0, k1, v1)
        b, kb, vb = filled(ctx, rng, 100)
        c, kc, vc = filled(ctx, rng, 77)
        entries = [(st, 0, lens[0], k, v), (b, 0, 100, kb, vb), (st, 0, lens[1], k, v), (c, 0, 77, kc, vc), (st, 1, lens[0], k1, v1)]
        qs = [rows(rng, Hq, R, D) for _ in entries]
        for turn in range(2):
            got = ctx.cross_attention([e[0] for e in entries], [e[1] for e in entries], qs, kv_lens=[e[2] for e in entries], weights=weights)
            outs, ws = got if weights else (got, [None] * len(entries))
            for (_, layer, m, kk, vv), q, out, w in zip(entries, qs, outs, ws):
                want, want_w = plain(q, kk[:, :m], vv[:, :m])
                near(out, want, f"R={R} m={m} layer={layer} turn={turn}")
                if weights:
                    near(w, want_w, f"weights R={R} m={m} layer={layer} turn={turn}", abs_tol=ABS * R)
        ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc", "auto"])
@pytest.mark.parametrize("ctas", [1, 8, 32, 64])
def test_reads_with_fewer_split_kv_blocks_than_sms(monkeypatch, path, ctas):
    """Long units cut over all SMs by the read of some rows, whatever the split-KV launches are bounded to."""
    monkeypatch.setenv("XORNET_ATTN_DECODE_CTAS", str(ctas))
    rng = np.random.default_rng(ctas)
    ctx = context(monkeypatch, path, 1, 8, 2, 64, pool_pages=300, shuffle_seed=4)
    made = [filled(ctx, rng, n) for n in (9001, 3000, 5500)]
    for R in (1, 3, 12):
        qs = [rows(rng, 8, R, 64) for _ in made]
        for _ in range(2):   # (the counters are left as they were found)
            outs, ws = ctx.cross_attention([st for st, _, _ in made], 0, qs, causal=R > 1, weights=True)
        for (st, k, v), q, out, w in zip(made, qs, outs, ws):
            want, want_w = plain(q, k, v, causal=R > 1)
            near(out, want, f"R={R}")
            near(w, want_w, f"weights R={R}", abs_tol=ABS * R)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
def test_account_adds_up_is_set_and_follows_writes(monkeypatch, path):
    rng = np.random.default_rng(8)
    Hq, Hkv, D, n = 6, 3, 64, 150
    ctx = context(monkeypatch, path, 2, Hq, Hkv, D, pool_pages=16, shuffle_seed=2)
    st, k, v = filled(ctx, rng, n, layer=1, cap=400)
    assert np.array_equal(st.account(1), np.zeros((Hkv, n), np.float32))
    total = np.zeros((Hkv, n))
    for R, m, causal in [(3, 100, False), (40, 150, True), (1, 20, False), (2, 150, False)]:
        q = rows(rng, Hq, R, D)
        _, (w,) = ctx.cross_attention([st], 1, [q], kv_lens=[m], causal=causal, account="add", weights=True)
        total[:, :m] += plain(q, k[:, :m], v[:, :m], causal)[1]
        near(st.account(1), total, abs_tol=1e-4)
        assert np.array_equal(w, st.account(1, 0, m))
    assert np.array_equal(st.account(0, 0, 0), np.zeros((Hkv, 0), np.float32))
    # without an account flag the weights are this call's own and nothing is kept
    before = st.account(1)
    q = rows(rng, Hq, 4, D)
    _, (w,) = ctx.cross_attention([st], 1, [q], weights=True)
    near(w, plain(q, k, v)[1], abs_tol=1e-4)
    assert np.array_equal(st.account(1), before)
    # set: starts afresh, positions behind the prefix have none
    ctx.cross_attention([st], 1, [q], kv_lens=[70], account="set")
    got = st.account(1)
    near(got[:, :70], plain(q, k[:, :70], v[:, :70])[1], abs_tol=1e-4)
    assert np.array_equal(got[:, 70:], np.zeros_like(got[:, 70:]))
    # rows written at 30 take the account from there on with them
    st.write(1, 30, k[:, 30:40], v[:, 30:40])
    after = st.account(1)
    assert np.array_equal(after[:, :30], got[:, :30]) and not after[:, 30:].any()
    # ... and so does an appending attention, also one that reuses the plan of the step before
    st.set_account(1, 0, np.ones((Hkv, n)))
    x = rows(rng, 1, Hq, 1, D)
    kv = rows(rng, 1, Hkv, 1, D)
    ctx.attention(st, 1, 140, x, kv, kv)
    assert st.account(1)[:, :140].all() and not st.account(1)[:, 140:].any()
    # set in the middle: what lies before and had none is zero, what lies behind is forgotten
    st.set_account(1, 145, np.full((Hkv, 3), 2.0))
    got = st.account(1)
    assert np.all(got[:, :140] == 1) and not got[:, 140:145].any() and np.all(got[:, 145:148] == 2) and not got[:, 148:].any()
    st.reset()
    assert st.length(1) == 0 and st.evicted(1) == 0
    ctx.close()


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 2), (100, 3, 3), (128, 8, 2), (16, 2, 1)])
def test_u8_cache_format(D, Hq, Hkv):
    rng = np.random.default_rng(D)
    ctx = xn.Context(1, Hq, Hkv, D, pool_pages=32, kv_format=xn.KV_U8, shuffle_seed=3)
    for n, R in [(1, 1), (70, 2), (200, 64), (131, 9)]:
        st, k, v = filled(ctx, rng, n)
        kd, vd = st.read_range(0, 0, n)   # the dequantised rows: what attention runs over
        q = rows(rng, Hq, R, D)
        for causal in (False, True):
            want, want_w = plain(q, kd, vd, causal)
            (out,), (w,) = ctx.cross_attention([st], 0, [q], causal=causal, weights=True, account="set")
            near(out, want, f"{n} {R}")
            near(w, want_w, abs_tol=ABS * R * Hq)
            (out,) = ctx.cross_attention([st], 0, [q], causal=causal)
            near(out, want, f"{n} {R} without weights")
        kept, ck, cv, cw = st.evict_copy(max(1, n // 3), recent=min(4, max(1, n // 3)))
        u = st.read_u8(0, 0, n)
        acct = st.account(0)
        for h in range(Hkv):
            assert np.array_equal(ck[0, h], kd[h, kept[0, h]]) and np.array_equal(cv[0, h], vd[h, kept[0, h]])
            assert np.array_equal(cw[0, h], acct[h, kept[0, h]])
        kept2 = st.evict(max(1, n // 3), recent=min(4, max(1, n // 3)))
        assert np.array_equal(kept, kept2)
        u2 = st.read_u8(0, 0, kept.shape[2])
        for h in range(Hkv):
            for x, y in zip(u, u2):
                assert np.array_equal(x[h][kept[0, h]], y[h])
        st.destroy()
    ctx.close()


def test_u8_weights_need_a_head_dim_the_tensor_cores_take():
    rng = np.random.default_rng(0)
    ctx = xn.Context(1, 2, 1, 200, pool_pages=4, kv_format=xn.KV_U8)
    st, _, _ = filled(ctx, rng, 10)
    q = rows(rng, 2, 3, 200)
    kd, vd = st.read_range(0, 0, 10)
    (out,) = ctx.cross_attention([st], 0, [q])
    near(out, plain(q, kd, vd)[0])
    with pytest.raises(xn.XnError) as e:
        ctx.cross_attention([st], 0, [q], account="add")
    assert e.value.code == 2
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
def test_values_over_many_orders_of_magnitude(monkeypatch, path):
    """K, V and Q rows of very different sizes (a page's largest element sets its scale), zero rows."""
    rng = np.random.default_rng(17)
    Hq, Hkv, D, n, R = 4, 1, 64, 200, 40
    ctx = context(monkeypatch, path, 1, Hq, Hkv, D, pool_pages=8)
    st = ctx.new_stream(n)
    k, v, q = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D), rows(rng, Hq, R, D)
    k *= np.exp2(rng.integers(-6, 2, size=(Hkv, n, 1))).astype(np.float32)
    v *= np.exp2(rng.integers(-12, 1, size=(Hkv, n, 1))).astype(np.float32)
    v[:, 64:128] *= np.float32(2.0 ** 14)
    k[:, 5] = 0
    v[:, 6] = 0
    k[:, 128:192] = 0
    q *= np.exp2(rng.integers(-20, 1, size=(Hq, R, 1))).astype(np.float32)
    q[:, 3] = 0
    q[0, 0] *= np.float32(1e-30)
    st.write(0, 0, k, v)
    (out,) = ctx.cross_attention([st], 0, [q], causal=True)
    want = plain(q, k, v, True)[0]
    near(out, want, abs_tol=4 * REL * np.abs(want).max())
    # row by row: every row's own norm, not the largest row's
    for h in range(Hq):
        for t in range(R):
            near(out[h, t], want[h, t], f"row {h} {t}", abs_tol=np.inf)
    ctx.close()


def spread_rows(rng, what, e):
    """256 positions and 190 causal query rows (the first sees 67), with values 2^e times the others' in a
    whole page of V, in one row of V or of K, or in every second row of them.  "behind": in positions that most query rows do not see;
    "unweighted": seen by all of them, with a score that leaves them no weight (exp(-200) and less).
    "faint": a page of zeros beside pages of 2^-e."""
    Hq, Hkv, D, n, R = 4, 2, 64, 256, 190
    k, v, q = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D), np.abs(rows(rng, Hq, R, D)) + np.float32(0.1)
    big = np.float32(2.0 ** e)
    if what == "faint":
        v /= big
        v[:, 64:128] = 0
        v[:, 130] = 0
        return k, v, q
    kind, how = what.split("_")
    at = {("page", "behind"): slice(192, 256), ("page", "unweighted"): slice(64, 128),
          ("row", "behind"): slice(200, 201), ("row", "unweighted"): slice(40, 41),
          ("krow", "behind"): slice(200, 201), ("krow", "unweighted"): slice(40, 41),
          ("rows", "unweighted"): slice(1, 256, 2), ("krows", "unweighted"): slice(1, 256, 2)}[kind, how]
    if kind == "rows":
        v[:, 64:128] /= 32                     # (and neighbouring pages of different sizes beside that)
    if kind in ("krow", "krows"):
        k[:, at] = -np.abs(k[:, at]) * big if how == "unweighted" else k[:, at] * big
    else:
        v[:, at] *= big
        if how == "unweighted":
            k[:, at] = -40 - np.abs(k[:, at])   # score below -(0.1 + 0) * 40 * 64 / 8 = -32, about -260
    return k, v, q


def check_spread(monkeypatch, path, what, e):
    """Row by row, each against its own norm: what a query row gives no weight to must not coarsen the rest
    of its output.  Rows that share a page and lie within 2^16 of one another have an element error of
    2^-23 of their own largest element from the scale they share, beside the 2^-23 of the split; that
    and the neighbours' factors (up to 2^10: 2^-29 of the weights) stay well inside the tolerance above."""
    rng = np.random.default_rng(1000 + e)
    ctx = context(monkeypatch, path, 1, 4, 2, 64, pool_pages=8, shuffle_seed=3)
    k, v, q = spread_rows(rng, what, e)
    st = ctx.new_stream(256)
    st.write(0, 0, k, v)
    (out,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True)
    want, want_w = plain(q, k, v, True)
    # (query rows that see a K row of 2^e: |score| is of order 2^e, and its rounding alone, 2^-24 of that in any
    # f32 arithmetic, may shift the weights by as much)
    seen_by = 200 - 66 if what == "krow_behind" else 190
    for h in range(4):
        for t in range(seen_by):
            near(out[h, t], want[h, t], f"{what} 2^{e} row {h} {t}", abs_tol=np.inf)
    if seen_by == 190:
        near(w, want_w, f"{what} 2^{e} weights", abs_tol=ABS * 190)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("e", [9, 11, 20, 30, 40])
@pytest.mark.parametrize("what", ["page_behind", "page_unweighted", "faint"])
def test_neighbouring_pages_of_very_different_sizes(monkeypatch, path, what, e):
    check_spread(monkeypatch, path, what, e)


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("e", [7, 9, 15, 17, 20, 30, 40])
@pytest.mark.parametrize("what", ["row_behind", "row_unweighted", "rows_unweighted", "krow_behind", "krow_unweighted", "krows_unweighted"])
def test_rows_of_one_page_of_very_different_sizes(monkeypatch, path, what, e):
    check_spread(monkeypatch, path, what, e)


@pytest.mark.parametrize("D", [64, 50])
@pytest.mark.parametrize("what", ["page_behind", "row_behind", "row_unweighted", "rows_unweighted", "krow_behind"])
def test_u8_rows_of_very_different_sizes(monkeypatch, what, D):
    """Over the u8 format, whose rows have a scale each, against the values that it holds; head sizes with and
    without padding bytes, queries that cannot be read four at a time."""
    rng = np.random.default_rng(D)
    ctx = context(monkeypatch, "tc", 1, 4, 2, D, pool_pages=8, shuffle_seed=3, kv_format=xn.KV_U8)
    k, v, q = (np.ascontiguousarray(x[..., :D]) for x in spread_rows(rng, what, 30))
    st = ctx.new_stream(256)
    st.write(0, 0, k, v)
    k, v = st.read_range(0, 0, 256)
    (out,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True)
    want, want_w = plain(q, k, v, True)
    seen_by = 200 - 66 if what == "krow_behind" else 190
    for h in range(4):
        for t in range(seen_by):
            near(out[h, t], want[h, t], f"{what} row {h} {t}", abs_tol=np.inf)
    if seen_by == 190:
        near(w, want_w, f"{what} weights", abs_tol=ABS * 190)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("e", [10, 20, 30])
def test_a_large_row_of_little_weight(monkeypatch, path, e):
    """A position that gets about e^-20 of the weight, with values of 2^e, in a page that is 2^-5 of its
    neighbour.  f32 arithmetic: REL of the weighted magnitudes.  Tensor cores: 2^-39 of the largest weight
    times the large values besides (the halves of P keep 2^-25 of 2^14), taken twice for its sum."""
    rng = np.random.default_rng(e)
    Hq, Hkv, D, n, R = 4, 2, 64, 256, 150
    ctx = context(monkeypatch, path, 1, Hq, Hkv, D, pool_pages=8)
    k, v = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D)
    q = np.abs(rows(rng, 1, 1, D)).repeat(Hq, 0).repeat(R, 1) + np.float32(0.1)
    k[:, 70] = -20 * np.sqrt(D) * q[0, 0] / np.sum(q[0, 0] ** 2)
    v[:, 64:128] /= 32
    v[:, 70] *= np.float32(2.0 ** (e + 5))
    st = ctx.new_stream(n)
    st.write(0, 0, k, v)
    (out,) = ctx.cross_attention([st], 0, [q])
    want = plain(q, k, v)[0]
    s = np.einsum("htd,hnd->htn", q.astype(np.float64), np.repeat(k, 2, 0).astype(np.float64)) / np.sqrt(D)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    mag = np.einsum("htn,hnd->htd", p, np.abs(np.repeat(v, 2, 0)).astype(np.float64))
    floor = 2.0 ** -38 * p.max(-1, keepdims=True) * np.abs(v).max() if path != "few" else 0.0
    assert np.all(np.abs(out - want) <= 4 * REL * mag.max(-1, keepdims=True) + floor)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("n,R", [(3, 4), (200, 9), (2000, 40)])
def test_scores_of_minus_infinity_throughout_are_no_numbers(monkeypatch, path, n, R):
    """0 / 0, as in a plain softmax; the causal rows that see nothing stay zeros."""
    rng = np.random.default_rng(n)
    ctx = context(monkeypatch, path, 1, 4, 2, 64, pool_pages=64)
    st = ctx.new_stream(n)
    k, v = rows(rng, 2, n, 64), rows(rng, 2, n, 64)
    k[0, :, 5] = -np.inf
    st.write(0, 0, k, v)
    q = np.abs(rows(rng, 4, R, 64)) + 0.1
    (out,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True)
    none = max(0, R - n)
    assert np.all(out[:, :none] == 0)
    assert np.all(np.isnan(out[:2, none:])) and np.all(np.isnan(w[0]))
    with np.errstate(invalid="ignore"):
        want, ww = plain(q, k, v, causal=True)
    near(out[2:], want[2:], "the other head")
    near(w[1], ww[1], "its weights", abs_tol=4e-6 * R * 2)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_infinities_and_nan_stay_where_they_are_seen(monkeypatch, path, value):
    rng = np.random.default_rng(4)
    Hq, Hkv, D, n, R = 4, 2, 64, 140, 70
    ctx = context(monkeypatch, path, 1, Hq, Hkv, D, pool_pages=8)
    k, v, q = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D), rows(rng, Hq, R, D)
    q = np.abs(q)   # (so that an infinite K element gives a score of one sign)
    for which in ("k", "v"):
        kb, vb = k.copy(), v.copy()
        (kb if which == "k" else vb)[1, 120, 7] = value
        st = ctx.new_stream(n)
        st.write(0, 0, kb, vb)
        (out,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True)
        with np.errstate(all="ignore"):
            want, want_w = plain(q, kb, vb, True)
        first = 120 - (n - R)   # rows from here on see the position
        near(out[:2], want[:2])                     # the other KV head
        near(out[2:, :first], want[2:, :first])     # rows before it
        got, ref = out[2:, first:], want[2:, first:]
        assert np.array_equal(np.isfinite(got), np.isfinite(ref)), which
        assert np.array_equal(np.isnan(got), np.isnan(ref)), which
        if which == "v":
            near(w, want_w, abs_tol=ABS * R)
            np.testing.assert_allclose(got[np.isfinite(ref)], ref[np.isfinite(ref)], atol=ABS, rtol=REL * 4)
        st.destroy()
    # behind the prefix anything may lie
    kb, vb = k.copy(), v.copy()
    kb[:, 100:], vb[:, 100:] = value, value
    st = ctx.new_stream(n)
    st.write(0, 0, kb, vb)
    (out,), (w,) = ctx.cross_attention([st], 0, [q], kv_lens=[100], weights=True)
    want, want_w = plain(q, k[:, :100], v[:, :100])
    near(out, want)
    near(w, want_w, abs_tol=ABS * R)
    # a query row with an infinity spoils itself alone
    st.write(0, 0, k, v)
    qb = q.copy()
    qb[0, 9, 3] = value
    (out,) = ctx.cross_attention([st], 0, [qb])
    want = plain(q, k, v)[0]
    assert not np.isfinite(out[0, 9]).any()
    keep = np.ones((Hq, R), bool)
    keep[0, 9] = False
    near(out[keep], want[keep])
    ctx.close()


def kept_of(account, keep, recent):
    """The definition: account [n] -> kept positions."""
    n = len(account)
    keep = min(keep, n)
    recent = min(recent, keep)
    a = np.where(np.isnan(account), -np.inf, account.astype(np.float64))
    nan = np.isnan(account)
    old = n - recent
    order = np.lexsort((np.arange(old), ~nan[:old] * -1, -a[:old]))   # value, then numbers before NaN, then position
    return np.concatenate([np.sort(order[: keep - recent]), np.arange(old, n)]).astype(np.int32)


@pytest.mark.parametrize("n,keep,recent", [(1, 1, 0), (10, 3, 0), (64, 64, 5), (65, 64, 0), (100, 40, 40), (130, 65, 64), (300, 299, 7),
                                           (1000, 1, 0), (1000, 700, 3), (5000, 5000, 10), (5000, 9000, 10), (9000, 4097, 4096),
                                           (20000, 777, 5), (70000, 33333, 1)])
def test_evict_keeps_what_the_account_says(n, keep, recent):
    rng = np.random.default_rng(n + keep)
    Hkv, D, L = 2, 12, 2
    ctx = xn.Context(L, 4, Hkv, D, pool_pages=(n + 63) // 64 + 3, shuffle_seed=9)
    st = ctx.new_stream(n + 100)
    k, v = rows(rng, L, Hkv, n, D), rows(rng, L, Hkv, n, D)
    w = np.exp(2 * rows(rng, L, Hkv, n))
    w[:, 0] = np.round(w[:, 0])            # many equal accounts, zeros among them
    w[1, 1] *= rng.choice([-1, 1], n).astype(np.float32)
    w[1, 1, rng.random(n) < 0.05] = np.nan
    w[0, 1, rng.random(n) < 0.05] = np.inf
    w[1, 0, rng.random(n) < 0.3] = -0.0
    for l in range(L):
        st.write(l, 0, k[l], v[l])
        st.set_account(l, 0, w[l])
    want = np.stack([np.stack([kept_of(w[l, h], keep, recent) for h in range(Hkv)]) for l in range(L)])
    kept, ck, cv, cw = st.evict_copy(keep, recent)
    assert np.array_equal(kept, want)
    for l in range(L):
        for h in range(Hkv):
            assert np.array_equal(ck[l, h], k[l, h, want[l, h]]) and np.array_equal(cv[l, h], v[l, h, want[l, h]])
            assert np.array_equal(cw[l, h], w[l, h, want[l, h]], equal_nan=True)
    assert [st.length(l) for l in range(L)] == [n] * L      # a copy changes nothing
    assert np.array_equal(st.read_range(1, 0, n)[0], k[1])
    in_use = ctx.stats()["pages_in_use"]
    one = st.evict(keep, recent, layer=1)                   # one layer: the other stays, and so do the pages
    assert np.array_equal(one[0], want[1]) and st.length(0) == n
    m = want.shape[2]
    assert st.length(1) == m and st.evicted(1) == n - m and st.evicted(0) == 0
    assert ctx.stats()["pages_in_use"] == in_use
    assert np.array_equal(st.evict(keep, recent, layer=0)[0], want[0])
    assert ctx.stats()["pages_in_use"] == (m + 63) // 64
    for l in range(L):
        gk, gv = st.read_range(l, 0, m)
        for h in range(Hkv):
            assert np.array_equal(gk[h], k[l, h, want[l, h]]) and np.array_equal(gv[h], v[l, h, want[l, h]])
            assert np.array_equal(st.account(l)[h], w[l, h, want[l, h]], equal_nan=True)
    ctx.close()


@pytest.mark.parametrize("n,keep,recent", [(262_200, 5, 0), (300_001, 1_000, 7), (270_000, 200_001, 63), (530_000, 3, 2)])
def test_evict_of_more_positions_than_the_selection_keeps_on_chip(n, keep, recent):
    """Above 262 144 candidates the selection reads its keys again in every pass."""
    rng = np.random.default_rng(n)
    Hkv, D = 2, 4
    ctx = xn.Context(1, 2, Hkv, D, pool_pages=(n + 63) // 64, shuffle_seed=9)
    st = ctx.new_stream(n)
    k, v = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D)
    w = np.exp(2 * rows(rng, Hkv, n))
    w[0] = np.round(w[0])
    w[1, rng.random(n) < 0.01] = np.nan
    st.write(0, 0, k, v)
    st.set_account(0, 0, w)
    want = np.stack([kept_of(w[h], keep, recent) for h in range(Hkv)])
    kept, ck, cv, cw = st.evict_copy(keep, recent)
    assert np.array_equal(kept[0], want)
    assert np.array_equal(st.evict(keep, recent)[0], want)
    gk, gv = st.read_range(0, 0, keep)
    for h in range(Hkv):
        assert np.array_equal(ck[0, h], k[h, want[h]]) and np.array_equal(cv[0, h], v[h, want[h]])
        assert np.array_equal(cw[0, h], w[h, want[h]], equal_nan=True)
        assert np.array_equal(gk[h], k[h, want[h]]) and np.array_equal(gv[h], v[h, want[h]])
        assert np.array_equal(st.account(0)[h], w[h, want[h]], equal_nan=True)
    ctx.close()


@pytest.mark.parametrize("fmt", [xn.KV_F32, xn.KV_U8])
def test_more_evictions_than_one_launch_takes_and_accounts_of_different_lengths(fmt):
    """31 streams of three layers, whose accounts are complete, end in the middle, or are not there."""
    rng = np.random.default_rng(31)
    L, Hkv, D, keep, recent = 3, 2, 32, 40, 9
    ctx = xn.Context(L, 4, Hkv, D, pool_pages=200, shuffle_seed=4, kv_format=fmt)
    made = []
    for i in range(31):
        n = int(rng.integers(1, 300))
        st = ctx.new_stream(n)
        w = np.zeros((L, Hkv, n), np.float32)
        for l in range(L):
            st.write(l, 0, rows(rng, Hkv, n, D), rows(rng, Hkv, n, D))
            ends = (n, n // 2, 0)[(l + i) % 3]
            if ends:
                w[l, :, :ends] = rows(rng, Hkv, ends)
                st.set_account(l, 0, w[l, :, :ends])
        made.append((st, n, w, [st.read_range(l, 0, n) for l in range(L)]))
    kepts = [np.zeros((L, Hkv, min(keep, n)), np.int32) for _, n, _, _ in made]
    ws = [np.zeros((L, Hkv, min(keep, n)), np.float32) for _, n, _, _ in made]
    ctx.submit_evict(ctx.make_evict_batch([(m[0], -1, keep, recent, a.ctypes.data, None, None, b.ctypes.data)
                                           for m, a, b in zip(made, kepts, ws)]))
    for (st, n, w, kv), kept, got_w in zip(made, kepts, ws):
        for l in range(L):
            gk, gv = st.read_range(l, 0, min(keep, n))
            for h in range(Hkv):
                want = kept_of(w[l, h], keep, recent)
                assert np.array_equal(kept[l, h], want), (n, l, h)
                assert np.array_equal(got_w[l, h], w[l, h, want])
                assert np.array_equal(gk[h], kv[l][0][h, want]) and np.array_equal(gv[h], kv[l][1][h, want])
                assert np.array_equal(st.account(l)[h], w[l, h, want])
    ctx.close()


def test_evict_without_an_account_keeps_the_first_and_the_last():
    rng = np.random.default_rng(1)
    ctx = xn.Context(1, 2, 1, 32, pool_pages=8)
    st, k, v = filled(ctx, rng, 100)
    assert np.array_equal(st.evict(10, recent=6)[0, 0], [0, 1, 2, 3, 94, 95, 96, 97, 98, 99])
    empty = ctx.new_stream(8)
    assert empty.evict(4).shape == (1, 1, 0)
    ctx.close()


def test_many_streams_in_one_eviction():
    import torch

    rng = np.random.default_rng(6)
    Hkv, D = 3, 64
    ctx = xn.Context(1, 3, Hkv, D, pool_pages=64, shuffle_seed=4)
    sts = []
    for i, n in enumerate([30, 200, 64, 131, 1]):
        st, k, v = filled(ctx, rng, n)
        w = rows(rng, Hkv, n)
        st.set_account(0, 0, w)
        sts.append((st, k, v, w, n))
    kept = [torch.full((Hkv * 64,), -1, dtype=torch.int32, device="cuda") for _ in sts]
    torch.cuda.synchronize()
    ctx.submit_evict(ctx.make_evict_batch([(st, 0, 64, 10, t.data_ptr(), None, None, None) for (st, *_), t in zip(sts, kept)],
                                          xn.REQ_DEVICE_PTRS))
    ctx.synchronize()
    for (st, k, v, w, n), t in zip(sts, kept):
        m = min(64, n)
        got = t.cpu().numpy()[: Hkv * m].reshape(Hkv, m)
        for h in range(Hkv):
            want = kept_of(w[h], 64, 10)
            assert np.array_equal(got[h], want)
            assert np.array_equal(st.read_range(0, 0, m)[0][h], k[h, want])
        assert np.all(t.cpu().numpy()[Hkv * m:] == -1)
    ctx.close()


@pytest.mark.parametrize("fmt", [xn.KV_F32, xn.KV_U8])
def test_prompt_account_eviction_and_decode_together(fmt):
    """A prompt is written and accounted, the cache cut down, and decoding goes on with the fused rotary
    path at the tokens' true positions, next to a second stream that takes the freed pages."""
    rng = np.random.default_rng(12)
    Hq, Hkv, D, n, keep, recent, R = 8, 2, 64, 260, 100, 16, 64
    cos, sin = xn.rope_tables(10000.0, D, 1024)
    ctx = xn.Context(1, Hq, Hkv, D, pool_pages=7, rope=(cos, sin), kv_format=fmt, shuffle_seed=1)
    st = ctx.new_stream(400)
    k, v = rows(rng, Hkv, n, D), rows(rng, Hkv, n, D)
    st.write(0, 0, k, v, rope=True)
    kd, vd = st.read_range(0, 0, n)

    def rot(x, pos):   # [..., D] at positions pos
        h = D // 2
        c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
        return np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)

    if fmt == xn.KV_F32:
        near(kd, rot(k.astype(np.float64), np.arange(n)), abs_tol=1e-6)
    q = rows(rng, Hq, R, D)
    (out,) = ctx.cross_attention([st], 0, [q], causal=True, account="set")
    want, want_w = plain(q, kd, vd, True)
    near(out, want)
    near(st.account(0), want_w, abs_tol=1e-4)
    acct = st.account(0)
    kept = st.evict(keep, recent)[0]
    for h in range(Hkv):
        assert np.array_equal(kept[h], kept_of(acct[h], keep, recent))
    assert st.evicted(0) == n - keep and st.length(0) == keep
    other, ko, vo = filled(ctx, rng, 300)   # five pages: only there because the eviction returned three
    ck = np.stack([kd[h, kept[h]] for h in range(Hkv)]).astype(np.float64)
    cv = np.stack([vd[h, kept[h]] for h in range(Hkv)]).astype(np.float64)
    for step in range(3):
        pos = n + step
        x, kn, vn = rows(rng, 1, Hq, 1, D), rows(rng, 1, Hkv, 1, D), rows(rng, 1, Hkv, 1, D)
        got = ctx.attention(st, 0, keep + step, x, kn, vn, rope=True)
        sk, sv = st.read_range(0, keep + step, 1)
        if fmt == xn.KV_F32:
            near(sk, rot(kn[0].astype(np.float64), np.array([pos])), abs_tol=1e-6)
            assert np.array_equal(sv, vn[0])
        ck, cv = np.concatenate([ck, sk], 1), np.concatenate([cv, sv], 1)
        near(got[0], plain(rot(x[0].astype(np.float64), np.array([pos])), ck, cv)[0], abs_tol=1e-4, rel=1e-5)
    # a prompt chunk on the evicted stream: its query rows are rotated by the prefill kernel or the append
    S = 150 if fmt == xn.KV_F32 else 5
    x, kn, vn = rows(rng, 1, Hq, S, D), rows(rng, 1, Hkv, S, D), rows(rng, 1, Hkv, S, D)
    other.destroy()
    got = ctx.attention(st, 0, keep + 3, x, kn, vn, rope=True)
    sk, sv = st.read_range(0, keep + 3, S)
    ck, cv = np.concatenate([ck, sk], 1), np.concatenate([cv, sv], 1)
    pos = n + 3 + np.arange(S)
    near(got[0], plain(rot(x[0].astype(np.float64), pos), ck, cv, True)[0], abs_tol=2e-2, rel=5e-3)  # TF32 prefill
    ctx.close()


def test_positions_past_the_rope_table_are_refused_by_true_position():
    rng = np.random.default_rng(2)
    cos, sin = xn.rope_tables(10000.0, 32, 100)
    ctx = xn.Context(1, 2, 1, 32, pool_pages=8, rope=(cos, sin))
    st, k, v = filled(ctx, rng, 100, cap=200)
    st.evict(20)
    x, kv = rows(rng, 1, 2, 1, 32), rows(rng, 1, 1, 1, 32)
    with pytest.raises(xn.XnError) as e:
        ctx.attention(st, 0, 20, x, kv, kv, rope=True)
    assert e.value.code == 5
    with pytest.raises(xn.XnError) as e:
        st.write(0, 20, kv[0], kv[0], rope=True)
    assert e.value.code == 5
    ctx.attention(st, 0, 20, x, kv, kv)   # rotated by the caller: no table, no limit
    ctx.close()


def test_plan_reuse_does_not_outlive_an_eviction():
    """Two decode submissions of one geometry: the second may reuse the first one's plan, but not across
    an eviction, nor on a layer whose positions are shifted differently."""
    import torch

    rng = np.random.default_rng(21)
    Hq, Hkv, D = 8, 2, 128
    cos, sin = xn.rope_tables(10000.0, D, 512)
    ctx = xn.Context(2, Hq, Hkv, D, pool_pages=16, rope=(cos, sin))
    st = ctx.new_stream(400)
    for l in range(2):
        st.write(l, 0, rows(rng, Hkv, 200, D), rows(rng, Hkv, 200, D))
    st.evict(64, layer=1)
    st.write(1, 64, rows(rng, Hkv, 136, D), rows(rng, Hkv, 136, D))
    x = torch.from_numpy(rows(rng, Hq, 1, D)).cuda()
    kv = torch.from_numpy(rows(rng, 2, Hkv, 1, D)).cuda()
    out = torch.zeros(2, Hq, 1, D, device="cuda")
    torch.cuda.synchronize()
    for l in range(2):
        ctx.submit(ctx.make_batch([(st, l, 200, 1, x.data_ptr(), kv[0].data_ptr(), kv[1].data_ptr(), out[l].data_ptr())],
                                  xn.REQ_DEVICE_PTRS | xn.REQ_ROPE))
    ctx.synchronize()
    h = D // 2
    for l in range(2):
        pos = 200 + st.evicted(l)
        a = kv[0].cpu().numpy().astype(np.float64)
        want = np.concatenate([a[..., :h] * cos[pos] - a[..., h:] * sin[pos], a[..., :h] * sin[pos] + a[..., h:] * cos[pos]], -1)
        near(st.read_range(l, 200, 1)[0], want, f"layer {l}", abs_tol=1e-6)
    # the same submission after an eviction that leaves it another length must not see the old plan
    st.evict(100)
    assert st.length(0) == 100
    with pytest.raises(xn.XnError):
        ctx.cross_attention([st], 0, [rows(rng, Hq, 1, D)], kv_lens=[201])
    ctx.close()


def test_folded_streams_and_bad_arguments_are_refused():
    rng = np.random.default_rng(0)
    ctx = xn.Context(2, 4, 2, 64, pool_pages=8)
    st, k, v = filled(ctx, rng, 60, cap=64)
    q = rows(rng, 4, 2, 64)

    def refused(code, fn, *a, **kw):
        with pytest.raises(xn.XnError) as e:
            fn(*a, **kw)
        assert e.value.code == code, str(e.value)

    read = lambda *e, flags=0: ctx.submit_reads(ctx.make_read_batch(list(e), flags))
    o = np.zeros_like(q)
    good = (st, 0, 2, 60, q.ctypes.data, o.ctypes.data, None, 0)
    read(good)
    refused(1, read, (st, 0, 2, 61, q.ctypes.data, o.ctypes.data, None, 0))
    refused(1, read, (st, 0, 2, -2, q.ctypes.data, o.ctypes.data, None, 0))
    refused(1, read, (st, 0, -1, 60, q.ctypes.data, o.ctypes.data, None, 0))
    refused(1, read, (st, 2, 2, 0, q.ctypes.data, o.ctypes.data, None, 0))
    refused(1, read, (st, 0, 2, 60, None, o.ctypes.data, None, 0))
    refused(1, read, (st, 0, 2, 60, q.ctypes.data, None, None, 0))
    refused(1, read, (st, 0, 2, 60, q.ctypes.data, o.ctypes.data, o.ctypes.data, 59))
    refused(1, read, good, flags=xn.REQ_ROPE)
    refused(1, read, good, good, flags=xn.READ_ACCOUNT)       # one account, twice in a call
    mixed = ctx.make_read_batch([good, good])
    mixed[1].flags = xn.REQ_DEVICE_PTRS
    refused(1, ctx.submit_reads, mixed)
    with pytest.raises(ValueError):
        ctx.cross_attention([st], 0, [q], account="maybe")
    refused(1, st.write, 0, 10, k, v)                         # 10 + 60 > 64
    refused(1, st.write, 5, 0, k, v)
    refused(8, st.write, 0, 0, k, v, rope=True)
    refused(1, st.account, 0, 50, 11)
    refused(1, st.set_account, 0, 59, np.zeros((2, 2)))
    refused(1, st.evict, 0)
    refused(1, st.evict, 5, recent=6)
    refused(1, st.evict, 5, recent=-1)
    refused(1, st.evict, 5, layer=2)
    refused(1, st.evict, 5)                                   # layers of 60 and 0 positions
    ev = lambda *e, flags=0: ctx.submit_evict(ctx.make_evict_batch(list(e), flags))
    refused(1, ev, (st, 0, 5, 0, None, None, None, None), (st, 1, 5, 0, None, None, None, None))
    refused(1, ev, (st, 0, 5, 0, None, o.ctypes.data, o.ctypes.data, None))
    refused(1, ev, (st, 0, 5, 0, None, None, None, None), flags=xn.EVICT_COPY)
    dead = ctx.new_stream(8)
    handle = dead.handle
    other = xn.Context(1, 4, 2, 64, pool_pages=2)
    foreign = other.new_stream(8)
    refused(3, read, (foreign, 0, 2, 0, q.ctypes.data, o.ctypes.data, None, 0))
    refused(3, ev, (foreign, 0, 5, 0, None, None, None, None))
    assert handle
    # nothing above changed the stream
    assert st.length(0) == 60 and np.array_equal(st.read_range(0, 0, 60)[0], k)
    # a stream that folds around its capacity: plain reads only
    x, kv = rows(rng, 1, 4, 10, 64), rows(rng, 1, 2, 10, 64)
    ctx.attention(st, 0, 60, x, kv, kv)
    fk, fv = st.read_range(0, 0, 64)
    (out,) = ctx.cross_attention([st], 0, [q])
    near(out, plain(q, fk, fv)[0])
    refused(5, ctx.cross_attention, [st], 0, [q], causal=True)
    refused(5, ctx.cross_attention, [st], 0, [q], account="add")
    refused(5, st.evict, 5, layer=0)
    refused(5, st.write, 0, 0, k[:, :1], v[:, :1])
    other.close()
    ctx.close()


@pytest.mark.parametrize("pos,S", [(60, 4), (60, 10), (63, 2), (64, 1)])
def test_an_append_that_folds_takes_the_whole_account_with_it(pos, S):
    """Positions 64.. of a stream of 64 overwrite slots 0..; an append that just reaches the end does not."""
    rng = np.random.default_rng(S)
    ctx = xn.Context(1, 4, 2, 64, pool_pages=8)
    st, k, v = filled(ctx, rng, 64, cap=64)
    st.set_account(0, 0, np.full((2, 64), 3.0))
    x, kv = rows(rng, 1, 4, S, 64), rows(rng, 1, 2, S, 64)
    ctx.attention(st, 0, pos, x, kv, kv)
    want = np.zeros((2, 64), np.float32)
    if pos + S <= 64:
        want[:, :pos] = 3
    assert np.array_equal(st.account(0), want)
    ctx.close()


def test_pool_exhaustion_by_a_write_leaves_the_stream_as_it_was():
    rng = np.random.default_rng(0)
    ctx = xn.Context(1, 2, 1, 16, pool_pages=2)
    st, k, v = filled(ctx, rng, 70, cap=1000)
    big = rows(rng, 1, 200, 16)
    with pytest.raises(xn.XnError) as e:
        st.write(0, 70, big, big)
    assert e.value.code == 4
    assert st.length(0) == 70 and len(st.pages()) == 2
    st.write(0, 100, big[:, :20], big[:, :20])    # positions 70..99 were skipped: zeros
    got = st.read_range(0, 0, 120)[0]
    assert np.array_equal(got[:, :70], k) and not got[:, 70:100].any() and np.array_equal(got[:, 100:], big[:, :20])
    ctx.close()


def test_calls_are_refused_inside_a_capture_and_work_after_it():
    import torch

    rng = np.random.default_rng(0)
    s = torch.cuda.Stream()
    ctx = xn.Context(1, 4, 2, 64, pool_pages=4, cuda_stream=s.cuda_stream)
    st, k, v = filled(ctx, rng, 100)
    q = torch.from_numpy(rows(rng, 4, 1, 64)).cuda()
    o = torch.zeros_like(q)
    reqs = ctx.make_read_batch([(st, 0, 1, 100, q.data_ptr(), o.data_ptr(), None, 0)], xn.REQ_DEVICE_PTRS)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    codes = []
    with torch.cuda.graph(g, stream=s):
        z = o + 1
        for fn in (lambda: ctx.submit_reads(reqs), lambda: st.evict(5), lambda: st.write(0, 0, k, v), lambda: st.account(0)):
            try:
                fn()
            except xn.XnError as e:
                codes.append(e.code)
    assert codes == [1, 1, 1, 1]
    g.replay()
    ctx.submit_reads(reqs)
    ctx.synchronize()
    near(o.cpu().numpy(), plain(q.cpu().numpy(), k, v)[0])
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
def test_same_bits_every_time_and_work_of_two_threads(monkeypatch, path):
    import threading

    rng = np.random.default_rng(14)
    ctx = context(monkeypatch, path, 1, 8, 2, 128, pool_pages=128, shuffle_seed=8)
    made = [filled(ctx, rng, n) + (rows(rng, 8, 48, 128),) for n in (1500, 700)]
    first = [ctx.cross_attention([st], 0, [q], causal=True, weights=True) for st, _, _, q in made]
    bad = []

    def work(i):
        st, _, _, q = made[i]
        for _ in range(10):
            (o,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True, account="set")
            if not (np.array_equal(o, first[i][0][0]) and np.array_equal(w, first[i][1][0])):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad
    for i, (st, k, v, q) in enumerate(made):
        want, want_w = plain(q, k, v, True)
        near(first[i][0][0], want)
        near(first[i][1][0], want_w, abs_tol=1e-3)
        assert np.array_equal(st.account(0), first[i][1][0])
    ctx.close()


def test_reads_between_appends_see_what_was_appended():
    rng = np.random.default_rng(30)
    Hq, Hkv, D = 6, 2, 64
    ctx = xn.Context(1, Hq, Hkv, D, pool_pages=8)
    st = ctx.new_stream(300)
    ref = xo.RingCache(1, Hkv, 300, D)
    for pos, S in [(0, 100), (100, 1), (101, 1), (102, 30)]:
        q, k, v = rows(rng, 1, Hq, S, D), rows(rng, 1, Hkv, S, D), rows(rng, 1, Hkv, S, D)
        got = ctx.attention(st, 0, pos, q, k, v)
        xo.fast_attention(q, k, v, 0, pos, ref, Hq, Hkv, D)
        # the causal read of the same rows is the appending attention
        (again,) = ctx.cross_attention([st], 0, [q[0]], causal=True)
        near(again, got[0], abs_tol=1e-4, rel=1e-5)
    kk, vv = st.read_range(0, 0, 132)
    q = rows(rng, Hq, 3, D)
    near(ctx.cross_attention([st], 0, [q])[0], plain(q, kk, vv)[0])
    ctx.close()


@pytest.mark.parametrize("R", [24, 40, 75])
def test_account_of_more_key_tiles_than_blocks(monkeypatch, R):
    """Resident blocks take several key tiles each, with one, two or three tiles of query rows to a key tile."""
    rng = np.random.default_rng(R)
    ctx = context(monkeypatch, "tc", 1, 16, 4, 64, pool_pages=400, shuffle_seed=3)
    made = [filled(ctx, rng, n) for n in (2900, 5001, 3333)]
    qs = [rows(rng, 16, R, 64) for _ in made]
    got, w = ctx.cross_attention([st for st, _, _ in made], 0, qs, causal=True, weights=True, account="set")
    for (st, k, v), q, out, acct in zip(made, qs, got, w):
        want, want_w = plain(q, k, v, causal=True)
        near(out, want)
        near(acct, want_w, abs_tol=ABS)
        assert np.array_equal(st.account(0, 0, k.shape[1]), acct)
    ctx.close()


@pytest.mark.parametrize("account", [None, "add"])
def test_many_requests_of_all_sizes_in_one_call(account):
    rng = np.random.default_rng(12)
    ctx = xn.Context(1, 6, 2, 64, pool_pages=600, shuffle_seed=2)
    sizes = [(int(n), int(r)) for n, r in zip(rng.integers(1, 400, 90), rng.choice([1, 1, 1, 2, 5, 17, 60], 90))] + [(130, 0), (200, 100)]
    made = [filled(ctx, rng, n) for n, _ in sizes]
    qs = [rows(rng, 6, r, 64) for _, r in sizes]
    for turn in range(2):
        got, w = ctx.cross_attention([st for st, _, _ in made], 0, qs, weights=True, account=account)
        for (n, r), (st, k, v), q, out, acct in zip(sizes, made, qs, got, w):
            want, want_w = plain(q, k, v)
            if r:
                near(out, want, f"n={n} r={r}")
            times = turn + 1 if account else 1
            near(acct, want_w * times, f"account n={n} r={r}", abs_tol=ABS * 3 * max(1, r)) if r else np.testing.assert_array_equal(acct, 0.0)
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
def test_pages_behind_the_32_bit_offsets_of_the_pools(monkeypatch, path):
    """The last layer of pools of 4.7 thousand million floats each, pages in shuffled order."""
    rng = np.random.default_rng(4)
    Hq, Hkv, D, L, n = 16, 8, 128, 8, 700
    ctx = context(monkeypatch, path, L, Hq, Hkv, D, pool_pages=9000, shuffle_seed=11)
    assert 9000 * L * Hkv * 64 * D > 2 ** 32
    st, k, v = filled(ctx, rng, n, layer=L - 1)
    for R in (1, 9, 70):
        q = rows(rng, Hq, R, D)
        (out,), (w,) = ctx.cross_attention([st], L - 1, [q], causal=True, weights=True, account="set")
        want, want_w = plain(q, k, v, causal=True)
        near(out, want, f"R={R}")
        near(w, want_w, f"weights R={R}", abs_tol=ABS * R)
    acct = st.account(L - 1)
    assert np.array_equal(acct, w)
    kept = st.evict(200, 50, layer=L - 1)[0]
    gk, gv = st.read_range(L - 1, 0, 200)
    for h in range(Hkv):
        want = kept_of(acct[h], 200, 50)
        assert np.array_equal(kept[h], want) and np.array_equal(gk[h], k[h, want]) and np.array_equal(gv[h], v[h, want])
        assert np.array_equal(st.account(L - 1)[h], acct[h, want])
    ctx.close()


@pytest.mark.parametrize("path", ["few", "mid", "tc"])
@pytest.mark.parametrize("D", [64, 256])
def test_the_account_of_thousands_of_like_weights(monkeypatch, path, D):
    """Equal weights of 1/n: every addition to a long running sum rounds the same way.  In blocks of 256 (32
    rows of 8 heads) the sums take at most 256 + 2000 / 32 roundings of 2^-24 one after the other, and the
    weight itself is off by 2^-21 (a logarithm below 8 and an exponential)."""
    n, R = 79, 2000
    ctx = context(monkeypatch, path, 1, 16, 2, D, pool_pages=2)
    st = ctx.new_stream(n)
    st.write(0, 0, np.zeros((2, n, D), np.float32), np.ones((2, n, D), np.float32))
    q = rows(np.random.default_rng(0), 16, R, D)
    _, (w,) = ctx.cross_attention([st], 0, [q], weights=True)
    assert np.abs(w / (R * 8 / n) - 1).max() <= (256 + 2000 / 32) * 2.0 ** -24 + 2.0 ** -21
    ctx.close()


def test_a_call_that_finds_no_memory_fails_alone():
    """The account's pool does not fit: that call is refused, the stream stays as it is, and the calls behind
    it, of the library and of others, do not inherit the error."""
    import torch

    rng = np.random.default_rng(3)
    Hkv, D, pages = 8, 4, 1 << 18     # account: 8 * 64 * 4 bytes a page, 512 MB
    ctx = xn.Context(1, Hkv, Hkv, D, pool_pages=pages)
    st, k, v = filled(ctx, rng, 100, cap=200)
    q = rows(rng, Hkv, 2, D)
    (before,) = ctx.cross_attention([st], 0, [q])
    x, kv = rows(rng, 1, Hkv, 1, D), rows(rng, 1, Hkv, 1, D)
    ctx.attention(st, 0, 100, x, kv, kv)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    hog = torch.empty(free - (256 << 20), dtype=torch.uint8, device="cuda")
    with pytest.raises(xn.XnError) as e:
        ctx.cross_attention([st], 0, [q], account="add")
    assert e.value.code == 6
    ctx.attention(st, 0, 101, x, kv, kv)
    assert np.array_equal(ctx.cross_attention([st], 0, [q], kv_lens=[100])[0], before)
    with pytest.raises(xn.XnError):
        st.account(0)
    hog[:16].zero_()                  # (a launch of another library, which looks for errors behind it)
    del hog
    torch.cuda.empty_cache()
    (out,) = ctx.cross_attention([st], 0, [q], kv_lens=[100], account="add")
    near(out, plain(q, k, v)[0])
    near(st.account(0, 0, 100), plain(q, k, v)[1])
    ctx.close()


def test_more_rows_with_weights_than_one_launch_takes(monkeypatch):
    """140 000 small causal reads (4.5 million units of work) in one call; and one of 70 000 rows."""
    import torch

    rng = np.random.default_rng(2)
    ctx = context(monkeypatch, "few", 1, 16, 16, 4, pool_pages=2)
    st, k, v = filled(ctx, rng, 2)
    qh = rows(rng, 16, 2, 4)
    want, want_w = plain(qh, k, v, causal=True)
    q = torch.from_numpy(qh).cuda()
    out, w = torch.zeros_like(q), torch.zeros(16, 2, device="cuda")
    torch.cuda.synchronize()
    one = (st, 0, 2, 2, q.data_ptr(), out.data_ptr(), w.data_ptr(), 0)
    ctx.submit_reads(ctx.make_read_batch([one] * 140_000, xn.REQ_DEVICE_PTRS | xn.READ_CAUSAL))
    ctx.synchronize()
    near(out.cpu().numpy(), want)
    near(w.cpu().numpy(), want_w)
    q = np.zeros((16, 70_000, 4), np.float32)
    q[:, -2:] = qh
    (o,), (w,) = ctx.cross_attention([st], 0, [q], causal=True, weights=True)
    assert not o[:, :-2].any()
    near(o[:, -2:], want)
    near(w, want_w)
    ctx.close()


def test_captured_attention_replays_after_reads_and_evictions():
    """A graph of another library's work on the caller's stream is not disturbed by calls made in between."""
    import torch

    rng = np.random.default_rng(5)
    ctx = xn.Context(1, 4, 2, 64, pool_pages=64)
    st, k, v = filled(ctx, rng, 300)
    q = torch.from_numpy(rows(rng, 4, 3, 64)).cuda()
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    x = torch.arange(64.0, device="cuda")
    with torch.cuda.stream(side):
        y = x * 2
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            y.copy_(x * 3)
    # the context's own stream is not the captured one: its calls go on
    ctx.submit_reads(ctx.make_read_batch([(st, 0, 3, 300, q.data_ptr(), out.data_ptr(), None, 0)], xn.REQ_DEVICE_PTRS))
    g.replay()
    ctx.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(y, x * 3)
    near(out.cpu().numpy(), plain(q.cpu().numpy(), k, v)[0])
    ctx.close()


def test_a_captured_decode_replays_beside_reads_that_grow_and_evictions():
    """The library's own call that can be captured (the allocation-free decode), replayed between reads whose
    workspaces and page tables grow, writes, and an eviction of the stream the cache rows came from."""
    import torch

    rng = np.random.default_rng(6)
    Hq, Hkv, D, n = 8, 2, 64, 400
    lib = xn.load()
    ctx = xn.Context(1, Hq, Hkv, D, pool_pages=200)
    st, k, v = filled(ctx, rng, n)
    kc, vc = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    q = torch.from_numpy(rows(rng, Hq, D)).cuda()
    out = torch.zeros(Hq, D, device="cuda")
    side = torch.cuda.Stream()
    call = lambda: lib.xn_decode_attention_static(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(), Hq, Hkv, D, n, n,
                                                  side.cuda_stream)
    torch.cuda.synchronize()
    assert call() == 0          # (the first call on a device comes before any capture)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        assert call() == 0

    def check_replay():
        x = rows(rng, Hq, D)
        q.copy_(torch.from_numpy(x))
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        near(out.cpu().numpy(), plain(x[:, None], k, v)[0][:, 0])

    check_replay()
    for m, R in [(50, 1), (300, 9), (2000, 150), (5000, 3)]:   # page tables, scores, images, partial records grow
        other, ok, ov = filled(ctx, rng, m)
        x = rows(rng, Hq, R, D)
        (o,), (w,) = ctx.cross_attention([other], 0, [x], causal=True, weights=True, account="set")
        want, want_w = plain(x, ok, ov, causal=True)
        near(o, want)
        near(w, want_w, abs_tol=ABS * R)
        check_replay()
        assert np.array_equal(other.evict(m // 2, m // 4)[0], np.stack([kept_of(w[h], m // 2, m // 4) for h in range(Hkv)]))
        check_replay()
        other.destroy()
    st.set_account(0, 0, np.ones((Hkv, n)))
    st.evict(100, 20)
    check_replay()
    ctx.close()
