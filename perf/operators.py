"""The operators that read and shrink a stream's KV cache: their cases, plain forms and exact values.

``cross``    attention of new query rows over what a stream holds, without appending (an encoder's
             states written once, or any cached prefix): every row sees the first ``len`` positions.
``account``  the same read with the causal rule of a decoder's own cache (row t of ``rows`` sees the
             positions up to ``len - rows + t``), which also adds up, per KV head and cached position,
             the attention weight that the rows and the group's query heads gave it.
``evict``    per layer and KV head, the ``recent`` last positions and those of the largest accumulated
             weight among the others (ties: the lowest position), ``keep`` in all, in their old order:
             the kept positions, their K and V rows and their weights.

With ``own`` false ``run`` computes them in elementary torch operations; with ``own`` true it makes the
library's calls on streams of a paged cache that ``prepare`` filled with the same rows.
"""
import math

import numpy as np
import torch

own = False

_shared = {}


def _lens(case):
    """The cached lengths of the batch: spread over [lo, hi], not sorted."""
    n, lo, hi = case["n"], case["lo"], case["hi"]
    return [lo + (hi - lo) * ((i * 7 + 3) % n if n % 7 else (i * 5 + 3) % n) // max(1, n - 1) for i in range(n)]


def _read(name, op, n, rows, hq, hkv, d, lo, hi):
    return {"name": name, "op": op, "n": n, "rows": rows, "hq": hq, "hkv": hkv, "d": d, "lo": lo, "hi": hi}


def _evict(name, layers, hkv, d, length, keep, recent):
    return {"name": name, "op": "evict", "layers": layers, "hkv": hkv, "d": d, "len": length, "keep": keep, "recent": recent}


def listed():
    return [
        # one generated token of one stream over a short encoded sentence: latency
        _read("cross_token_1x197", "cross", 1, 1, 20, 5, 128, 197, 197),
        # one generated token of each of 32 streams, sources from a sentence to a long article
        _read("cross_token_32x4096", "cross", 32, 1, 32, 8, 128, 133, 4096),
        # full multi-head shape with a head_dim off the powers of two: a few dozen rows over short sources
        _read("cross_rows_4x37_d100", "cross", 4, 37, 32, 32, 100, 130, 1501),
        # a long prompt against a long document
        _read("cross_prompt_1024x8192", "cross", 1, 1024, 32, 8, 128, 8192, 8192),
        # decode of one stream that keeps the account
        _read("account_token_1x1025", "account", 1, 1, 20, 5, 128, 1025, 1025),
        # batched decode over long caches
        _read("account_token_16x8192", "account", 16, 1, 32, 8, 128, 2048, 8192),
        # the observation window: the last rows of a prompt decide what the cache keeps
        _read("account_window_2x64", "account", 2, 64, 32, 8, 128, 4097, 6001),
        # a whole prompt accounted while it is prefilled
        _read("account_prompt_2048", "account", 1, 2048, 20, 5, 128, 2048, 2048),
        # a short stream of one layer
        _evict("evict_1x300", 1, 5, 128, 300, 128, 32),
        # several layers of a long stream cut to a quarter
        _evict("evict_8x8192", 8, 8, 128, 8192, 2048, 256),
        # many KV heads, odd sizes
        _evict("evict_2x3999_d100", 2, 32, 100, 3999, 1001, 77),
        # one layer of a very long stream
        _evict("evict_1x131072", 1, 8, 128, 131072, 16384, 1024),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        hq, hkv = rng.choice([(20, 5), (32, 8), (32, 32), (8, 8), (16, 2), (6, 1), (24, 8)])
        d = rng.choice([64, 80, 100, 128, 128, 128])
        op = rng.choice(["cross", "account", "evict"])
        if op == "evict":
            length = _span(rng, 65, 140000)
            keep = min(length - 1, _span(rng, 16, length))
            case = {"op": op, "layers": _span(rng, 1, 16), "hkv": hkv, "d": d, "len": length, "keep": keep,
                    "recent": rng.randrange(0, keep + 1)}
            if case["layers"] * hkv * length * d > 3e8:
                continue
        else:
            rows = rng.choice([1, 1, _span(rng, 2, 64), _span(rng, 64, 2048)])
            hi = max(rows, _span(rng, 16, 16384))
            case = {"op": op, "n": _span(rng, 1, 32), "rows": rows, "hq": hq, "hkv": hkv, "d": d,
                    "lo": rng.randrange(min(rows, hi), hi + 1), "hi": hi}
            padded = case["n"] * hi  # the plain form's score matrix and padded cache
            if padded * hq * rows > 3e8 or padded * hkv * d > 3e8:
                continue
        if _cost(case) <= most:
            return case


def work(case):
    d, hkv = case["d"], case["hkv"]
    if case["op"] == "evict":
        heads = case["layers"] * hkv
        return {"bytes": heads * (4 * case["len"] + case["keep"] * (4 + 4 + 4 * 4 * d)), "flops": heads * case["len"]}
    b = f = 0
    for length in _lens(case):
        rows, hq = case["rows"], case["hq"]
        pairs = rows * length - (rows * (rows - 1) // 2 if case["op"] == "account" else 0)
        b += 4 * (2 * hkv * length * d + 2 * hq * rows * d + (hkv * length if case["op"] == "account" else 0))
        f += 4 * hq * d * pairs
    return {"bytes": b, "flops": f}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 6e13)


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    hkv, d = case["hkv"], case["d"]
    if case["op"] == "evict":
        layers, length = case["layers"], case["len"]
        # accumulated weights spread over orders of magnitude; every ninth position or so was never looked at
        w = torch.exp(2 * normal(layers, hkv, length))
        w = w * (torch.rand(layers, hkv, length, generator=gen, device="cuda") > 0.11)
        return {"k": normal(layers, hkv, length, d), "v": normal(layers, hkv, length, d), "w": w}
    n, hi = case["n"], case["hi"]
    k, v = normal(n, hkv, hi, d), normal(n, hkv, hi, d)
    return {"q": normal(n, case["hq"], case["rows"], d), "k": k, "v": v}


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] != "evict":
        s["lens"] = _lens(case)
        s["len"] = torch.tensor(s["lens"], device="cuda")
    if own:
        _bind(s, seed)
    return s


def _bind(s, seed):
    """The handles a program keeps: the context, the streams with their cached rows, and the request
    descriptors that name the caller's own buffers."""
    import xor_net_b200 as xn

    case, k, v = s["case"], s["k"], s["v"]
    hkv, d = case["hkv"], case["d"]
    if "stream" not in _shared:
        _shared["stream"] = torch.cuda.Stream()
    at = _shared["stream"].cuda_stream
    torch.cuda.synchronize()
    if case["op"] == "evict":
        layers, length, keep = case["layers"], case["len"], case["keep"]
        ctx = xn.Context(layers, hkv, hkv, d, pool_pages=(length + 63) // 64, shuffle_seed=seed + 1, cuda_stream=at)
        st = ctx.new_stream(length)
        for i in range(layers):
            st.write_device(i, 0, length, k[i].data_ptr(), v[i].data_ptr())
            st.set_account_device(i, 0, length, s["w"][i].data_ptr())
        out = (torch.empty(layers, hkv, keep, dtype=torch.int32, device="cuda"), torch.empty(layers, hkv, keep, d, device="cuda"),
               torch.empty(layers, hkv, keep, d, device="cuda"), torch.empty(layers, hkv, keep, device="cuda"))
        s["reqs"] = ctx.make_evict_batch([(st, -1, keep, case["recent"], *[t.data_ptr() for t in out])],
                                         xn.REQ_DEVICE_PTRS | xn.EVICT_COPY)
    else:
        pages = sum((x + 63) // 64 for x in s["lens"])
        ctx = xn.Context(1, case["hq"], hkv, d, pool_pages=pages, shuffle_seed=seed + 1, cuda_stream=at)
        out = (torch.empty_like(s["q"]), torch.zeros(case["n"], hkv, case["hi"], device="cuda"))
        account = case["op"] == "account"
        torch.cuda.synchronize()
        entries = []
        for i, length in enumerate(s["lens"]):
            st = ctx.new_stream(length)
            rows_k, rows_v = k[i, :, :length].contiguous(), v[i, :, :length].contiguous()
            torch.cuda.synchronize()
            st.write_device(0, 0, length, rows_k.data_ptr(), rows_v.data_ptr())
            ctx.synchronize()
            entries.append((st, 0, case["rows"], length, s["q"][i].data_ptr(), out[0][i].data_ptr(),
                            out[1][i].data_ptr() if account else 0, case["hi"]))
        flags = xn.REQ_DEVICE_PTRS | (xn.READ_CAUSAL | xn.READ_ACCOUNT_SET if account else 0)
        s["reqs"] = ctx.make_read_batch(entries, flags)
        out = out if account else out[:1]
    ctx.synchronize()
    s["ctx"], s["out"] = ctx, out


def run(s):
    case = s["case"]
    if own:
        if case["op"] == "evict":
            s["ctx"].submit_evict(s["reqs"])
        else:
            s["ctx"].submit_reads(s["reqs"])
        return s["out"]
    return _evict_plain(s, case) if case["op"] == "evict" else _read_plain(s, case)


def _read_plain(s, case):
    q, k, v = s["q"], s["k"], s["v"]
    n, hq, rows, d = q.shape
    hkv, hi = case["hkv"], case["hi"]
    scores = torch.matmul(q.reshape(n, hkv, hq // hkv * rows, d), k.transpose(-1, -2)).reshape(n, hq, rows, hi) / math.sqrt(d)
    pos = torch.arange(hi, device="cuda")
    last = s["len"].reshape(n, 1, 1, 1) - 1
    if case["op"] == "account":
        last = last - rows + 1 + torch.arange(rows, device="cuda").reshape(1, 1, rows, 1)
    scores = scores.masked_fill(pos > last, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n, hkv, hq // hkv * rows, hi), v).reshape(n, hq, rows, d)
    if case["op"] == "cross":
        return (out,)
    return out, p.reshape(n, hkv, hq // hkv * rows, hi).sum(2)


def _evict_plain(s, case):
    w, k, v = s["w"], s["k"], s["v"]
    length, keep, recent = case["len"], case["keep"], case["recent"]
    order = torch.sort(w[..., : length - recent], dim=-1, descending=True, stable=True).indices[..., : keep - recent]
    tail = torch.arange(length - recent, length, device="cuda").expand(*w.shape[:2], recent)
    kept = torch.sort(torch.cat([order, tail], -1), dim=-1).values
    rows = kept.unsqueeze(-1).expand(*kept.shape, case["d"])
    return kept.to(torch.int32), torch.gather(k, 2, rows), torch.gather(v, 2, rows), torch.gather(w, 2, kept)


def exact(case, seed):
    """The definitions, head by head, in 64 bits."""
    s = _inputs(case, seed)
    if case["op"] == "evict":
        length, keep, recent = case["len"], case["keep"], case["recent"]
        w = s["w"].cpu().numpy()
        kept = np.empty(w.shape[:2] + (keep,), dtype=np.int32)
        for i in range(w.shape[0]):
            for h in range(w.shape[1]):
                old = w[i, h, : length - recent].astype(np.float64)
                first = np.lexsort((np.arange(length - recent), -old))[: keep - recent]
                kept[i, h] = np.concatenate([np.sort(first), np.arange(length - recent, length)])
        at = torch.from_numpy(kept.astype(np.int64)).cuda()
        pick = [torch.stack([torch.stack([x[i, h][at[i, h]] for h in range(at.shape[1])]) for i in range(at.shape[0])]) for x in (s["k"], s["v"], s["w"])]
        return [torch.from_numpy(kept)] + [x.double() for x in pick]
    q, group = s["q"], case["hq"] // case["hkv"]
    n, hq, rows, d = q.shape
    out = torch.zeros(n, hq, rows, d, dtype=torch.float64, device="cuda")
    weight = torch.zeros(n, case["hkv"], case["hi"], dtype=torch.float64, device="cuda")
    for i, length in enumerate(_lens(case)):
        for h in range(hq):
            k, v = (s[x][i, h // group, :length].double() for x in "kv")
            a = q[i, h].double() @ k.T / math.sqrt(d)
            if case["op"] == "account":
                a += torch.full_like(a, -math.inf).triu(length - rows + 1)
            p = torch.softmax(a, -1)
            out[i, h] = p @ v
            weight[i, h // group, :length] += p.sum(0)
    return [out, weight] if case["op"] == "account" else [out]
