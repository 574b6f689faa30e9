"""CPU-only checks of the calls that read, write, account and evict without appending: the layout of
their request structures, and their refusal of handles that are not live."""
import ctypes as C
import os
import subprocess

import pytest

import xor_net_b200 as xn
from xor_net_b200._ffi import EvictReq, ReadReq


@pytest.mark.parametrize("struct,name", [(ReadReq, "xn_read_req"), (EvictReq, "xn_evict_req")])
def test_request_layout_matches_the_header(tmp_path, repo_root, struct, name):
    fields = [f for f, _ in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "xn_attn.h"\nint main(void) {\n'
                   f'    printf("%zu", sizeof({name}));\n'
                   + "".join(f'    printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "    return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(repo_root, "include"), "-o", exe, src], check=True)
    want = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert [C.sizeof(struct)] + [getattr(struct, f).offset for f in fields] == want


def test_flag_values_match_the_header(tmp_path, repo_root):
    names = ["XN_READ_CAUSAL", "XN_READ_ACCOUNT", "XN_READ_ACCOUNT_SET", "XN_EVICT_COPY"]
    src = tmp_path / "flags.c"
    src.write_text('#include <stdio.h>\n#include "xn_attn.h"\nint main(void) {\n'
                   + "".join(f'    printf("%u ", (unsigned){n});\n' for n in names) + "    return 0;\n}\n")
    exe = tmp_path / "flags"
    subprocess.run(["gcc", "-I", os.path.join(repo_root, "include"), "-o", exe, src], check=True)
    want = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert [xn.READ_CAUSAL, xn.READ_ACCOUNT, xn.READ_ACCOUNT_SET, xn.EVICT_COPY] == want
    # none of them is a flag that the appending calls know
    assert not any(f & (xn.REQ_DEVICE_PTRS | xn.REQ_ROPE | xn.REQ_SEQ_MAJOR) for f in want)


def test_contexts_that_are_not_live_are_refused():
    lib = xn.load()
    dead = C.create_string_buffer(1 << 16)   # zeros: no context, no stream
    for ctx in (None, C.cast(dead, C.c_void_p)):
        read, evict = ReadReq(), EvictReq()
        assert lib.xn_kv_write(ctx, None, 0, 0, 1, None, None, 0) == 3
        assert lib.xn_cross_attention(ctx, 1, C.byref(read)) == 3
        assert lib.xn_cross_attention(ctx, 0, None) == 3
        assert lib.xn_kv_account_get(ctx, None, 0, 0, 1, None, 0) == 3
        assert lib.xn_kv_account_set(ctx, None, 0, 0, 1, None, 0) == 3
        assert lib.xn_kv_evict(ctx, 1, C.byref(evict)) == 3
        assert lib.xn_stream_evicted(ctx, None, 0) == -1


def test_arrival_counters_cover_every_launch(tmp_path, repo_root):
    """A launch of b blocks over c chunks counts arrivals in words 2 .. 1 + max(b, c) of the context's array,
    also where the split-KV launches are cut into fewer chunks than there are SMs."""
    src = tmp_path / "counters.cpp"
    src.write_text('#include <cstdio>\n#include "xn_plan.hpp"\nint main() {\n'
                   "    for (int c : {1, 8, 32, 64, 147, 148, 149, 296, 1000})\n"
                   "        for (int b : {1, 132, 148}) printf(\"%d %d %zu\\n\", c, b, xn::sync_words(c, b));\n}\n")
    exe = tmp_path / "counters"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(repo_root, "xor-net_b200", "csrc"), "-o", exe, src], check=True)
    for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines():
        chunks, blocks, words = map(int, line.split())
        assert words >= 2 + max(chunks, blocks)


class FakeLib:
    """Stands in for the library: records a request, writes what a call on a stream of `length` would."""

    def __init__(self, length, layers, heads, dim):
        self.length, self.layers, self.heads, self.dim = length, layers, heads, dim

    def xn_kv_evict(self, ctx, n, reqs):
        r = reqs[0]
        m = min(r.keep, self.length)
        heads = (self.layers if r.layer < 0 else 1) * self.heads
        for ptr, kind, width in ((r.kept, C.c_int32, 1), (r.weights_out, C.c_float, 1), (r.k_out, C.c_float, self.dim)):
            if ptr:
                (kind * (heads * m * width)).from_address(ptr)[:] = [kind(i % 100).value for i in range(heads * m * width)]
        return 0

    def xn_stream_len(self, ctx, stream, layer):
        return 3          # what it was before another thread appended


@pytest.mark.parametrize("length,keep,layer", [(3, 2, -1), (3, 8, 0), (50, 40, -1), (0, 4, -1), (64, 1000, 1)])
def test_eviction_buffers_hold_what_the_call_keeps(length, keep, layer):
    """... also when the stream has grown since its length was last asked for."""
    ctx = object.__new__(xn.Context)
    ctx.lib, ctx.handle = FakeLib(length, 2, 3, 4), None
    ctx.num_layers, ctx.num_kv_heads, ctx.num_heads, ctx.head_dim = 2, 3, 3, 4
    st = xn.Stream(ctx, 0, 64)
    layers, m = 2 if layer < 0 else 1, min(keep, length)
    assert st.evict(keep, layer=layer).shape == (layers, 3, m)
    kept, k, v, w = st.evict_copy(keep, layer=layer)
    assert kept.shape == w.shape == (layers, 3, m) and k.shape == v.shape == (layers, 3, m, 4)
    assert k.ravel().tolist() == [i % 100 for i in range(layers * 3 * m * 4)]


def test_lists_of_different_lengths_are_refused():
    import numpy as np

    ctx = object.__new__(xn.Context)
    ctx.lib, ctx.handle = FakeLib(3, 1, 1, 4), None
    ctx.num_layers = ctx.num_kv_heads = ctx.num_heads = 1
    ctx.head_dim = 4
    st, q = xn.Stream(ctx, 0, 64), np.zeros((1, 1, 4), np.float32)
    for streams, layer, qs, lens in [([st], 0, [q, q], None), ([st, st], 0, [q], None), ([st], [0, 0], [q], None), ([st], 0, [q], [1, 2])]:
        with pytest.raises(ValueError):
            ctx.cross_attention(streams, layer, qs, kv_lens=lens)
