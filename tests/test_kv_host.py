"""Rotary positions, the quantised KV cache, attention over it and log probabilities: what
is refused before any device is touched, and where a batch's rows go (the kernels' own
location rules, on the host)."""
import ctypes as C

import numpy as np
import pytest

from onnx_runtime_dart_amd import ops
from onnx_runtime_dart_amd.errors import ArgumentError, UnsupportedError

lib = ops.lib


class Handle:
    """Stands in for a context or a cache where only argument checks run: zeroed memory
    with a cache's leading fields (device, format, log2 page, heads, head size, padded)."""

    def __init__(self, *fields):
        self.mem = (C.c_int32 * 2048)(*fields)
        self.ptr = C.cast(self.mem, C.c_void_p)


CTX = Handle()
CACHE = Handle(0, 0, 6, 2, 64, 64)
BUF = np.zeros(4096, np.float32)
P = BUF.ctypes.data


def seqs(**kw):
    base = dict(batch=1, rows=4, max_new=4, max_len=100, row_start_ptr=P, past_ptr=P,
                page_table_ptr=P, table_stride=2)
    return ops.SeqBatch(**{**base, **kw})


def rope(**kw):
    base = dict(cos_ptr=P, sin_ptr=P, max_pos=10, half_rot=8)
    return ops.Rope(**{**base, **kw})


BAD_SEQS = [dict(batch=-1), dict(batch=65536), dict(rows=-1), dict(max_new=101), dict(max_new=-1),
            dict(max_len=3), dict(max_new=2**31, max_len=2**31), dict(max_len=2**31),
            dict(rows=2**31), dict(table_stride=-1),
            dict(table_stride=2**31),
            dict(row_start_ptr=0), dict(past_ptr=0), dict(page_table_ptr=0)]
BAD_ROPE = [dict(half_rot=0), dict(half_rot=33), dict(max_pos=0), dict(max_pos=2**31),
            dict(cos_ptr=0), dict(sin_ptr=0)]


def append(s=None, k=P, v=P, ks=0, vs=0, r=None, cache=CACHE):
    return lib.mg_kv_cache_append_f32_dev(CTX.ptr, cache.ptr, C.byref(s or seqs()), k, ks, v, vs,
                                          None if r is None else C.byref(r))


def read(s=None, k=P, v=P, ks=0, vs=0):
    return lib.mg_kv_cache_read_f32_dev(CTX.ptr, CACHE.ptr, C.byref(s or seqs()), k, ks, v, vs)


def attend(s=None, q=P, y=P, heads=4, qs=0, ys=0, r=None, tree=None, words=0, cache=CACHE):
    return lib.mg_kv_cache_attention_f32_dev(CTX.ptr, cache.ptr, C.byref(s or seqs()), q, qs, heads,
                                             None if r is None else C.byref(r), tree, words, 0,
                                             0.0, y, ys)


@pytest.mark.parametrize("bad", BAD_SEQS, ids=str)
def test_batches_out_of_bounds(bad):
    for call in (append, read, attend):
        assert call(seqs(**bad)) == 1


@pytest.mark.parametrize("bad", BAD_ROPE, ids=str)
def test_tables_out_of_bounds(bad):
    assert append(r=rope(**bad)) == 1
    assert attend(r=rope(**bad)) == 1
    st = lib.mg_rotary_embedding_f32_dev(CTX.ptr, P, 1, 1, 1, 64, None, C.byref(rope(**bad)), P, None)
    assert st == 1


def test_null_buffers_strides_and_heads():
    assert append(k=None) == append(v=None) == append(ks=127) == append(vs=1) == append(ks=-1) == 1
    assert read(k=None) == read(v=None) == read(ks=127) == read(vs=127) == 1
    assert attend(q=None) == attend(y=None) == attend(qs=255) == attend(ys=255) == 1
    assert attend(heads=3) == attend(heads=0) == attend(heads=-2) == 1
    assert attend(tree=P, words=0) == attend(seqs(rows=65, max_new=65), tree=P, words=1) == 1
    other = Handle(1, 0, 6, 2, 64, 64)
    assert append(cache=other) == attend(cache=other) == 1


def test_more_rows_than_a_launch_takes():
    n = 67108857
    s = seqs(rows=n, max_new=n, max_len=n)
    assert append(s) == read(s) == 2


def test_nothing_to_do_needs_no_device():
    none = seqs(batch=0, row_start_ptr=0, past_ptr=0, page_table_ptr=0)
    empty = seqs(rows=0, max_new=0, row_start_ptr=0, past_ptr=0, page_table_ptr=0)
    loose = seqs(rows=0, max_new=7)
    for s in (none, empty, loose):
        assert append(s, k=None, v=None) == read(s, k=None, v=None) == attend(s, q=None, y=None) == 0


def create(fmt=0, pages=4, page=64, heads=2, d=64):
    out = C.c_void_p()
    return lib.mg_kv_cache_create(CTX.ptr, fmt, pages, page, heads, d, C.byref(out))


def test_cache_shapes():
    assert create(fmt=3) == create(fmt=-1) == create(page=8) == create(page=48) == create(page=512) == 1
    assert create(pages=0) == create(heads=0) == create(pages=2**31) == create(heads=5000) == 1
    assert create(pages=2**31 - 300, page=256, heads=4096) == 1
    assert create(d=0) == create(d=257) == 2
    with pytest.raises(ArgumentError):
        ops.KvCache(1, kv_heads=1, head_size=64, fmt="int3", ctx=object())
    assert lib.mg_kv_cache_release(None) == 1


def tables(first=0, count=4, half=8, base=1e4, s=None, c=P):
    return lib.mg_rotary_tables_f32_dev(CTX.ptr, first, count, half, base,
                                        None if s is None else C.byref(s), c, P)


def test_rotary_tables_refusals():
    assert tables(first=-1) == tables(count=-1) == tables(half=0) == tables(half=129) == 1
    assert tables(first=2**31 - 2, count=4) == tables(base=1.0) == tables(base=float("nan")) == 1
    assert tables(c=None) == 1 and tables(count=0, c=None) == 0
    S = ops.RopeScaling
    for bad in (S("linear", factor=0.5), S("ntk", factor=float("inf")), S("yarn", factor=4.0),
                S("bands", factor=4.0, original_length=100, low=4.0, high=4.0),
                S("bands", factor=4.0, original_length=100, low=0.0),
                S("none", value_factor=0.0), S("none", value_factor=float("nan"))):
        assert tables(s=bad, count=0) == 1
    assert tables(half=1, s=S("ntk", factor=2.0), count=0) == 1
    odd = S("none")
    odd.kind = 9
    assert tables(s=odd, count=0) == 1
    with pytest.raises(ArgumentError):
        S("cubic")


def rotary(batch=1, seq=1, heads=1, d=64, xs=None, ys=None, x=P, y=P + 8192):
    arr = lambda s: None if s is None else (C.c_int64 * 3)(*s)  # noqa: E731
    return lib.mg_rotary_embedding_f32_dev(CTX.ptr, x, batch, seq, heads, d, arr(xs),
                                           C.byref(rope()), y, arr(ys))


def test_rotary_refusals():
    assert rotary(batch=-1) == rotary(seq=-1) == rotary(heads=-1) == rotary(d=0) == rotary(d=15) == 1
    assert rotary(batch=2**20, seq=2**20) == rotary(batch=2, seq=2, heads=2**38) == 1
    assert rotary(x=None) == rotary(y=None) == 1
    assert rotary(heads=2, xs=(0, 0, -64)) == rotary(heads=2, ys=(0, 0, 63)) == 1
    assert rotary(heads=2, x=P, y=P, xs=(64, 64, 128)) == 1
    assert rotary(batch=0, x=None, y=None) == rotary(heads=0, x=None) == 0


def logprobs(rows=1, vocab=100, stride=0, tokens=P, lp=P, ent=P, top=2, ids=P, lps=P, x=P):
    return lib.mg_token_logprobs_f32_dev(CTX.ptr, x, rows, vocab, stride, tokens, lp, ent, top, ids,
                                         lps)


def test_logprobs_refusals():
    assert logprobs(rows=-1) == logprobs(rows=2**23) == logprobs(vocab=0) == logprobs(vocab=2**31 - 10) == 1
    assert logprobs(top=-1) == logprobs(top=65) == logprobs(vocab=1, top=2) == logprobs(stride=99) == 1
    assert logprobs(x=None) == logprobs(lp=None) == logprobs(ids=None) == logprobs(lps=None) == 1
    assert logprobs(rows=0, x=None) == 0
    assert logprobs(tokens=None, lp=None, ent=None, top=0, ids=None, lps=None) == 0
    with pytest.raises(ArgumentError):
        ops.op_token_logprobs(np.zeros((2, 5), np.float32), np.zeros(3, np.int64), ctx=object())


def test_host_array_shapes():
    cache = ops.KvCache.__new__(ops.KvCache)
    cache.kv_heads, cache.head_size, cache.ctx = 2, 8, None
    k = np.zeros((3, 2, 8), np.float32)
    where = dict(row_start=[0, 3], past=[0], page_table=[[0]])
    for bad in (dict(where, row_start=[0, 4]), dict(where, past=[-1]), dict(where, row_start=[1, 0]),
                dict(where, past=[0, 1]), dict(where, page_table=[0])):
        with pytest.raises(ArgumentError):
            cache.append(k, k, **bad)
    with pytest.raises(ArgumentError):
        cache.append(k, k[:, :1], **where)
    with pytest.raises(ArgumentError):
        cache.attend(np.zeros((3, 2, 9), np.float32), **where)
    with pytest.raises(ArgumentError):
        cache.attend(k, tree=np.zeros((2, 1), np.uint64), **where)


# ------------------------------------------------------------------ locations


def slots(row_start, past, table, **kw):
    base = dict(rows=8, max_new=8, max_len=64, pages=5, page_size=16)
    return ops.kv_cache_slots(row_start, past, table, **{**base, **kw})


def test_slots_follow_the_page_table():
    got, refused = slots([0, 3, 3, 7], [14, 5, 0], [[4, 1], [0, 0], [3, 2]])
    assert not refused
    np.testing.assert_array_equal(got, [4 * 16 + 14, 4 * 16 + 15, 16, 48, 49, 50, 51, -1])


def test_bad_pages_are_refused_row_by_row():
    for bad in (-1, 5, 2**31 - 1, -2**31):
        got, refused = slots([0, 3], [15], [[bad, 1]])
        assert refused
        np.testing.assert_array_equal(got[:3], [-1, 16, 17])
    got, refused = slots([0, 3], [30], [[4, 1]])  # past the table
    assert refused
    np.testing.assert_array_equal(got[:3], [16 + 14, 16 + 15, -1])
    got, refused = slots([0, 3], [0], np.zeros((1, 0), np.int32))
    assert refused and (got == -1).all()


@pytest.mark.parametrize("row_start, past, kw", [
    ([0, 9], [0], {}), ([-1, 3], [0], {}), ([3, 1], [0], {}), ([0, 5], [0], dict(max_new=4)),
    ([0, 2], [-1], {}), ([0, 2], [63], {}), ([0, 2**31 - 1], [0], {}), ([0, 2], [2**31 - 1], {})],
    ids=str)
def test_a_sequence_that_breaks_a_bound_is_refused_whole(row_start, past, kw):
    got, refused = slots(row_start, past, [[0, 1, 2, 3]], **kw)
    assert refused and (got == -1).all()


def test_other_sequences_of_such_a_batch_go_on():
    got, refused = slots([0, 2, 2, 4], [0, -5, 0], [[0], [1], [2]])
    assert refused
    np.testing.assert_array_equal(got[:4], [0, 1, 32, 33])


def test_slots_beyond_32_bits():
    got, refused = slots([0, 1], [0], [[2**31 - 300]], pages=2**31 - 256, page_size=256)
    assert not refused and got[0] == (2**31 - 300) * 256


def test_slots_refusals():
    s = seqs()
    one = C.c_int32(0)
    assert lib.mg_kv_cache_slots(None, 1, 16, P, C.byref(one)) == 1
    assert lib.mg_kv_cache_slots(C.byref(s), 0, 16, P, None) == 1
    assert lib.mg_kv_cache_slots(C.byref(s), 1, 24, P, None) == 1
    assert lib.mg_kv_cache_slots(C.byref(s), 1, 16, None, None) == 1
    with pytest.raises(ArgumentError):
        ops.kv_cache_slots([0, 1], [0, 0], [[0]], rows=1, max_new=1, max_len=1, pages=1, page_size=16)


def test_large_heads_are_unsupported():
    with pytest.raises(UnsupportedError):
        ops.check(create(d=300))


def test_host_code_under_sanitizers():
    # This file's calls on the host code built with AddressSanitizer and
    # UndefinedBehaviorSanitizer.
    import os

    import test_sanitizers as ts
    if "MIGEMM_LIBRARY" in os.environ:
        pytest.skip("already on the sanitized build")
    import build as B  # onnx_runtime_dart_amd/csrc/build.py
    srcs = [B.CSRC / n for n in ("api.hip", "kv_common.h", "rope_common.h", "logprobs_common.h")]
    if not B.SAN_LIB.exists() or B.SAN_LIB.stat().st_mtime < max(p.stat().st_mtime for p in srcs):
        B.build_sanitized()
    out = ts._child({"LD_PRELOAD": str(B.asan_runtime()), "MIGEMM_LIBRARY": str(B.SAN_LIB)},
                    ["test_kv_host.py"])
    assert " passed" in out


def test_numbers_beyond_32_bits_do_not_wrap():
    # past 2^32 + 1 is not 1, nor is page 2^32 page 0.
    slots, refused = ops.kv_cache_slots([0, 1], [2**32 + 1], [[0]], rows=1, max_new=1, max_len=8,
                                        pages=1, page_size=16)
    assert refused and (slots == -1).all()
    slots, refused = ops.kv_cache_slots([0, 1], [1], [[2**32]], rows=1, max_new=1, max_len=8,
                                        pages=1, page_size=16)
    assert refused and (slots == -1).all()
    with pytest.raises(ArgumentError):
        ops.kv_cache_slots([0, 1], [1.5], [[0]], rows=1, max_new=1, max_len=8, pages=1, page_size=16)


def test_rotary_heads_beyond_32_bits():
    # Within the elements that a call takes, but not within the kernel's index of a head.
    for heads in (2**31 - 3, 2**31, 2**33):
        assert rotary(heads=heads, d=16) == 1


@pytest.mark.parametrize("sizes, ys, ok", [
    ((2, 2, 1), (64, 64, 64), False), ((2, 2, 2), (128, 64, 64), False), ((2, 3, 1), (128, 64, 64), False),
    ((3, 2, 2), (128, 4096, 64), True), ((2, 1, 2), (64, 0, 64), False), ((1, 4, 2), (0, 64, 100), False),
    ((2, 3, 4), (768, 256, 64), True), ((2, 3, 4), (64, 512, 128), True), ((2, 3, 4), (767, 256, 64), False),
    ((1, 1, 1), (0, 0, 0), True), ((1, 5, 1), (1, 64, 1), True), ((2, 3, 4), (64, 128, 384), True),
    ((2, 3, 4), (64, 128, 383), False)], ids=str)
def test_rotary_outputs_that_overlap(sizes, ys, ok):
    # Vectors of 64: each stride passes all that the smaller ones span.
    refused = rotary(*sizes, d=64, xs=(1, 1, 1), ys=ys) == 1
    assert refused != ok


def test_rotary_cache_shapes():
    x = np.zeros((2, 3, 32), np.float32)
    three = np.ones((2, 3, 8), np.float32)
    for cos, kw in ((three, dict(position_ids=np.zeros((2, 3), np.int64))), (three[:1], {}), (three[:, :2], {}),
                    (three[0, 0], {}), (three[None], {})):
        with pytest.raises(ArgumentError):
            ops.op_rotary_embedding(x, cos, cos, num_heads=2, ctx=object(), **kw)
    with pytest.raises(ArgumentError):
        ops.op_rotary_embedding(x, three, three[..., :4], num_heads=2, ctx=object())


class Memory:
    """Device buffers of which the n-th cannot be had."""

    def __init__(self, n):
        self.left, self.held = n, []

    def __call__(self, nbytes, ctx=None):
        self.left -= 1
        if self.left < 0:
            raise MemoryError
        buf = type("Buffer", (), dict(ptr=P, free=lambda b: self.held.remove(b)))()
        self.held.append(buf)
        return buf

    def from_array(self, arr, ctx=None):
        return self(arr.nbytes, ctx)


def test_buffers_of_a_call_that_fails_are_freed(monkeypatch):
    # At once, not when the exception is let go.
    cache = ops.KvCache.__new__(ops.KvCache)
    cache.kv_heads, cache.head_size, cache.ctx = 2, 16, object()
    k = np.zeros((3, 2, 16), np.float32)
    cos = np.zeros((4, 8), np.float32)
    where = dict(row_start=[0, 3], past=[0], page_table=[[0]])
    rope = (cos, cos, False, [0, 1, 2])
    calls = [(lambda: cache.append(k, k, **where, rope=rope), 8),
             (lambda: cache.read(3, **where), 5),
             (lambda: cache.attend(k, **where, tree=np.ones((3, 1), np.uint64), rope=rope), 9),
             (lambda: ops.op_token_logprobs(k[..., 0], np.zeros(3, np.int64), top=1, ctx=object()), 6),
             (lambda: ops.op_rotary_embedding(k, cos, cos, np.zeros((3, 2)), num_heads=1, ctx=object()), 5)]
    for call, most in calls:
        for n in range(most):
            memory = Memory(n)
            monkeypatch.setattr(ops, "DeviceBuffer", memory)
            with pytest.raises(MemoryError) as held:
                call()
            assert memory.held == [], (call, n, held)
