"""CPU tests of the paged cache: refusals of the C entry points (made before any device work), of the
Python side, and the oracle against an independent statement."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import paged as po
from transmuter_b200 import _lib, paged
from transmuter_b200.deferred import ArgumentError

P = ctypes.c_void_p
# Addresses that are never followed: every call below is refused first.
K, V, TABLE, X, Y, Z, W = (P(1 << 32), P(2 << 32), P(3 << 32), P(4 << 32), P(5 << 32), P(6 << 32), P(7 << 32))


def desc(**kw):
    d = _lib.PagedDesc()
    d.dtype, d.kv_heads, d.head_dim, d.page_size = kw.get("dtype", _lib.F16), kw.get("kv", 2), kw.get("d", 64), kw.get("page", 16)
    d.num_pages, d.max_seqs, d.max_pages = kw.get("pages", 10), kw.get("seqs", 4), kw.get("max_pages", 5)
    return d


def create(d, k=K, v=V, table=TABLE, device=0):
    h = P()
    st = _lib.load().tq4_paged_create(ctypes.byref(d), k, v, table, device, ctypes.byref(h))
    return st, h


@pytest.fixture
def cache():
    st, h = create(desc())
    assert st == 0
    yield h
    assert _lib.load().tq4_paged_destroy(h) == 0


@pytest.mark.parametrize("kw,status,msg", [
    ({"dtype": _lib.U8}, 2, "f32, f16 or bf16"), ({"d": 0}, 1, "head_dim"), ({"d": 264}, 1, "head_dim"),
    ({"d": 60}, 1, "16 bytes"), ({"d": 62, "dtype": _lib.F32}, 1, "16 bytes"), ({"page": 0}, 1, "power of two"),
    ({"page": 24}, 1, "power of two"), ({"kv": 0}, 1, "positive"), ({"kv": 16385}, 1, "16384"), ({"max_pages": (1 << 26) + 1}, 1, "2^30"),
    ({"pages": (1 << 31) - 1, "kv": 8, "page": 1}, 1, "2^32"), ({"pages": 0}, 1, "positive"),
    ({"pages": 1 << 31}, 1, "2^31"), ({"seqs": 0}, 1, "positive"), ({"max_pages": 1 << 27}, 1, "2^31"),
])
def test_create_refuses(kw, status, msg):
    st, h = create(desc(**kw))
    assert st == status and msg in _lib.last_error() and not h.value


def test_create_refuses_pointers():
    for kw in ({"k": None}, {"v": None}, {"table": None}, {"device": -1}, {"k": P((1 << 32) + 8)}, {"table": P(6)}):
        st, h = create(desc(), **kw)
        assert st == 1 and _lib.last_error() and not h.value


@pytest.mark.parametrize("d,dtype", [(8, _lib.F16), (4, _lib.F32), (256, _lib.BF16), (72, _lib.F16), (12, _lib.F32)])
def test_create_accepts_head_dims(d, dtype):
    st, h = create(desc(d=d, dtype=dtype, page=1))
    assert st == 0
    _lib.load().tq4_paged_destroy(h)


def test_null_handles():
    lib = _lib.load()
    n = ctypes.c_int64()
    assert lib.tq4_paged_destroy(None) == 0
    assert lib.tq4_paged_append(None, X, 1, X, 1, X, 1, 1, 1, X, X, X, None, Y, None) == 1
    assert lib.tq4_paged_attention(None, X, 1, 1, X, 1, 1.0, 0, None, None, Y, W, 1, None) == 1
    assert lib.tq4_paged_attention_workspace(None, 4, 1, 0, ctypes.byref(n)) == 1
    assert lib.tq4_paged_evict(None, X, 1, X, 1, 0, X, 1, X, X, None, 0, None) == 1


def rotary(**kw):
    r = _lib.RotaryDesc()
    r.cos_table, r.sin_table, r.max_pos = kw.get("cos", 1 << 36), kw.get("sin", 1 << 36), kw.get("max_pos", 100)
    r.pairs, r.axes, r.eps = kw.get("pairs", 32), kw.get("axes", 1), 1e-6
    r._axis = (ctypes.c_uint8 * 32)(*([kw.get("axis", 0)] * 32))
    r.pair_axis = ctypes.addressof(r._axis)
    return r


@pytest.mark.parametrize("kw,msg", [
    ({"tokens": -1}, "tokens"), ({"tokens": 1 << 40}, "tokens"), ({"heads": 0}, "heads"), ({"q": None}, "heads"),
    ({"heads": -4}, "heads"), ({"out": None}, "q_out"), ({"k": None}, "null"), ({"seq": None}, "null"),
    ({"slot": None}, "null"), ({"qs": 255}, "strides"), ({"ks": 127}, "strides"), ({"vs": 127}, "strides"),
    ({"out": X}, "overlaps"), ({"out": P((4 << 32) + 2 * (2 * 300 + 255))}, "overlaps"),
    ({"out": Z}, "overlaps"), ({"v": Y}, "overlaps"), ({"heads": 65536, "qs": 1 << 23}, "heads"),
    ({"rot": {"pairs": 33}}, "pairs"), ({"rot": {"pairs": -1}}, "pairs"), ({"rot": {"cos": None}}, "tables"),
    ({"rot": {"max_pos": 0}}, "tables"), ({"rot": {"axes": 5}}, "axes"), ({"rot": {"axes": 0}}, "axes"),
    ({"rot": {"axis": 1}}, "axis"), ({"rot": {}, "pos": None}, "positions"),
])
def test_append_refuses(cache, kw, msg):
    r = rotary(**kw["rot"]) if "rot" in kw else None
    st = _lib.load().tq4_paged_append(
        cache, kw.get("q", X), kw.get("qs", 300), kw.get("k", Z), kw.get("ks", 128), kw.get("v", Z), kw.get("vs", 128),
        kw.get("heads", 4), kw.get("tokens", 3), kw.get("seq", W), kw.get("slot", W), kw.get("pos", W),
        ctypes.byref(r) if r is not None else None, kw.get("out", Y), None)
    assert st == 1 and msg in _lib.last_error()


@pytest.mark.parametrize("kw,msg", [
    ({"heads": 0}, "heads"), ({"heads": 3}, "heads"), ({"heads": 65538}, "heads"), ({"batch": -1}, "sequences"),
    ({"batch": 5}, "sequences"), ({"q": None}, "null"), ({"len": None}, "null"), ({"out": None}, "null"),
    ({"ws": None}, "workspace"), ({"sc": X}, "only one"), ({"new": X}, "only one"), ({"window": -1}, "window"),
    ({"qs": 255}, "q_stride"), ({"bytes": -1}, "workspace"), ({"ws": P((7 << 32) + 4)}, "workspace"),
    ({"out": X}, "overlaps"), ({"out": P((4 << 32) + 2 * (3 * 256 - 1))}, "overlaps"),
    ({"sc": P(8 << 32), "new": P((8 << 32) + 4)}, "overlaps"),
])
def test_attention_refuses(kw, msg):
    lib = _lib.load()
    st, cache = create(desc(max_pages=5000))  # room for long sequences: a workspace is needed
    assert st == 0
    n = ctypes.c_int64()
    assert lib.tq4_paged_attention_workspace(cache, 4, 3, 0, ctypes.byref(n)) == 0 and n.value > 0
    st = lib.tq4_paged_attention(
        cache, kw.get("q", X), kw.get("qs", 256), kw.get("heads", 4), kw.get("len", Z), kw.get("batch", 3), 0.125,
        kw.get("window", 0), kw.get("sc"), kw.get("new"), kw.get("out", Y), kw.get("ws", W), n.value + kw.get("bytes", 0), None)
    assert st == 1 and msg in _lib.last_error()
    lib.tq4_paged_destroy(cache)


def test_attention_workspace_holds_the_scores(cache):
    lib = _lib.load()
    a, b = ctypes.c_int64(), ctypes.c_int64()
    lib.tq4_paged_attention_workspace(cache, 4, 3, 0, ctypes.byref(a))
    lib.tq4_paged_attention_workspace(cache, 4, 3, 1, ctypes.byref(b))
    assert a.value == 0 and b.value == 3 * 4 * 5 * 16 * 4  # few short rows: nothing but the scores
    st, wide = create(desc(max_pages=5000))
    lib.tq4_paged_attention_workspace(wide, 4, 3, 0, ctypes.byref(a))
    lib.tq4_paged_attention_workspace(wide, 4, 3, 1, ctypes.byref(b))
    assert a.value > 0 and b.value >= a.value + 3 * 4 * 5000 * 16 * 4
    lib.tq4_paged_destroy(wide)
    assert lib.tq4_paged_attention_workspace(cache, 4, 3, 1, None) == 1


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.F16])
@pytest.mark.parametrize("d", [8, 72, 128, 256])
@pytest.mark.parametrize("max_pages", [1, 5000, 1 << 20])
@pytest.mark.parametrize("seqs,kv,group", [(1, 1, 64), (64, 8, 4), (5000, 2, 16), (7, 64, 1), (3, 1, 5)])
def test_attention_workspace_is_bounded_as_documented(dtype, d, max_pages, seqs, kv, group):
    st, h = create(desc(dtype=dtype, d=d, max_pages=max_pages, seqs=seqs, kv=kv))
    assert st == 0
    n, heads = ctypes.c_int64(), kv * group
    for scores in (0, 1):
        assert _lib.load().tq4_paged_attention_workspace(h, heads, seqs, scores, ctypes.byref(n)) == 0
        assert 0 <= n.value <= 119e6 + seqs * (heads + 1) * 8 + scores * seqs * heads * max_pages * 16 * 4
    _lib.load().tq4_paged_destroy(h)


@pytest.mark.parametrize("kw,msg", [
    ({"batch": -1}, "sequences"), ({"batch": 5}, "sequences"), ({"keep": 0}, "keep"), ({"keep": 33}, "keep"),
    ({"recent": -1}, "recent"), ({"recent": 9}, "recent"), ({"len": None}, "null"), ({"sc": None}, "null"),
    ({"nt": None}, "null"), ({"nl": None}, "null"), ({"kept": None}, "null"), ({"stride": 7}, "new_score_stride"),
    ({"new": W}, "two outputs"), ({"nl": P(9 << 32)}, "two outputs"),
    ({"nl": X}, "overlaps"), ({"new": Y}, "overlaps"), ({"kept": TABLE}, "overlaps"), ({"nl": Z}, "overlaps"),
])
def test_evict_refuses(cache, kw, msg):
    st = _lib.load().tq4_paged_evict(
        cache, kw.get("len", X), kw.get("batch", 3), kw.get("sc", Y), kw.get("keep", 8), kw.get("recent", 2), kw.get("nt", Z), 2,
        kw.get("nl", P(8 << 32)), kw.get("kept", W), kw.get("new", P(9 << 32)), kw.get("stride", 8), None)
    assert st == 1 and msg in _lib.last_error()


def test_empty_calls_are_done(cache):
    lib = _lib.load()
    assert lib.tq4_paged_append(cache, X, 256, Z, 128, Z, 128, 4, 0, W, W, W, None, Y, None) == 0
    assert lib.tq4_paged_attention(cache, X, 256, 4, Z, 0, 1.0, 0, None, None, Y, W, 0, None) == 0
    assert lib.tq4_paged_evict(cache, X, 0, Y, 8, 2, Z, 2, P(8 << 32), W, None, 0, None) == 0


def test_empty_calls_take_the_null_addresses_of_empty_tensors(cache):
    lib = _lib.load()
    r = rotary()
    for heads, rot in ((4, None), (4, ctypes.byref(r)), (0, None)):
        assert lib.tq4_paged_append(cache, None, 256, None, 128, None, 128, heads, 0, None, None, None, rot, None, None) == 0
    assert lib.tq4_paged_attention(cache, None, 256, 4, None, 0, 1.0, 0, None, None, None, None, 0, None) == 0
    assert lib.tq4_paged_evict(cache, None, 0, None, 8, 2, None, 2, None, None, None, 0, None) == 0
    assert lib.tq4_paged_append(cache, None, 256, None, 128, None, 128, -1, 0, None, None, None, None, None, None) == 1


def test_python_side_refuses_cpu_tensors():
    pages = torch.zeros(4, 2, 16, 64)
    with pytest.raises(ArgumentError, match="CUDA"):
        paged.PagedCache(pages, pages, torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ArgumentError, match="CUDA"):
        paged.Rotary(torch.zeros(4, 32), torch.zeros(4, 32))


# ---- the oracle ------------------------------------------------------------------------------

def test_oracle_attention_is_softmax_over_the_gathered_rows():
    r = np.random.default_rng(0)
    k, v = r.standard_normal((2, 6, 2, 4, 8))
    q = r.standard_normal((2, 6, 8))
    table = np.array([[3, 0, 5], [1, 4, -1]])
    lengths, window = [11, 6], 5
    scores = r.random((2, 2, 12))
    out, _, new, _ = po.attention(q, k, v, table, lengths, 0.3, window, scores)
    for b in range(2):
        kk = torch.from_numpy(np.concatenate([k[p] for p in table[b] if p >= 0], 1))[:, lengths[b] - window:lengths[b]]
        vv = torch.from_numpy(np.concatenate([v[p] for p in table[b] if p >= 0], 1))[:, lengths[b] - window:lengths[b]]
        w = torch.softmax(torch.einsum("hgd,hnd->hgn", torch.from_numpy(q[b]).view(2, 3, 8), kk) * 0.3, -1)
        np.testing.assert_allclose(out[b], torch.einsum("hgn,hnd->hgd", w, vv).reshape(6, 8).numpy(), rtol=1e-12)
        want = scores[b].copy()
        want[:, lengths[b] - window:lengths[b]] += w.sum(1).numpy()
        np.testing.assert_allclose(new[b], want, rtol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation_is_a_complex_product(interleaved):
    r = np.random.default_rng(1)
    ang = r.standard_normal((9, 3))
    x = r.standard_normal(8)
    y, _ = po.norm_rotate(x, None, 0, np.cos(ang), np.sin(ang), [0, 1, 1], [4, 7], interleaved)
    a, b = (x[0:6:2], x[1:6:2]) if interleaved else (x[:3], x[3:6])
    z = (a + 1j * b) * np.exp(1j * np.array([ang[4, 0], ang[7, 1], ang[7, 2]]))
    got = y[0:6:2] + 1j * y[1:6:2] if interleaved else y[:3] + 1j * y[3:6]
    np.testing.assert_allclose(got, z, rtol=1e-12)
    assert np.array_equal(y[6:], x[6:])


def test_oracle_norm():
    x = np.array([3.0, 4.0, 0.0, 0.0])
    y, _ = po.norm_rotate(x, [1, 2, 1, 1], 0, np.zeros((1, 0)), np.zeros((1, 0)), [], [], False)
    np.testing.assert_allclose(y, [3 / 2.5, 2 * 4 / 2.5, 0, 0])


def test_oracle_keeps_by_score_then_slot():
    s = [1.0, 5.0, math.nan, 5.0, -math.inf, 0.0, -0.0, 2.0]
    assert po.keep_slots(s, 8, 3, 1) == [1, 3, 7]
    assert po.keep_slots(s, 8, 2, 1) == [1, 7]
    assert po.keep_slots(s, 8, 5, 1) == [0, 1, 3, 5, 7]      # 0.0 and -0.0 are equal: the lower slot
    assert po.keep_slots(s, 8, 7, 1) == [0, 1, 3, 4, 5, 6, 7]  # NaN goes first
    assert po.keep_slots(s, 8, 3, 3) == [5, 6, 7]
    assert po.keep_slots(s, 3, 4, 1) == [0, 1, 2]
