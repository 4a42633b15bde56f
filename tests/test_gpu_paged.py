"""GPU tests of the paged key-value cache (include/tq4_paged.h, transmuter_b200.paged) against the
float64 oracle (oracle/paged.py).

Tolerances: a 16-bit output is off by at most half a step of its type (torch.finfo(t).eps / 2 relative)
beyond the oracle's bound of a 32-bit evaluation; an attention over a 16-bit cache also rounds each
softmax weight once to that type before it multiplies the values, half a step of each weight more.
Cache rows outside the sequences hold NaN throughout, so that a row read too many shows.
"""

import math

import numpy as np
import pytest
import torch

from oracle import paged as po
from transmuter_b200 import _lib, paged
from transmuter_b200.deferred import ArgumentError

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
BAD = 0x200


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def f64(x):
    return x.detach().double().cpu().numpy()


def device_status():
    import ctypes
    code = ctypes.c_int32()
    _lib.check(_lib.load().tq4_device_status(0, ctypes.byref(code)))
    return code.value


@pytest.fixture(autouse=True)
def clean_status():
    device_status()
    yield
    assert device_status() == 0, "a device-side check fired"


def make_pool(lengths, kv, ps, d, dtype, seed=0, spare=3, width=None, fresh=0):
    """Shuffled pages whose rows in use are normal and whose others are NaN; `fresh` unlisted pages a
    sequence in a second table."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // ps) for n in lengths]
    total = sum(need) + spare + fresh * len(lengths)
    order = torch.randperm(total, generator=g).int()
    width = width or max(need + [1])
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    k = torch.full((total, kv, ps, d), math.nan)
    v = torch.full((total, kv, ps, d), math.nan)
    at = 0
    for s, n in enumerate(lengths):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
        for j in range(n):
            k[table[s, j // ps], :, j % ps] = torch.randn(kv, d, generator=g)
            v[table[s, j // ps], :, j % ps] = torch.randn(kv, d, generator=g)
    new = order[at:at + fresh * len(lengths)].reshape(len(lengths), fresh).to(DEV)
    return k.to(DEV, dtype), v.to(DEV, dtype), table.to(DEV), new


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- append -----------------------------------------------------------------------------------

APPENDS = [
    # dtype, heads, kv, d, page, pairs, axes, interleaved, norm
    (F32, 16, 8, 128, 16, 64, 1, False, True),
    (BF16, 32, 8, 128, 16, 64, 1, False, False),
    (BF16, 28, 4, 128, 32, 64, 3, False, True),
    (F16, 6, 2, 80, 8, 40, 3, True, True),
    (F16, 3, 3, 72, 1, 36, 1, False, True),
    (F32, 5, 1, 12, 2, 3, 2, True, False),
    (BF16, 4, 2, 256, 16, 64, 4, False, True),
    (F32, 4, 2, 256, 64, 128, 1, True, True),
    (F16, 2, 1, 8, 4, 4, 1, False, False),
    (F16, 2, 1, 40, 4, 0, 1, False, True),
    (BF16, 40, 2, 64, 16, 10, 1, True, False),
    # rows in chunks of 8 and 4 bytes, and of single values
    (BF16, 9, 3, 72, 8, 36, 3, False, True),
    (F16, 10, 1, 40, 8, 10, 1, False, True),
    (F32, 4, 2, 72, 8, 18, 3, False, True),
    (F16, 4, 2, 256, 4, 6, 2, False, True),
    (BF16, 4, 2, 72, 4, 9, 2, True, True),
    (F32, 4, 2, 12, 4, 5, 1, False, True),
]


def run_append(dtype, heads, kv, d, ps, pairs, axes, interleaved, norm, tokens=7, strided=True, offset=0, seed=1):
    g = torch.Generator().manual_seed(seed)
    max_pos = 50
    lengths = [5, 0, 20]
    k_pages, v_pages, table, _ = make_pool([9, 4, 30], kv, ps, d, dtype, seed)
    seq = [s for _, s in zip(range(tokens), [0, 2, 1, 2, 0, 2, 1] * 10)]
    slot = []
    for s in seq:  # the next free slot of each sequence
        slot.append(lengths[s])
        lengths[s] += 1
    width = (heads + 2 * kv) * d
    qkv = torch.randn(tokens + 1, width + (5 if strided else 0) + offset, generator=g).to(DEV, dtype)[:tokens]
    row = qkv[:, offset:offset + width]
    q, k, v = (x.unflatten(1, (-1, d)) for x in (row[:, :heads * d], row[:, heads * d:(heads + kv) * d], row[:, (heads + kv) * d:]))
    positions = torch.randint(0, max_pos, (axes, tokens), generator=g).int().to(DEV)
    ang = torch.randn(max_pos, pairs, generator=g)
    pair_axis = [i % axes for i in range(pairs)]
    w = [torch.rand(d, generator=g).add(0.5).to(DEV) if norm else None for _ in range(2)]
    rot = paged.Rotary(ang.cos().to(DEV), ang.sin().to(DEV), pair_axis=pair_axis, interleaved=interleaved, q_weight=w[0],
                       k_weight=w[1], eps=1e-6)
    rot.axes, rot._desc.axes = axes, axes  # also where the last axes have no pair
    cache = paged.PagedCache(k_pages, v_pages, table)
    want_k, want_v = f64(k_pages), f64(v_pages)
    out = cache.append(q, k, v, ints(seq), ints(slot), positions, rot)
    torch.cuda.synchronize()
    got_k, got_v, got_q = f64(k_pages), f64(v_pages), f64(out)
    eps = half_step(dtype) if dtype != F32 else 0.0
    tiny = 2.0 ** -25 if dtype == F16 else 0.0  # half of f16's subnormal step
    args = (1e-6, f64(ang.cos()), f64(ang.sin()), pair_axis)
    pos, tab = positions.cpu().numpy(), table.cpu().numpy()

    def check(got, x, wt, t):
        y, bound = po.norm_rotate(f64(x), None if wt is None else f64(wt), *args, pos[:, t], interleaved)
        assert np.all(np.abs(got - y) <= bound * (1 + eps) + np.abs(y) * eps + tiny)

    for t in range(tokens):
        for h in range(heads):
            check(got_q[t, h], q[t, h], w[0], t)
        page, r = po.place(tab, ps, seq[t], slot[t])
        for h in range(kv):
            check(got_k[page, h, r], k[t, h], w[1], t)
            want_k[page, h, r] = got_k[page, h, r]
            want_v[page, h, r] = f64(v[t, h])
    # every other row is as it was, and values are copied bit for bit
    assert np.array_equal(got_k, want_k, equal_nan=True) and np.array_equal(got_v, want_v, equal_nan=True)


@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_append(case):
    run_append(*case)


@pytest.mark.parametrize("tokens", [1, 2, 33])
@pytest.mark.parametrize("case", [APPENDS[0], APPENDS[2]], ids=str)
def test_append_token_counts(case, tokens):
    run_append(*case, tokens=tokens if tokens < 33 else 12, strided=tokens == 2)


@pytest.mark.parametrize("offset", [1, 2, 8])
def test_append_reads_unaligned_views(offset):
    run_append(BF16, 4, 2, 64, 16, 32, 1, False, True, offset=offset)


def simple_cache(dtype=BF16, lengths=(5, 3), kv=2, ps=4, d=64, width=None):
    k, v, table, _ = make_pool(list(lengths), kv, ps, d, dtype, 3, width=width)
    return paged.PagedCache(k, v, table)


def test_append_without_queries_fills_the_cache():
    c = simple_cache()
    k, v = torch.randn(2, 3, 2, 64, device=DEV).to(BF16)
    assert c.append(None, k, v, ints([0, 1, 1]), ints([4, 0, 2])) is None
    for t, (s, j) in enumerate([(0, 4), (1, 0), (1, 2)]):
        p = c.page_table[s, j // 4]
        assert torch.equal(c.k_pages[p, :, j % 4], k[t]) and torch.equal(c.v_pages[p, :, j % 4], v[t])


def test_append_leaves_padding_alone():
    c = simple_cache()
    q, out = torch.randn(3, 4, 64, device=DEV).to(BF16), torch.full((3, 4, 64), 7.0, device=DEV, dtype=BF16)
    k, v = torch.randn(2, 3, 2, 64, device=DEV).to(BF16)
    before = c.k_pages.clone(), c.v_pages.clone()
    c.append(q, k, v, ints([-1, 0, -1]), ints([0, 1, -5]), out=out)
    assert torch.equal(out[1], q[1]) and (out[0] == 7).all() and (out[2] == 7).all()
    p = c.page_table[0, 0]
    before[0][p, :, 1], before[1][p, :, 1] = k[1], v[1]
    assert torch.equal(c.k_pages.nan_to_num(9), before[0].nan_to_num(9))
    assert torch.equal(c.v_pages.nan_to_num(9), before[1].nan_to_num(9))


@pytest.mark.parametrize("seq,slot,pos", [(2, 0, 0), (0, 8, 0), (0, -1, 0), (0, 0, 20), (0, 0, -1), (1, 7, 0)])
def test_append_flags_what_is_out_of_range(seq, slot, pos):
    c = simple_cache(width=2)  # sequence 1 has no second page: its entry is -1
    q, out = torch.randn(1, 4, 64, device=DEV).to(BF16), torch.zeros(1, 4, 64, device=DEV, dtype=BF16)
    k, v = torch.randn(2, 1, 2, 64, device=DEV).to(BF16)
    ang = torch.randn(20, 32, device=DEV)
    before = c.k_pages.nan_to_num(9), c.v_pages.nan_to_num(9)
    c.append(q, k, v, ints([seq]), ints([slot]), ints([pos]), paged.Rotary(ang.cos(), ang.sin()), out=out)
    assert device_status() == BAD
    assert torch.equal(c.k_pages.nan_to_num(9), before[0]) and torch.equal(c.v_pages.nan_to_num(9), before[1])
    assert not out.any()


# ---- attention --------------------------------------------------------------------------------

ATTENTIONS = [
    # dtype, heads, kv, d, page, lengths, window, scores
    (F32, 16, 8, 128, 16, [257], 0, False),
    (BF16, 32, 8, 128, 16, [1, 0, 15, 16, 17, 100, 333], 0, True),
    (F16, 32, 8, 128, 64, [1000, 3], 0, True),
    (F16, 28, 4, 80, 16, [300, 0, 31, 32, 33], 100, True),
    (F32, 8, 8, 64, 32, [63, 64, 65, 1], 0, True),
    (BF16, 8, 1, 256, 8, [130, 7], 0, True),
    (F32, 6, 2, 256, 8, [70], 3, True),
    (F16, 20, 1, 72, 1, [40, 5], 0, True),
    (BF16, 32, 2, 40, 128, [200, 129], 1, True),
    (F16, 2, 2, 8, 2, [19, 1], 0, False),
    (F32, 3, 1, 12, 4, [37, 0, 0], 36, True),
    (BF16, 15, 3, 96, 16, [90, 500], 500, False),
    (F32, 16, 1, 64, 16, [200], 0, True),
    (BF16, 17, 1, 64, 16, [77], 0, True),
    (BF16, 64, 1, 128, 16, [160], 0, True),
]


def check_attention(out, new, c, q, lengths, window, scores, scale=None):
    dtype = c.dtype
    scale = 1 / math.sqrt(c.head_dim) if scale is None else scale
    k, v = f64(c.k_pages), f64(c.v_pages)
    want, bound, want_new, new_bound = po.attention(f64(q), k, v, c.page_table.cpu().numpy(), lengths, scale, window,
                                                    None if scores is None else f64(scores))
    tol = bound
    if dtype != F32:
        mean_abs = po.attention(f64(q), k, np.abs(v), c.page_table.cpu().numpy(), lengths, scale, window)[0]
        tol = bound + half_step(dtype) * (mean_abs + np.abs(want)) + (2.0 ** -24 if dtype == F16 else 0.0)
    else:
        tol = tol + np.abs(want) * po.U
    got = f64(out)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) - tol)
    if scores is not None:
        assert np.all(np.abs(f64(new) - want_new) <= new_bound), np.max(np.abs(f64(new) - want_new) - new_bound)


# A page table with room for these sequences alone, and one for 40000 slots: few sequences of a tight table
# are a cluster's each, those of a wide one share a line of work whatever their lengths.
TABLES = pytest.mark.parametrize("wide", [False, True], ids=["tight", "wide"])


def width_of(wide, lengths, ps):
    return -(-(40000 if wide else max(lengths)) // ps) + 2


def run_attention(dtype, heads, kv, d, ps, lengths, window, with_scores, seed=2, gain=2.0, scale=None, wide=False):
    k, v, table, _ = make_pool(lengths, kv, ps, d, dtype, seed, width=width_of(wide, lengths, ps))
    c = paged.PagedCache(k, v, table)
    g = torch.Generator(DEV).manual_seed(seed)
    q = (torch.randn(len(lengths), heads, d, device=DEV, generator=g) * gain).to(dtype)
    scores = torch.rand(len(lengths), kv, c.max_slots, device=DEV, generator=g) if with_scores else None
    new = torch.full_like(scores, -7.0) if with_scores else None
    out = c.attention(q, ints(lengths), scale=scale, window=window, scores=scores, new_scores=new)
    if with_scores:  # behind each sequence nothing is written
        for b, n in enumerate(lengths):
            assert (new[b, :, n:] == -7).all()
            new[b, :, n:] = scores[b, :, n:]
    check_attention(out, new, c, q, lengths, window, scores, scale)
    return c, q, out


@TABLES
@pytest.mark.parametrize("case", ATTENTIONS, ids=str)
def test_attention(case, wide):
    run_attention(*case, wide=wide)


@TABLES
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gain,scale", [(40.0, None), (1.0, 0.0), (2.0, -0.3), (1e-3, 2.0)])
def test_attention_scales(dtype, gain, scale, wide):
    run_attention(dtype, 8, 2, 64, 16, [100, 1, 33], 0, True, gain=gain, scale=scale, wide=wide)


@pytest.mark.parametrize("dtype,heads", [(F32, 4), (BF16, 4), (F16, 32)])
def test_attention_many_sequences(dtype, heads):
    lengths = [(i * 37) % 61 for i in range(700)]  # more rows than CTAs, some empty
    run_attention(dtype, heads, 2, 16, 4, lengths, 0, True)


@TABLES
@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_in_place_scores_and_strided_queries(dtype, wide):
    lengths, kv, d = [50, 20], 2, 64
    k, v, table, _ = make_pool(lengths, kv, 16, d, dtype, 5, width=width_of(wide, lengths, 16))
    c = paged.PagedCache(k, v, table)
    wide = torch.randn(2, 500, device=DEV).to(dtype)
    q = wide[:, 3:3 + 4 * d].unflatten(1, (4, d))
    scores = torch.rand(2, kv, c.max_slots, device=DEV)
    old = scores.clone()
    a = c.attention(q, ints(lengths))
    b = c.attention(q, ints(lengths), scores=scores)
    assert torch.equal(a, b)
    check_attention(b, scores, c, q, lengths, 0, old)


@TABLES
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_is_deterministic_and_independent_of_the_workspace(dtype, wide):
    lengths = [1500, 3, 700]
    k, v, table, _ = make_pool(lengths, 2, 16, 128, dtype, 6, width=width_of(wide, lengths, 16))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(3, 8, 128, device=DEV).to(dtype)
    first = c.attention(q, ints(lengths))
    n = c._workspace[(8, 3, False)]
    assert n > 0 or not wide
    for _ in range(3):
        junk = torch.full((max(n, 1),), 0xFF, dtype=torch.uint8, device=DEV)  # NaN wherever a float is read unwritten
        del junk
        assert torch.equal(c.attention(q, ints(lengths)), first)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_shared_prefix_pages(dtype):
    k, v, table, _ = make_pool([40, 40], 2, 16, 64, dtype, 7)
    table[1, 0] = table[0, 0]
    c = paged.PagedCache(k, v, table)
    q = torch.randn(2, 4, 64, device=DEV).to(dtype)
    check_attention(c.attention(q, ints([40, 33])), None, c, q, [40, 33], 0, None)


@TABLES
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_flags_bad_lengths_and_pages(dtype, wide):
    k, v, table, _ = make_pool([20, 20, 20, 20], 2, 4, 64, dtype, 8, width=width_of(wide, [20], 4))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(4, 4, 64, device=DEV).to(dtype)
    good = c.attention(q, ints([20, 20, 20, 20]))
    out = c.attention(q, ints([20, -1, c.max_slots + 1, 20]))
    assert device_status() == BAD
    assert torch.equal(out[0], good[0]) and torch.equal(out[3], good[3]) and not out[1:3].any()
    table[1, 2], table[2, 2] = c.num_pages, -1  # slots 8 to 11 of these are left out
    out = c.attention(q, ints([20, 20, 20, 20]))
    assert device_status() == BAD
    assert torch.equal(out[0], good[0]) and torch.equal(out[3], good[3])
    rest = paged.PagedCache(k, v, torch.cat([table[:, :2], table[:, 3:]], 1).contiguous())
    check_attention(out[1:3], None, rest_rows(rest, 1, 3), q[1:3], [16, 16], 0, None)


def rest_rows(c, lo, hi):
    return paged.PagedCache(c.k_pages, c.v_pages, c.page_table[lo:hi].contiguous())


@TABLES
@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_infinite_values_stay_in_their_rows(dtype, wide):
    """An infinite or NaN value in one sequence reaches no other."""
    k, v, table, _ = make_pool([30, 30], 1, 16, 64, dtype, 9, width=width_of(wide, [30], 16))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(2, 2, 64, device=DEV).to(dtype)
    good = c.attention(q, ints([30, 30]))
    v[table[0, 1], 0, 3, 5] = math.inf
    k[table[0, 0], 0, 3] = math.nan
    out = c.attention(q, ints([30, 30]))
    assert torch.equal(out[1], good[1]) and out[0].isnan().any()


def check_attention_long(c, q, lengths, out, old=None, new=None):
    """check_attention in float64 on the GPU, for lengths that the oracle is too slow for. The bound is the
    oracle's: scores off by delta, sums in four chains and their joins."""
    kv, d, ps = c.kv_heads, c.head_dim, c.page_size
    eps = half_step(c.dtype)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any()
            continue
        rows = lambda x: x[c.page_table[b, :-(-n // ps)].long()].transpose(0, 1).flatten(1, 2)[:, :n].double()
        k, v, qb = rows(c.k_pages), rows(c.v_pages), q[b].double().view(kv, -1, d)
        w = torch.softmax(qb @ k.transpose(1, 2) / math.sqrt(d), -1)
        delta = (qb.abs() @ k.abs().transpose(1, 2) / math.sqrt(d)).amax(-1, keepdim=True) * (d + 4) * po.U
        rel = 2 * delta + (n / 4 + 200) * po.U
        want, near = w @ v, w @ v.abs()
        tol = near * rel + (0 if c.dtype == F32 else near * eps) + want.abs() * eps + 2.0 ** -24
        assert ((out[b].double().view(kv, -1, d) - want).abs() <= tol).all()
        if new is not None:
            target = old[b, :, :n].double() + w.sum(1)
            assert ((new[b, :, :n].double() - target).abs() <= (w * rel).sum(1) + target * po.U * 20).all()


@pytest.mark.parametrize("dtype,heads,kv,d,ps,most,count", [
    (BF16, 16, 4, 128, 16, 1500, 60), (F16, 32, 2, 64, 64, 5000, 40), (F32, 8, 8, 64, 32, 900, 50),
    (F32, 4, 4, 128, 8, 700, 64), (F32, 24, 3, 128, 16, 3000, 20), (BF16, 8, 2, 256, 16, 4000, 20),
    (F32, 4, 2, 256, 16, 3000, 16), (F16, 28, 4, 80, 16, 2000, 40), (BF16, 20, 1, 128, 4, 9000, 40),
    (BF16, 12, 1, 128, 128, 200000, 1),
], ids=str)
@pytest.mark.parametrize("room", [1, 12])
def test_attention_many_chunks(dtype, heads, kv, d, ps, most, count, room):
    """Lines of several chunks a CTA, with rows of every length across their borders; with a table `room` times
    as wide as it need be, which the chunks must not follow."""
    g = torch.Generator().manual_seed(most)
    lengths = [int(most * (i + 1) / count) for i in torch.randperm(count, generator=g).tolist()]
    lengths[0], lengths[-1] = (0, 1) if count > 1 else (most, most)
    need = [-(-n // ps) for n in lengths]
    order = torch.randperm(sum(need), generator=g).int()
    table = torch.full((count, max(need) * room), -1, dtype=torch.int32)
    for b, (at, n) in enumerate(zip(np.cumsum([0] + need), need)):
        table[b, :n] = order[at:at + n]
    gen = torch.Generator(DEV).manual_seed(3)
    k, v = (torch.randn(sum(need), kv, ps, d, device=DEV, dtype=dtype, generator=gen) for _ in range(2))
    c = paged.PagedCache(k, v, table.to(DEV))
    q = torch.randn(count, heads, d, device=DEV, dtype=dtype, generator=gen)
    old = torch.rand(count, kv, c.max_slots, device=DEV, generator=gen)
    new = torch.zeros_like(old)
    out = c.attention(q, ints(lengths), scores=old, new_scores=new)
    check_attention_long(c, q, lengths, out, old, new)
    assert torch.equal(c.attention(q, ints(lengths)), out)


def test_attention_short_sequences_in_a_wide_table():
    """A table for 65536 slots with a few rows in use: most of the grid has nothing to do."""
    lengths = [3, 0, 500, 17, 1, 260]
    k, v, table, _ = make_pool(lengths, 8, 16, 128, BF16, 3, width=4096)
    c = paged.PagedCache(k, v, table)
    q = torch.randn(6, 32, 128, device=DEV).to(BF16)
    for _ in range(20):
        out = c.attention(q, ints(lengths))
    check_attention(out, None, c, q, lengths, 0, None)


def test_attention_past_2_31_values():
    """Pages beyond 2^31 values from the pool's start, and a sequence beyond 2^16 slots."""
    kv, ps, d, n = 2, 64, 128, 70000
    need = -(-n // ps)
    total = (1 << 31) // (kv * ps * d) + need + 5
    k = torch.empty(total, kv, ps, d, dtype=F16, device=DEV)
    v = torch.empty_like(k)
    k[-need - 1:].normal_(generator=torch.Generator(DEV).manual_seed(1))
    v[-need - 1:].normal_(generator=torch.Generator(DEV).manual_seed(2))
    table = torch.arange(total - need, total, device=DEV).int().flip(0).contiguous()[None]
    c = paged.PagedCache(k, v, table)
    q = torch.randn(1, 8, d, device=DEV).to(F16)
    scores = torch.zeros(1, kv, c.max_slots, device=DEV)
    old = scores.clone()
    out = c.attention(q, ints([n]), scores=scores)
    check_attention_long(c, q, [n], out, old, scores)


@TABLES
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_step_replays_with_new_lengths(dtype, wide):
    """Append and attention captured once; lengths, slots and pages change between replays, and two
    graphs replayed on two streams at once do not disturb each other."""
    kv, d, ps, heads = 2, 64, 16, 4
    states = []
    for seed in (1, 2):
        k, v, table, _ = make_pool([90, 90], kv, ps, d, dtype, seed, width=width_of(wide, [90], ps))
        c = paged.PagedCache(k, v, table)
        s = {"c": c, "q": torch.randn(2, heads, d, device=DEV).to(dtype), "k": torch.randn(2, kv, d, device=DEV).to(dtype),
             "v": torch.randn(2, kv, d, device=DEV).to(dtype), "len": ints([40, 7]), "slot": ints([39, 6]), "seq": ints([0, 1]),
             "stream": torch.cuda.Stream(), "graph": torch.cuda.CUDAGraph()}

        def step(s=s):
            qo = s["c"].append(s["q"], s["k"], s["v"], s["seq"], s["slot"])
            return s["c"].attention(qo, s["len"])

        s["step"] = step
        torch.cuda.synchronize()
        with torch.cuda.stream(s["stream"]):
            step()
        torch.cuda.synchronize()
        with torch.cuda.graph(s["graph"], stream=s["stream"]):
            s["out"] = step()
        states.append(s)
    for lengths in ([41, 8], [90, 1], [64, 0]):
        for s in states:
            s["len"].copy_(ints(lengths))
            s["slot"].copy_(ints([max(n - 1, 0) for n in lengths]))
            s["seq"].copy_(ints([i if n else -1 for i, n in enumerate(lengths)]))
            s["q"].normal_()
            s["k"].normal_()
        torch.cuda.synchronize()
        for _ in range(5):
            for s in states:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in states:
            got = s["out"].clone()
            assert torch.equal(got[0], s["step"]()[0])
            live = [i for i, n in enumerate(lengths) if n]
            check_attention(got[live], None, rest_rows(s["c"], 0, len(live)), s["q"][live], [lengths[i] for i in live], 0, None)


# ---- evict ------------------------------------------------------------------------------------

EVICTIONS = [
    # dtype, kv, d, page, lengths, keep, recent
    (F32, 8, 128, 16, [257], 128, 32),
    (BF16, 2, 128, 32, [300, 0, 40, 99, 100, 101, 1], 100, 10),
    (F16, 1, 72, 1, [33, 5], 7, 7),
    (F16, 3, 40, 8, [64, 65], 64, 0),
    (F32, 2, 12, 4, [50, 50], 1, 0),
    (F32, 2, 12, 4, [50, 50], 1, 1),
    (BF16, 2, 256, 128, [1000, 2500], 700, 100),
    (F16, 2, 8, 2, [4000], 3999, 1),
]


def run_evict(dtype, kv, d, ps, lengths, keep, recent, scores=None, seed=4):
    k, v, table, new = make_pool(lengths, kv, ps, d, dtype, seed, fresh=-(-keep // ps) + 1, width=-(-max(lengths) // ps) + 1)
    c = paged.PagedCache(k, v, table)
    if scores is None:
        g = torch.Generator(DEV).manual_seed(seed)
        scores = (torch.rand(len(lengths), kv, c.max_slots, device=DEV, generator=g) * 20).round() / 4  # many equal
    before = k.clone(), v.clone()
    kept, new_len, new_sc = c.evict(ints(lengths), scores, keep, recent, new)
    assert new_len.tolist() == [min(n, keep) for n in lengths]
    want = before
    for b, n in enumerate(lengths):
        m = min(n, keep)
        for h in range(kv):
            idx = po.keep_slots(scores[b, h].tolist(), n, keep, recent)
            assert kept[b, h].tolist() == idx + [-1] * (keep - m)
            i = torch.tensor(idx, dtype=torch.long, device=DEV)
            assert torch.equal(new_sc[b, h, :m].nan_to_num(77), scores[b, h, i].nan_to_num(77)) and not new_sc[b, h, m:].any()
            j = torch.arange(m, device=DEV)
            src, dst = table[b].long()[i // ps], new[b].long()[j // ps]
            for was, pages in zip(want, (k, v)):
                assert torch.equal(pages[dst, h, j % ps], was[src, h, i % ps])
                was[dst, h, j % ps] = pages[dst, h, j % ps]
    for was, pages in zip(want, (k, v)):  # nothing else is written
        assert torch.equal(was.nan_to_num(9), pages.nan_to_num(9))
    return c, new, new_len, new_sc


@pytest.mark.parametrize("case", EVICTIONS, ids=str)
def test_evict(case):
    run_evict(*case)


def test_evict_orders_every_kind_of_score():
    vals = [0.0, -0.0, 1.0, math.inf, -math.inf, math.nan, 1e-45, -1e-45, 3e38, -3e38, 1.0, math.nan, -math.inf, math.inf]
    for keep, recent in ((1, 0), (2, 0), (3, 1), (5, 0), (7, 0), (9, 2), (12, 0), (13, 0)):
        n = len(vals)
        sc = torch.tensor(vals, device=DEV)
        sc = torch.cat([sc, torch.full((2 * 8 - n,), 5e30, device=DEV)])  # behind the length: must not count
        scores = torch.zeros(1, 2, 24, device=DEV)
        scores[0, 0, :16], scores[0, 1, :16] = sc, torch.cat([sc[:n].flip(0), sc[n:]])
        run_evict(F32, 2, 8, 8, [n], keep, recent, scores)


@pytest.mark.parametrize("value", [0.0, -1.5, math.nan, math.inf])
def test_evict_equal_scores_keep_the_first(value):
    run_evict(F16, 1, 8, 4, [3000], 1100, 50, torch.full((1, 1, 3004), value, device=DEV))


def test_evict_long_sequence():
    n, keep, recent = 100003, 9001, 128
    k = torch.arange(n + 13, device=DEV, dtype=F32)[:, None].expand(-1, 4).reshape(-1, 1, 16, 4).contiguous()
    pool = torch.cat([k, torch.zeros(600, 1, 16, 4, device=DEV)])
    table = torch.arange(k.shape[0], device=DEV).int()[None]
    new = torch.arange(k.shape[0], k.shape[0] + 563, device=DEV).int()[None].contiguous()
    c = paged.PagedCache(pool, -pool, table)
    scores = torch.rand(1, 1, c.max_slots, device=DEV).half().float()  # ties at every value
    kept, length, sc = c.evict(ints([n]), scores, keep, recent, new)
    idx = po.keep_slots(scores[0, 0].tolist(), n, keep, recent)
    assert kept[0, 0].tolist() == idx and length.tolist() == [keep]
    moved = pool[new[0].long()].reshape(-1, 4)[:keep, 0]
    assert moved.tolist() == [float(i) for i in idx]
    assert torch.equal(sc[0, 0, :keep], scores[0, 0, kept[0, 0].long()])


def test_evict_flags_bad_lengths_and_pages():
    k, v, table, new = make_pool([20, 20, 20], 1, 4, 64, F16, 8, fresh=3)
    c = paged.PagedCache(k, v, table)
    scores = torch.rand(1, device=DEV).expand(3, 1, c.max_slots).contiguous()
    kept, length, _ = c.evict(ints([-2, 20, c.max_slots + 1]), scores, 10, 2, new)
    assert device_status() == BAD and length.tolist() == [0, 10, 0]
    assert (kept[0] == -1).all() and (kept[2] == -1).all()
    new[1, 0] = c.num_pages
    before = k.clone()
    c.evict(ints([0, 20, 0]), scores, 10, 2, new)
    assert device_status() == BAD
    same = [p for p in range(c.num_pages) if p not in new[1].tolist()]
    assert torch.equal(before[same].nan_to_num(9), k[same].nan_to_num(9))


def test_python_side_refuses():
    c = simple_cache(BF16)
    q = torch.zeros(2, 4, 64, device=DEV, dtype=BF16)
    k = torch.zeros(2, 2, 64, device=DEV, dtype=BF16)
    n, i = ints([5, 3]), ints([0, 1])
    bad = [
        lambda: c.attention(q.float(), n), lambda: c.attention(q[:, :3], n), lambda: c.attention(q, n.long()),
        lambda: c.attention(q, n[:1]), lambda: c.attention(q, n.cpu()), lambda: c.attention(torch.cat([q, q]), ints([1] * 4)),
        lambda: c.attention(q, n, new_scores=torch.zeros(2, 2, c.max_slots, device=DEV)),
        lambda: c.attention(q, n, scores=torch.zeros(2, 2, c.max_slots + 1, device=DEV)),
        lambda: c.attention(q, n, out=torch.zeros(2, 4, 64, device=DEV)), lambda: c.attention(q[..., :32], n),
        lambda: c.append(q, k, k[:1], i, i), lambda: c.append(q[:1], k, k, i, i), lambda: c.append(q, k, k, i, i[:1]),
        lambda: c.append(None, k, k, i, i, out=q), lambda: c.append(q, k[:, :1], k, i, i),
        lambda: c.append(q, k, k, i, i, i, paged.Rotary(torch.zeros(4, 33, device=DEV), torch.zeros(4, 33, device=DEV))),
        lambda: c.append(q, k, k, i, i, None, paged.Rotary(torch.zeros(4, 32, device=DEV), torch.zeros(4, 32, device=DEV))),
        lambda: c.append(q, k, k, i, i, i, paged.Rotary(*torch.zeros(2, 4, 32, device=DEV), q_weight=torch.ones(63, device=DEV))),
        lambda: paged.Rotary(*torch.zeros(2, 4, 32, device=DEV), sections=(16, 8)),
        lambda: c.evict(n, torch.zeros(2, 2, c.max_slots, device=DEV), 5, 6, ints([[0], [1]])),
        lambda: c.evict(n, torch.zeros(2, 2, c.max_slots, device=DEV), 5, 1, ints([[0], [1]])),
        lambda: paged.PagedCache(c.k_pages, c.v_pages[:1], c.page_table),
        lambda: paged.PagedCache(c.k_pages, c.v_pages, c.page_table.long()),
    ]
    for f in bad:
        with pytest.raises(ArgumentError):
            f()
    with pytest.raises(_lib.Tq4Error, match="overlaps"):
        c.append(q, k, k, i, i, out=q)


# ---- together, as they are used ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
def test_served_batch_prompts_steps_and_eviction(dtype):
    """Prompts appended at once, then decode steps of a ragged batch that accumulate attention
    weights, an eviction in between, and steps over the trimmed cache: every step's output against the
    oracle over the rows that the cache should hold."""
    heads, kv, d, ps, pairs = 4, 2, 64, 8, 32
    g = torch.Generator(DEV).manual_seed(3)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)
    prompts = [21, 1, 33]
    width = 8
    pool_k, pool_v = (torch.full((64, kv, ps, d), math.nan, device=DEV, dtype=dtype) for _ in range(2))
    table = torch.randperm(64, generator=torch.Generator().manual_seed(1)).int().to(DEV)[:3 * width].view(3, width).contiguous()
    free = torch.tensor(sorted(set(range(64)) - set(table.flatten().tolist())), dtype=torch.int32, device=DEV)
    ang = torch.arange(80, dtype=torch.float64)[:, None] * (1e4 ** (-torch.arange(pairs, dtype=torch.float64) / pairs))[None]
    rot = paged.Rotary(ang.cos().float().to(DEV), ang.sin().float().to(DEV), sections=(8, 12, 12),
                       q_weight=torch.rand(d, device=DEV) + 0.5, k_weight=torch.rand(d, device=DEV) + 0.5)
    c = paged.PagedCache(pool_k, pool_v, table)
    seq = [s for s, n in enumerate(prompts) for _ in range(n)]
    slot = [j for n in prompts for j in range(n)]
    t = len(seq)
    c.append(None, rand(t, kv, d), rand(t, kv, d), ints(seq), ints(slot), ints([slot, slot, slot]), rot)
    lengths, position = list(prompts), list(prompts)
    scores = torch.zeros(3, kv, c.max_slots, device=DEV)
    for step in range(8):
        if step == 4:
            keep, recent = 12, 4
            new = free[:3 * 2].view(3, 2).contiguous()
            order = [[po.keep_slots(scores[b, h].tolist(), lengths[b], keep, recent) for h in range(kv)] for b in range(3)]
            rows = lambda pages, b, h: torch.stack([pages[table[b, j // ps], h, j % ps] for j in order[b][h]])
            want = [[(rows(pool_k, b, h).clone(), rows(pool_v, b, h).clone()) for h in range(kv)] for b in range(3)]
            kept, new_len, new_sc = c.evict(ints(lengths), scores, keep, recent, new)
            lengths = new_len.tolist()
            # the sequences go on over the new pages, with room for more
            table = torch.cat([new, free[6:12].view(3, 2)], 1).contiguous()
            c = paged.PagedCache(pool_k, pool_v, table)
            scores = torch.zeros(3, kv, c.max_slots, device=DEV)
            scores[:, :, :new_sc.shape[2]] = new_sc
            for b in range(3):
                for h in range(kv):
                    for j in range(lengths[b]):
                        assert torch.equal(pool_k[table[b, j // ps], h, j % ps], want[b][h][0][j])
                        assert torch.equal(pool_v[table[b, j // ps], h, j % ps], want[b][h][1][j])
        qkv = rand(3, (heads + 2 * kv) * d)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([heads * d, kv * d, kv * d], 1))
        p = ints([position] * 3)
        qo = c.append(q, k, v, ints([0, 1, 2]), ints(lengths), p, rot)
        lengths = [n + 1 for n in lengths]
        position = [n + 1 for n in position]
        old = scores.clone()
        out = c.attention(qo, ints(lengths), scores=scores)
        check_attention(out, scores, c, qo, lengths, 0, old)
        # each sequence's weights of a step add up to one a query head
        assert torch.allclose((scores - old).sum(-1), torch.full((3, kv), float(heads // kv), device=DEV), atol=1e-4)


# ---- the workspace ------------------------------------------------------------------------------

def attention_in(c, q, lengths, ws, scores=None, new=None, window=0):
    """The C entry with a workspace of the caller's and an output between guards: (output, whether the guards held)."""
    import ctypes
    batch, heads, d = q.shape
    n = ctypes.c_int64()
    _lib.check(c._lib.tq4_paged_attention_workspace(c._handle, heads, batch, int(scores is not None), ctypes.byref(n)))
    assert ws.numel() >= n.value
    guard = 1 << 14
    room = torch.full((q.numel() + 2 * guard,), 3.0, device=DEV, dtype=q.dtype)
    out = room[guard:-guard].view(q.shape)
    _lib.check(c._lib.tq4_paged_attention(
        c._handle, q.data_ptr(), heads * d, heads, lengths.data_ptr(), batch, 1 / math.sqrt(d), window,
        scores.data_ptr() if scores is not None else None, new.data_ptr() if new is not None else None, out.data_ptr(),
        ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    return out, bool((room[:guard] == 3).all() and (room[-guard:] == 3).all())


# what a workspace may hold before a call: zeros, ones, the largest and all bits set
FILLS = [0, 1, 0x7F, 0xFF]


@pytest.mark.parametrize("dtype,heads,kv,lengths", [
    (BF16, 8, 2, [3000, 0, 900, 1, 5000]), (F32, 16, 2, [700, 2, 1500]), (F16, 40, 2, [20000]), (BF16, 4, 4, [0, 0]),
    (F32, 6, 2, [(i * 37) % 90 for i in range(400)]),
], ids=lambda x: str(x)[:40])
def test_attention_reads_nothing_that_an_earlier_call_left(dtype, heads, kv, lengths):
    k, v, table, _ = make_pool(lengths, kv, 16, 64, dtype, 21, width=width_of(True, lengths, 16))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(len(lengths), heads, 64, device=DEV).to(dtype)
    old = torch.rand(len(lengths), kv, c.max_slots, device=DEV)
    n = ints(lengths)
    new = torch.zeros_like(old)
    want, want_s = c.attention(q, n), c.attention(q, n, scores=old, new_scores=new)
    most = torch.empty(c._workspace[(heads, len(lengths), True)], dtype=torch.uint8, device=DEV)
    for fill in FILLS:
        out, held = attention_in(c, q, n, most.fill_(fill))
        assert held and torch.equal(out, want)
        got = torch.zeros_like(old)
        out, held = attention_in(c, q, n, most.fill_(fill), old, got)
        assert held and torch.equal(out, want_s) and torch.equal(got, new)


ATTENTION_TIMEOUT = 0x107


@pytest.mark.parametrize("dtype,heads,kv,count,most", [
    (BF16, 8, 2, 20000, 70), (F32, 8, 1, 20000, 40), (F16, 32, 2, 60, 9000), (F32, 4, 2, 3, 9000),
], ids=str)
def test_attention_of_which_a_wait_runs_out(dtype, heads, kv, count, most):
    """With the shortest wait limit, warps give up waiting for their next chunk (a chunk among 20000 sequences takes longer
    to find than that): the call says so or is right, writes nothing outside its outputs whatever the workspace held, and
    the next call is as ever."""
    ps, d, pages = 16, 64, 600
    g = torch.Generator(DEV).manual_seed(31)
    k, v = (torch.randn(pages, kv, ps, d, device=DEV, generator=g).to(dtype) for _ in range(2))
    table = torch.randint(0, pages, (count, -(-most // ps)), device=DEV, generator=g, dtype=torch.int32)  # pages are shared
    c = paged.PagedCache(k, v, table)
    q = torch.randn(count, heads, d, device=DEV, generator=g).to(dtype)
    n = torch.randint(0, most + 1, (count,), device=DEV, generator=g, dtype=torch.int32)
    old = torch.rand(count, kv, c.max_slots, device=DEV, generator=g)
    new = torch.zeros_like(old)
    want, want_s = c.attention(q, n), c.attention(q, n, scores=old, new_scores=new)
    ws = torch.empty(c._workspace[(heads, count, True)], dtype=torch.uint8, device=DEV)
    small = ws.view(torch.int32)[:ws.numel() // 4]
    codes = []
    for fill in FILLS + [None]:
        for scores in (False, True):
            if fill is None:
                small.fill_(1)  # numbers that could be a row's
            else:
                ws.fill_(fill)
            got = torch.zeros_like(old) if scores else None
            torch.cuda.synchronize()
            _lib.check(_lib.load().tq4_set_wait_limit(0, 1000))
            try:
                out, held = attention_in(c, q, n, ws, old if scores else None, got)
                torch.cuda.synchronize()
                codes.append(device_status())
            finally:
                _lib.check(_lib.load().tq4_set_wait_limit(0, 0))
            assert held and codes[-1] in (0, ATTENTION_TIMEOUT)
            if scores:
                behind = torch.arange(c.max_slots, device=DEV) >= n[:, None, None]
                assert not got[behind.expand_as(got)].any()
            if codes[-1] == 0:
                assert torch.equal(out, want_s if scores else want)
            assert torch.equal(c.attention(q, n), want)  # the default limit is back
    print(codes)
    assert count < 20000 or ATTENTION_TIMEOUT in codes


# ---- values that are not finite -----------------------------------------------------------------

def bits(x):
    return x.contiguous().view(torch.int32 if x.dtype == F32 else torch.int16)


def append_into(c, q, k, v, rot=None, pos=None):
    """One append of q, k, v [tokens, heads, d] to the first slots of sequence 0: (queries, keys, values) as they then stand."""
    n = q.shape[0]
    out = c.append(q, k, v, ints([0] * n), ints(range(n)), pos, rot)
    at = [(c.page_table[0, j // c.page_size].item(), j % c.page_size) for j in range(n)]
    return out, torch.stack([c.k_pages[p, :, r] for p, r in at]), torch.stack([c.v_pages[p, :, r] for p, r in at])


# dtype, d, pairs, interleaved, offset of the views
UNTURNED = [
    (BF16, 128, 32, False, 0), (BF16, 128, 32, True, 0), (F16, 128, 0, False, 0), (F32, 64, 16, False, 0), (F32, 64, 16, True, 0),
    (F16, 72, 18, False, 0), (BF16, 72, 9, True, 0), (F16, 128, 32, False, 2), (BF16, 128, 32, True, 1), (F32, 256, 5, False, 0),
]


def special_rows(n, heads, d, dtype, offset, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads * d + offset, generator=g)
    for i, value in enumerate([math.inf, -math.inf, math.nan, -0.0, 1e-45, math.inf]):
        x[:, offset + i * 7 + 3::53] = value
    return x.to(DEV, dtype)[:, offset:].unflatten(1, (heads, d))


@pytest.mark.parametrize("case", UNTURNED, ids=str)
def test_append_copies_what_is_not_turned(case):
    """Without a norm, values that no pair turns come out bit for bit, whatever stands beside them: infinities, NaN, -0."""
    dtype, d, pairs, interleaved, offset = case
    c = simple_cache(dtype, lengths=(12, 1), kv=2, ps=4, d=d)
    q, k, v = (special_rows(9, h, d, dtype, offset, i) for i, h in enumerate((5, 2, 2)))
    ang = torch.randn(9, pairs, device=DEV)
    rot = paged.Rotary(ang.cos(), ang.sin(), interleaved=interleaved)
    for r, rest in ((rot, 2 * pairs), (None, 0)):
        for x, y in zip((q, k, v), append_into(c, q, k, v, r, ints(range(9)) if r else None)):
            assert torch.equal(bits(x[..., d if x is v else rest:]), bits(y[..., d if x is v else rest:]))
        assert torch.equal(bits(v), bits(y))


@pytest.mark.parametrize("case", UNTURNED, ids=str)
def test_append_keeps_an_infinity_in_its_pair(case):
    """An infinite value of a head changes its own output and its partner's, with or without a norm of zero angles; with a norm
    it makes the head's finite values 0."""
    dtype, d, pairs, interleaved, offset = case
    c = simple_cache(dtype, lengths=(12, 1), kv=2, ps=4, d=d)
    g = torch.Generator().manual_seed(5)
    clean = [torch.randn(8, h * d + offset, generator=g).to(DEV, dtype) for h in (5, 2, 2)]
    ang = torch.randn(8, pairs, device=DEV)
    w = torch.rand(d, device=DEV) + 0.5
    pos = ints(range(8))
    for i in sorted({0, 1, pairs, 2 * pairs, 2 * pairs + 1, d // 2, d - 1} & set(range(d))):
        other = i if i >= 2 * pairs else i ^ 1 if interleaved else (i + pairs) % (2 * pairs)
        hot = [x.clone() for x in clean]
        for x in hot[:2]:
            x[:, offset + i::d] = math.inf
        view = lambda x: x[:, offset:].unflatten(1, (-1, d))
        rot = paged.Rotary(ang.cos(), ang.sin(), interleaved=interleaved)
        want, got = ([y.clone() for y in append_into(c, *map(view, x), rot, pos)] for x in (clean, hot))
        for x, y in zip(want, got):
            rest = [e for e in range(d) if e not in (i, other)]
            assert torch.equal(bits(x[..., rest]), bits(y[..., rest]))
        rot = paged.Rotary(ang.cos(), ang.sin(), interleaved=interleaved, q_weight=w, k_weight=w)
        for y in append_into(c, *map(view, hot), rot, pos)[:2]:
            rest = [e for e in range(d) if e not in (i, other)]
            assert not y[..., rest].any() and y[..., i].isnan().all()


@TABLES
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4), (20, 1)])
def test_attention_nan_of_a_query_head_stays_nan(dtype, heads, kv, wide):
    """A head whose every score is NaN gives NaN, however its row is cut; every other head and sequence keeps its bits."""
    lengths = [5000, 3, 700, 0]
    k, v, table, _ = make_pool(lengths, kv, 16, 64, dtype, 11, width=width_of(wide, lengths, 16))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(4, heads, 64, device=DEV).to(dtype)
    old = torch.rand(4, kv, c.max_slots, device=DEV)
    hot, h = q.clone(), heads - 2
    hot[:3, h, 5] = math.nan
    for scores in (False, True):
        new = [torch.zeros_like(old) for _ in range(2)] if scores else [None] * 2
        good, out = (c.attention(x, ints(lengths), scores=old if scores else None, new_scores=n) for x, n in zip((q, hot), new))
        rest = [i for i in range(heads) if i != h]
        assert torch.equal(out[:, rest], good[:, rest]) and not out[3].any()
        assert out[:3, h].isnan().all()
        if scores:
            own = h // (heads // kv)
            rest = [i for i in range(kv) if i != own]
            assert torch.equal(new[1][:, rest], new[0][:, rest])
            for b, n in enumerate(lengths):
                assert new[1][b, own, :n].isnan().all() and torch.equal(new[1][b, own, n:], new[0][b, own, n:])


@TABLES
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_nan_keys_of_one_part_are_seen(dtype, wide):
    """A stretch of NaN keys that fills whole parts of a row makes its output NaN, beside finite parts too."""
    lengths = [5000, 700]
    k, v, table, _ = make_pool(lengths, 2, 16, 64, dtype, 12, width=width_of(wide, lengths, 16))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(2, 8, 64, device=DEV).to(dtype)
    good = c.attention(q, ints(lengths))
    k[table[0, 100:200].long(), 1] = math.nan
    out = c.attention(q, ints(lengths))
    assert torch.equal(out[0, :4], good[0, :4]) and torch.equal(out[1], good[1]) and out[0, 4:].isnan().all()


@TABLES
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_large_scores(dtype, d, wide):
    """Scores of 2^26 and more, where f32 cannot tell neighbours 15 apart: the two slots that share the largest have half the
    weight each, and all products are exact."""
    n, pair = 300, (20, 250)
    k, v, table, _ = make_pool([n], 1, 16, d, dtype, 13, width=width_of(wide, [n], 16))
    c = paged.PagedCache(k, v, table)
    g = torch.Generator().manual_seed(13)
    values = torch.randint(-100, 100, (n, d), generator=g).float() * 2
    for j in range(n):
        p = table[0, j // 16].item()
        k[p, 0, j % 16] = 1024.0 if j in pair else 512.0
        v[p, 0, j % 16] = values[j].to(DEV, dtype)
    want = ((values[pair[0]] + values[pair[1]]) / 2).to(DEV)
    for gain in (256.0, 512.0, 1024.0, 4096.0):
        q = torch.full((1, 4, d), gain, device=DEV, dtype=dtype)
        scores = torch.zeros(1, 1, c.max_slots, device=DEV)
        out = c.attention(q, ints([n]), scale=1.0, scores=scores)
        assert torch.equal(out[0].float(), want.expand(4, d))
        assert torch.equal(scores[0, 0].nonzero()[:, 0], torch.tensor(pair, device=DEV)) and (scores[0, 0, list(pair)] == 2).all()


@TABLES
@pytest.mark.parametrize("gain,scale", [(40.0, None), (1.0, 0.0), (2.0, -0.3), (1e-3, 2.0), (40.0, 30.0)])
def test_attention_scales_of_f16(gain, scale, wide):
    run_attention(F16, 8, 2, 64, 16, [100, 1, 33], 0, True, gain=gain, scale=scale, wide=wide)


# ---- the edges of the arguments -------------------------------------------------------------------

def test_calls_without_tokens_or_sequences():
    c = simple_cache(BF16)
    q, k = torch.zeros(0, 4, 64, device=DEV, dtype=BF16), torch.zeros(0, 2, 64, device=DEV, dtype=BF16)
    none = ints([])
    ang = torch.randn(4, 32, device=DEV)
    for rot in (None, paged.Rotary(ang.cos(), ang.sin())):
        assert c.append(q, k, k, none, none, none, rot).shape == (0, 4, 64)
        assert c.append(None, k, k, none, none, none, rot) is None
    assert c.attention(q, none).shape == (0, 4, 64)
    kept, lengths, _ = c.evict(none, torch.zeros(0, 2, c.max_slots, device=DEV), 2, 1, torch.zeros(0, 1, dtype=torch.int32, device=DEV))
    assert kept.shape == (0, 2, 2) and lengths.shape == (0,)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n", [40, 9000])
def test_attention_windows_longer_than_any_sequence(dtype, n):
    """A window that no sequence reaches is no window, up to the largest number: the same kernels, the same bits."""
    k, v, table, _ = make_pool([n], 2, 64, 64, dtype, 14)
    c = paged.PagedCache(k, v, table)
    q = torch.randn(1, 4, 64, device=DEV).to(dtype)
    old = torch.rand(1, 2, c.max_slots, device=DEV)
    want, new = c.attention(q, ints([n])), torch.zeros_like(old)
    want_s = c.attention(q, ints([n]), scores=old, new_scores=new)
    for window in (c.max_slots, c.max_slots + 1, 1 << 31, (1 << 63) - 33, (1 << 63) - 1):
        assert torch.equal(c.attention(q, ints([n]), window=window), want)
        got = torch.zeros_like(old)
        assert torch.equal(c.attention(q, ints([n]), window=window, scores=old, new_scores=got), want_s) and torch.equal(got, new)


# ---- sizes at which the kernels take other paths --------------------------------------------------

# dtype, heads, kv, d, pairs, axes, interleaved, norm, offset of the views: rows in chunks of 16, 8 and 4 bytes and of single
# values; 36, 40, 15 and 29 rows a token, so that a warp's steps mix queries, keys and values and the last is not full
PROMPTS = [
    (BF16, 28, 4, 128, 64, 3, False, True, 0), (F16, 32, 4, 128, 32, 1, True, False, 0), (F32, 9, 3, 128, 64, 3, False, True, 0),
    (BF16, 28, 4, 72, 36, 3, False, True, 0), (F16, 9, 3, 40, 10, 1, False, True, 0), (BF16, 21, 4, 64, 32, 3, True, True, 2),
    (F16, 9, 3, 64, 32, 1, False, True, 1), (F32, 21, 4, 256, 6, 2, False, False, 0),
]


@pytest.mark.parametrize("tokens", [33, 700, 2500])
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_append_prompts(case, tokens):
    """Prompts of ragged sequences packed one after another with padding between them, in float64 on the GPU; the bounds are
    the oracle's (oracle/paged.py)."""
    dtype, heads, kv, d, pairs, axes, interleaved, norm, offset = case
    ps, gen = 16, torch.Generator().manual_seed(tokens + d)
    lengths = [tokens // 7, tokens // 2, 1, tokens - tokens // 7 - tokens // 2 - 1]
    start = [5, 0, 30, 16]
    need = [-(-(s + n) // ps) for s, n in zip(start, lengths)]
    order = torch.randperm(sum(need) + 3, generator=gen).int()
    table = torch.full((4, max(need)), -1, dtype=torch.int32)
    for s, at in enumerate(np.cumsum([0] + need)[:4]):
        table[s, :need[s]] = order[at:at + need[s]]
    table = table.to(DEV)
    seq = torch.cat([torch.cat([torch.full((n,), s), torch.full((s,), -1)]) for s, n in enumerate(lengths)])
    slot = torch.cat([torch.cat([torch.arange(n) + start[s], torch.full((s,), -9)]) for s, n in enumerate(lengths)])
    rows = len(seq)
    pools = [torch.randn(sum(need) + 3, kv, ps, d, generator=gen).to(DEV, dtype) for _ in range(2)]
    c = paged.PagedCache(*pools, table)
    width = (heads + 2 * kv) * d
    x = torch.randn(rows, width + offset, generator=gen).to(DEV, dtype)[:, offset:].unflatten(1, (-1, d))
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    positions = torch.randint(0, 4000, (axes, rows), generator=gen).int().to(DEV)
    ang = torch.arange(4000, dtype=torch.float64)[:, None] * (1e4 ** (-torch.arange(pairs, dtype=torch.float64) / pairs))[None]
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    axis = torch.arange(pairs, device=DEV) % axes
    w = [torch.rand(d, generator=gen).add(0.5).to(DEV) if norm else None for _ in range(2)]
    rot = paged.Rotary(cos, sin, pair_axis=axis.tolist(), interleaved=interleaved, q_weight=w[0], k_weight=w[1], eps=1e-6)
    want_pools = [p.clone() for p in pools]
    out = torch.full((rows, heads, d), 3.0, device=DEV, dtype=dtype)
    c.append(q, k, v, seq.int().to(DEV), slot.int().to(DEV), positions, rot, out=out)
    j = torch.arange(pairs, device=DEV)
    one, two = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    at = positions.long()[axis].T  # [rows, pairs]
    cs, sn = cos.double()[at, j][:, None], sin.double()[at, j][:, None]

    def check(got, x, w):
        y = x.double()
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        bound = y.abs() * (20 * po.U)
        a, b = y[..., one], y[..., two]
        bound[..., one] = bound[..., two] = torch.hypot(a, b) * (20 * po.U)
        y[..., one], y[..., two] = a * cs[live] - b * sn[live], b * cs[live] + a * sn[live]
        eps = 0.0 if dtype == F32 else half_step(dtype)
        tiny = 2.0 ** -25 if dtype == F16 else 0.0
        assert ((got.double() - y).abs() <= bound * (1 + eps) + y.abs() * eps + tiny).all()

    live = (seq >= 0).to(DEV)
    check(out[live], q[live], w[0])
    assert (out[~live] == 3).all()
    s, r = seq.to(DEV)[live], slot.to(DEV)[live]
    page, row = table.long()[s, r // ps], r % ps
    check(pools[0][page, :, row], k[live], w[1])
    want_pools[0][page, :, row], want_pools[1][page, :, row] = pools[0][page, :, row], v[live]
    assert torch.equal(want_pools[0], pools[0]) and torch.equal(want_pools[1], pools[1])


def kept_of(scores, n, keep, recent):
    """oracle.paged.keep_slots on the GPU, for finite scores."""
    if n <= keep:
        return torch.arange(n, device=DEV)
    best = scores[:n - recent].sort(descending=True, stable=True).indices[:keep - recent]
    return torch.cat([best.sort().values, torch.arange(n - recent, n, device=DEV)])


@pytest.mark.parametrize("lengths,kv,keep,recent", [
    ([340001, 12, 340000, 0], 2, 30001, 77),       # clusters of eight, each CTA with more keys than it holds
    ([20000, 9000, 1, 8999, 20011], 3, 9000, 0),   # clusters of four, some rows without a selection
    ([41300, 40000] + [100] * 100, 2, 500, 50),    # one CTA a row, with more keys than it holds
    ([340001], 1, 340000, 339999),                 # one slot goes
], ids=str)
def test_evict_wide_tables(lengths, kv, keep, recent):
    """Sequences over the same pages (the old rows are only read), in tables wide enough for each way that a row's keys are
    shared out; with few values, so that most scores have equals."""
    ps, d, count = 128, 4, len(lengths)
    width, new_width = -(-max(lengths) // ps), -(-keep // ps)
    old = torch.arange(width * kv * ps, device=DEV, dtype=F32)[:, None].expand(-1, d).reshape(width, kv, ps, d)
    fresh = torch.zeros(count * new_width, kv, ps, d, device=DEV)
    pool = torch.cat([old, fresh])
    table = torch.arange(width, device=DEV).int().expand(count, width).contiguous()
    new = torch.arange(width, width + count * new_width, device=DEV).int().view(count, new_width)
    c = paged.PagedCache(pool, -pool, table)
    scores = torch.randint(0, 400, (count, kv, c.max_slots), device=DEV, generator=torch.Generator(DEV).manual_seed(9)).float()
    kept, new_len, new_sc = c.evict(ints(lengths), scores, keep, recent, new)
    assert new_len.tolist() == [min(n, keep) for n in lengths]
    assert torch.equal(pool[:width], old)
    for b, n in enumerate(lengths):
        m = min(n, keep)
        for h in range(kv):
            idx = kept_of(scores[b, h], n, keep, recent)
            assert torch.equal(kept[b, h, :m].long(), idx) and (kept[b, h, m:] == -1).all()
            assert torch.equal(new_sc[b, h, :m], scores[b, h, idx]) and not new_sc[b, h, m:].any()
            j = torch.arange(m, device=DEV)
            for pages, sign in ((pool, 1), (c.v_pages, -1)):
                assert torch.equal(pages[new[b].long()[j // ps], h, j % ps], sign * old[idx // ps, h, idx % ps])


@TABLES
@pytest.mark.parametrize("dtype,heads,kv", [(F16, 20, 1), (BF16, 96, 2), (F32, 24, 2)])
def test_attention_of_several_head_tiles_with_and_without_scores(dtype, heads, kv, wide):
    """Scores may choose another kernel, whose sums run in another order: both within the bounds."""
    lengths = [200, 1, 90]
    k, v, table, _ = make_pool(lengths, kv, 16, 64, dtype, 15, width=width_of(wide, lengths, 16))
    c = paged.PagedCache(k, v, table)
    q = torch.randn(3, heads, 64, device=DEV).to(dtype)
    old = torch.rand(3, kv, c.max_slots, device=DEV)
    new = old.clone()
    check_attention(c.attention(q, ints(lengths)), None, c, q, lengths, 0, None)
    check_attention(c.attention(q, ints(lengths), scores=old, new_scores=new), new, c, q, lengths, 0, old)


def test_calls_on_two_streams_at_once():
    """Eager steps of two caches side by side, without waiting for one another: each gives the bits that it gives alone."""
    def make(seed, dtype, lengths):
        k, v, table, new = make_pool(lengths, 2, 16, 64, dtype, seed, width=width_of(True, lengths, 16), fresh=20)
        c = paged.PagedCache(k, v, table)
        g = torch.Generator(DEV).manual_seed(seed)
        q = torch.randn(len(lengths), 8, 64, device=DEV, generator=g).to(dtype)
        return c, q, ints(lengths), torch.rand(len(lengths), 2, c.max_slots, device=DEV, generator=g), new

    def step(c, q, n, scores, new):
        s = scores.clone()
        out = c.attention(q, n, scores=s)
        return (out, s, *c.evict(n, s, 300, 40, new))

    cases = [make(41, BF16, [4000, 900, 0, 2500]), make(42, F32, [3000, 1, 1700])]
    alone = [step(*x) for x in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for x, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append([step(*x) for _ in range(3)])
        torch.cuda.synchronize()
        for want, three in zip(alone, got):
            for one in three:
                assert all(torch.equal(a, b) for a, b in zip(want, one))
