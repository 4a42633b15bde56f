"""The paged key-value cache's operators as timed cases: what fills the cache (`append`: per-head
RMSNorm, rotary positions of one or several axes, the write into pages), what reads it
(`attention` of one new token a sequence) and what trims it (`evict` by accumulated attention
weight).

A pool of pages [num_pages, kv_heads, page_size, head_dim] is shared by all sequences; row s of
the page table lists the pages of sequence s in order, -1 behind the last one.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 1e6
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------

def _append(name, dtype, heads, kv_heads, head_dim, page, tokens, batch, start, norm, axes, interleaved=False,
            rotary_dim=0, padding=0):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "tokens": tokens, "batch": batch, "start": start, "norm": norm, "axes": axes,
            "interleaved": interleaved, "rotary_dim": rotary_dim or head_dim, "padding": padding}


def _attention(name, dtype, heads, kv_heads, head_dim, page, batch, length, ragged, window, scores):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "batch": batch, "length": length, "ragged": ragged, "window": window,
            "scores": scores}


def _evict(name, dtype, kv_heads, head_dim, page, batch, length, ragged, keep, recent):
    return {"name": name, "op": "evict", "dtype": dtype, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "batch": batch, "length": length, "ragged": ragged, "keep": keep, "recent": recent}


def listed():
    return [
        # one decode step of the framework's own decoder: one token, query/key norm, f32
        _append("append_decoder_token", "f32", 16, 8, 128, 16, 1, 1, 256, True, 1),
        # one decode step of a served batch, padded to a fixed number of rows for a captured graph
        _append("append_batch_tokens", "bf16", 32, 8, 128, 16, 64, 64, 1500, False, 1, padding=3),
        # prompts with images, packed one after another: time, height and width positions
        _append("append_video_prompts", "bf16", 28, 4, 128, 32, 8191, 5, 37, True, 3),
        # the framework's own decoder at the end of its default context
        _attention("attention_decoder_token", "f32", 16, 8, 128, 16, 1, 257, 0, 0, False),
        # a served batch of chats of every length
        _attention("attention_chats", "bf16", 32, 8, 128, 16, 32, 4096, 11, 0, False),
        # a single long document: few rows, the length is all there is to split
        _attention("attention_long_document", "f16", 32, 8, 128, 64, 1, 131071, 0, 0, False),
        # a full card: long ragged contexts, with the weights that eviction needs
        _attention("attention_full_batch_scores", "bf16", 32, 8, 128, 32, 64, 8192, 12, 0, True),
        # odd head counts and sizes with a sliding window
        _attention("attention_window_odd", "f16", 28, 4, 80, 16, 7, 1999, 13, 1000, True),
        # as many key heads as query heads, f32
        _attention("attention_ungrouped", "f32", 8, 8, 64, 32, 24, 2900, 14, 0, False),
        # one short sequence trimmed to half
        _evict("evict_decoder", "f32", 8, 128, 16, 1, 257, 0, 128, 32),
        # a served batch trimmed to a budget (the shorter sequences only move)
        _evict("evict_batch", "bf16", 8, 128, 32, 16, 8192, 15, 2047, 256),
        # long documents trimmed to an eighth
        _evict("evict_long_documents", "f16", 8, 128, 64, 2, 131072, 0, 16384, 1000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "evict"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    kv_heads, group = rng.choice([(8, 2), (8, 4), (4, 7), (8, 1), (2, 6), (1, 8), (4, 8), (3, 5), (2, 16), (1, 20)])
    head_dim = rng.choice([128, 128, 64, 80, 96, 72, 256, 40])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    size = 4 if dtype == "f32" else 2
    row = kv_heads * head_dim * size * 2
    if op == "append":
        batch = _log(rng, 1, 64)
        tokens = max(batch, _log(rng, 1, 8191))
        axes = rng.choice([1, 1, 3])
        rotary = rng.choice([head_dim, head_dim, head_dim // 2])
        return _append("drawn", dtype, kv_heads * group, kv_heads, head_dim, page, tokens, batch,
                       _log(rng, 1, 4000), rng.random() < 0.5, axes, rng.random() < 0.3, rotary,
                       rng.choice([0, 0, 5]))
    if op == "attention":
        length = _log(rng, 1, min(131072, (1 << 30) // row))
        most = min(64, (1 << 30) // (row * length))
        batch = _log(rng, 1, max(1, most))
        window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        return _attention("drawn", dtype, kv_heads * group, kv_heads, head_dim, page, batch, length,
                          rng.choice([0, rng.randint(1, 1 << 20)]), window, rng.random() < 0.4)
    length = _log(rng, 2, min(131072, (1 << 29) // row))
    batch = _log(rng, 1, max(1, min(32, (1 << 29) // (row * length))))
    keep = max(1, int(length * rng.uniform(0.05, 0.9)))
    return _evict("drawn", dtype, kv_heads, head_dim, page, batch, length, rng.choice([0, rng.randint(1, 1 << 20)]),
                  keep, int(keep * rng.choice([0.0, 0.1, 0.5, 1.0])))


def _lengths(case):
    """Slots in use of each sequence, the new token's among them; a ragged batch of four and more
    has one row without a sequence."""
    n, most = case["batch"], case["length"]
    if not case["ragged"]:
        return [most] * n
    rnd = random.Random(case["ragged"])
    out = [rnd.randint(1, most) for _ in range(n)]
    out[rnd.randrange(n)] = most
    if n >= 4:
        out[out.index(min(out))] = 0
    return out


def _spans(case):
    """(first slot, tokens) of each sequence of an append."""
    rnd = random.Random(case["tokens"] * 131 + case["batch"])
    cuts = sorted(rnd.sample(range(1, case["tokens"]), case["batch"] - 1)) if case["batch"] > 1 else []
    edges = [0] + cuts + [case["tokens"]]
    return [(rnd.randint(0, case["start"]), b - a) for a, b in zip(edges, edges[1:])]


def _sections(case):
    """Pairs of each axis: a quarter turns with time, the rest half and half with height and width."""
    half = case["rotary_dim"] // 2
    if case["axes"] == 1:
        return [half]
    t = half // 4
    return [t, (half - t) // 2, half - t - (half - t) // 2]


# ---- inputs -----------------------------------------------------------------------------------

def _pool(case, gen, lengths, fresh=0):
    """Pages in a shuffled order, as a pool in use has them, and the table. `fresh`: pages a row
    for an eviction's destination."""
    page, n = case["page"], len(lengths)
    need = [-(-x // page) for x in lengths]
    total = sum(need) + n * fresh + 8
    shape = (total, case["kv_heads"], page, case["head_dim"])
    dt = DTYPES[case["dtype"]]
    k = torch.randn(shape, device=DEVICE, dtype=dt, generator=gen)
    v = torch.randn(shape, device=DEVICE, dtype=dt, generator=gen)
    order = torch.randperm(total, device=DEVICE, generator=gen).to(torch.int32)
    width = max(need) + 1
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEVICE)
    starts = torch.tensor([sum(need[:i]) for i in range(n)], device=DEVICE)[:, None]
    col = torch.arange(width, device=DEVICE)[None, :]
    used = col < torch.tensor(need, device=DEVICE)[:, None]
    table[used] = order[(starts + col)[used]]
    new = order[sum(need):sum(need) + n * fresh].reshape(n, fresh).contiguous()
    return k, v, table, new


def _tables(max_pos, half):
    inv = THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    ang = torch.arange(max_pos, device=DEVICE, dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float(), ang.sin().float()


def _prepare_append(case, gen):
    spans = _spans(case)
    t, pad = case["tokens"], case["padding"]
    seq, slot = [], []
    for s, (first, count) in enumerate(spans):
        seq += [s] * count
        slot += range(first, first + count)
    pos = torch.tensor(slot, device=DEVICE, dtype=torch.int32)
    if case["axes"] == 3:
        # stretches of 512 tokens: every second one is a frame of 16 x 32 patches
        j = torch.arange(t, device=DEVICE, dtype=torch.int32)
        base = pos - j % 512
        frame = (j // 512) % 2 == 1
        base = torch.where(frame & (base >= 0), base, pos)
        inside = torch.where(base == pos, 0, j % 512)
        pos = torch.stack([base, base + inside // 32, base + inside % 32])
    else:
        pos = pos[None]
    tail = torch.full((pad,), -1, dtype=torch.int32, device=DEVICE)
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    dt = DTYPES[case["dtype"]]
    # the merged projection's rows: q, k and v are views of it
    qkv = torch.randn((t + pad, (h + 2 * kv) * d), device=DEVICE, dtype=dt, generator=gen)
    k_pages, v_pages, table, _ = _pool(case, gen, [a + b for a, b in spans])
    half = case["rotary_dim"] // 2
    cos, sin = _tables(case["start"] + t + 1, half)
    s = {"q": qkv[:, :h * d].view(t + pad, h, d), "k": qkv[:, h * d:(h + kv) * d].view(t + pad, kv, d),
         "v": qkv[:, (h + kv) * d:].view(t + pad, kv, d), "seq": torch.cat([torch.tensor(seq, device=DEVICE, dtype=torch.int32), tail]),
         "slot": torch.cat([torch.tensor(slot, device=DEVICE, dtype=torch.int32), tail]),
         "positions": torch.cat([pos, tail.expand(pos.shape[0], pad)], 1).contiguous(), "cos": cos, "sin": sin,
         "k_pages": k_pages, "v_pages": v_pages, "table": table, "tokens": t,
         "q_out": torch.zeros((t + pad, h, d), device=DEVICE, dtype=dt), "q_w": None, "k_w": None}
    if case["norm"]:
        s["q_w"] = torch.rand(d, device=DEVICE, generator=gen) + 0.5
        s["k_w"] = torch.rand(d, device=DEVICE, generator=gen) + 0.5
    return s


def _prepare_attention(case, gen):
    lengths = _lengths(case)
    k_pages, v_pages, table, _ = _pool(case, gen, lengths)
    dt = DTYPES[case["dtype"]]
    # twice the unit variance: some slots stand out, as with trained heads
    q = torch.randn((case["batch"], case["heads"], case["head_dim"]), device=DEVICE, dtype=dt, generator=gen) * 2
    s = {"q": q, "k_pages": k_pages, "v_pages": v_pages, "table": table, "host_lengths": lengths,
         "lengths": torch.tensor(lengths, device=DEVICE, dtype=torch.int32), "scores": None, "new_scores": None}
    if case["scores"]:
        shape = (case["batch"], case["kv_heads"], table.shape[1] * case["page"])
        s["scores"] = torch.rand(shape, device=DEVICE, generator=gen)
        s["new_scores"] = torch.zeros(shape, device=DEVICE)
    return s


def _prepare_evict(case, gen):
    lengths = _lengths(case)
    k_pages, v_pages, table, new = _pool(case, gen, lengths, -(-case["keep"] // case["page"]))
    shape = (case["batch"], case["kv_heads"], table.shape[1] * case["page"])
    # a few slots hold most of the weight; the f16 grid makes equal scores common
    scores = (torch.rand(shape, device=DEVICE, generator=gen).clamp_min(1e-6).log() ** 2).half().float()
    scores[torch.rand(shape, device=DEVICE, generator=gen) < 0.1] = 0
    return {"k_pages": k_pages, "v_pages": v_pages, "table": table, "new_table": new, "host_lengths": lengths,
            "lengths": torch.tensor(lengths, device=DEVICE, dtype=torch.int32), "scores": scores,
            "new_scores": torch.zeros((case["batch"], case["kv_heads"], case["keep"]), device=DEVICE)}


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    s = {"append": _prepare_append, "attention": _prepare_attention, "evict": _prepare_evict}[case["op"]](case, gen)
    s["case"] = case
    if own:
        from transmuter_b200 import paged
        s["cache"] = paged.PagedCache(s["k_pages"], s["v_pages"], s["table"])
        if case["op"] == "append":
            s["rotary"] = paged.Rotary(s["cos"], s["sin"], sections=_sections(case), interleaved=case["interleaved"],
                                       q_weight=s["q_w"], k_weight=s["k_w"], eps=EPS)
    return s


# ---- the plain forms --------------------------------------------------------------------------

def _rotated(x, w, s):
    """x [T, heads, D] of the real tokens: norm, then each pair of the rotated part turned."""
    case, t = s["case"], s["tokens"]
    x = x[:t].float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    half = case["rotary_dim"] // 2
    axis = torch.cat([torch.full((n,), i) for i, n in enumerate(_sections(case))]).to(DEVICE)
    row = s["positions"][:, :t].long()[axis]                     # [half, T]
    col = torch.arange(half, device=DEVICE)[:, None]
    c, n = s["cos"][row, col].T[:, None, :], s["sin"][row, col].T[:, None, :]
    if case["interleaved"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_append(s):
    t, page = s["tokens"], s["case"]["page"]
    seq, slot = s["seq"][:t].long(), s["slot"][:t].long()
    s["q_out"][:t] = _rotated(s["q"], s["q_w"], s).to(s["q_out"].dtype)
    where = s["table"][seq, slot // page].long()
    s["k_pages"][where, :, slot % page] = _rotated(s["k"], s["k_w"], s).to(s["k_pages"].dtype)
    s["v_pages"][where, :, slot % page] = s["v"][:t]
    return s["q_out"], s["k_pages"], s["v_pages"]


def _rows(pages, table, b, lo, hi, page):
    """Slots lo..hi of sequence b: [kv_heads, hi - lo, head_dim]."""
    first = lo // page
    at = table[b, first:-(-hi // page)].long()
    x = pages[at].transpose(0, 1).flatten(1, 2)
    return x[:, lo - first * page:hi - first * page]


def _plain_attention(s):
    case, q = s["case"], s["q"]
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros_like(q)
    for b, n in enumerate(s["host_lengths"]):
        lo = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        k = _rows(s["k_pages"], s["table"], b, lo, n, page).float()
        v = _rows(s["v_pages"], s["table"], b, lo, n, page).float()
        x = q[b].float().view(kv, -1, d) @ k.transpose(1, 2) / math.sqrt(d)
        e = torch.exp(x - x.max(-1, keepdim=True).values)
        p = e / e.sum(-1, keepdim=True)
        out[b] = (p @ v).reshape(-1, d).to(q.dtype)
        if case["scores"]:
            s["new_scores"][b, :, :lo] = s["scores"][b, :, :lo]
            s["new_scores"][b, :, lo:n] = s["scores"][b, :, lo:n] + p.sum(1)
    return (out, s["new_scores"]) if case["scores"] else out


def _plain_evict(s):
    case = s["case"]
    kv, page, keep, recent = case["kv_heads"], case["page"], case["keep"], case["recent"]
    kept = torch.full((case["batch"], kv, keep), -1, dtype=torch.int32, device=DEVICE)
    for b, n in enumerate(s["host_lengths"]):
        if n == 0:
            continue
        idx = torch.arange(n, device=DEVICE).expand(kv, n)
        if n > keep:
            best = s["scores"][b, :, :n - recent].sort(dim=-1, descending=True, stable=True).indices[:, :keep - recent]
            idx = torch.cat([best.sort(-1).values, idx[:, n - recent:]], 1)
        m = idx.shape[1]
        kept[b, :, :m] = idx.int()
        s["new_scores"][b, :, :m] = s["scores"][b].gather(1, idx)
        to = torch.arange(m, device=DEVICE)
        at = s["new_table"][b, to // page].long()
        for pages in (s["k_pages"], s["v_pages"]):
            x = _rows(pages, s["table"], b, 0, n, page)
            moved = x.gather(1, idx[:, :, None].expand(-1, -1, x.shape[2]))
            pages[at, :, to % page] = moved.transpose(0, 1)
    return kept, s["lengths"].clamp(max=keep), s["new_scores"], s["k_pages"], s["v_pages"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict}[op](s)
    cache, case = s["cache"], s["case"]
    if op == "append":
        cache.append(s["q"], s["k"], s["v"], s["seq"], s["slot"], s["positions"], s["rotary"], out=s["q_out"])
        return s["q_out"], s["k_pages"], s["v_pages"]
    if op == "attention":
        if case["scores"]:
            return cache.attention(s["q"], s["lengths"], window=case["window"], scores=s["scores"],
                                   new_scores=s["new_scores"]), s["new_scores"]
        return cache.attention(s["q"], s["lengths"], window=case["window"])
    kept, lengths, scores = cache.evict(s["lengths"], s["scores"], case["keep"], case["recent"], s["new_table"],
                                        new_scores=s["new_scores"])
    return kept, lengths, scores, s["k_pages"], s["v_pages"]


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kv, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        t, h = case["tokens"], case["heads"]
        positions = sum(count for _, count in _spans(case)) * case["axes"]
        return {"bytes": t * (h + 2 * kv) * d * size * 2 + positions * 4 + t * (8 + 4 * case["rotary_dim"]),
                "flops": t * (h + kv) * (3 * case["rotary_dim"] + (4 * d if case["norm"] else 0))}
    lengths = _lengths(case)
    if case["op"] == "attention":
        seen = [min(n, case["window"]) if case["window"] else n for n in lengths]
        moved = 2 * sum(seen) * kv * d * size + 2 * case["batch"] * case["heads"] * d * size
        if case["scores"]:
            moved += 8 * sum(lengths) * kv
        return {"bytes": moved, "flops": 4 * sum(seen) * case["heads"] * d}
    rows = sum(min(n, case["keep"]) for n in lengths) * kv
    return {"bytes": sum(n for n in lengths if n > case["keep"]) * kv * 4 + rows * (4 * d * size + 12),
            "flops": sum(n for n in lengths if n > case["keep"]) * kv}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _exact_append(s):
    case = s["case"]
    t, page, half = s["tokens"], case["page"], case["rotary_dim"] // 2
    j = torch.arange(half, device=DEVICE)
    if case["interleaved"]:
        one, two = 2 * j, 2 * j + 1
    else:
        one, two = j, j + half
    bounds = torch.tensor(_sections(case), device=DEVICE).cumsum(0)
    axis = torch.bucketize(j, bounds, right=True)
    at = s["positions"].long()[axis, :t].T                        # [T, half]
    phase = torch.complex(s["cos"].double()[at, j], s["sin"].double()[at, j])[:, None]

    def turn(x, w):
        x = x[:t].double()
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        z = torch.complex(x[..., one], x[..., two]) * phase
        x = x.clone()
        x[..., one], x[..., two] = z.real, z.imag
        return x

    q = s["q_out"].double()
    q[:t] = turn(s["q"], s["q_w"])
    k, v = s["k_pages"].double(), s["v_pages"].double()
    flat = s["slot"][:t].long()
    pages = s["table"].long()[s["seq"][:t].long()].gather(1, (flat // page)[:, None])[:, 0]
    k.transpose(1, 2)[pages, flat % page] = turn(s["k"], s["k_w"])
    v.transpose(1, 2)[pages, flat % page] = s["v"][:t].double()
    return q, k, v


def _exact_attention(s):
    case = s["case"]
    d, page, group = case["head_dim"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    total = s["new_scores"].double() if case["scores"] else None
    for b, n in enumerate(s["host_lengths"]):
        lo = max(0, n - case["window"]) if case["window"] else 0
        slots = torch.arange(lo, n, device=DEVICE)
        if total is not None:
            total[b, :, :n] = s["scores"][b, :, :n].double()
        if n == 0:
            continue
        at, off = s["table"][b].long()[slots // page], slots % page
        for g in range(case["kv_heads"]):
            k, v = s["k_pages"][at, g, off].double(), s["v_pages"][at, g, off].double()
            w = torch.softmax((k @ s["q"][b, g * group:(g + 1) * group].double().T) * d ** -0.5, 0)
            out[b, g * group:(g + 1) * group] = w.T @ v
            if total is not None:
                total[b, g, lo:n] += w.sum(1)
    return (out, total) if case["scores"] else out


def _exact_evict(s):
    case = s["case"]
    page, keep, recent = case["page"], case["keep"], case["recent"]
    kept = torch.full((case["batch"], case["kv_heads"], keep), -1, dtype=torch.int32, device=DEVICE)
    scores = s["new_scores"].double()
    k, v = s["k_pages"].double(), s["v_pages"].double()
    for b, n in enumerate(s["host_lengths"]):
        m = min(n, keep)
        for g in range(case["kv_heads"] if n else 0):
            key = s["scores"][b, g, :n].double()
            if n > keep:
                key = torch.where(torch.arange(n, device=DEVICE) >= n - recent, math.inf, key)
            # the m-th largest: what lies above it stays, and the first of its equals up to m
            edge = key.kthvalue(n - m + 1).values
            above, equal = key > edge, key == edge
            stay = above | (equal & (equal.cumsum(0) <= m - above.sum()))
            idx = stay.nonzero()[:, 0]
            kept[b, g, :m] = idx.int()
            scores[b, g, :m] = s["scores"][b, g, idx].double()
            to = torch.arange(m, device=DEVICE)
            src, dst = s["table"][b].long()[idx // page], s["new_table"][b].long()[to // page]
            k[dst, g, to % page] = s["k_pages"][src, g, idx % page].double()
            v[dst, g, to % page] = s["v_pages"][src, g, idx % page].double()
    return kept, torch.tensor([min(n, keep) for n in s["host_lengths"]], dtype=torch.int32, device=DEVICE), scores, k, v


def exact(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    s = {"append": _prepare_append, "attention": _prepare_attention, "evict": _prepare_evict}[case["op"]](case, gen)
    s["case"] = case
    return {"append": _exact_append, "attention": _exact_attention, "evict": _exact_evict}[case["op"]](s)
