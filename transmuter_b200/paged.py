"""The paged key-value cache of a served q4 decoder (include/tq4_paged.h): a pool of pages that holds
the rows of many sequences, what fills it (``PagedCache.append``: per-head RMSNorm, rotary positions
of one or several axes, the write into pages), what reads it (``attention`` of one new token of each
sequence) and what trims it (``evict`` by accumulated attention weight).

``decoder.Q4Decoder`` runs one sequence over a contiguous f32 cache; between the projections of
``quantized.PackedWeight`` a batch of sequences runs over this one. All tensors are CUDA tensors of
the cache's device, calls enqueue on the current torch stream and can be captured into a CUDA graph
(lengths, slots and page tables are read on the device). Errors follow ``quantized``: wrong arguments
raise ``ArgumentError``; what only the device can see (a length, slot or page number out of range) is
skipped and sets the device status (``tq4_device_status``).
"""

import ctypes
import math

import torch

from . import _lib
from .deferred import ArgumentError
from .quantized import TORCH_TO_TQ4

FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _need(ok, message):
    if not ok:
        raise ArgumentError(message)


def _pointer(x, name, shape, dtype, device):
    """The address of a contiguous tensor of exactly this shape, type and device."""
    # (a call makes up to nine of these checks in the time of one launch: the message is only made for a refusal)
    if not (isinstance(x, torch.Tensor) and x.dtype is dtype and x.shape == shape and x.device == device
            and x.is_contiguous()):
        got = f"{x.dtype} {tuple(x.shape)} on {x.device}" if isinstance(x, torch.Tensor) else type(x).__name__
        raise ArgumentError(f"paged cache: {name} must be a contiguous {dtype} {tuple(shape)} on {device}, got {got}")
    return x.data_ptr()


# The stream's address without the Stream object around it (2.2 us of a call otherwise).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class Rotary:
    """The rotary embedding of ``PagedCache.append`` and the per-head RMSNorm before it.

    ``cos`` and ``sin`` are f32 tables [max_pos, pairs] (``decoder.rope_tables``), ``sections`` the
    number of pairs that follow each axis of the positions, in order (time, height, width), or
    ``pair_axis`` each pair's axis; one axis by default. ``interleaved`` pairs values (2i, 2i + 1)
    instead of (i, i + pairs), and heads wider than 2 * pairs keep the rest unturned. ``q_weight`` and
    ``k_weight`` are f32 norm weights [head_dim], None for no norm.
    """

    def __init__(self, cos, sin, sections=None, pair_axis=None, interleaved=False, q_weight=None, k_weight=None,
                 eps=1e-6):
        _need(isinstance(cos, torch.Tensor) and cos.dim() == 2 and cos.is_cuda,
              "Rotary: cos must be a CUDA tensor [max_pos, pairs]")
        max_pos, pairs = cos.shape
        self.device, self.pairs = cos.device, pairs
        _pointer(cos, "cos", (max_pos, pairs), torch.float32, self.device)
        _pointer(sin, "sin", (max_pos, pairs), torch.float32, self.device)
        _need(sections is None or pair_axis is None, "Rotary: sections or pair_axis, not both")
        if sections is not None:
            _need(sum(sections) == pairs and min(sections, default=0) >= 0,
                  f"Rotary: sections {tuple(sections)} do not add up to {pairs} pairs")
            pair_axis = [i for i, n in enumerate(sections) for _ in range(n)]
            self.axes = len(sections)
        elif pair_axis is not None:
            _need(len(pair_axis) == pairs, f"Rotary: {len(pair_axis)} axes for {pairs} pairs")
            self.axes = max(pair_axis, default=0) + 1
        else:
            pair_axis, self.axes = [0] * pairs, 1
        _need(1 <= self.axes <= 4 and min(pair_axis, default=0) >= 0, "Rotary: 1 to 4 axes")
        for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if w is not None:
                _pointer(w, name, (w.numel(),), torch.float32, self.device)
        self.widths = {w.numel() for w in (q_weight, k_weight) if w is not None}
        self._keep = (cos, sin, q_weight, k_weight, (ctypes.c_uint8 * max(1, pairs))(*pair_axis))
        r = _lib.RotaryDesc()
        r.cos_table, r.sin_table, r.max_pos, r.pairs, r.axes = cos.data_ptr(), sin.data_ptr(), max_pos, pairs, self.axes
        r.pair_axis = ctypes.addressof(self._keep[4])
        r.interleaved, r.eps = int(bool(interleaved)), eps
        r.q_w = q_weight.data_ptr() if q_weight is not None else None
        r.k_w = k_weight.data_ptr() if k_weight is not None else None
        self._desc = r
        self._ref = ctypes.byref(r)


class PagedCache:
    """A pool ``k_pages`` / ``v_pages`` [num_pages, kv_heads, page_size, head_dim] (f32, f16 or bf16)
    with the page table int32 [max_seqs, max_pages] of the sequences in it: slot j of sequence s is
    row j % page_size of page ``page_table[s, j // page_size]``. The tensors stay the caller's, who
    hands out pages by writing the table."""

    def __init__(self, k_pages, v_pages, page_table):
        _need(isinstance(k_pages, torch.Tensor) and k_pages.is_cuda and k_pages.dim() == 4 and k_pages.dtype in FLOATS,
              "PagedCache: k_pages must be a CUDA tensor [num_pages, kv_heads, page_size, head_dim], f32, f16 or bf16")
        self.device, self.dtype = k_pages.device, k_pages.dtype
        _pointer(k_pages, "k_pages", k_pages.shape, self.dtype, self.device)
        _pointer(v_pages, "v_pages", k_pages.shape, self.dtype, self.device)
        _need(isinstance(page_table, torch.Tensor) and page_table.dim() == 2, "PagedCache: page_table must be [max_seqs, max_pages]")
        _pointer(page_table, "page_table", page_table.shape, torch.int32, self.device)
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k_pages.shape
        self.max_seqs, self.max_pages = page_table.shape
        self.max_slots = self.max_pages * self.page_size
        d = _lib.PagedDesc()
        d.dtype, d.kv_heads, d.head_dim, d.page_size = TORCH_TO_TQ4[self.dtype], self.kv_heads, self.head_dim, self.page_size
        d.num_pages, d.max_seqs, d.max_pages = self.num_pages, self.max_seqs, self.max_pages
        self._lib = _lib.load()
        self._handle = None
        handle = ctypes.c_void_p()
        _lib.check(self._lib.tq4_paged_create(ctypes.byref(d), k_pages.data_ptr(), v_pages.data_ptr(),
                                              page_table.data_ptr(), self.device.index or 0, ctypes.byref(handle)))
        self._handle = handle
        self._index = self.device.index or 0
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._workspace = {}  # (heads, batch, with scores) -> bytes

    def close(self):
        if getattr(self, "_handle", None):
            self._lib.tq4_paged_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _rows(self, x, name, heads):
        """x [tokens, heads, head_dim] with each token's heads contiguous, copied where they are not; the
        distance of its tokens, and tokens and heads."""
        shape = x.shape if isinstance(x, torch.Tensor) else ()
        if len(shape) != 3 or not (x.dtype is self.dtype and shape[2] == self.head_dim and heads in (None, shape[1])
                                   and x.device == self.device):
            raise ArgumentError(f"paged cache: {name} must be {self.dtype} [tokens, {heads or 'heads'}, {self.head_dim}] "
                                f"on {self.device}")
        tokens, heads, d = shape
        width = heads * d
        if not x.is_contiguous():
            s0, s1, s2 = x.stride()
            if s2 == 1 and (s1 == d or heads == 1) and (s0 >= width or tokens <= 1):
                return x, max(s0, width), tokens, heads
            x = x.contiguous()
        return x, width, tokens, heads

    def append(self, q, k, v, seq, slot, positions=None, rotary=None, out=None):
        """Writes the keys and values of new tokens into the cache (token t is slot ``slot[t]`` of
        sequence ``seq[t]``; seq -1 is padding and nothing of it is touched) and returns their queries,
        both normed and turned by ``rotary`` at ``positions`` (int32 [tokens], or [axes, tokens]; what no
        pair turns is copied bit for bit where there is no norm).
        q [tokens, heads, head_dim], or None when only the cache is filled; k and v [tokens, kv_heads,
        head_dim]; views of a merged projection are read in place. ``out`` may not overlap them."""
        device = self.device
        k, ks, tokens, _ = self._rows(k, "k", self.kv_heads)
        v, vs, values, _ = self._rows(v, "v", self.kv_heads)
        if values != tokens:
            raise ArgumentError(f"paged cache: {values} values for {tokens} keys")
        heads = qs = 0
        q_p = out_p = pos_p = ref = None
        if q is not None:
            q, qs, queries, heads = self._rows(q, "q", None)
            if queries != tokens or heads == 0:
                raise ArgumentError(f"paged cache: {queries} queries of {heads} heads for {tokens} keys")
            q_p = q.data_ptr()
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                out_p = out.data_ptr()
            else:
                out_p = _pointer(out, "out", q.shape, self.dtype, device)
        elif out is not None:
            raise ArgumentError("paged cache: out without q")
        seq_p = _pointer(seq, "seq", (tokens,), torch.int32, device)
        slot_p = _pointer(slot, "slot", (tokens,), torch.int32, device)
        if rotary is not None:
            if rotary.device != device or 2 * rotary.pairs > self.head_dim or not rotary.widths <= {self.head_dim}:
                raise ArgumentError(f"paged cache: the rotary embedding does not fit heads of {self.head_dim} values on {device}")
            ref = rotary._ref
            if rotary.pairs:
                flat = rotary.axes == 1 and isinstance(positions, torch.Tensor) and positions.dim() == 1
                pos_p = _pointer(positions, "positions", (tokens,) if flat else (rotary.axes, tokens), torch.int32, device)
        _lib.check(self._lib.tq4_paged_append(self._handle, q_p, qs, k.data_ptr(), ks, v.data_ptr(), vs, heads, tokens,
                                              seq_p, slot_p, pos_p, ref, out_p, _raw_stream(self._index)))
        return out

    def attention(self, q, lengths, scale=None, window=0, scores=None, new_scores=None, out=None):
        """Attention of one new token of each sequence b < batch over its ``lengths[b]`` slots (int32
        [batch]; the new token's own among them), or the last ``window`` of them: [batch, heads,
        head_dim]. Length 0 gives zeros; ``scale`` is 1 / sqrt(head_dim) by default. Sums are f32; over a
        16-bit cache each softmax weight is rounded once to its type before it multiplies its value.
        ``out`` may not overlap another tensor of the call. With ``scores``
        (f32 [batch, kv_heads, max_pages * page_size]) each slot's softmax weights, summed over the
        query heads of a KV head, are added to them: in place, or into ``new_scores``."""
        device = self.device
        q, qs, batch, heads = self._rows(q, "q", None)
        if heads == 0 or heads % self.kv_heads:
            raise ArgumentError(f"paged cache: {heads} query heads are not a multiple of {self.kv_heads} KV heads")
        if batch > self.max_seqs:
            raise ArgumentError(f"paged cache: {batch} sequences, the page table has {self.max_seqs}")
        len_p = _pointer(lengths, "lengths", (batch,), torch.int32, device)
        in_p = new_p = None
        if scores is not None:
            shape = (batch, self.kv_heads, self.max_slots)
            in_p = _pointer(scores, "scores", shape, torch.float32, device)
            new_p = in_p if new_scores is None else _pointer(new_scores, "new_scores", shape, torch.float32, device)
        elif new_scores is not None:
            raise ArgumentError("paged cache: new_scores without scores")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            out_p = out.data_ptr()
        else:
            out_p = _pointer(out, "out", q.shape, self.dtype, device)
        key = (heads, batch, scores is not None)
        nbytes = self._workspace.get(key)
        if nbytes is None:
            n = ctypes.c_int64()
            _lib.check(self._lib.tq4_paged_attention_workspace(self._handle, heads, batch, int(key[2]), ctypes.byref(n)))
            nbytes = self._workspace[key] = n.value
        # a workspace of its own for each call, from torch's allocator: calls on several streams and
        # captured graphs never share one
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.check(self._lib.tq4_paged_attention(
            self._handle, q.data_ptr(), qs, heads, len_p, batch, self._scale if scale is None else scale, window, in_p, new_p,
            out_p, ws.data_ptr() if nbytes else None, nbytes, _raw_stream(self._index)))
        return out

    def evict(self, lengths, scores, keep, recent, new_table, new_scores=None):
        """Trims every sequence longer than ``keep`` to ``keep`` slots a KV head: the last ``recent``
        and, of those before, the ones with the highest scores (equal scores: the lower slot). What
        stays moves to the pages of ``new_table`` (int32 [batch, new_max_pages], pages that no sequence
        of the call lists). Returns (kept slots int32 [batch, kv_heads, keep], -1 behind the last;
        new lengths int32 [batch]; the kept slots' scores). ``new_scores`` may be given, f32 [batch,
        kv_heads, keep or more]; a new one has 0 behind the kept slots and the width of the new table's
        slots, as ``attention`` over it wants."""
        device = self.device
        batch = lengths.shape[0] if isinstance(lengths, torch.Tensor) and lengths.dim() == 1 else -1
        if not 0 <= batch <= self.max_seqs:
            raise ArgumentError(f"paged cache: lengths must be int32 [batch] of at most {self.max_seqs} sequences")
        pages = new_table.shape[1] if isinstance(new_table, torch.Tensor) and new_table.dim() == 2 else -1
        if not (0 <= recent <= keep and 0 < keep <= pages * self.page_size):
            raise ArgumentError(f"paged cache: recent {recent} of keep {keep} slots, and a new_table [batch, pages] of int32 "
                                f"with room for them on pages of {self.page_size}")
        len_p = _pointer(lengths, "lengths", (batch,), torch.int32, device)
        score_p = _pointer(scores, "scores", (batch, self.kv_heads, self.max_slots), torch.float32, device)
        table_p = _pointer(new_table, "new_table", (batch, pages), torch.int32, device)
        if new_scores is None:
            new_scores = torch.zeros((batch, self.kv_heads, pages * self.page_size), dtype=torch.float32, device=device)
        width = new_scores.shape[2] if isinstance(new_scores, torch.Tensor) and new_scores.dim() == 3 else 0
        new_p = _pointer(new_scores, "new_scores", (batch, self.kv_heads, max(width, keep)), torch.float32, device)
        kept = torch.empty((batch, self.kv_heads, keep), dtype=torch.int32, device=device)
        new_lengths = torch.empty_like(lengths)
        _lib.check(self._lib.tq4_paged_evict(self._handle, len_p, batch, score_p, keep, recent, table_p, pages,
                                             new_lengths.data_ptr(), kept.data_ptr(), new_p, width, _raw_stream(self._index)))
        return kept, new_lengths, new_scores
