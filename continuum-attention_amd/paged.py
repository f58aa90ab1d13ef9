"""Generation over a paged key/value cache: appending new tokens, Continuum
Attention of them over everything cached, eviction by accumulated weight.

A cache holds the keys and values of one layer in pages
``k_pages, v_pages [pages, kv_heads, page_size, head_dim]`` (any strides with
contiguous rows).  ``page_table [B, pages per sequence]`` names a sequence's
pages in order, ``lengths [B]`` counts its cached slots with the new tokens, and
``starts [B + 1]`` delimits its new tokens among the token tensors' rows, all
32-bit integers on the device and read there, so a captured graph replays with
whatever they hold then.  Token rows behind ``starts[B]`` belong to no sequence:
the kernels leave their outputs as they were.

The training operator's contract holds: a token at slot p sees slots 0..p with
the weights that ``continuum_attention`` gives it over the same keys.  These
entry points are for inference and have no backward pass.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _native
from . import cpu as _cpu
from .ops import _clear_hooks
from .rotary import _DTYPES, _argument, _positions, _rows, _turn_cpu


def _require(cond, message):
    if not cond:
        raise ValueError(message)


def _refuse_grad(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no backward pass; call it under torch.no_grad()")


def _on_gpu(t):
    return isinstance(t, torch.Tensor) and t.is_cuda and not torch.compiler.is_compiling()


def _int32(name, t, shape, device):
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32, f"{name} must be a tensor of 32-bit integers")
    _require(t.dim() == len(shape) and all(s is None or s == n for s, n in zip(shape, t.shape)),
             f"{name} has shape {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on the device of the cache")
    _require(t.numel() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1, f"{name} must be contiguous")


def _cache(k_pages, v_pages, page_table, lengths, starts, tokens):
    """The C description of a cache, its tensors checked."""
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        _require(isinstance(t, torch.Tensor) and t.dim() == 4, f"{name} must be [pages, heads, page_size, head_dim]")
    _require(k_pages.dtype in _DTYPES, f"unsupported cache dtype {k_pages.dtype}")
    _require(k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype
             and k_pages.stride() == v_pages.stride(), "k_pages and v_pages must share shape, dtype and strides")
    dev = k_pages.device
    if v_pages.device != dev:
        raise RuntimeError("k_pages and v_pages must be on one device")
    _require(not (k_pages.is_neg() or v_pages.is_neg()), "pages must not be views of negated values")
    pages, heads, page_size, D = k_pages.shape
    _require(min(pages, heads, page_size, D) > 0, f"empty cache {tuple(k_pages.shape)}")
    _require(k_pages.stride(-1) == 1, "cache rows must be contiguous")
    _int32("page_table", page_table, (None, None), dev)
    B = page_table.shape[0]
    _require(B > 0 and page_table.shape[1] > 0, "page_table must not be empty")
    _int32("lengths", lengths, (B,), dev)
    c = _native.PagedCache()
    c.k, c.v = k_pages.data_ptr(), v_pages.data_ptr()
    c.page_stride, c.head_stride, c.row_stride, _ = k_pages.stride()
    c.table, c.table_stride = page_table.data_ptr(), max(page_table.stride(0), page_table.shape[1])
    _require(B == 1 or page_table.stride(0) >= page_table.shape[1], "page_table rows must not overlap")
    c.lengths = lengths.data_ptr()
    if starts is not None:
        _int32("starts", starts, (B + 1,), dev)
        c.starts = starts.data_ptr()
    c.dtype, c.heads, c.head_dim, c.page_size, c.num_pages = _DTYPES[k_pages.dtype], heads, D, page_size, pages
    c.pages_per_seq, c.batch, c.tokens = page_table.shape[1], B, tokens
    return c


def _disjoint(t):
    """No two elements in one place (as far as nested strides show it)."""
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < span:
            return False
        span += stride * (size - 1)
    return True


def _gpu(name, dev):
    if dev.type != "cuda":
        raise RuntimeError(f"{name} runs on ROCm GPU and CPU tensors; got one on {dev}")


def _spans(page_table, lengths, starts, page_size, tokens):
    """Host view of the sequences for the CPU path: (length, first, count)."""
    room = page_table.shape[1] * page_size
    out = []
    for b in range(page_table.shape[0]):
        t0 = min(max(int(starts[b]), 0), tokens)
        t1 = min(max(int(starts[b + 1]), t0), tokens)
        out.append((min(max(int(lengths[b]), 0), room), t0, t1 - t0))
    return out


def _row_ids(table, page_size, slots, num_pages):
    """(page, row) of slots and whether the page is one of the cache's."""
    pages = table[torch.div(slots, page_size, rounding_mode="floor")].long()
    good = (pages >= 0) & (pages < num_pages)
    return pages.clamp(0, num_pages - 1), slots % page_size, good


def rotary_append(q, k, v, positions, rotary, k_pages, v_pages, page_table, lengths, starts, max_new=None,
                  out=None):
    """Rotates new tokens and writes them to the cache: k, turned to its
    positions, and v go to slots ``lengths[b] - n_b ..`` of their sequence
    (``n_b = starts[b + 1] - starts[b]``), and q, turned, is returned.

    q ``[tokens, heads, D]``, k and v ``[tokens, kv_heads, D]`` of the cache's
    dtype, positions ``[tokens]`` integers (they need not be the slots, and after
    an eviction are not).  One launch.  Two new tokens must not share a slot.
    Slots without a page of the cache are not written.  ``out`` (no other
    argument's memory) receives q;
    without it rows that belong to no sequence are undefined.  ``max_new`` is
    accepted for symmetry with paged_attention and not needed."""
    # the plain case runs in native code (csrc/ca_torch.cpp); what it does not take is checked here
    if _on_gpu(q) and q.shape[-1] == rotary.head_dim:
        y = _native.torch_ext().append(q, k, v, positions, rotary.turns, rotary.magnitude, rotary.layout == "half",
                                       rotary.rotary_dim, k_pages, v_pages, page_table, lengths, starts, out)
        if y is not None:
            return y
    _refuse_grad("rotary_append", q, k, v, k_pages, v_pages)
    q3, k3 = _rows("q", q, rotary), _rows("k", k, rotary, q)
    v3 = _rows("v", v, rotary, q)
    _require(starts is not None, "starts must be given")
    _require(q.dim() == 3 and k.dim() == 3, "q, k and v must be [tokens, heads, head_dim]")
    _require(v.shape == k.shape, "k and v must share their shape")
    N = q.shape[0]
    c = _cache(k_pages, v_pages, page_table, lengths, starts, N)
    _require(q.dtype == k_pages.dtype, f"q is {q.dtype}, the cache {k_pages.dtype}")
    _require((c.heads, c.head_dim) == tuple(k.shape[1:]), "the cache's heads and head dim differ from k's")
    _require(_disjoint(k_pages) and k_pages.data_ptr() != v_pages.data_ptr(),
             "k_pages and v_pages must be apart, and their rows too")
    if q.device != k_pages.device:
        raise RuntimeError("q must be on the device of the cache")
    p = _positions(positions, q.shape[:1], q.device)
    if out is None:
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    else:
        _check_out(out, q)
    if N == 0:
        return out
    if q.device.type == "cpu":
        kr = _turn_cpu(k3, p, rotary)
        qr = _turn_cpu(q3, p, rotary)
        for b, (length, t0, n) in enumerate(_spans(page_table, lengths, starts, c.page_size, N)):
            slots = torch.arange(length - n, length)
            seen = slots >= 0
            pages, rows, good = _row_ids(page_table[b], c.page_size, slots.clamp(min=0), c.num_pages)
            good = good & seen
            tok = torch.arange(t0, t0 + n)[good]
            k_pages[pages[good], :, rows[good]] = kr[tok]
            v_pages[pages[good], :, rows[good]] = v3[tok]
            out[t0:t0 + n] = qr[t0:t0 + n]
        return out
    _gpu("rotary_append", q.device)
    r = _argument(q3, k3, out, None, p, rotary, False)
    with _native.on_device(q.device):
        _native.check(_native.load().ca_rotary_append(ctypes.byref(r), v3.data_ptr(), v3.stride(0), v3.stride(1),
                                                      ctypes.byref(c), _native.stream_handle(q.device)))
    return out


def _check_out(out, q):
    _require(isinstance(out, torch.Tensor) and out.shape == q.shape and out.dtype == q.dtype,
             "out must have q's shape and dtype")
    if out.device != q.device:
        raise RuntimeError("out must be on the device of q")
    _require(out.numel() == 0 or (out.stride(-1) == 1 and _disjoint(out)) and not out.is_neg(),
             "out rows must be contiguous and apart")
    if torch.is_grad_enabled() and out.requires_grad:
        raise RuntimeError("out must not require grad")
    _require(out.numel() == 0 or out.untyped_storage().data_ptr() != q.untyped_storage().data_ptr(),
             "out must not share memory with q")


@functools.lru_cache(maxsize=256)
def _workspace_bytes(*args):
    return int(_native.load().ca_paged_attention_workspace_bytes(*args))


_clear_hooks.append(_workspace_bytes.cache_clear)


def paged_attention(q, k_pages, v_pages, page_table, lengths, starts, log_gain, max_new=None,
                    max_length=None, weight_sums=None, out=None):
    """Continuum Attention of each sequence's new tokens over its paged cache,
    ``[tokens, heads, head_dim]`` in q's dtype (the cache's: fp32, bf16, fp16).

    q ``[tokens, heads, head_dim]`` with heads a multiple of the cache's (query
    head i reads key head ``i // (heads // kv_heads)``); log_gain ``[heads]``;
    head_dim a multiple of 8 up to 128.  The new tokens' keys and values are in
    the cache already (rotary_append).  ``max_new`` and ``max_length``, the most
    new tokens and the longest cached length to expect (default: all of q, the
    whole page table), size the grid and the workspace: results do not depend on
    them but for the order of sums, times do.  ``weight_sums`` (fp32 ``[B,
    kv_heads, slots]``) is added to: the weights each slot got from the new
    tokens, over the query heads of its key head, which evict ranks by.

    A token that sees no slot gets zeros; one that reads a page number outside
    the cache gets NaN.  Of keys and values that are not finite, those a token does
    not see change nothing in its row; from those it sees the row may get
    NaN where the formula has an infinity.  ``out`` (no other argument's memory)
    receives the result; without it rows that belong to no sequence are
    undefined."""
    if _on_gpu(q):  # as in rotary_append
        y = _native.torch_ext().attend(q, k_pages, v_pages, page_table, lengths, starts, log_gain,
                                       -1 if max_new is None else int(max_new),
                                       -1 if max_length is None else int(max_length),
                                       weight_sums, out)
        if y is not None:
            return y
    _refuse_grad("paged_attention", q, k_pages, v_pages, log_gain)
    _require(isinstance(q, torch.Tensor) and q.dim() == 3, "q must be [tokens, heads, head_dim]")
    N, H, D = q.shape
    c = _cache(k_pages, v_pages, page_table, lengths, starts, N)
    _require(starts is not None, "starts must be given")
    _require(q.dtype == k_pages.dtype, f"q is {q.dtype}, the cache {k_pages.dtype}")
    _require(D == c.head_dim and D % 8 == 0 and D <= 128,
             f"head dim {D} (the cache's {c.head_dim}; multiples of 8 up to 128)")
    _require(H > 0 and H % c.heads == 0, f"{H} query heads over {c.heads} key heads")
    _require(isinstance(log_gain, torch.Tensor) and log_gain.numel() == H, f"log_gain must have {H} entries")
    dev = q.device
    if dev != k_pages.device or log_gain.device != dev:
        raise RuntimeError("q, log_gain and the cache must be on one device")
    max_new = N if max_new is None else int(max_new)
    capacity = c.pages_per_seq * c.page_size
    max_length = capacity if max_length is None else int(max_length)
    _require(max_new >= 0 and max_length >= 0, "max_new and max_length must not be negative")
    if weight_sums is not None:
        _require(isinstance(weight_sums, torch.Tensor) and weight_sums.dtype == torch.float32
                 and weight_sums.dim() == 3 and weight_sums.shape[:2] == (c.batch, c.heads),
                 f"weight_sums must be fp32 [{c.batch}, {c.heads}, slots]")
        _require(weight_sums.numel() == 0 or weight_sums.stride(2) == 1 or weight_sums.shape[2] == 1,
                 "weight_sums rows must be contiguous")
        _require(_disjoint(weight_sums), "weight_sums rows must be apart")
        _require(not weight_sums.requires_grad or not torch.is_grad_enabled(), "weight_sums must not require grad")
        if weight_sums.device != dev:
            raise RuntimeError("weight_sums must be on the device of q")
    if out is None:
        out = torch.empty(q.shape, device=dev, dtype=q.dtype)
    else:
        _check_out(out, q)
    if N == 0:
        return out
    if dev.type == "cpu":
        _attention_cpu(q, k_pages, v_pages, page_table, lengths, starts, log_gain, weight_sums, out)
        return out
    _gpu("paged_attention", dev)
    q = q.detach().resolve_neg()
    esize = q.element_size()
    if q.stride(2) != 1 or q.data_ptr() % 16 or q.stride(0) * esize % 16 or q.stride(1) * esize % 16:
        q = q.contiguous() if not q.is_contiguous() else q.clone()
    g = log_gain.detach().resolve_neg()
    if g.dtype != torch.float32 or not g.is_contiguous():
        g = g.float().contiguous()
    sums = weight_sums if weight_sums is not None and weight_sums.numel() else None
    max_length = min(max_length, capacity)
    nbytes = _workspace_bytes(c.dtype, c.batch, c.heads, H, D, N, max_new, max_length, int(sums is not None))
    ws = torch.empty(max(nbytes, 1), device=dev, dtype=torch.uint8)
    with _native.on_device(dev):
        _native.check(_native.load().ca_paged_attention(
            ctypes.byref(c), q.data_ptr(), q.stride(0), q.stride(1), H, g.data_ptr(), out.data_ptr(),
            out.stride(0), out.stride(1), sums.data_ptr() if sums is not None else None,
            sums.stride(0) if sums is not None else 0, sums.stride(1) if sums is not None else 0,
            sums.shape[2] if sums is not None else 0, max_new, max_length, ws.data_ptr(), nbytes,
            _native.stream_handle(dev)))
    return out


def _attention_cpu(q, k_pages, v_pages, page_table, lengths, starts, log_gain, sums, out):
    N, H, D = q.shape
    num_pages, heads, page_size, _ = k_pages.shape
    group = H // heads
    scale = (torch.exp(log_gain.detach().reshape(H).float()) * D ** -0.5).view(heads, group, 1, 1)
    for b, (length, t0, n) in enumerate(_spans(page_table, lengths, starts, page_size, N)):
        blind = max(0, n - length)  # tokens before slot 0 see nothing
        out[t0:t0 + blind] = 0
        if n == blind:
            continue
        pages, rows, good = _row_ids(page_table[b], page_size, torch.arange(length), num_pages)
        k, v = (torch.where(good[:, None, None], p[pages, :, rows].float(), math.nan).transpose(0, 1)
                for p in (k_pages, v_pages))
        first = length - n + blind
        for t in range(t0 + blind, t0 + n):
            seen = first + (t - t0 - blind) + 1
            s = (q[t].detach().float().view(heads, group, 1, D) * scale) @ k[:, None, :seen].transpose(2, 3)
            w = _cpu.tile_weights(s.reshape(heads * group, 1, seen), seen - 1).view(heads, group, seen)
            out[t] = (w @ v[:, :seen]).reshape(H, D).to(out.dtype)
            if sums is not None:
                m = min(seen, sums.shape[2])
                sums[b, :, :m] += w.sum(1)[:, :m]


def evict(k_pages, v_pages, page_table, lengths, weight_sums, new_table, budget, sinks=0, recent=0):
    """Cuts every sequence's cache to ``budget`` slots: of each key head the first
    ``sinks``, the last ``recent`` and, of those between, the slots with the
    largest ``weight_sums`` (``[B, kv_heads, slots]`` fp32; of equal ones the first;
    NaN counts as the largest).  Shorter sequences are kept whole; slots that
    ``weight_sums`` does not reach are not kept.

    The kept rows are copied, in their order, to slots 0, 1, ... of the pages that
    ``new_table [B, new pages per sequence]`` names in the same cache; these must be
    pages that no sequence's table names and that occur once.  The old pages are
    left as they were.  Returns ``(kept, new_lengths, new_sums)``: the kept
    slots' former numbers ``[B, kv_heads, budget]`` int32 (-1 behind the last),
    the new lengths ``[B]`` int32 and the kept slots' sums (0 behind the last)."""
    if _on_gpu(k_pages):  # as in rotary_append
        y = _native.torch_ext().evict(k_pages, v_pages, page_table, lengths, weight_sums, new_table, int(budget),
                                      int(sinks), int(recent))
        if y is not None:
            return y
    _refuse_grad("evict", k_pages, v_pages, weight_sums)
    c = _cache(k_pages, v_pages, page_table, lengths, None, 0)
    dev = k_pages.device
    _require(c.head_dim % 8 == 0 and c.head_dim <= 128, f"head dim {c.head_dim} (multiples of 8 up to 128)")
    _require(isinstance(weight_sums, torch.Tensor) and weight_sums.dtype == torch.float32 and weight_sums.dim() == 3
             and weight_sums.shape[:2] == (c.batch, c.heads), f"weight_sums must be fp32 [{c.batch}, {c.heads}, slots]")
    if weight_sums.device != dev:
        raise RuntimeError("weight_sums must be on the device of the cache")
    _require(_disjoint(k_pages), "the cache's rows must be apart")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    _require(budget > 0 and sinks >= 0 and recent >= 0 and sinks + recent <= budget,
             f"budget {budget} must be positive and hold {sinks} sinks and {recent} recent slots")
    _int32("new_table", new_table, (c.batch, None), dev)
    _require(c.batch == 1 or new_table.stride(0) >= new_table.shape[1], "new_table rows must not overlap")
    _require(new_table.shape[1] * c.page_size >= budget,
             f"{new_table.shape[1]} new pages of {c.page_size} slots do not hold {budget}")
    s = weight_sums.detach().resolve_neg()
    if s.shape[2] > 1 and s.stride(2) != 1:
        s = s.contiguous()
    kept = torch.empty(c.batch, c.heads, budget, device=dev, dtype=torch.int32)
    sums = torch.empty(c.batch, c.heads, budget, device=dev, dtype=torch.float32)
    new_lengths = torch.empty(c.batch, device=dev, dtype=torch.int32)
    if dev.type == "cpu":
        _evict_cpu(k_pages, v_pages, page_table, lengths, s, new_table, budget, sinks, recent, kept, sums, new_lengths)
        return kept, new_lengths, sums
    _gpu("evict", dev)
    with _native.on_device(dev):
        _native.check(_native.load().ca_evict(
            ctypes.byref(c), s.data_ptr() if s.numel() else kept.data_ptr(), s.stride(0), s.stride(1), s.shape[2],
            budget, sinks, recent, new_table.data_ptr(), max(new_table.stride(0), new_table.shape[1]),
            kept.data_ptr(), sums.data_ptr(), new_lengths.data_ptr(), _native.stream_handle(dev)))
    return kept, new_lengths, sums


def _evict_cpu(k_pages, v_pages, table, lengths, sums, new_table, budget, sinks, recent, kept, new_sums, new_lengths):
    num_pages, heads, page_size, _ = k_pages.shape
    kept.fill_(-1)
    new_sums.zero_()
    for b in range(table.shape[0]):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page_size, sums.shape[2])
        m = min(n, budget)
        new_lengths[b] = m
        if m == 0:
            continue
        if n <= budget:
            idx = torch.arange(n).expand(heads, n)
        else:
            between = sums[b, :, sinks:n - recent]
            order = torch.sort(between, dim=-1, descending=True, stable=True).indices[:, :budget - sinks - recent] + sinks
            ends = torch.cat((torch.arange(sinks), torch.arange(n - recent, n))).expand(heads, -1)
            idx = torch.sort(torch.cat((order, ends), 1), -1).values
        kept[b, :, :m] = idx.to(torch.int32)
        new_sums[b, :, :m] = sums[b].gather(1, idx)
        to, to_rows, to_good = _row_ids(new_table[b], page_size, torch.arange(m), num_pages)
        for h in range(heads):
            src, rows, good = _row_ids(table[b], page_size, idx[h], num_pages)
            for pages in (k_pages, v_pages):
                x = torch.where(good[:, None], pages[src, h, rows], math.nan)
                pages[to[to_good], h, to_rows[to_good]] = x[to_good].to(pages.dtype)


class PagedCache:
    """Keys and values of a decoder's layers in pages, with the tables and
    counts that rotary_append, paged_attention and evict read.

    ``pages`` pages of ``page_size`` slots per layer serve ``batch`` sequences of at
    most ``max_length`` slots; all layers share one page table.  ``weight_sums``
    keeps each slot's accumulated attention weight (for evict)."""

    def __init__(self, layers, batch, kv_heads, head_dim, max_length, pages=None, page_size=64,
                 dtype=torch.bfloat16, device="cuda", weight_sums=False):
        _require(min(layers, batch, kv_heads, head_dim, max_length, page_size) > 0, "sizes must be positive")
        _require(dtype in _DTYPES, f"unsupported cache dtype {dtype}")
        self.page_size, self.batch = int(page_size), int(batch)
        self.pages_per_seq = -(-int(max_length) // self.page_size)
        self.max_length = self.pages_per_seq * self.page_size
        self.pages = self.batch * self.pages_per_seq if pages is None else int(pages)
        shape = (layers, 2, self.pages, kv_heads, self.page_size, head_dim)
        self.data = torch.zeros(shape, dtype=dtype, device=device)
        self.device = self.data.device
        self.weight_sums = (torch.zeros(layers, batch, kv_heads, self.max_length, device=device)
                            if weight_sums else None)
        self.table = torch.zeros(batch, self.pages_per_seq, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.starts = torch.zeros(batch + 1, dtype=torch.int32, device=device)
        self.positions = torch.zeros(0, dtype=torch.int64, device=device)
        self.free = list(range(self.pages - 1, -1, -1))
        self.owned = [[] for _ in range(batch)]  # pages of each sequence
        self.counts = [0] * batch                # cached slots
        self.next = [0] * batch                  # next token's position
        self.max_new = 0

    def k(self, layer):
        return self.data[layer, 0]

    def v(self, layer):
        return self.data[layer, 1]

    def _take(self, need):
        return [self.free.pop() for _ in range(need)]

    def _upload(self):
        rows = [o + [0] * (self.pages_per_seq - len(o)) for o in self.owned]
        self.table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.lengths.copy_(torch.tensor(self.counts, dtype=torch.int32))

    def extend(self, new):
        """Makes room for ``new[b]`` new tokens of every sequence b and sets
        lengths, starts and positions for the pass that brings them."""
        new = [int(n) for n in new]
        _require(len(new) == self.batch and min(new) >= 0, f"new must hold {self.batch} counts")
        for b, n in enumerate(new):
            _require(self.counts[b] + n <= self.max_length,
                     f"sequence {b}: {self.counts[b]} + {n} slots exceed {self.max_length}")
        need = [max(0, -(-(c + n) // self.page_size) - len(o)) for c, n, o in zip(self.counts, new, self.owned)]
        if sum(need) > len(self.free):
            raise RuntimeError(f"the cache is out of pages: {sum(need)} needed, {len(self.free)} free")
        starts, positions = [0], []
        for b, n in enumerate(new):
            self.owned[b] += self._take(need[b])
            positions += range(self.next[b], self.next[b] + n)
            self.counts[b] += n
            self.next[b] += n
            starts.append(starts[-1] + n)
        self._upload()
        self.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        self.positions = torch.tensor(positions, dtype=torch.int64).to(self.device)
        self.max_new = max(new)

    def evict(self, budget, sinks=0, recent=0):
        """Cuts every layer's cache to ``budget`` slots per sequence (see evict)
        and frees the pages no longer needed.  Positions go on counting."""
        _require(self.weight_sums is not None, "the cache was made without weight_sums")
        if max(self.counts) <= budget:
            return
        # every sequence moves, also those within the budget
        need = [-(-min(c, budget) // self.page_size) for c in self.counts]
        if sum(need) > len(self.free):
            raise RuntimeError(f"the cache has no free pages to evict into: {sum(need)} needed, {len(self.free)} free")
        new = [self._take(n) for n in need]
        width = -(-budget // self.page_size)
        table = torch.tensor([n + [-1] * (width - len(n)) for n in new], dtype=torch.int32).to(self.device)
        for layer in range(self.data.shape[0]):
            _, _, sums = evict(self.k(layer), self.v(layer), self.table, self.lengths, self.weight_sums[layer],
                               table, budget, sinks, recent)
            self.weight_sums[layer].zero_()
            self.weight_sums[layer, :, :, :budget] = sums[:, :, :self.max_length]
        for b, n in enumerate(new):
            self.free += reversed(self.owned[b])
            self.owned[b] = n
            self.counts[b] = min(self.counts[b], budget)
        self._upload()

    def release(self, b):
        """Frees sequence b's pages; it starts anew at position 0."""
        self.free += reversed(self.owned[b])
        self.owned[b], self.counts[b], self.next[b] = [], 0, 0
        if self.weight_sums is not None:
            self.weight_sums[:, b].zero_()
        self._upload()
