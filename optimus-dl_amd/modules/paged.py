"""A cache of keys and values in pages, and the two steps of a decoder that work on it: what goes into it, and attention over it.

A sequence's tokens lie in pages of a fixed number of tokens, anywhere in the cache; a table says which.  A step brings some new tokens of each of
several sequences, one behind the other: single tokens of a decode step, drafted tokens that are to be verified, chunks of prompts, or all of
them at once.  The reference runs whole sequences through PyTorch's attention and keeps nothing (optimus_dl/modules/model/blocks/attention.py:128-170).

For inference: inputs that want gradients are refused.
"""

from __future__ import annotations

from itertools import accumulate
from typing import NamedTuple

import torch

from .. import native
from .calls import untraced, untransformed

E4M3_MAX = 448.0


def _refuse_gradients(what: str, *tensors: "torch.Tensor | None") -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} is for inference; an input wants a gradient (torch.no_grad() around the call, or detach it)")


def refuse_transforms(what: str) -> None:
    if not untransformed():
        raise native.NativeError(f"{what} on the GPU is a call that torch does not see into: no forward-mode derivative, functorch rule or trace of it")


def _check(what: str, q, keys, values, pages, offsets, lengths, key_scale, value_scale) -> None:
    if keys.dim() != 4 or not (keys.shape[1] and keys.shape[3]) or values.shape != keys.shape or values.dtype != keys.dtype:
        raise ValueError(f"{what}: keys {keys.dtype} {tuple(keys.shape)} and values {values.dtype} {tuple(values.shape)}, expected [pages, kv heads, page size, "
                         "head_dim] of one type")
    if q.dim() != 3 or q.shape[2] != keys.shape[3] or q.shape[1] % keys.shape[1]:
        raise ValueError(f"{what}: q {tuple(q.shape)} for a cache of {keys.shape[1]} heads of {keys.shape[3]}, expected [rows, a multiple of the heads, head_dim]")
    if any(t.dtype != torch.int32 for t in (pages, offsets, lengths)) or pages.dim() != 2 or lengths.shape != pages.shape[:1] or offsets.shape != (lengths.numel() + 1,):
        raise ValueError(f"{what}: pages {pages.dtype} {tuple(pages.shape)}, offsets {offsets.dtype} {tuple(offsets.shape)} and lengths {lengths.dtype} "
                         f"{tuple(lengths.shape)}, expected int32 [sequences, width], [sequences + 1], [sequences]")
    if keys.shape[2] < 1 or keys.shape[2] & (keys.shape[2] - 1):
        raise ValueError(f"{what}: pages of {keys.shape[2]} tokens (a power of two)")
    for scale in (key_scale, value_scale):
        if (keys.dtype == torch.float8_e4m3fn) != (scale is not None) or (scale is not None and scale.shape != (keys.shape[1],)):
            raise ValueError(f"{what}: a float8_e4m3fn cache has a scale for each of {keys.shape[1]} heads of keys and of values, others have none")


def _sequences(offsets, lengths, rows: int):
    """(first row, new tokens, position of the first) of every sequence, on the CPU."""
    at = offsets.tolist()
    for s, length in enumerate(lengths.tolist()):
        first = min(max(at[s], 0), rows)
        n = max(min(at[s + 1], rows) - first, 0)
        yield s, first, n, length - n


def _slots(pages_row, position, n_pages: int, page_size: int):
    """Page and place in it of every position; which of them there are."""
    inside = (position >= 0) & (position < pages_row.numel() * page_size)
    at = torch.where(inside, position, torch.zeros_like(position))
    page = pages_row.long()[at // page_size] if pages_row.numel() else torch.full_like(at, -1)
    held = inside & (page >= 0) & (page < n_pages)
    return torch.where(held, page, torch.zeros_like(page)), at % page_size, held


def _append_plain(q, k, v, keys, values, pages, offsets, lengths, cos, sin, interleaved, q_weight, k_weight, eps, key_scale, value_scale):
    wide = torch.promote_types(q.dtype, torch.float32)
    out = torch.zeros(q.shape, dtype=q.dtype)

    def turned(x, weight, position):
        x = x.to(wide)
        if weight is not None:
            x = x * (1.0 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()).to(wide) * weight.to(wide)
        if cos is None:
            return x
        c, s = cos[position].to(wide).unsqueeze(1), sin[position].to(wide).unsqueeze(1)
        half = c.shape[-1]
        a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
        a, b = a * c - b * s, a * s + b * c
        return torch.cat((torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1), x[..., 2 * half:]), -1)

    for s, first, n, before in _sequences(offsets, lengths, q.shape[0]):
        position = torch.arange(before, before + n)
        inside = (position >= 0) & (position < pages.shape[1] * keys.shape[2])
        rows, position = torch.arange(first, first + n)[inside], position[inside]
        page, slot, held = _slots(pages[s], position, keys.shape[0], keys.shape[2])
        out[rows] = turned(q[rows], q_weight, position).to(q.dtype)
        for cache, x, scale in ((keys, turned(k[rows], k_weight, position), key_scale), (values, v[rows].to(wide), value_scale)):
            if scale is not None:
                scale = scale.view(1, -1, 1)
                x = torch.where(scale == 0, torch.where(x.isnan(), x, torch.zeros_like(x)), (x / scale).clamp(-E4M3_MAX, E4M3_MAX))
            x = x.to(cache.dtype)
            bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[cache.element_size()]
            cache.view(bits)[page[held], :, slot[held]] = x.view(bits)[held]
    return out


def _attention_plain(q, keys, values, pages, offsets, lengths, scale, window, softcap, key_scale, value_scale):
    wide = torch.promote_types(q.dtype, torch.float32)
    out = torch.zeros(q.shape, dtype=q.dtype)
    group, size = q.shape[1] // keys.shape[1], keys.shape[2]
    for s, first, n, before in _sequences(offsets, lengths, q.shape[0]):
        if n == 0:
            continue
        place = torch.arange(min(max(before + n, 0), pages.shape[1] * size))
        page, slot, held = _slots(pages[s], place, keys.shape[0], size)

        def read(cache, scale):
            x = cache.to(wide)[page, :, slot]                                # [positions, kv heads, head_dim]
            x = x if scale is None else x * scale.to(wide).view(1, -1, 1)
            return x.repeat_interleave(group, dim=1).transpose(0, 1)

        score = torch.matmul(q[first:first + n].to(wide).transpose(0, 1), read(keys, key_scale).transpose(1, 2)) * scale
        if softcap:
            score = softcap * torch.tanh(score / softcap)
        position = torch.arange(before, before + n).unsqueeze(1)
        seen = (place <= position) & held
        if window:
            seen = seen & (place > position - window)
        score = score.masked_fill(~seen, float("-inf"))
        some = (score != float("-inf")).any(-1, keepdim=True)
        weight = torch.where(some, torch.softmax(score, -1), torch.zeros_like(score))
        v = read(values, value_scale).unsqueeze(1)                           # (an unseen value does not reach a row, not even a NaN)
        odd = ~v.isfinite()
        y = torch.matmul(weight.unsqueeze(2), torch.where(odd, torch.zeros_like(v), v)).squeeze(2)
        if odd.any():
            y = y + torch.where(odd & seen.view(1, *seen.shape, 1) & some.unsqueeze(2), v, torch.zeros_like(v)).sum(2)
        out[first:first + n] = y.transpose(0, 1).to(q.dtype)
    return out


@untraced
def append_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor,
              lengths: torch.Tensor, *, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, interleaved: bool = True,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6, key_scale: torch.Tensor | None = None,
              value_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Puts the keys and values of new tokens into a paged cache, with the norm and the rotation of queries and keys on the way.  -> the queries.

    q [rows, heads, head_dim], k and v [rows, kv heads, head_dim]: the new tokens of sequence s are rows ``offsets[s]`` to ``offsets[s + 1]``.  keys, values
    [pages, kv heads, page size, head_dim]: the cache, bf16, or float8_e4m3fn with ``key_scale`` and ``value_scale`` [kv heads] (fp32; a code stands for
    code * scale, larger values are clamped, and all are 0 where the scale is).  lengths: tokens of each sequence in the cache, with the new ones; position p of sequence s is in slot
    ``p % page size`` of page ``pages[s, p // page size]``.  pages, offsets, lengths int32.

    cos, sin: fp32 [positions, pairs], of every position that the table reaches; the first 2 * pairs elements of a head are rotated, as pairs (2 i, 2 i + 1)
    where ``interleaved``, else (i, pairs + i).  q_weight, k_weight [head_dim]: norms by root mean square in front of the rotation, in fp32 or bf16 without a cast.
    Rows of no sequence, in front of the first or behind the last, are not read: their queries are 0.  Tokens whose page is none of the cache are not written, those behind the
    table's reach neither, and their queries are 0.  Two rows of a call must not share a slot.

    bf16 on the GPU, one kernel, in head dimensions of 16 to 128 (a multiple of 16).  CPU tensors run as torch operations, in any floating type."""
    if q.is_cuda and untransformed():
        out = native.plain_append_kv(q, k, v, keys, values, pages, offsets, lengths, cos, sin, interleaved, q_weight, k_weight, eps, key_scale, value_scale)
        if out is not None:
            return out
    _check("append_kv", q, keys, values, pages, offsets, lengths, key_scale, value_scale)
    if k.shape != v.shape or k.shape != (q.shape[0], keys.shape[1], keys.shape[3]) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"append_kv: k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} beside q {q.dtype} {tuple(q.shape)}, expected "
                         f"[{q.shape[0]}, {keys.shape[1]}, {keys.shape[3]}]")
    if (cos is None) != (sin is None) or (cos is not None and (cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > q.shape[2]
                                                              or cos.shape[0] < pages.shape[1] * keys.shape[2])):
        raise ValueError(f"append_kv: cos and sin of {pages.shape[1] * keys.shape[2]} positions, [positions, up to {q.shape[2] // 2}] of both")
    for weight in (q_weight, k_weight):
        if weight is not None and weight.shape != q.shape[2:]:
            raise ValueError(f"append_kv: norms of heads have {q.shape[2]} weights")
    _refuse_gradients("append_kv", q, k, v, keys, values, q_weight, k_weight, cos, sin)
    if not q.is_cuda:
        return _append_plain(q, k, v, keys, values, pages, offsets, lengths, cos, sin, interleaved, q_weight, k_weight, eps, key_scale, value_scale)
    refuse_transforms("append_kv")
    return native.append_kv(q, k, v, keys, values, pages, offsets, lengths, cos, sin, interleaved, q_weight, k_weight, eps, key_scale, value_scale)


@untraced
def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, pages: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor, *,
                    max_new: int | None = None, scale: float | None = None, window: int = 0, softcap: float = 0.0,
                    key_scale: torch.Tensor | None = None, value_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over a paged cache that holds them (see :func:`append_kv` for both).  -> [rows, heads, head_dim].

    A token at position p sees positions ``max(0, p - window + 1)`` to p (window 0: from 0).  Scores are ``scale * q . key`` (1 / sqrt(head_dim) by
    default), and ``softcap * tanh(score / softcap)`` where softcap is not 0.  Heads in groups share a head of the cache.
    max_new: the most new tokens of a sequence, where the program knows it: it chooses kernels, results hold without.
    Keys and values that a token does not see do not reach it, NaN and infinities included.  A token that sees nothing, or
    no score above -inf, and rows of no sequence answer 0.

    bf16 on the GPU: one kernel for up to 32 rows (tokens times heads of a group) a sequence, another for more, and one that joins parts; sums and maxima
    in fp32, weights rounded to bf16.  The same call answers the same bits.  CPU tensors run as torch operations, in any floating type."""
    scale = q.shape[-1] ** -0.5 if scale is None and q.dim() and q.shape[-1] else scale
    if q.is_cuda and untransformed() and scale is not None:
        out = native.plain_paged_attention(q, keys, values, pages, offsets, lengths, max_new, scale, window, softcap, key_scale, value_scale)
        if out is not None:
            return out
    _check("paged_attention", q, keys, values, pages, offsets, lengths, key_scale, value_scale)
    if not 0.0 < scale <= 1e30 or window < 0 or not (softcap == 0.0 or 1e-3 <= softcap <= 1e6) or (max_new is not None and max_new < 0):
        raise ValueError(f"paged_attention: scale {scale} (above 0, up to 1e30), window {window} (0 or more), softcap {softcap} (0, or 1e-3 to 1e6), max_new {max_new}")
    _refuse_gradients("paged_attention", q, keys, values)
    if not q.is_cuda:
        return _attention_plain(q, keys, values, pages, offsets, lengths, scale, window, softcap, key_scale, value_scale)
    refuse_transforms("paged_attention")
    return native.paged_attention(q, keys, values, pages, offsets, lengths, max_new, scale, window, softcap, key_scale, value_scale)


class PagedBatch(NamedTuple):
    """The new tokens of a step: what :func:`append_kv` and :func:`paged_attention` are told of them.  ``max_new``: the most of a sequence, None where the
    program does not know (a captured step whose tensors change)."""

    pages: torch.Tensor
    offsets: torch.Tensor
    lengths: torch.Tensor
    max_new: int | None = None

    def positions(self, rows: int) -> torch.Tensor:
        """The position of every row's token, 0 for rows behind the last sequence."""
        row, offsets = torch.arange(rows, device=self.offsets.device), self.offsets.long()
        first = torch.nn.functional.pad(self.lengths - offsets[1:], (0, 1), value=-rows)         # position 0's row, negative; none behind the last sequence
        return first[torch.searchsorted(offsets[1:], row, right=True)].add_(row).clamp_(min=0)


class PagedLayer(NamedTuple):
    """One layer's part of a cache, and a batch."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scale: torch.Tensor | None
    value_scale: torch.Tensor | None
    batch: PagedBatch
    cache: "PagedKVCache"


class PagedKVCache:
    """Keys and values of all layers of a decoder in pages, and which sequence has which of them.

    ``max_tokens`` bounds a sequence: tables have room for that many.  dtype: bf16 or float8_e4m3fn on the GPU; a code of the latter stands for code *
    ``key_scale`` (``value_scale``), by default 1 / 16, at which values of up to 28 are kept and a normal one has three bits behind its leading one down to
    2^-10.  The book-keeping is the host's; pages are handed out when a batch is made of new tokens."""

    def __init__(self, n_layer: int, kv_heads: int, head_dim: int, *, pages: int, page_size: int = 64, max_tokens: int | None = None,
                 dtype: torch.dtype = torch.bfloat16, device: "torch.device | str" = "cuda", key_scale: float = 1 / 16, value_scale: float = 1 / 16):
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError(f"pages of {page_size} tokens (a power of two)")
        if n_layer < 1 or kv_heads < 1 or head_dim < 1 or pages < 1:
            raise ValueError(f"a cache of {n_layer} layers, {kv_heads} heads of {head_dim} and {pages} pages")
        self.page_size, self.device = page_size, torch.device(device)
        self.max_tokens = pages * page_size if max_tokens is None else max_tokens
        self.width = -(-self.max_tokens // page_size)
        shape = (n_layer, pages, kv_heads, page_size, head_dim)
        self.keys, self.values = (torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(2))
        scales = dtype == torch.float8_e4m3fn
        self.key_scale = torch.full((n_layer, kv_heads), key_scale, dtype=torch.float32, device=self.device) if scales else None
        self.value_scale = torch.full((n_layer, kv_heads), value_scale, dtype=torch.float32, device=self.device) if scales else None
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._rows: dict[int, torch.Tensor] = {}       # the same as rows of a table, 0 behind the last
        self._length: dict[int, int] = {}
        self._next = 0
        self._angles: dict[tuple, tuple] = {}

    def add(self) -> int:
        """A new sequence without tokens."""
        s, self._next = self._next, self._next + 1
        self._pages[s], self._length[s], self._rows[s] = [], 0, torch.zeros(self.width, dtype=torch.int32)
        return s

    def length(self, sequence: int) -> int:
        return self._length[sequence]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def shorten(self, sequence: int, length: int) -> None:
        """The sequence's first ``length`` tokens are kept (drafts that were refused go, say); pages that hold none of them are free again."""
        if not 0 <= length <= self._length[sequence]:
            raise ValueError(f"sequence {sequence} has {self._length[sequence]} tokens, not {length}")
        self._length[sequence] = length
        kept = -(-length // self.page_size)
        self._rows[sequence][kept:len(self._pages[sequence])] = 0
        while len(self._pages[sequence]) > kept:
            self._free.append(self._pages[sequence].pop())

    def remove(self, sequence: int) -> None:
        self.shorten(sequence, 0)
        del self._pages[sequence], self._length[sequence], self._rows[sequence]

    def batch(self, sequences: "list[int]", new: "list[int]") -> PagedBatch:
        """Room for ``new`` more tokens of each of ``sequences``, and the batch of them in this order.  Refused as a whole where pages run out.

        The tokens count from here on.  Where the step that puts them into the cache raises, ``shorten`` takes them out again; until then later steps
        would see what their pages held before."""
        if len(sequences) != len(new) or len(set(sequences)) != len(sequences) or any(n < 0 for n in new):
            raise ValueError(f"{len(sequences)} sequences, each once, and {len(new)} numbers of new tokens")
        need = []
        for s, n in zip(sequences, new):
            if self._length[s] + n > self.max_tokens:
                raise ValueError(f"sequence {s}: {self._length[s]} tokens and {n} new ones, of {self.max_tokens}")
            need.append(-(-(self._length[s] + n) // self.page_size) - len(self._pages[s]))
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages wanted, {len(self._free)} are free")
        for s, n, k in zip(sequences, new, need):
            self._length[s] += n
            if k > 0:
                pages = [self._free.pop() for _ in range(k)]
                held = len(self._pages[s])
                self._rows[s][held:held + k] = torch.tensor(pages, dtype=torch.int32)
                self._pages[s] += pages
        seqs, offsets = len(sequences), list(accumulate(new, initial=0))
        numbers = torch.tensor(offsets + [self._length[s] for s in sequences], dtype=torch.int32)
        # one tensor of everything, which goes to the GPU in one copy
        everything = torch.cat([self._rows[s] for s in sequences] + [numbers]).to(self.device)
        table, offsets, lengths = everything.split((seqs * self.width, seqs + 1, seqs))
        return PagedBatch(table.view(seqs, self.width), offsets, lengths, max(new, default=0))

    def layer(self, i: int, batch: PagedBatch) -> PagedLayer:
        scale = lambda t: None if t is None else t[i]
        return PagedLayer(self.keys[i], self.values[i], scale(self.key_scale), scale(self.value_scale), batch, self)

    def angles(self, tables, head_dim: int, theta: float) -> tuple[torch.Tensor, torch.Tensor]:
        """``tables(head_dim, positions, theta, device)`` for every position that the tables reach, made once."""
        key = (tables, head_dim, theta)
        if key not in self._angles:
            on_gpu = self.device.type == "cuda"
            if on_gpu and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a cache makes its angles in its first step: run one before a step is captured")
            self._angles[key] = tables(head_dim, self.width * self.page_size, theta, self.device)
            if on_gpu:                                 # (steps on other streams use them too)
                torch.cuda.current_stream(self.device).synchronize()
        return self._angles[key]
