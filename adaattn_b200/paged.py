"""The paged key-value cache: attention of one new token per sequence over it,
the append that fills it, and the operations on its pages.

A cache is a pool of pages. ``k_pages`` and ``v_pages`` are [P, Hkv, page, D]
(any strides, the innermost 1); ``page_table`` int32 [S, W] lists the pages of
each sequence in order, ``seq_lens`` int32 [S] how many tokens it has and
``ref_counts`` int32 [P] how many sequences hold a page (0: free). Everything
is device memory and every call enqueues on the current CUDA stream without a
host synchronisation, so a decoding step can be captured in a CUDA graph.

``PagedKVCache`` owns such a pool for the layers of a model; the functions
work on tensors of any origin. Ids that a kernel finds out of range in device
memory are left out and recorded in the library's status word
(``_lib.poll_device_status`` raises for it).
"""

from __future__ import annotations

import functools
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.autograd.forward_ad as _fwd

from . import _lib
from .config import ShapeError

# Workspace sizes follow from the shapes alone; a decoding loop asks for the same ones again and again.
@functools.lru_cache(maxsize=256)
def _attn_workspace(b: int, h: int, hkv: int, d: int) -> int:
    return max(_lib.load().ada_paged_attn_workspace_bytes(b, h, hkv, d), 1)


@functools.lru_cache(maxsize=256)
def _pages_workspace(num_pages: int, num_sequences: int, n: int) -> int:
    return _lib.load().ada_pages_workspace_bytes(num_pages, num_sequences, n)


Ids = Union[torch.Tensor, Sequence[int]]


def _device_of(first: torch.Tensor, *rest: Optional[torch.Tensor]) -> torch.device:
    index = first.get_device()
    if index < 0:
        raise RuntimeError(f"adaattn_b200 runs on CUDA devices only (sm_100a); got a tensor on {first.device}. "
                           "There is no CPU path.")
    for t in rest:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"all tensors must be on {first.device}; got one on {t.device}")
    return first.device


def _no_tangent(what: str, *ts: Optional[torch.Tensor]) -> None:
    """Refuses dual tensors, whose tangents the kernels would drop (they need no requires_grad)."""
    if _fwd._current_level >= 0 and any(
            t is not None and t.is_floating_point() and _fwd.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it outside dual levels or on the primals")


def _no_grad(what: str, *ts: Optional[torch.Tensor]) -> None:
    _no_tangent(what, *ts)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _opt(t: Optional[torch.Tensor]):
    return None if t is None else _lib.packed(t)


def _call(what: str, dev: torch.device, fn, *args) -> None:
    """One C call on the current stream of `dev`, with that device current."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, what)


def _ids(x: Ids, dev: torch.device) -> torch.Tensor:
    if isinstance(x, torch.Tensor):
        return x
    return torch.tensor(list(x), dtype=torch.int32, device=dev)


_MASK_DTYPES = (torch.bool, torch.uint8, torch.float32, torch.float16, torch.bfloat16)


def _mask32(m: torch.Tensor) -> torch.Tensor:
    """A mask of another floating type in 32 bits; only infinities become infinite (the type's lowest value hides nothing)."""
    if not m.is_floating_point():
        raise TypeError(f"key_mask must be bool (True keeps) or floating point (added), got {m.dtype}")
    top = torch.finfo(torch.float32).max
    return torch.where(m.isinf(), m, m.clamp(-top, top)).float() if m.dtype == torch.float64 else m.float()


def _unit_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    page_table: torch.Tensor, seq_lens: torch.Tensor, *, scale: Optional[float] = None,
                    seqs: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of one new token per sequence over its cached keys and values
    (``ada_paged_attn``): q [B, H, D] -> [B, H, D] in q's dtype.

    Sequence b is row ``seqs[b]`` (int32; row b when omitted) of page_table
    and seq_lens, and sees all its seq_lens keys. H is a multiple of the
    pages' Hkv: groups of H / Hkv query heads share a key/value head. The
    pages have q's dtype (fp32, fp16 or bf16) or are float8_e4m3fn holding
    value / scale with ``k_scale`` / ``v_scale`` float32 [Hkv] (1 when
    omitted). ``key_mask`` [B, L] or [1, L] covers the first L keys, bool
    (True keeps; uint8 counts as bool) or floating point (added; -inf hides;
    float64 beyond float32's range counts as its ends); later keys are open
    and what hidden keys hold does not matter. ``scale`` defaults to D ** -0.5.

    Scores, softmax and sums are fp32, the result is rounded once. On the
    tensor cores (16- and 8-bit pages, heads of 64 or 128) a probability is
    held to 16 bits over bf16 pages, to 22 bits and 2^-40 of the largest one
    over the others, and q over 8-bit pages to fp16's bits after a power of two
    per head; a visible infinite value may come out as NaN there. A sequence
    without a visible key gives zeros. With ``return_lse`` also the fp32
    [B, H] log-sum-exp of the scores (-inf there). ``out`` shares no memory with
    the inputs or with itself. No autograd. Up to 4096
    sequences per call (whose tables cover less than 2^36 keys), head dims up
    to 128.
    """
    dev = _device_of(q, k_pages, v_pages, page_table, seq_lens, seqs, key_mask, k_scale, v_scale, out)
    _no_grad("paged_attention", q, k_pages, v_pages, key_mask)
    _no_tangent("paged_attention", k_scale, v_scale)
    if q.dim() != 3:
        raise ShapeError(f"q must be 3-D [B, H, D], got {q.dim()}-D")
    if k_pages.dim() != 4:
        raise ShapeError(f"k_pages must be 4-D [P, Hkv, page, D], got {k_pages.dim()}-D")
    b, h, d = q.shape
    if out is None:
        out = torch.empty(b, h, d, dtype=q.dtype, device=dev)
    lse = torch.empty(b, h, dtype=torch.float32, device=dev) if return_lse else None
    if key_mask is not None and key_mask.dtype not in _MASK_DTYPES:
        key_mask = _mask32(key_mask)
    lib = _lib.load()
    ws = torch.empty(_attn_workspace(b, h, max(1, k_pages.shape[1]), d), dtype=torch.uint8, device=dev)
    _call("ada_paged_attn", dev, lib.ada_paged_attn, _lib.packed(_unit_last(q)), _lib.packed(k_pages),
          _lib.packed(v_pages), _lib.packed(page_table), _lib.packed(seq_lens), _opt(seqs), _opt(key_mask),
          _opt(k_scale), _opt(v_scale), float(d ** -0.5 if scale is None else scale), _lib.packed(out),
          None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel())
    return out if lse is None else (out, lse)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor,
                 new_tokens: Optional[torch.Tensor] = None, *, seqs: Optional[torch.Tensor] = None,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 prompts: bool = False) -> None:
    """Write new keys and values into their pages in place (``ada_paged_append``).

    k, v [B, Hkv, N, D] views (unit innermost stride): token t <
    new_tokens[b] (int32; N when omitted) goes to position seq_lens -
    new_tokens[b] + t of table row ``seqs[b]`` (row b when omitted);
    ``seq_lens`` already count the new tokens, as ``reserve_pages`` leaves
    them. The pages written must be held by their sequence alone (which
    ``reserve_pages`` sees to). k and v have the pages' dtype, or the pages are
    float8_e4m3fn and receive value / scale, rounded once and saturated at 448.
    With ``prompts`` the new tokens must be all that their sequence holds; one
    that holds others too is left out and recorded in the status word.
    """
    dev = _device_of(k, v, k_pages, v_pages, page_table, seq_lens, new_tokens, seqs, k_scale, v_scale)
    _no_grad("paged_append", k, v, k_pages, v_pages)
    _no_tangent("paged_append", k_scale, v_scale)
    lib = _lib.load()
    _call("ada_paged_append", dev, lib.ada_paged_append_prompts if prompts else lib.ada_paged_append,
          _lib.packed(_unit_last(k)),
          _lib.packed(_unit_last(v)), _lib.packed(k_pages), _lib.packed(v_pages), _lib.packed(page_table),
          _lib.packed(seq_lens), _opt(new_tokens), _opt(seqs), _opt(k_scale), _opt(v_scale))


def _planes(pages: torch.Tensor) -> bytes:
    """[planes, P, ...] as [planes, P, elements of a page] (page blocks must be contiguous)."""
    if pages.dim() < 3:
        raise ShapeError(f"pages must be [planes, P, ...], got {pages.dim()}-D")
    shape, stride = pages.shape, pages.stride()
    inner = 1
    for i in range(len(shape) - 1, 1, -1):
        if shape[i] > 1 and stride[i] != inner:
            raise ShapeError("the pages' blocks must be contiguous")
        inner *= shape[i]
    return _lib.packed(pages.as_strided((shape[0], shape[1], inner), (stride[0], stride[1], 1)))


def _page_size(pages: torch.Tensor, page_size: Optional[int]) -> int:
    if page_size is not None:
        return int(page_size)
    if pages.dim() != 5:
        raise ShapeError("page_size is needed unless pages are [planes, P, Hkv, page, D]")
    return pages.shape[3]


def _workspace(page_table: torch.Tensor, ref_counts: torch.Tensor, n: int) -> torch.Tensor:
    if page_table.dim() != 2 or ref_counts.dim() != 1:
        raise ShapeError("page_table must be 2-D [S, W] and ref_counts 1-D [P]")
    return torch.empty(_pages_workspace(ref_counts.shape[0], page_table.shape[0], n), dtype=torch.uint8,
                       device=page_table.device)


def reserve_pages(pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                  ref_counts: torch.Tensor, seqs: torch.Tensor, new_tokens: torch.Tensor, *,
                  page_size: Optional[int] = None) -> torch.Tensor:
    """Make room for new_tokens[i] more tokens of sequence seqs[i] (int32) and
    add them to its length (``ada_pages_reserve``). A part-full last page that
    other sequences hold too is copied first (the last of the call's sequences
    that share it keeps it when they are all its holders). Returns int32
    [n]: the tokens granted, new_tokens[i], or 0 for a sequence that was left
    as it was because the needs up to and including its own exceed the free
    pages, or (recorded in the status word) because they exceed its table row
    or it was named before. Free pages are handed out lowest id first."""
    dev = _device_of(pages, page_table, seq_lens, ref_counts, seqs, new_tokens)
    granted = torch.empty(seqs.shape, dtype=torch.int32, device=dev)
    ws = _workspace(page_table, ref_counts, seqs.numel())
    _call("ada_pages_reserve", dev, _lib.load().ada_pages_reserve, _planes(pages), _lib.packed(page_table),
          _lib.packed(seq_lens), _lib.packed(ref_counts), _page_size(pages, page_size), _lib.packed(seqs),
          _lib.packed(new_tokens), _lib.packed(granted), ws.data_ptr(), ws.numel())
    return granted


def fork_pages(page_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
               src: torch.Tensor, dst: torch.Tensor, *, page_size: int) -> None:
    """Sequence dst[i] gives its pages up and holds src[i]'s pages with it
    (``ada_pages_fork``); no data moves. A dst named twice counts once, one
    that is also a src of the call is left out."""
    dev = _device_of(page_table, seq_lens, ref_counts, src, dst)
    _call("ada_pages_fork", dev, _lib.load().ada_pages_fork, _lib.packed(page_table), _lib.packed(seq_lens),
          _lib.packed(ref_counts), int(page_size), _lib.packed(src), _lib.packed(dst))


def copy_pages(pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
               ref_counts: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, *,
               page_size: Optional[int] = None) -> torch.Tensor:
    """Sequence dst[i] gives its pages up and gets its own copy of src[i]'s
    (``ada_pages_copy``). Returns int32 [n]: dst[i]'s length, 0 where the free
    pages did not suffice and it was left empty."""
    dev = _device_of(pages, page_table, seq_lens, ref_counts, src, dst)
    granted = torch.empty(src.shape, dtype=torch.int32, device=dev)
    ws = _workspace(page_table, ref_counts, src.numel())
    _call("ada_pages_copy", dev, _lib.load().ada_pages_copy, _planes(pages), _lib.packed(page_table),
          _lib.packed(seq_lens), _lib.packed(ref_counts), _page_size(pages, page_size), _lib.packed(src),
          _lib.packed(dst), _lib.packed(granted), ws.data_ptr(), ws.numel())
    return granted


def free_pages(page_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
               seqs: torch.Tensor, *, page_size: int) -> None:
    """The sequences give their pages up: length 0, table entries -1
    (``ada_pages_free``). A sequence named twice is freed once."""
    dev = _device_of(page_table, seq_lens, ref_counts, seqs)
    _call("ada_pages_free", dev, _lib.load().ada_pages_free, _lib.packed(page_table), _lib.packed(seq_lens),
          _lib.packed(ref_counts), int(page_size), _lib.packed(seqs))


def compact_pages(pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                  ref_counts: torch.Tensor, *, page_size: Optional[int] = None) -> torch.Tensor:
    """Move the live pages into the ids 0 .. live - 1 and rewrite the table
    (``ada_pages_compact``): live pages above move, in order, into the free
    ids below. Returns live as int32 [1]."""
    dev = _device_of(pages, page_table, seq_lens, ref_counts)
    live = torch.empty(1, dtype=torch.int32, device=dev)
    ws = _workspace(page_table, ref_counts, 0)
    _call("ada_pages_compact", dev, _lib.load().ada_pages_compact, _planes(pages), _lib.packed(page_table),
          _lib.packed(seq_lens), _lib.packed(ref_counts), _page_size(pages, page_size), _lib.packed(live),
          ws.data_ptr(), ws.numel())
    return live


class PagedKVCache:
    """Pages for the keys and values of a model's layers, shared by up to
    ``max_sequences`` sequences of up to ``max_pages_per_sequence`` pages.

    ``data`` [2 * num_layers, num_pages, num_kv_heads, page_size, head_dim]
    holds layer l's keys in plane 2 l and its values in plane 2 l + 1; a page id
    means the same page in every plane, so the accounting is done once for all
    layers. A decoding step is one ``reserve`` and, per layer, one ``append``
    and one ``attend``. Sequences are named by int32 device tensors (or lists).
    With ``dtype=torch.float8_e4m3fn`` the pages hold value / scale;
    ``k_scale`` / ``v_scale`` float32 [num_layers, num_kv_heads] (default 1).
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *,
                 max_sequences: int, max_pages_per_sequence: int, dtype: torch.dtype = torch.bfloat16,
                 device: Optional[torch.device] = None, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None) -> None:
        for name, n in (("num_layers", num_layers), ("num_pages", num_pages), ("page_size", page_size),
                        ("num_kv_heads", num_kv_heads), ("head_dim", head_dim),
                        ("max_sequences", max_sequences), ("max_pages_per_sequence", max_pages_per_sequence)):
            if n < 1:
                raise ValueError(f"{name} must be positive, got {n}")
        if dtype not in (torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn):
            raise TypeError(f"the cache holds fp32, fp16, bf16 or float8_e4m3fn, got {dtype}")
        if head_dim > 128:
            raise ShapeError(f"head dims go up to 128, got {head_dim}")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if s is None:
                continue
            if dtype != torch.float8_e4m3fn:
                raise TypeError(f"{name} goes with float8_e4m3fn pages only")
            if tuple(s.shape) != (num_layers, num_kv_heads) or s.dtype != torch.float32:
                raise ShapeError(f"{name} must be float32 [{num_layers}, {num_kv_heads}]")
        self.num_layers, self.page_size = num_layers, page_size
        self.data = torch.zeros(2 * num_layers, num_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=dev)
        self.page_table = torch.full((max_sequences, max_pages_per_sequence), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(max_sequences, dtype=torch.int32, device=dev)
        self.ref_counts = torch.zeros(num_pages, dtype=torch.int32, device=dev)
        self.k_scale = None if k_scale is None else k_scale.to(dev).contiguous()
        self.v_scale = None if v_scale is None else v_scale.to(dev).contiguous()

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def dtype(self) -> torch.dtype:
        return self.data.dtype

    def keys(self, layer: int) -> torch.Tensor:
        """[P, Hkv, page, D] of a layer."""
        return self.data[2 * self._layer(layer)]

    def values(self, layer: int) -> torch.Tensor:
        return self.data[2 * self._layer(layer) + 1]

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.num_layers:
            raise IndexError(f"layer {layer} outside [0, {self.num_layers})")
        return layer

    def _pool(self):
        return self.page_table, self.seq_lens, self.ref_counts

    def _scales(self, layer: int) -> dict:
        return dict(k_scale=None if self.k_scale is None else self.k_scale[layer],
                    v_scale=None if self.v_scale is None else self.v_scale[layer])

    def reserve(self, seqs: Ids, new_tokens: Ids) -> torch.Tensor:
        """Room for new_tokens[i] more tokens of seqs[i]; the tokens granted (``reserve_pages``)."""
        return reserve_pages(self.data, *self._pool(), _ids(seqs, self.device), _ids(new_tokens, self.device))

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, new_tokens: Optional[Ids] = None, *,
               seqs: Optional[Ids] = None, prompts: bool = False) -> None:
        """Write k, v [B, Hkv, N, D] of the newest tokens of seqs (``paged_append``)."""
        paged_append(k, v, self.keys(layer), self.values(layer), self.page_table, self.seq_lens,
                     None if new_tokens is None else _ids(new_tokens, self.device),
                     seqs=None if seqs is None else _ids(seqs, self.device), prompts=prompts, **self._scales(layer))

    def attend(self, layer: int, q: torch.Tensor, *, seqs: Optional[Ids] = None, **kwargs):
        """Attention of q [B, H, D], the newest tokens of seqs, over the layer's cache (``paged_attention``)."""
        return paged_attention(q, self.keys(layer), self.values(layer), self.page_table, self.seq_lens,
                               seqs=None if seqs is None else _ids(seqs, self.device), **self._scales(layer),
                               **kwargs)

    def fork(self, src: Ids, dst: Ids) -> None:
        """dst[i] shares src[i]'s pages until either grows (``fork_pages``)."""
        fork_pages(*self._pool(), _ids(src, self.device), _ids(dst, self.device), page_size=self.page_size)

    def copy(self, src: Ids, dst: Ids) -> torch.Tensor:
        """dst[i] gets its own copy of src[i]; its length, 0 when the pool ran out (``copy_pages``)."""
        return copy_pages(self.data, *self._pool(), _ids(src, self.device), _ids(dst, self.device))

    def free(self, seqs: Ids) -> None:
        """The sequences give their pages up (``free_pages``)."""
        free_pages(*self._pool(), _ids(seqs, self.device), page_size=self.page_size)

    def compact(self) -> torch.Tensor:
        """Live pages to the front of the pool; their number as int32 [1] (``compact_pages``)."""
        return compact_pages(self.data, *self._pool())


__all__ = ["paged_attention", "paged_append", "reserve_pages", "fork_pages", "copy_pages", "free_pages",
           "compact_pages", "PagedKVCache"]
