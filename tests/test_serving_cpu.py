"""Refusals of the serving operators that need no GPU: the C entry points
answer bad arguments with a status code before they touch a device, the Python
functions refuse host tensors, and the workspace sizes come from shapes alone."""

import os

import pytest
import torch

import adaattn_b200 as ada
from adaattn_b200 import _lib
from adaattn_b200.host_model import AdaptiveTransformer
from adaattn_b200.paged import _planes
from adaattn_b200.scoring import _rows3, token_logprobs_backward
from serving_util import PoolModel, attend64, build_pool

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")

INVALID, SHAPE, DTYPE, LAYOUT, WORKSPACE, UNSUPPORTED = -1, -2, -3, -5, -8, -9
T = _lib.packed


def _attn(q=None, k=None, v=None, table=None, lens=None, seqs=None, mask=None, ks=None, vs=None, out=None, ws=0):
    q = torch.zeros(2, 4, 64) if q is None else q
    k = torch.zeros(5, 2, 16, 64) if k is None else k
    v = torch.zeros_like(k) if v is None else v
    table = torch.zeros(2, 3, dtype=torch.int32) if table is None else table
    lens = torch.zeros(table.shape[0], dtype=torch.int32) if lens is None else lens
    out = torch.zeros_like(q) if out is None else out
    o = lambda t: None if t is None else T(t)
    buf = torch.zeros(max(ws, 1), dtype=torch.uint8)
    return _lib.load().ada_paged_attn(T(q), T(k), T(v), T(table), T(lens), o(seqs), o(mask), o(ks), o(vs), 0.125, T(out),
                                      None, buf.data_ptr() if ws else None, ws, None)


def test_attention_refuses_before_any_device_work():
    z = torch.zeros
    assert _lib.load().ada_paged_attn(None, None, None, None, None, None, None, None, None, 1.0, None, None, None, 0,
                                      None) == INVALID
    assert _attn() == WORKSPACE and _attn(ws=64) == WORKSPACE
    assert _attn(q=z(2, 4, 2, 64)) == SHAPE
    assert _attn(q=z(2, 3, 64)) == SHAPE                       # 3 heads over 2
    assert _attn(q=z(2, 4, 64, dtype=torch.float64)) == DTYPE
    assert _attn(q=z(2, 4, 64, dtype=torch.float16)) == DTYPE  # pages are fp32
    assert _attn(q=z(2, 4, 32)) == SHAPE
    assert _attn(q=z(2, 4, 64), out=z(2, 4, 63)) == SHAPE
    assert _attn(q=z(2, 64, 4).transpose(1, 2)) == LAYOUT
    assert _attn(q=z(2, 4, 256), k=z(5, 2, 16, 256)) == UNSUPPORTED
    assert _attn(k=z(5, 2, 0, 64)) == UNSUPPORTED
    assert _attn(k=z(5, 2, 16, 64), v=z(5, 2, 8, 64)) == SHAPE
    assert _attn(k=z(5, 2, 16, 64), v=z(5, 2, 16, 64, dtype=torch.float16)) == DTYPE
    assert _attn(table=z(2, 3, dtype=torch.int64)) == DTYPE
    assert _attn(table=z(3, 3, dtype=torch.int32)) == SHAPE    # a row per sequence unless picked
    assert _attn(lens=z(3, dtype=torch.int32)) == SHAPE
    assert _attn(seqs=z(3, dtype=torch.int32)) == SHAPE
    assert _attn(seqs=z(2, dtype=torch.int64)) == DTYPE
    assert _attn(mask=torch.ones(3, 40, dtype=torch.bool)) == SHAPE
    assert _attn(mask=torch.ones(2, 40, dtype=torch.int32)) == DTYPE
    assert _attn(ks=torch.ones(2)) == UNSUPPORTED              # scales go with 8-bit pages
    k8 = z(5, 2, 16, 64).to(torch.float8_e4m3fn)
    assert _attn(k=k8, ks=torch.ones(3)) == SHAPE
    assert _attn(k=k8, ks=torch.ones(2, dtype=torch.float64)) == DTYPE
    big = z(1, 4, 64).expand(5000, 4, 64)
    assert _attn(q=big, table=z(5000, 1, dtype=torch.int32), out=big) == UNSUPPORTED


def test_workspaces_come_from_shapes():
    lib = _lib.load()
    assert lib.ada_paged_attn_workspace_bytes(1, 32, 8, 128) > 0
    assert lib.ada_paged_attn_workspace_bytes(1, 3, 2, 128) == 0
    assert lib.ada_paged_attn_workspace_bytes(5000, 8, 8, 128) == 0
    assert lib.ada_paged_attn_workspace_bytes(1, 8, 8, 129) == 0
    a, b = lib.ada_pages_workspace_bytes(100, 10, 5), lib.ada_pages_workspace_bytes(1000, 10, 5)
    assert 0 < a < b and lib.ada_pages_workspace_bytes(-1, 1, 1) == 0


def _append(k=None, pages=None, table=None, lens=None, new=None, seqs=None, ks=None, v=None):
    k = torch.zeros(2, 2, 3, 64) if k is None else k
    pages = torch.zeros(5, 2, 16, 64) if pages is None else pages
    table = torch.zeros(2, 3, dtype=torch.int32) if table is None else table
    lens = torch.zeros(table.shape[0], dtype=torch.int32) if lens is None else lens
    o = lambda t: None if t is None else T(t)
    return _lib.load().ada_paged_append(T(k), T(k if v is None else v), T(pages), T(pages), T(table), T(lens), o(new),
                                        o(seqs), o(ks), None, None)


def test_append_refuses_before_any_device_work():
    z = torch.zeros
    assert _lib.load().ada_paged_append(*[None] * 11) == INVALID
    assert _append(k=z(2, 2, 64)) == SHAPE
    assert _append(k=z(2, 3, 3, 64)) == SHAPE
    assert _append(v=z(2, 2, 4, 64)) == SHAPE
    assert _append(k=z(2, 2, 3, 64, dtype=torch.bfloat16)) == DTYPE
    assert _append(k=z(2, 2, 64, 3).transpose(2, 3)) == LAYOUT
    assert _append(new=z(1, dtype=torch.int32)) == SHAPE
    assert _append(new=z(2, dtype=torch.int64)) == DTYPE
    assert _append(table=z(3, 3, dtype=torch.int32)) == SHAPE
    assert _append(ks=torch.ones(2)) == UNSUPPORTED
    assert _append(k=z(0, 2, 3, 64), table=z(0, 3, dtype=torch.int32)) == 0


def test_page_operations_refuse_before_any_device_work():
    lib, i32 = _lib.load(), torch.int32
    table, lens, refs = torch.zeros(4, 3, dtype=i32), torch.zeros(4, dtype=i32), torch.zeros(7, dtype=i32)
    one, two = torch.zeros(1, dtype=i32), torch.zeros(2, dtype=i32)
    data = torch.zeros(2, 7, 2, 16, 8)
    pool = (T(table), T(lens), T(refs))
    assert lib.ada_pages_free(None, None, None, 16, None, None) == INVALID
    assert lib.ada_pages_free(*pool, 0, T(one), None) == UNSUPPORTED
    assert lib.ada_pages_free(*pool, 70000, T(one), None) == UNSUPPORTED
    assert lib.ada_pages_free(T(table.long()), T(lens), T(refs), 16, T(one), None) == DTYPE
    assert lib.ada_pages_free(T(table), T(lens[:3]), T(refs), 16, T(one), None) == SHAPE
    assert lib.ada_pages_free(T(table[:, ::2]), T(lens), T(refs), 16, T(one), None) == LAYOUT
    assert lib.ada_pages_free(T(table[:1].expand(4, 3)), T(lens), T(refs), 16, T(one), None) == LAYOUT
    assert lib.ada_pages_free(*pool, 16, T(one.float()), None) == DTYPE
    assert lib.ada_pages_fork(*pool, 16, T(one), T(two), None) == SHAPE
    assert lib.ada_pages_fork(*pool, 16, T(one[:0]), T(one[:0]), None) == 0
    p = _planes(data)
    assert lib.ada_pages_reserve(p, *pool, 16, T(one), T(two), T(one), None, 0, None) == SHAPE
    assert lib.ada_pages_reserve(p, *pool, 16, T(one), T(one), T(one), None, 0, None) == WORKSPACE
    assert lib.ada_pages_reserve(_planes(data[:, :5]), *pool, 16, T(one), T(one), T(one), None, 0, None) == SHAPE
    assert lib.ada_pages_copy(p, *pool, 16, T(one), T(one), T(two), None, 0, None) == SHAPE
    assert lib.ada_pages_compact(p, *pool, 16, T(two), None, 0, None) == SHAPE
    assert lib.ada_pages_compact(_planes(data.expand(2, 7, 2, 16, 8)[:1].expand(2, 7, 2, 16, 8)), *pool, 16, T(one),
                                 None, 0, None) == LAYOUT
    both = torch.zeros(14 * 256)  # planes and pages a page apart: they overlap
    assert lib.ada_pages_compact(_planes(both.as_strided((2, 7, 2, 16, 8), (256, 256, 128, 8, 1))), *pool, 16, T(one),
                                 None, 0, None) == LAYOUT
    wide = torch.zeros(1, dtype=i32).expand(2 ** 16, 1).as_strided((2 ** 16, 2 ** 15), (0, 0))
    assert lib.ada_pages_free(T(wide), T(torch.zeros(2 ** 16, dtype=i32)), T(refs), 16, T(one), None) in (LAYOUT, UNSUPPORTED)
    with pytest.raises(ada.ShapeError):
        _planes(data.transpose(3, 4))


def test_an_empty_batch_of_picked_sequences_is_none():
    """A serving loop with nothing to do: no rows of q or k and an empty list of
    sequences, whatever the table's size. Without a list the table has to be empty as well."""
    z, none = torch.zeros, torch.zeros(0, dtype=torch.int32)
    table, mask = z(3, 2, dtype=torch.int32), z(0, 40, dtype=torch.bool)
    assert _attn(q=z(0, 4, 64), table=table, seqs=none) == 0
    assert _attn(q=z(0, 4, 64), table=table, seqs=none, mask=mask) == 0
    assert _attn(q=z(0, 4, 64), table=table) == SHAPE and _attn(q=z(2, 4, 64), table=table, seqs=none) == SHAPE
    assert _append(k=z(0, 2, 3, 64), table=table, seqs=none) == 0
    assert _append(k=z(0, 2, 3, 64), table=table, seqs=none, new=none) == 0
    assert _append(k=z(0, 2, 3, 64), table=table) == SHAPE


def test_empty_options_are_no_omitted_ones():
    """A list, mask or scale without elements is refused where elements are due, not taken for None."""
    z, none = torch.zeros, torch.zeros(0, dtype=torch.int32)
    assert _attn(seqs=none) == SHAPE and _append(seqs=none) == SHAPE and _append(new=none) == SHAPE
    assert _attn(mask=z(0, 40, dtype=torch.bool)) == SHAPE
    assert _attn(mask=z(2, 0, dtype=torch.bool)) == WORKSPACE  # covers no key: like none
    k8 = z(5, 2, 16, 64).to(torch.float8_e4m3fn)
    assert _attn(k=k8, ks=z(0)) == SHAPE and _append(pages=k8, ks=z(0)) == SHAPE
    absent = bytes(_lib.AdaTensor())
    lib, t, p = _lib.load(), torch.zeros(2, 4, 64), torch.zeros(5, 2, 16, 64)
    table, lens = z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32)
    assert lib.ada_paged_attn(T(t), T(p), T(p), T(table), T(lens), absent, absent, absent, absent, 1.0, T(t.clone()), None,
                              None, 0, None) == WORKSPACE


def test_batches_whose_places_pass_32_bits_are_refused():
    """Tiles of 32 keys and 6 places for each sequence, summed over the batch in
    32 bits. (The tables are described over a small buffer and never read:
    every call is refused on the host.)"""

    def table(s, w):
        t = _lib.AdaTensor.from_buffer_copy(T(torch.zeros(1, 1, dtype=torch.int32)))
        t.shape[0], t.shape[1], t.stride[0] = s, w, w
        return bytes(t)

    def call(b, w, page=16):
        q, k = torch.zeros(1, 1, 64).expand(b, 1, 64), torch.zeros(1, 1, page, 64)
        return _lib.load().ada_paged_attn(T(q), T(k), T(k), table(b, w), T(torch.zeros(b, dtype=torch.int32)), None, None,
                                          None, None, 1.0, T(torch.zeros(b, 1, 64)), None, None, 0, None)

    at = (2 ** 31 - 1) // 4096 - 6  # tiles per sequence that still fit
    assert call(4096, 2 * at) == WORKSPACE and call(4096, 2 * at + 1) == UNSUPPORTED
    assert call(4096, 2 ** 27 - 1) == UNSUPPORTED and call(33, 2 ** 27 - 1) == UNSUPPORTED
    assert call(1, 2 ** 27 - 1) == WORKSPACE and call(31, 2 ** 27 - 1) == WORKSPACE


def test_needs_that_would_reach_the_flags_are_refused():
    """2^29 - 1 table entries and more: a need of that many pages would set the
    bits that stand beside it. (The tables are never read: one row of them is
    described over a small buffer, and every call is refused on the host.)"""
    lib, i32 = _lib.load(), torch.int32
    lens, refs = torch.zeros(1, dtype=i32), torch.zeros(7, dtype=i32)
    one, data = torch.zeros(1, dtype=i32), torch.zeros(2, 7, 2, 1, 8)

    def table(w):
        t = _lib.AdaTensor.from_buffer_copy(T(torch.zeros(1, 1, dtype=i32)))
        t.shape[1] = w
        return bytes(t)

    p = _planes(data)
    for w, rc in ((2 ** 29 - 1, UNSUPPORTED), (2 ** 29, UNSUPPORTED), (2 ** 30, UNSUPPORTED), (2 ** 29 - 2, WORKSPACE)):
        pool = (table(w), T(lens), T(refs))
        assert lib.ada_pages_reserve(p, *pool, 1, T(one), T(one), T(one), None, 0, None) == rc
        assert lib.ada_pages_copy(p, *pool, 1, T(one), T(one), T(one), None, 0, None) == rc
        assert lib.ada_pages_compact(p, *pool, 1, T(one), None, 0, None) == rc
    assert lib.ada_pages_free(table(2 ** 29), T(lens), T(refs), 1, T(one), None) == UNSUPPORTED


def test_scores_refuse_before_any_device_work():
    lib = _lib.load()
    z, t = torch.zeros(1, 3, 10), torch.zeros(3, dtype=torch.int64)
    outs = [torch.zeros(30) for _ in range(6)]
    p = [o.data_ptr() for o in outs]

    def call(z=z, t=t, k=0, nulls=False):
        a = [None] * 6 if nulls else p
        return lib.ada_token_logprobs(T(z), T(t), -100, k, *a, None)

    assert lib.ada_token_logprobs(None, None, -100, 0, *[None] * 6, None) == INVALID
    assert call(z=z[0]) == SHAPE and call(t=t[:2]) == SHAPE
    assert call(z=z.double()) == DTYPE and call(t=t.float()) == DTYPE
    assert call(z=z.transpose(1, 2)) in (SHAPE, LAYOUT)
    assert call(k=65) == UNSUPPORTED and call(k=-1) == UNSUPPORTED and call(k=11) == SHAPE
    assert call(z=z[:, :, :0]) == UNSUPPORTED
    assert call(nulls=True) == INVALID
    assert call(z=z[:, :0], t=t[:0]) == 0
    grad = torch.zeros(1, 3, 9)
    assert lib.ada_token_logprobs_bwd(T(z), T(t), -100, p[0], p[1], None, None, None, T(grad), None) == SHAPE
    assert lib.ada_token_logprobs_bwd(T(z), T(t), -100, p[0], p[1], None, None, None, T(z.half()), None) == DTYPE
    assert lib.ada_token_logprobs_bwd(T(z), T(t), -100, None, p[1], None, None, None, T(z), None) == INVALID


def test_what_is_written_may_not_overlap_itself():
    """Expanded or interlaced outputs, pages and gradients (several elements in one place) and an output in q's
    memory are refused; transposed, sliced and padded ones are not."""
    z = torch.zeros
    q = z(2, 4, 64)
    assert _attn(out=z(1, 4, 64).expand(2, 4, 64)) == LAYOUT and _attn(out=z(2, 1, 64).expand(2, 4, 64)) == LAYOUT
    assert _attn(out=z(1000).as_strided((2, 4, 64), (128, 64, 1))) == LAYOUT
    assert _attn(out=z(1000).as_strided((2, 4, 64), (256, 63, 1))) == LAYOUT
    assert _attn(q=q, out=q) == LAYOUT
    for out in (z(4, 2, 64).transpose(0, 1), z(2, 8, 64)[:, ::2], z(2, 4, 80)[..., :64], z(2, 4, 2, 64)[:, :, 1]):
        assert _attn(out=out) == WORKSPACE
    for pages in (z(1, 2, 16, 64).expand(5, 2, 16, 64), z(5, 1, 16, 64).expand(5, 2, 16, 64), z(5, 2, 1, 64).expand(5, 2, 16, 64)):
        assert _append(pages=pages) == LAYOUT
    assert _append(k=z(2, 2, 0, 64), pages=z(5, 16, 2, 64).transpose(1, 2)) == 0
    lib, t, zl, o = _lib.load(), z(3, dtype=torch.int64), z(1, 3, 10), z(3, 2)
    assert lib.ada_token_logprobs_bwd(T(zl), T(t), -100, o.data_ptr(), o.data_ptr(), None, None, None,
                                      T(z(1, 1, 10).expand(1, 3, 10)), None) == LAYOUT


@pytest.mark.parametrize("lead", [(0, 2, 3), (2, 0, 3), (2, 3, 0), (0, 0, 0), (2, 3, 4), (2, 0), (0,), ()])
def test_rows_of_any_leading_dimensions(lead):
    """Logits without rows have three dimensions like all others."""
    z = torch.zeros(*lead, 9)
    rows = _rows3(z)
    assert rows.dim() == 3 and rows.shape[0] * rows.shape[1] == z.numel() // 9 and rows.shape[2] == 9
    if len(lead) > 1:
        assert rows.shape[0] == lead[0]


def test_gradient_arguments_are_checked():
    """The kernel reads a statistic pair, an entropy and an upstream gradient per row, whatever their tensors hold."""
    z, t = torch.zeros(2, 3, 10), torch.zeros(6, dtype=torch.int64)
    stats, ent, up = torch.zeros(6, 2), torch.zeros(6), torch.zeros(6)

    def call(z=z, stats=stats, ent=ent, **ups):
        return token_logprobs_backward(z, t, stats, ent, **ups)

    for bad in (dict(z=z[0]), dict(stats=stats[:5]), dict(stats=stats[:, 0]), dict(stats=stats.double()),
                dict(ent=ent[:1]), dict(ent=ent.half()), dict(ent=ent[:, None]), dict(grad_logprobs=up[:2]),
                dict(grad_entropy=up.view(2, 3)), dict(grad_lse=torch.zeros(()))):
        with pytest.raises(ada.ShapeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="CUDA"):  # all right but for the device
        call(grad_logprobs=up.double())


def test_host_tensors_are_refused():
    i32 = torch.int32
    table, lens, refs = torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(5, dtype=i32)
    pages, ids = torch.zeros(5, 2, 16, 64), torch.zeros(1, dtype=i32)
    for call in (lambda: ada.paged_attention(torch.zeros(2, 4, 64), pages, pages, table, lens),
                 lambda: ada.paged_append(torch.zeros(2, 2, 1, 64), torch.zeros(2, 2, 1, 64), pages, pages, table, lens),
                 lambda: ada.reserve_pages(pages[None], table, lens, refs, ids, ids),
                 lambda: ada.fork_pages(table, lens, refs, ids, ids, page_size=16),
                 lambda: ada.copy_pages(pages[None], table, lens, refs, ids, ids),
                 lambda: ada.free_pages(table, lens, refs, ids, page_size=16),
                 lambda: ada.compact_pages(pages[None], table, lens, refs),
                 lambda: ada.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        ada.PagedKVCache(1, 0, 16, 2, 64, max_sequences=1, max_pages_per_sequence=1, device="cpu")
    with pytest.raises(TypeError):
        ada.PagedKVCache(1, 4, 16, 2, 64, max_sequences=1, max_pages_per_sequence=1, device="cpu", dtype=torch.float64)
    with pytest.raises(TypeError):
        ada.PagedKVCache(1, 4, 16, 2, 64, max_sequences=1, max_pages_per_sequence=1, device="cpu",
                         k_scale=torch.ones(1, 2))
    c = ada.PagedKVCache(2, 4, 16, 2, 64, max_sequences=1, max_pages_per_sequence=1, device="cpu")
    assert c.keys(1).data_ptr() != c.values(1).data_ptr() and c.keys(0).shape == (4, 2, 16, 64)
    with pytest.raises(IndexError):
        c.keys(2)


def test_the_references_themselves():
    """The model of the page operations and the 64-bit attention agree with hand-made answers."""
    g = torch.Generator().manual_seed(0)
    k, v, table, ln = build_pool([3], 2, 1, 4, torch.float32, g)
    q = torch.zeros(1, 2, 4)
    out, lse = attend64(q, k, v, table, ln, 1.0)
    rows = torch.cat([v[table[0, 0], 0], v[table[0, 1], 0, :1]]).double()
    assert torch.allclose(out[0, 1], rows.mean(0)) and abs(lse[0, 0].item() - 1.0986122886681098) < 1e-12
    m = PoolModel(torch.tensor([[4, 1], [-1, -1], [-1, -1]], dtype=torch.int32), torch.tensor([3, 0, 0], dtype=torch.int32),
                  torch.tensor([0, 1, 0, 0, 1], dtype=torch.int32), torch.arange(10.).view(1, 5, 2), 2)
    m.fork([0], [1])
    assert m.refs.tolist() == [0, 2, 0, 0, 2]
    assert m.reserve([0, 1], [1, 1]) == [1, 1]          # 0 copies the part-full page, 1 keeps it
    assert m.table.tolist() == [[4, 0], [4, 1], [-1, -1]] and m.refs.tolist() == [1, 1, 0, 0, 2]
    assert m.data[0, 0].tolist() == m.data[0, 1].tolist()
    assert m.compact() == 3 and m.table.tolist() == [[2, 0], [2, 1], [-1, -1]]
    m.free([0, 1])
    assert m.refs.sum() == 0


def test_scores_of_a_decoder_that_sees_ahead_are_refused():
    """A decoder built without causal=True gives a token's position the token itself; a mask may close it."""
    m = AdaptiveTransformer(50, 32, 2, 2, 64, max_seq_len=16, dropout=0.0)
    ids = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="causal"):
        m.score(ids)
    m.forward = lambda ids, attention_mask=None: torch.zeros(*ids.shape, 50)  # (the attention has no CPU path)
    for kw in (dict(attention_mask=torch.ones(4, 4).tril()[None, None]),):
        with pytest.raises(RuntimeError, match="CUDA"):
            m.score(ids, **kw)
