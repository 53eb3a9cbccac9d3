"""Attention over a paged key-value cache (ada_paged_attn) and the append
(ada_paged_append) against 64-bit evaluations of their formulas.

Attention's tolerance, for outputs o = sum p v with sum p = 1 and values of
size up to A = max |v|: the result's rounding, half a step of its type
relative to the value; and fp32 arithmetic: scores |s| <= S err by the sum
over D products and their rounding to the order of (D / 2 + 4) 2^-24 S', with
S' = sum |q k| scale, which changes p by that factor, the exponential by
2^-21 relative and sums over n keys in at most n / 256 + 40 dependent steps of
2^-24 each: A (2 (D / 2 + 4) 2^-24 S' + 2^-20 + (n / 256 + 40) 2^-23).
Probabilities that enter a 16-bit product as two 16-bit parts keep 2^-16
relative (bf16: 8 + 8 bits), half a step 2^-17, times A.
"""

import math

import pytest
import torch

import adaattn_b200 as ada
from adaattn_b200 import _lib
from serving_util import attend64, build_pool

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def _bar(q, k, v, lens, scale, ks, vs, want):
    d = q.shape[-1]
    a = v.float()[torch.isfinite(v.float())].abs().max().item() * (1 if vs is None else vs.max().item())
    kmax = k.float()[torch.isfinite(k.float())].abs().max().item() * (1 if ks is None else ks.max().item())
    s1 = q.float().abs().sum(-1).max().item() * kmax * scale
    n = max(1, int(lens.max()))
    fp32 = a * (2 * (d / 2 + 4) * 2.0 ** -24 * s1 + 2.0 ** -20 + (n / 256 + 40) * 2.0 ** -23 + 2.0 ** -17)
    return want.abs() * HALF[q.dtype] + fp32


def _check(lens, page, h, hkv, d, dtype, dev, *, qdtype=None, mask=None, scales=False, seed=0, fill=None, seqs=None):
    g = torch.Generator().manual_seed(seed * 1000 + d + page + h)
    k, v, table, ln = build_pool(lens, page, hkv, d, dtype, g, fill=fill)
    b = len(lens) if seqs is None else len(seqs)
    q = torch.randn(b, h, d, generator=g).to(qdtype or dtype)
    ks = (0.5 + torch.rand(hkv, generator=g)) if scales else None
    vs = (0.5 + torch.rand(hkv, generator=g)) if scales else None
    m = mask(b, max(1, max(lens)), g) if mask is not None else None
    sq = None if seqs is None else torch.tensor(seqs, dtype=torch.int32)
    scale = d ** -0.5
    up = (lambda t: None if t is None else t.to(dev))
    out, lse = ada.paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ln.to(dev), seqs=up(sq),
                                   key_mask=up(m), k_scale=up(ks), v_scale=up(vs), return_lse=True)
    torch.cuda.synchronize()
    _lib.poll_device_status(dev)
    want, want_lse = attend64(q, k, v, table, ln, scale, m, ks, vs, seqs)
    err = (out.cpu().double() - want).abs()
    bar = _bar(q, k, v, ln, scale, ks, vs, want)
    assert (err <= bar).all(), f"off by up to {(err / bar).max().item():.2f} of the bar"
    fin = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), fin)
    lerr = (lse.cpu().double() - want_lse)[fin].abs()
    if lerr.numel():
        assert lerr.max().item() <= 1e-5 * max(1.0, want_lse[fin].abs().max().item())
    return out


SHAPES = [  # lens, page, H, Hkv, D
    ([1], 16, 1, 1, 64), ([0], 16, 4, 2, 64), ([0, 5, 0, 17, 0], 16, 4, 4, 128), ([187], 16, 12, 12, 64),
    ([31, 32, 33, 64, 65], 16, 8, 2, 128), ([1000, 3, 700, 1, 129], 64, 8, 1, 128), ([257, 4000], 128, 32, 8, 128),
    ([100, 90], 24, 10, 2, 64), ([77, 300], 5, 7, 1, 80), ([50, 129], 1, 6, 3, 33), ([513], 8, 16, 1, 128),
    ([15, 16, 17], 16, 3, 3, 1), ([40, 41], 256, 18, 2, 64), ([3000], 32, 4, 4, 32), ([600, 2], 48, 40, 2, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", SHAPES)
def test_attention_matches_formula(case, dtype, cuda_device):
    _check(*case, dtype, cuda_device)


@pytest.mark.parametrize("qdtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", SHAPES)
@pytest.mark.parametrize("scales", [False, True])
def test_attention_over_8bit_pages(case, qdtype, scales, cuda_device):
    _check(*case, torch.float8_e4m3fn, cuda_device, qdtype=qdtype, scales=scales)


def _bool_mask(b, n, g):
    m = torch.rand(b, n, generator=g) < 0.6
    m[0] = False  # a sequence with no visible key
    return m


def _float_mask(b, n, g):
    m = torch.randn(b, n, generator=g) * 2
    return m.masked_fill(torch.rand(b, n, generator=g) < 0.3, -math.inf)


def _short_mask(b, n, g):  # covers half of the keys, for all sequences alike
    return torch.rand(1, max(1, n // 2), generator=g) < 0.5


@pytest.mark.parametrize("mask", [_bool_mask, _float_mask, _short_mask])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("case", [([40, 100, 7, 256], 16, 8, 2, 128), ([33, 500], 5, 3, 3, 48), ([70, 64], 64, 12, 12, 64)])
def test_masks(case, dtype, mask, cuda_device):
    _check(*case, dtype, cuda_device, qdtype=None if dtype != torch.float8_e4m3fn else torch.bfloat16, mask=mask)


@pytest.mark.parametrize("mdtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lowest_value_masks_leave_a_uniform_row(mdtype, cuda_device):
    """A mask of the type's lowest finite value everywhere hides nothing: in
    fp32 it absorbs the scores (bf16, fp32) and the keys count alike."""
    g = torch.Generator().manual_seed(1)
    k, v, table, ln = build_pool([50], 16, 2, 64, torch.float32, g)
    q = torch.randn(1, 4, 64, generator=g)
    m = torch.full((1, 50), torch.finfo(mdtype).min, dtype=mdtype)
    dev = cuda_device
    out = ada.paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ln.to(dev), key_mask=m.to(dev)).cpu()
    want, _ = attend64(q, k, v, table, ln, 0.125, m)
    if mdtype != torch.float16:  # 64-bit sums still see the scores beside -3.4e38 only in part; fp32 does not
        for h in range(4):
            ids = table[0, :4].long()
            want[0, h] = v[ids, h // 2].reshape(-1, 64)[:50].double().mean(0)
        assert (out.double() - want).abs().max().item() <= 2.0 ** -20 * v.abs().max().item()
    else:  # scores lose what 65504 + s rounds away: s to half of 2^-8, p to e^(2^-8) - 1 relative
        assert (out.double() - want).abs().max().item() <= 2 * (math.exp(2.0 ** -8) - 1) * v.abs().max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("mdtype", [torch.float32, torch.bfloat16])
def test_lowest_value_masks_on_the_tensor_cores(mdtype, dtype, cuda_device):
    """As above where the scores come from the tensor cores: -3.4e38 absorbs every score in fp32, all keys count alike."""
    dev = cuda_device
    g = torch.Generator().manual_seed(12)
    k, v, table, ln = build_pool([50, 200], 16, 2, 64, dtype, g)
    qd = torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype
    q = torch.randn(2, 4, 64, generator=g).to(qd)
    m = torch.full((2, 200), torch.finfo(mdtype).min, dtype=mdtype)
    out = ada.paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ln.to(dev), key_mask=m.to(dev)).cpu()
    want, _ = attend64(torch.zeros_like(q), k, v, table, ln, 0.125)
    err = (out.double() - want).abs()
    assert (err <= _bar(torch.zeros_like(q), k, v, ln, 0.125, None, None, want)).all()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float8_e4m3fn, 128),
                                     (torch.float8_e4m3fn, 64), (torch.float32, 64)])
@pytest.mark.parametrize("b", [700, 4096])
def test_large_batches(b, dtype, d, cuda_device):
    """More sequences than a block has threads, and the most that a call takes (whose prefix leaves less shared memory)."""
    g = torch.Generator().manual_seed(b)
    lens = torch.randint(0, 41, (b,), generator=g).tolist()
    _check(lens, 16, 2, 1, d, dtype, cuda_device, qdtype=None if dtype != torch.float8_e4m3fn else torch.bfloat16)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [(16, 4, 2, 128), (8, 2, 2, 64), (5, 4, 2, 96)])
def test_what_is_behind_the_last_token_does_not_matter(shape, dtype, bad, cuda_device):
    if dtype == torch.float8_e4m3fn:
        bad = math.nan
    _check([1, 17, 40, 31], *shape, dtype, cuda_device, qdtype=None if dtype != torch.float8_e4m3fn else torch.bfloat16,
           fill=bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_hidden_keys_may_hold_nan(dtype, cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(2)
    k, v, table, ln = build_pool([90], 16, 2, 128, dtype, g)
    q = torch.randn(1, 6, 128, generator=g).to(dtype)
    for m in (torch.rand(1, 90, generator=g) < 0.5,
              torch.zeros(1, 90).masked_fill(torch.rand(1, 90, generator=g) < 0.5, -math.inf)):
        hidden = ~m if m.dtype == torch.bool else m == -math.inf
        want, _ = attend64(q, k, v, table, ln, 128 ** -0.5, m)
        k2, v2 = k.clone(), v.clone()
        for j in range(90):
            if hidden[0, j]:
                k2[table[0, j // 16], :, j % 16] = math.nan
                v2[table[0, j // 16], :, j % 16] = math.inf
        out = ada.paged_attention(q.to(dev), k2.to(dev), v2.to(dev), table.to(dev), ln.to(dev), key_mask=m.to(dev))
        err = (out.cpu().double() - want).abs()
        assert (err <= _bar(q, k, v, ln, 128 ** -0.5, None, None, want)).all()


def test_visible_nan_and_infinity_reach_the_output(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(3)
    k, v, table, ln = build_pool([40, 40], 16, 1, 128, torch.bfloat16, g)
    k[table[1, 0], 0, 3, 5] = math.nan
    q = torch.randn(2, 2, 128, generator=g).to(torch.bfloat16)
    out = ada.paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ln.to(dev)).cpu()
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_picked_sequences_and_repeats(dtype, cuda_device):
    _check([100, 5, 0, 333], 16, 8, 2, 128, dtype, cuda_device, seqs=[3, 0, 3, 2, 1, 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
def test_large_scores(dtype, cuda_device):
    """Scores in the hundreds: the softmax is nearly one-hot and the maximum moves along the cache."""
    dev = cuda_device
    g = torch.Generator().manual_seed(4)
    k, v, table, ln = build_pool([700, 65], 16, 2, 64, dtype, g)
    qd = torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype
    q = (torch.randn(2, 4, 64, generator=g) * 8).to(qd)
    out = ada.paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ln.to(dev), scale=1.0).cpu()
    want, _ = attend64(q, k, v, table, ln, 1.0)
    err = (out.double() - want).abs()
    assert (err <= _bar(q, k, v, ln, 1.0, None, None, want)).all()


def test_strided_pages_heads_and_outputs(cuda_device):
    """Pages as [P, page, H, D] storage in a two-tensor buffer, q from a wider
    projection, out into every second head of a buffer, a table with spare columns."""
    dev = cuda_device
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.bfloat16, torch.float32):
        k, v, table, ln = build_pool([70, 10, 200], 16, 2, 64, dtype, g)
        store = torch.full((k.shape[0], 16, 2, 2, 64), math.nan, dtype=dtype)
        store[:, :, 0], store[:, :, 1] = k.transpose(1, 2), v.transpose(1, 2)
        store = store.to(dev)
        kp, vp = store[:, :, 0].transpose(1, 2), store[:, :, 1].transpose(1, 2)
        wide = torch.randn(3, 8 * 64 + 16, generator=g).to(dtype).to(dev)
        q = wide[:, 16:].view(3, 8, 64)
        buf = torch.full((3, 16, 64), 7.0, dtype=dtype, device=dev)
        tab = torch.cat([table, torch.full((3, 5), -1, dtype=torch.int32)], 1).to(dev)
        got = ada.paged_attention(q, kp, vp, tab, ln.to(dev), out=buf[:, ::2])
        want, _ = attend64(q.cpu(), k, v, table, ln, 0.125)
        err = (got.cpu().double() - want).abs()
        assert (err <= _bar(q.cpu(), k, v, ln, 0.125, None, None, want)).all()
        assert (buf[:, 1::2] == 7).all()
    # rows that start on odd elements
    k, v, table, ln = build_pool([70], 16, 2, 64, torch.bfloat16, g)
    odd = torch.zeros(k.numel() + 1, dtype=torch.bfloat16, device=dev)[1:].view(k.shape)
    odd.copy_(k)
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16)
    got = ada.paged_attention(q.to(dev), odd, v.to(dev), table.to(dev), ln.to(dev))
    want, _ = attend64(q, k, v, table, ln, 0.125)
    assert ((got.cpu().double() - want).abs() <= _bar(q, k, v, ln, 0.125, None, None, want)).all()


def test_offsets_past_32_bits(cuda_device):
    """A pool of more than 2^32 elements whose used pages are its last ones."""
    dev = cuda_device
    pages, hkv, page, d = 2 ** 20 + 64, 8, 8, 64 + 0
    assert pages * hkv * page * d > 2 ** 32
    k = torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(6)
    ks, vs, table, ln = build_pool([60], page, hkv, d, torch.bfloat16, g, spare=0)
    n = ks.shape[0]
    k[-n:] = ks.to(dev)
    v = torch.zeros_like(k)
    v[-n:] = vs.to(dev)
    q = torch.randn(1, 8, d, generator=g).to(torch.bfloat16)
    got = ada.paged_attention(q.to(dev), k, v, (table + (pages - n) * (table >= 0).int()).to(dev), ln.to(dev))
    want, _ = attend64(q, ks, vs, table, ln, d ** -0.5)
    assert ((got.cpu().double() - want).abs() <= _bar(q, ks, vs, ln, d ** -0.5, None, None, want)).all()
    nk = torch.randn(1, hkv, 1, d, generator=g).to(torch.bfloat16).to(dev)
    ada.paged_append(nk, nk, k, v, (table + (pages - n) * (table >= 0).int()).to(dev), ln.to(dev))
    p = int(table[0, 59 // page]) + pages - n
    assert torch.equal(k[p, :, 59 % page], nk[0, :, 0])
    del k, v


@pytest.mark.parametrize("dtype,page,width", [(torch.float32, 42966, 49981), (torch.bfloat16, 38872, 55245)])
def test_lengths_up_to_the_last_32_bit_number(dtype, page, width, cuda_device):
    """2^31 - 2 and 2^31 - 8 keys, all of them the one page's: keys of 0 and values
    of 1 give 1 and log n. Every sum within a warp counts ones exactly (below
    2^24 a lane); the 296 x 8 pieces join in as many roundings of 2^-24 at most,
    lse rounds its logarithm to 2^-23 of itself besides."""
    dev = cuda_device
    n = page * width
    assert 2 ** 31 - 32 < n < 2 ** 31
    d = 8 if dtype == torch.float32 else 64
    k = torch.zeros(1, 1, page, d, dtype=dtype, device=dev)
    out, lse = ada.paged_attention(torch.ones(1, 1, d, dtype=dtype, device=dev), k, torch.ones_like(k),
                                   torch.zeros(1, width, dtype=torch.int32, device=dev),
                                   torch.tensor([n], dtype=torch.int32, device=dev), return_lse=True)
    _lib.poll_device_status(dev)
    joins = 296 * 8 * 2.0 ** -24
    assert (out.double() - 1).abs().max().item() <= joins + HALF[dtype]
    assert abs(lse.item() - math.log(n)) <= joins + 2.0 ** -22 * math.log(n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_longer_than_any_sequence(dtype, cuda_device):
    """A mask described over 2^31 + 5 keys (one element, expanded) hides them all."""
    dev = cuda_device
    g = torch.Generator().manual_seed(14)
    k, v, table, ln = (t.to(dev) for t in build_pool([40], 16, 2, 64, dtype, g))
    q = torch.randn(1, 4, 64, generator=g).to(dtype).to(dev)
    m = torch.zeros(1, 1, dtype=torch.bool, device=dev).expand(1, 2 ** 31 + 5)
    out, lse = ada.paged_attention(q, k, v, table, ln, key_mask=m, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    open_ = ada.paged_attention(q, k, v, table, ln, key_mask=~m[:, :1].expand(1, 2 ** 31 + 5))
    assert torch.equal(open_, ada.paged_attention(q, k, v, table, ln))


def test_bad_ids_are_left_out_and_recorded(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(7)
    for dtype in (torch.bfloat16, torch.float32):
        k, v, table, ln = build_pool([40, 40, 40], 16, 2, 64, dtype, g)
        q = torch.randn(3, 4, 64, generator=g).to(dtype)
        want, _ = attend64(q, k, v, table, ln, 0.125)
        keep = torch.ones(1, 40, dtype=torch.bool)
        keep[0, 16:32] = False
        want[1:2], _ = attend64(q[1:2], k, v, table[1:2], ln[1:2], 0.125, keep)
        bad = table.clone()
        bad[1, 1] = 2 ** 30  # the sequence's middle page
        args = (q.to(dev), k.to(dev), v.to(dev))
        got = ada.paged_attention(*args, bad.to(dev), ln.to(dev)).cpu()
        with pytest.raises(ada.KernelError):
            _lib.poll_device_status(dev)
        assert ((got.double() - want).abs() <= _bar(q, k, v, ln, 0.125, None, None, want)).all()
        got = ada.paged_attention(*args, table.to(dev), ln.to(dev),
                                  seqs=torch.tensor([0, 9, -1], dtype=torch.int32, device=dev)).cpu()
        with pytest.raises(ada.KernelError):
            _lib.poll_device_status(dev)
        assert (got[1:] == 0).all() and torch.isfinite(got[0]).all()
        long = ln.clone()
        long[2], long[0] = 10 ** 6, -4
        got = ada.paged_attention(*args, table.to(dev), long.to(dev)).cpu()
        with pytest.raises(ada.KernelError):
            _lib.poll_device_status(dev)
        assert (got[0] == 0).all()
    _lib.poll_device_status(dev)  # read and cleared


def test_results_repeat_and_replay(cuda_device):
    """The same bits again, on another stream and from two captured graphs in turn;
    a replay sees new lengths and tables."""
    dev = cuda_device
    g = torch.Generator().manual_seed(8)
    k, v, table, ln = (t.to(dev) for t in build_pool([900, 33, 2000, 0], 16, 2, 128, torch.bfloat16, g))
    q = torch.randn(4, 16, 128, generator=g).to(torch.bfloat16).to(dev)
    first = ada.paged_attention(q, k, v, table, ln)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        again = ada.paged_attention(q, k, v, table, ln)
    torch.cuda.synchronize()
    assert torch.equal(first, again)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ada.paged_attention(q, k, v, table, ln))
        graphs.append(gr)
    short = torch.tensor([9, 33, 1000, 0], dtype=torch.int32, device=dev)
    full = ln.clone()
    want_short = ada.paged_attention(q, k, v, table, short)
    for lens, want in ((full, first), (short, want_short), (full, first)):
        ln.copy_(lens)
        for gr, out in zip(graphs, outs):
            out.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_no_gradient_and_device_refusals(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(9)
    k, v, table, ln = (t.to(dev) for t in build_pool([20], 16, 2, 64, torch.float32, g))
    q = torch.randn(1, 4, 64, generator=g).to(dev)
    with pytest.raises(RuntimeError, match="no gradient"):
        ada.paged_attention(q.requires_grad_(), k, v, table, ln)
    q = q.detach()
    with pytest.raises(RuntimeError):
        ada.paged_attention(q.cpu(), k, v, table, ln)
    with pytest.raises(RuntimeError):
        ada.paged_attention(q, k, v, table.cpu(), ln)
    with pytest.raises(TypeError):
        ada.paged_attention(q, k, v, table.long(), ln)
    with pytest.raises(TypeError):
        ada.paged_attention(q.half(), k, v, table, ln)
    with pytest.raises(ada.ShapeError):
        ada.paged_attention(q[:, :3], k, v, table, ln)
    with pytest.raises(ada.ShapeError):
        ada.paged_attention(q, k, v, table, ln, key_mask=torch.ones(2, 20, dtype=torch.bool, device=dev))
    assert ada.paged_attention(q[:0], k, v, table[:0], ln[:0]).shape == (0, 4, 64)


# ---- append --------------------------------------------------------------------

def _append64(x, pages, table, lens, new, scale, seqs=None):
    want = pages.float().double()
    page = pages.shape[2]
    for b in range(x.shape[0]):
        s = b if seqs is None else seqs[b]
        for t in range(int(new[b])):
            pos = int(lens[s]) - int(new[b]) + t
            y = x[b, :, t].float()
            if pages.dtype == torch.float8_e4m3fn:
                if scale is not None:
                    y = y / scale[:, None]
                y = y.clamp(-448, 448).to(torch.float8_e4m3fn).float()
            want[int(table[s, pos // page]), :, pos % page] = y.double()
    return want


@pytest.mark.parametrize("src,dst", [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None),
                                     (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.float8_e4m3fn),
                                     (torch.float32, torch.float8_e4m3fn)])
@pytest.mark.parametrize("b,hkv,n,d,page", [(1, 1, 1, 64, 16), (5, 2, 1, 128, 16), (3, 4, 70, 64, 8), (2, 3, 33, 33, 5),
                                            (4, 12, 100, 80, 24), (2, 1, 9, 1, 1)])
def test_append_writes_its_tokens_and_nothing_else(b, hkv, n, d, page, src, dst, cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(b + n + d)
    dst = dst or src
    new = torch.randint(0, n + 1, (b,), generator=g, dtype=torch.int32)
    new[0] = n
    past = torch.randint(0, 40, (b,), generator=g, dtype=torch.int32)
    lens = (past + new).tolist()
    kp, vp, table, ln = build_pool(lens, page, hkv, d, dst, g)
    x = torch.randn(b, n, 2, hkv, d, generator=g)
    x[0, 0, 0, 0, 0] = math.inf  # saturates in 8 bits
    x[0, 0, 1, 0, 0] = -1e9 if src != torch.float16 else -6e4
    x = x.to(src)
    k, v = x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)
    scale = (0.01 + torch.rand(hkv, generator=g)) if dst == torch.float8_e4m3fn and b > 1 else None
    xd = x.to(dev)
    gk, gv = kp.to(dev), vp.to(dev)
    ada.paged_append(xd[:, :, 0].transpose(1, 2), xd[:, :, 1].transpose(1, 2), gk, gv, table.to(dev), ln.to(dev),
                     new.to(dev), k_scale=None if scale is None else scale.to(dev),
                     v_scale=None if scale is None else scale.to(dev))
    torch.cuda.synchronize()
    _lib.poll_device_status(dev)
    for got, x0, old in ((gk, k, kp), (gv, v, vp)):
        want = _append64(x0, old, table, ln, new, scale)
        assert torch.equal(got.cpu().float().double(), want)


def test_append_picks_refuses_and_bounds(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(11)
    kp, vp, table, ln = build_pool([20, 40, 9], 16, 2, 64, torch.bfloat16, g)
    k = torch.randn(3, 2, 4, 64, generator=g).to(torch.bfloat16)
    # sequence 1 twice: the first row writes it; a row outside the table writes nothing
    gk, gv = kp.to(dev), vp.to(dev)
    ada.paged_append(k.to(dev), k.to(dev), gk, gv, table.to(dev), ln.to(dev),
                     seqs=torch.tensor([1, 1, 7], dtype=torch.int32, device=dev))
    with pytest.raises(ada.KernelError):
        _lib.poll_device_status(dev)
    want = _append64(k[:1], kp, table, ln, [4], None, [1])
    assert torch.equal(gk.cpu().double(), want)
    # more tokens than the sequence has, more than given, negative: left out
    for new in (50, 5, -1):
        gk = kp.to(dev)
        ada.paged_append(k.to(dev), k.to(dev), gk, vp.to(dev), table.to(dev), ln.to(dev),
                         torch.tensor([0, new, 0], dtype=torch.int32, device=dev))
        with pytest.raises(ada.KernelError):
            _lib.poll_device_status(dev)
        assert torch.equal(gk.cpu(), kp)
    # a page id outside the pool: its tokens are left out
    bad = table.clone()
    bad[1, 2] = -7
    gk = kp.to(dev)
    ada.paged_append(k.to(dev), k.to(dev), gk, vp.to(dev), bad.to(dev), ln.to(dev),
                     torch.tensor([0, 4, 0], dtype=torch.int32, device=dev))
    with pytest.raises(ada.KernelError):
        _lib.poll_device_status(dev)
    assert torch.equal(gk.cpu(), kp)
    with pytest.raises(TypeError):
        ada.paged_append(k.to(dev).half(), k.to(dev).half(), kp.to(dev), vp.to(dev), table.to(dev), ln.to(dev))
    with pytest.raises(ada.ShapeError):
        ada.paged_append(k.to(dev)[:, :1], k.to(dev)[:, :1], kp.to(dev), vp.to(dev), table.to(dev), ln.to(dev))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 16])
@pytest.mark.parametrize("above", [14.0, 18.0, 20.0])
def test_what_stands_behind_an_attention_sink_is_kept(above, group, d, dtype, cuda_device):
    """One key with a score far above all others and a value of 0 (a sink): the
    output is the others' sum alone, (n - 1) e^-a / (1 + (n - 1) e^-a). A
    probability enters a 16-bit product with 2^-16 of itself (bf16) or with
    2^-22 of itself and 2^-40 of the largest one (fp16), the fp32 exponent and
    exponential add 2^-19, the output half a step (below the type's normal
    values, as fp16's output at 20 is, half of its smallest). 300 sequences of 4096 keys
    (over the same pages) make units that one warp takes whole: its sums of n
    equal terms take up to n dependent fp32 additions, each off by at most 2^-24
    of a running sum that is no larger than the final one, n 2^-24 in all. The
    sum of p has the same error, lse that much absolutely beside its own 2^-23."""
    dev = cuda_device
    n, page, hkv, b = 4096, 64, 4, 300
    k, v = torch.zeros(n // page, hkv, page, d), torch.ones(n // page, hkv, page, d)
    k[0, :, 0, 0], v[0, :, 0] = above, 0.0
    qd = torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype
    q = torch.zeros(b, hkv * group, d, dtype=qd)
    q[:, :, 0] = 1.0
    table = torch.arange(n // page, dtype=torch.int32).expand(b, -1).contiguous()
    ln = torch.full((b,), n, dtype=torch.int32)
    out, lse = ada.paged_attention(q.to(dev), k.to(dtype).to(dev), v.to(dtype).to(dev), table.to(dev), ln.to(dev),
                                   scale=1.0, return_lse=True)
    rest = (n - 1) * math.exp(-above)
    want = rest / (1 + rest)
    lost = {torch.bfloat16: 2.0 ** -16, torch.float32: 0.0}.get(dtype, 2.0 ** -22 + 2.0 ** -40 * math.exp(above))
    step = torch.finfo(qd).smallest_normal * HALF[qd]
    assert (out.double() - want).abs().max().item() <= step + want * (HALF[qd] + lost + 2.0 ** -19 + n * 2.0 ** -24)
    assert (lse.double() - above - math.log1p(rest)).abs().max().item() <= 2.0 ** -19 + n * 2.0 ** -24 + 2.0 ** -23 * above


def test_forward_mode_is_refused(cuda_device):
    fwd = torch.autograd.forward_ad
    dev = cuda_device
    g = torch.Generator().manual_seed(13)
    k, v, table, ln = (t.to(dev) for t in build_pool([20], 16, 2, 64, torch.float32, g))
    q = torch.randn(1, 4, 64, generator=g).to(dev)
    m = torch.zeros(1, 20, device=dev)
    new = torch.randn(1, 2, 1, 64, generator=g).to(dev)
    want = ada.paged_attention(q, k, v, table, ln, key_mask=m)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for args, kw in (((dual(q), k, v), {}), ((q, dual(k), v), {}), ((q, k, dual(v)), {}),
                         ((q, k, v), dict(key_mask=dual(m)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ada.paged_attention(*args, table, ln, **kw)
        before = k.clone()
        with pytest.raises(RuntimeError, match="forward-mode"):
            ada.paged_append(dual(new), new, k, v, table, ln)
        assert torch.equal(k, before)
        assert torch.equal(ada.paged_attention(q, k, v, table, ln, key_mask=m), want)
        c = ada.PagedKVCache(1, 4, 8, 2, 32, max_sequences=1, max_pages_per_sequence=4)
        att = ada.AdaAttention(embed_dim=64, num_heads=2, causal=True, enable_adaptive_rank=False).to(dev).eval()
        with pytest.raises(RuntimeError, match="forward-mode"):
            att.forward_cached(dual(torch.randn(1, 1, 64, device=dev)), c, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_other_mask_types(dtype, cuda_device):
    """0/1 masks of whole numbers are refused (added, they would hide nothing),
    uint8 is bool, and a float64 mask of its lowest value everywhere leaves a uniform row as in 32 bits."""
    dev = cuda_device
    g = torch.Generator().manual_seed(15)
    k, v, table, ln = build_pool([50], 16, 2, 64, dtype, g)
    q = torch.randn(1, 4, 64, generator=g).to(dtype)
    m = torch.rand(1, 50, generator=g) < 0.5
    up = [t.to(dev) for t in (q, k, v, table, ln)]
    run = lambda mask, **kw: ada.paged_attention(*up, key_mask=mask.to(dev), **kw)
    for whole in (torch.int64, torch.int32, torch.int16, torch.int8):
        with pytest.raises(TypeError):
            run(m.to(whole))
    assert torch.equal(run(m.to(torch.uint8)), run(m))
    want, want_lse = run(torch.full((1, 50), torch.finfo(torch.float32).min), return_lse=True)
    got, lse = run(torch.full((1, 50), torch.finfo(torch.float64).min, dtype=torch.float64), return_lse=True)
    assert torch.equal(got, want) and torch.equal(lse, want_lse) and (got != 0).any()
    f = torch.randn(1, 50, generator=g).masked_fill(~m, -math.inf)
    assert torch.equal(run(f.double()), run(f))
    assert (run(torch.full((1, 50), -math.inf, dtype=torch.float64)) == 0).all()
    assert torch.isnan(run(torch.full((1, 50), math.nan, dtype=torch.float64)).float()).all()
