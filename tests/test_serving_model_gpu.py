"""The serving operators together, as the decoder uses them: prefill, decoding
over a paged cache with forks, copies, frees and compaction in between, and
scores, against the decoder's own full forward.

Tolerance: the cached path computes the same layers with attention in another
order of sums and one rounding per layer that may tip (16-bit types). Logits of
this small model with 0.02-size weights stay below 1; a layer adds a few
roundings of values of size up to 4, half a step of 2^-8 (bf16) each, so two
paths differ by at most layers * 8 roundings * 4 * 2^-9 through the head's
0.02 sqrt(E) gain.
"""

import pytest
import torch

import adaattn_b200 as ada
from adaattn_b200 import PrecisionMode, _lib
from adaattn_b200.host_model import AdaptiveTransformer

pytestmark = pytest.mark.gpu

V, E, H, LAYERS = 211, 256, 4, 3


def _model(dev, dtype, **kw):
    torch.manual_seed(0)
    m = AdaptiveTransformer(V, E, H, LAYERS, 512, max_seq_len=96, dropout=0.0, enable_adaptive_rank=False,
                            enable_adaptive_precision=False, causal=True,
                            default_precision={torch.float32: PrecisionMode.FP32, torch.bfloat16: PrecisionMode.BF16,
                                               torch.float16: PrecisionMode.FP16}[dtype], **kw)
    m.init_gpt2_weights()
    return m.to(dev).to(dtype).eval()


def _bar(dtype):
    return {torch.bfloat16: LAYERS * 8 * 4 * 2.0 ** -9, torch.float16: LAYERS * 8 * 4 * 2.0 ** -12,
            torch.float32: 1e-5}[dtype] * 0.02 * E ** 0.5


def _ids(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decoding_follows_the_full_forward(dtype, cuda_device):
    dev = cuda_device
    m = _model(dev, dtype)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (4, 60), generator=g).to(dev)
    lengths = [17, 1, 32, 9]
    cache = m.make_cache(64, 8, max_sequences=8)
    seqs = _ids([5, 0, 3, 6], dev)
    logits, granted = m.prefill(ids[:, :32], cache, seqs, _ids(lengths, dev))
    assert granted.tolist() == lengths
    with torch.no_grad():
        full = m(ids)
    at = torch.tensor(lengths, device=dev)
    rows = torch.arange(4, device=dev)
    assert (logits.float() - full[rows, at - 1].float()).abs().max().item() <= _bar(dtype)
    for step in range(20):
        if step == 7:      # room is made: a sequence comes and goes, the pool closes up
            m.prefill(ids[:1, :30], cache, _ids([1], dev))
            cache.copy([3], [2])
            cache.free([1, 2])
            cache.compact()
        if step == 12:     # the sequence in row 3 goes on in row 7, from the pages it shares with it
            cache.fork([3], [7])
            cache.free([3])
            seqs = _ids([5, 0, 7, 6], dev)
        logits, granted = m.decode_step(ids[rows, at], cache, seqs)
        assert granted.tolist() == [1, 1, 1, 1]
        assert (logits.float() - full[rows, at].float()).abs().max().item() <= _bar(dtype)
        at = at + 1
    _lib.poll_device_status(dev)
    assert cache.seq_lens[seqs.long()].tolist() == at.tolist()
    cache.free([0, 1, 2, 3, 4, 5, 6, 7])
    assert int(cache.ref_counts.abs().sum()) == 0


def test_branches_diverge_from_shared_pages(cuda_device):
    """Two branches of one prompt continue differently; each follows its own full forward."""
    dev, dtype = cuda_device, torch.bfloat16
    m = _model(dev, dtype)
    g = torch.Generator().manual_seed(2)
    a = torch.randint(0, V, (1, 40), generator=g).to(dev)
    b = a.clone()
    b[:, 21:] = torch.randint(0, V, (1, 19), generator=g).to(dev)
    cache = m.make_cache(24, 8, max_sequences=4)
    m.prefill(a[:, :21], cache, _ids([0], dev))
    cache.fork([0], [1])
    assert int((cache.ref_counts == 2).sum()) == 3
    with torch.no_grad():
        fa, fb = m(a), m(b)
    for t in range(21, 40):
        logits, granted = m.decode_step(torch.stack([a[0, t], b[0, t]]), cache, _ids([0, 1], dev))
        assert granted.tolist() == [1, 1]
        want = torch.stack([fa[0, t], fb[0, t]])
        assert (logits.float() - want.float()).abs().max().item() <= _bar(dtype)
    assert int((cache.ref_counts == 2).sum()) == 2  # the two full pages of the common prompt


def test_eight_bit_cache(cuda_device):
    """An E4M3 cache: keys and values off by up to 2^-4 of themselves, so the
    attention's change is bounded by its inputs' size; the logits stay close."""
    dev = cuda_device
    m = _model(dev, torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, V, (3, 30), generator=g).to(dev)
    cache = m.make_cache(32, 16, max_sequences=3, dtype=torch.float8_e4m3fn,
                         k_scale=torch.full((LAYERS, H), 0.01), v_scale=torch.full((LAYERS, H), 0.01))
    m.prefill(ids[:, :20], cache, _ids([0, 1, 2], dev))
    with torch.no_grad():
        full = m(ids)
    for t in range(20, 30):
        logits, _ = m.decode_step(ids[:, t], cache, _ids([0, 1, 2], dev))
        err = (logits.float() - full[:, t].float()).abs().max().item()
        assert err <= _bar(torch.bfloat16) + LAYERS * 2.0 ** -4 * 0.02 * E ** 0.5


def test_a_captured_step_replays(cuda_device):
    """One captured decoding step, replayed token by token, against eager steps on a second cache."""
    dev, dtype = cuda_device, torch.bfloat16
    m = _model(dev, dtype)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, V, (2, 40), generator=g).to(dev)
    seqs = _ids([0, 1], dev)
    caches = [m.make_cache(24, 8, max_sequences=2) for _ in range(2)]
    for c in caches:
        m.prefill(ids[:, :13], c, seqs)
    token = ids[:, 13].clone()
    side = torch.cuda.Stream(dev)
    scratch = m.make_cache(24, 8, max_sequences=2)
    with torch.cuda.stream(side):
        m.prefill(ids[:, :13], scratch, seqs)
        m.decode_step(token, scratch, seqs)  # warm-up on a cache of its own
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        logits, granted = m.decode_step(token, caches[0], seqs)
    for t in range(13, 33):
        token.copy_(ids[:, t])
        gr.replay()
        want, _ = m.decode_step(ids[:, t], caches[1], seqs)
        torch.cuda.synchronize()
        assert granted.tolist() == [1, 1]
        assert torch.equal(logits, want)
    assert torch.equal(caches[0].data.view(torch.uint8), caches[1].data.view(torch.uint8))


def test_a_pool_that_runs_out(cuda_device):
    dev = cuda_device
    m = _model(dev, torch.bfloat16)
    ids = torch.randint(0, V, (2, 30), generator=torch.Generator().manual_seed(5)).to(dev)
    cache = m.make_cache(5, 8, max_sequences=2)
    _, granted = m.prefill(ids[:, :16], cache, _ids([0, 1], dev))
    assert granted.tolist() == [16, 16]
    seqs = _ids([0, 1], dev)
    _, granted = m.decode_step(ids[:, 16], cache, seqs)
    assert granted.tolist() == [1, 0]
    before = cache.data[:, cache.page_table[1, :2].long()].clone()
    _, granted = m.decode_step(ids[:, 17], cache, seqs)
    assert granted.tolist() == [1, 0] and cache.seq_lens.tolist() == [18, 16]
    assert torch.equal(before, cache.data[:, cache.page_table[1, :2].long()])
    _lib.poll_device_status(dev)


def test_sequences_end_at_the_models_length(cuda_device):
    """max_seq_len 96 in pages of 20: the fifth page has room for four more tokens than the model has positions."""
    dev = cuda_device
    m = _model(dev, torch.bfloat16)
    ids = torch.randint(0, V, (2, 96), generator=torch.Generator().manual_seed(7)).to(dev)
    cache = m.make_cache(12, 20, max_sequences=3)
    _, granted = m.prefill(ids[:, :95], cache, _ids([0, 2], dev), _ids([95, 200], dev))
    assert granted.tolist() == [95, 95]
    seqs = _ids([0, 2], dev)
    assert m.decode_step(ids[:, 95], cache, seqs)[1].tolist() == [1, 1]
    assert m.decode_step(ids[:, 95], cache, seqs)[1].tolist() == [0, 0]
    assert cache.seq_lens.tolist() == [96, 0, 96]
    _lib.poll_device_status(dev)
    assert m.decode_step(ids[:, 0], cache, _ids([1, 9], dev))[1].tolist() == [1, 0]  # row 9 does not exist
    with pytest.raises(ada.KernelError):
        _lib.poll_device_status(dev)
    with pytest.raises(ada.ShapeError):
        m.prefill(torch.zeros(1, 97, dtype=torch.int64, device=dev), cache, _ids([0], dev))


def test_score_and_its_gradient(cuda_device):
    """score() against log_softmax of the same logits; its gradient reaches the
    weights like that of the plain formula, to the roundings of the bf16 logits' gradient."""
    dev = cuda_device
    m = _model(dev, torch.bfloat16)
    ids = torch.randint(0, V, (3, 25), generator=torch.Generator().manual_seed(6)).to(dev)
    with torch.no_grad():  # (with autograd the forward takes other LayerNorm kernels: other bf16 logits)
        r = m.score(ids, top_k=4)
        logp = torch.log_softmax(m(ids)[:, :-1].double(), -1)
    assert r.logprobs.shape == (3, 24) and r.top_tokens.shape == (3, 24, 4)
    want = logp.gather(-1, ids[:, 1:, None])[..., 0]
    assert (r.logprobs.double() - want).abs().max().item() <= 1e-5
    assert (r.entropy.double() + (logp.exp() * logp).sum(-1)).abs().max().item() <= 1e-5
    w = m.blocks[1].ff[0].weight
    g1, = torch.autograd.grad(m.score(ids).logprobs.sum(), w)
    plain = torch.log_softmax(m(ids)[:, :-1].float(), -1).gather(-1, ids[:, 1:, None]).sum()
    g2, = torch.autograd.grad(plain, w)
    assert ((g1.float() - g2.float()).norm() / g2.float().norm()).item() <= 2.0 ** -6


def test_refusals(cuda_device):
    dev = cuda_device
    x = torch.randn(1, 1, 64, device=dev, dtype=torch.bfloat16)
    c = ada.PagedKVCache(1, 4, 8, 2, 32, max_sequences=1, max_pages_per_sequence=4)
    for kw, err in ((dict(causal=False, enable_adaptive_rank=False), "causal"),
                    (dict(causal=True), "enable_adaptive_rank")):
        m = ada.AdaAttention(embed_dim=64, num_heads=2, **kw).to(dev).bfloat16().eval()
        with pytest.raises(RuntimeError, match=err):
            m.forward_cached(x, c, 0)
    m = ada.AdaAttention(embed_dim=64, num_heads=2, causal=True, enable_adaptive_rank=False,
                         dropout=0.1).to(dev).bfloat16()
    with pytest.raises(RuntimeError, match="eval"):
        m.forward_cached(x, c, 0)
    with pytest.raises(ada.ShapeError):
        m.eval().forward_cached(x[..., :32], c, 0)
    with pytest.raises(IndexError):
        m.forward_cached(x, c, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_several_tokens_after_cached_ones_are_recorded(dtype, cuda_device):
    """N > 1 attends within its own tokens: a sequence that holds others is left
    out and recorded, its neighbours in the batch and empty rows are not; token by token it goes on."""
    dev = cuda_device
    prec = {torch.float32: PrecisionMode.FP32, torch.bfloat16: PrecisionMode.BF16}[dtype]
    att = ada.AdaAttention(embed_dim=E, num_heads=H, causal=True, enable_adaptive_rank=False, dropout=0.0,
                           enable_adaptive_precision=False, default_precision=prec).to(dev).to(dtype).eval()
    x = torch.randn(3, 12, E, generator=torch.Generator().manual_seed(8)).to(dev).to(dtype)
    cache = ada.PagedKVCache(1, 16, 8, H, E // H, max_sequences=4, max_pages_per_sequence=4, dtype=dtype)
    cache.reserve([0], [5])
    att.forward_cached(x[:1, :5], cache, 0, seqs=_ids([0], dev))
    _lib.poll_device_status(dev)
    # row 0 holds five tokens; row 2 is new; row 3 takes part with no token at all
    cache.reserve([0, 2], [7, 12])
    before, full = cache.data.clone(), att.forward_cached(x[1:2], _fresh(cache), 0, seqs=_ids([1], dev))
    got = att.forward_cached(x, cache, 0, seqs=_ids([0, 2, 3], dev), new_tokens=_ids([7, 12, 0], dev))
    with pytest.raises(ada.KernelError):
        _lib.poll_device_status(dev)
    # (the library's fp32 products add 256 terms in another order for another batch)
    tol = {torch.bfloat16: 2.0 ** -7, torch.float32: 1e-5}[dtype]
    assert (got[1].float() - full[0].float()).abs().max().item() <= tol * full.float().abs().max().item()
    pages = cache.page_table[0, :2].long()
    assert torch.equal(cache.data[:, pages], before[:, pages])
    # the refused tokens one by one, as the documentation puts it
    cache.free([0])
    whole = att(x[:1], x[:1], x[:1])[0]
    for t in range(12):
        cache.reserve([0], [1])
        y = att.forward_cached(x[:1, t:t + 1], cache, 0, seqs=_ids([0], dev))
        assert (y[0, 0].float() - whole[0, t].float()).abs().max().item() <= tol * whole.float().abs().max().item()
    _lib.poll_device_status(dev)


def _fresh(cache):
    """A cache of the same shape with room for 12 tokens in row 1."""
    p, hkv, page, d = cache.data.shape[1:]
    c = ada.PagedKVCache(1, p, page, hkv, d, max_sequences=4, max_pages_per_sequence=4, dtype=cache.dtype)
    c.reserve([1], [12])
    return c


def test_score_through_a_mask(cuda_device):
    """A decoder without causal=True scores through a causal mask; without one it is refused."""
    dev = cuda_device
    m = _model(dev, torch.float32)
    ids = torch.randint(0, V, (2, 20), generator=torch.Generator().manual_seed(10)).to(dev)
    with torch.no_grad():
        want = m.score(ids)
        for b in m.blocks:
            b.attention.causal = False
        with pytest.raises(RuntimeError, match="causal"):
            m.score(ids)
        got = m.score(ids, attention_mask=torch.ones(2, 1, 20, 20, dtype=torch.bool, device=dev).tril())
    # the same sums of 20 keys; logits of size below 1 to fp32 roundings through three layers
    assert (got.logprobs - want.logprobs).abs().max().item() <= 2 * _bar(torch.float32) + 2.0 ** -20
