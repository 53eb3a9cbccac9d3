"""Log probabilities of given tokens (ada_token_logprobs) and their gradient
against 64-bit evaluations.

Tolerances. Forward, with x = z - max of size up to X and V terms: the sums
hold each term with the exponential's 2^-21 (its argument x log2 e is rounded
to 2^-24 X) and at most V / 256 / parts + 40 dependent additions; so s is off
by r = 2^-21 + X 2^-23 + (V / 256 + 40) 2^-24 relative, a log by as much
absolutely plus 2^-23 of its value, and the entropy by r times the mean of
|x| as well. The values then carry fp32 roundings of numbers up to |z|.
Gradient: fp32 terms off by the same r of their size, rounded once to the
logits' type (half a step).
"""

import math

import pytest
import torch

import adaattn_b200 as ada
from adaattn_b200 import _lib
from adaattn_b200.scoring import token_logprobs_backward

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _make(rows, vocab, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + rows + vocab)
    z = torch.randn(rows, vocab, generator=g) * spread * (0.2 + torch.rand(rows, 1, generator=g))
    t = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 2:
        t[1] = -100
    return z.to(dtype), t


def _exact(z, t, ignore=-100):
    z = z.double()
    lse = torch.logsumexp(z, -1)
    logp = z - lse[:, None]
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    lp = logp.gather(1, t.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    return torch.where(t == ignore, torch.zeros_like(lp), lp), ent, lse, logp


def _r(z):
    zf = z.double()
    zf = zf[torch.isfinite(zf)]
    x = (zf.max() - zf.min()).item() if zf.numel() else 0.0
    return 2.0 ** -21 + min(x, 120.0) * 2.0 ** -23 + (z.shape[-1] / 256 + 40) * 2.0 ** -24, x


def _top(z, k):
    o = torch.sort(z.double(), dim=-1, descending=True, stable=True).indices
    return o[..., :k]


def _off(got, want):
    """Largest difference; equal infinities differ by nothing."""
    got = got.cpu().double()
    return torch.where(got == want, torch.zeros_like(want), (got - want).abs()).max().item()


def _check(z, t, dev, top=0, zd=None):
    zd = z.to(dev) if zd is None else zd
    got = ada.token_logprobs(zd, t.to(dev), top_k=top)
    torch.cuda.synchronize()
    _lib.poll_device_status(dev)
    lp, ent, lse, logp = _exact(z, t)
    r, x = _r(z)
    big = z.double()[torch.isfinite(z.double())].abs().max().item() + math.log(z.shape[1])
    bar = 2 * r + 2.0 ** -22 * big
    assert _off(got.logprobs, lp) <= bar
    assert _off(got.lse, lse) <= bar
    assert _off(got.entropy, ent) <= bar + 2 * r * (ent.max().item() + 1)
    if top:
        ids = _top(z, top)
        assert torch.equal(got.top_tokens.cpu(), ids)
        assert _off(got.top_logprobs, logp.gather(1, ids)) <= bar
    else:
        assert got.top_tokens is None and got.top_logprobs is None
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 7, 3), (3, 64, 64), (5, 1000, 20), (2, 4096, 5), (4, 4097, 0),
                                            (1, 50257, 20), (37, 50257, 5), (300, 5003, 1), (2, 131072, 64),
                                            (3, 200003, 7), (160, 8192, 32), (700, 300, 64)])
def test_matches_formula(rows, vocab, top, dtype, cuda_device):
    z, t = _make(rows, vocab, dtype)
    _check(z, t, cuda_device, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(47, 0), (1, 0), (0, 1), (3, 5), (8, 7)])
def test_row_strides_and_alignment(pad, offset, dtype, cuda_device):
    z, t = _make(9, 2043, dtype)
    buf = torch.full((9 * (2043 + pad) + offset + 8,), math.nan, dtype=dtype, device=cuda_device)
    zd = buf[offset:offset + 9 * (2043 + pad)].view(9, 2043 + pad)[:, :2043]
    zd.copy_(z)
    _check(z, t, cuda_device, 10, zd)


def test_leading_dimensions(cuda_device):
    """The next-token slice of a decoder's padded logits, one row, four
    dimensions, a transposed layout. Layouts of other alignment add a row's
    terms in another order, so each result is within the forward's bar of the
    64-bit value and two of them within twice that of one another."""
    dev = cuda_device
    z, t = _make(4 * 6, 1003, torch.bfloat16)
    r, _ = _r(z)
    bar = 2 * (2 * r + 2.0 ** -22 * (z.double().abs().max().item() + math.log(1003))) + 4 * r * math.log(1003)
    near = lambda a, b: a.shape == b.shape and (a - b).abs().max().item() <= bar
    store = torch.full((4, 7, 1024), math.nan, dtype=torch.bfloat16, device=dev)
    view = store[:, :-1, :1003]
    view.copy_(z.view(4, 6, 1003))
    got = ada.token_logprobs(view, t.view(4, 6).to(dev), top_k=3)
    flat = ada.token_logprobs(z.to(dev), t.to(dev), top_k=3)
    assert near(got.logprobs.reshape(-1), flat.logprobs) and got.logprobs.shape == (4, 6)
    assert torch.equal(got.top_tokens.reshape(-1, 3), flat.top_tokens) and got.top_tokens.shape == (4, 6, 3)
    got = ada.token_logprobs(z[0].to(dev), t[0].to(dev), top_k=3)
    assert got.logprobs.shape == () and torch.equal(got.top_tokens, flat.top_tokens[0])
    got = ada.token_logprobs(view.unflatten(1, (2, 3)), t.view(4, 2, 3).to(dev))
    assert near(got.lse.reshape(-1), flat.lse) and got.lse.shape == (4, 2, 3)
    got = ada.token_logprobs(z.to(dev).t().contiguous().t(), t.to(torch.int32).to(dev))
    assert near(got.entropy, flat.entropy)
    empty = ada.token_logprobs(z[:0].to(dev), t[:0].to(dev), top_k=3)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_take_the_lowest_tokens(dtype, cuda_device):
    dev = cuda_device
    for vocab in (100, 5000, 50257):
        z = torch.zeros(4, vocab, dtype=dtype)
        z[1, vocab // 2:] = 1.0              # a tie of half the row
        z[2] = torch.arange(vocab) % 7       # many ties at every value
        z[3] = -0.0
        z[3, ::2] = 0.0                      # both zeros are one value
        t = torch.zeros(4, dtype=torch.int64)
        _check(z, t, dev, 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [4099, 50257])
def test_orders_that_fill_the_candidate_list(dtype, vocab, cuda_device):
    up = torch.linspace(-20, 20, vocab)
    z = torch.stack([up, up.flip(0), up.abs(), -up.abs()]).to(dtype)
    _check(z, torch.full((4,), vocab - 1), cuda_device, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_vocabularies(dtype, cuda_device):
    """-inf over most of a row, all of it but one or fewer entries than alternatives."""
    dev = cuda_device
    vocab = 9000
    z, t = _make(6, vocab, dtype)
    z[0, 5:] = -math.inf
    z[1, :-1] = -math.inf
    z[2, :4096] = -math.inf
    z[3, ::2] = -math.inf
    t[:] = torch.tensor([3, vocab - 1, 8000, 1, 0, 4])
    got = _check(z, t, dev, 64)
    assert abs(got.entropy[1].item()) <= 1e-6 and abs(got.logprobs[1].item()) <= 1e-6
    t[0] = 10  # a hidden token
    assert ada.token_logprobs(z.to(dev), t.to(dev)).logprobs[0].item() == -math.inf
    lowest = torch.full((1, vocab), torch.finfo(dtype).min, dtype=dtype)
    got = ada.token_logprobs(lowest.to(dev), t[:1].to(dev), top_k=2)
    assert abs(got.entropy.item() - math.log(vocab)) <= 1e-5
    assert abs(got.logprobs.item() + math.log(vocab)) <= 1e-5 and got.top_tokens.tolist() == [[0, 1]]


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_a_distribution(dtype, cuda_device):
    dev = cuda_device
    z, t = _make(5, 6000, dtype)
    z[0] = -math.inf
    z[1, 77] = math.nan
    z[2, 4500] = math.inf
    z[3, :4200] = math.nan
    x = z.to(dev).requires_grad_()
    t = t.clamp_min(0)
    got = ada.token_logprobs(x, t.to(dev), top_k=3)
    assert torch.isnan(got.logprobs[:4]).all() and torch.isnan(got.entropy[:4]).all()
    assert got.lse[0].item() == -math.inf and torch.isfinite(got.logprobs[4])
    assert got.top_tokens[1, 0].item() == 77 and got.top_tokens[2, 0].item() == 4500
    assert got.top_tokens[3].tolist() == [0, 1, 2] and got.top_tokens[0].tolist() == [0, 1, 2]
    grad, = torch.autograd.grad(got.logprobs.sum(), x)
    assert torch.isnan(grad[:4].float()).all(-1).all() and torch.isfinite(grad[4].float()).all()


def test_tokens_outside_the_vocabulary(cuda_device):
    dev = cuda_device
    z, t = _make(4, 500, torch.float32)
    t = torch.tensor([-1, 500, 3, -100])
    x = z.to(dev).requires_grad_()
    got = ada.token_logprobs(x, t.to(dev))
    with pytest.raises(ada.KernelError):
        _lib.poll_device_status(dev)
    assert torch.isnan(got.logprobs[:2]).all() and torch.isfinite(got.logprobs[2:]).all()
    assert got.logprobs[3].item() == 0
    grad, = torch.autograd.grad(got.logprobs.sum(), x)
    assert torch.isnan(grad[:2]).all() and torch.isfinite(grad[2:]).all() and (grad[3] == 0).all()
    assert torch.equal(ada.token_logprobs(z.to(dev), t.to(dev).clamp_min(0).clamp_max(499), ignore_index=3).logprobs[2:3],
                       torch.zeros(1, device=dev))


def _grad64(z, t, g_lp, g_ent, g_lse):
    z = z.double()
    _, ent, lse, logp = _exact(z, t)
    p = logp.exp()
    hit = torch.zeros_like(z)
    hit[torch.arange(len(t)), t.clamp_min(0)] = 1
    g = g_lp.double() * (t != -100)
    plogp = torch.where(p > 0, logp, torch.zeros_like(p))
    return (g[:, None] * (hit - p) - g_ent.double()[:, None] * p * (plogp + ent[:, None])
            + g_lse.double()[:, None] * p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 17, 0), (6, 1000, 0), (5, 4099, 0), (4, 50257, 47),
                                            (3, 50257, 0), (400, 515, 13)])
def test_gradient_matches_formula(rows, vocab, pad, dtype, cuda_device):
    dev = cuda_device
    z, t = _make(rows, vocab, dtype)
    if rows > 2:
        z[0, vocab // 2:] = -math.inf
        t[0] = 0
    g = torch.Generator().manual_seed(3)
    ups = [torch.randn(rows, generator=g) for _ in range(3)]
    store = torch.zeros(rows, vocab + pad, dtype=dtype, device=dev)
    x = store[:, :vocab]
    x.copy_(z)
    x = x.requires_grad_()
    got = ada.token_logprobs(x, t.to(dev))
    grad, = torch.autograd.grad((got.logprobs, got.entropy, got.lse), x, [u.to(dev) for u in ups])
    assert grad.shape == x.shape and grad.dtype == dtype
    want = _grad64(z, t, *ups)
    r, _ = _r(z)
    _, ent, _, logp = _exact(z, t)
    p = logp.exp()
    size = p * (sum(u.abs().double() for u in ups)[:, None]
                * (1 + torch.where(p > 0, logp.abs(), torch.zeros_like(p)) + ent.abs()[:, None]))
    hit = torch.zeros_like(want)
    hit[torch.arange(rows), t.clamp_min(0)] = ups[0].abs().double()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bar = want.abs() * torch.finfo(dtype).eps / 2 + 4 * r * (size + hit) + tiny
    assert ((grad.cpu().double() - want).abs() <= bar).all()


def test_gradient_matches_differences(cuda_device):
    """Central differences of the forward in steps of 2^-6: truncation h^2 / 6 of
    third derivatives (at most 1 for log p and lse, (1 + |log p|) for H here) and
    the forward's error over h."""
    dev = cuda_device
    z, t = _make(2, 40, torch.float32, spread=1.0)
    x = z.to(dev).requires_grad_()
    f = lambda y: (lambda r: (r.logprobs * 1.5 + r.entropy * 0.7 - r.lse * 0.4).sum())(ada.token_logprobs(y, t.to(dev)))
    grad, = torch.autograd.grad(f(x), x)
    h = 2.0 ** -6
    for i in range(2):
        for j in range(0, 40, 7):
            e = torch.zeros_like(x)
            e[i, j] = h
            num = ((f(x + e) - f(x - e)) / (2 * h)).item()
            assert abs(num - grad[i, j].item()) <= 8 * h * h / 6 * 4 + 2e-5 / h


def test_partial_upstream_gradients(cuda_device):
    """Only some outputs used; an entropy gradient reaches an ignored row, a log probability's does not."""
    dev = cuda_device
    z, t = _make(4, 300, torch.float32)
    x = z.to(dev).requires_grad_()
    zero = torch.zeros(4)
    one = torch.ones(4)
    for pick, ups in (("logprobs", (one, zero, zero)), ("entropy", (zero, one, zero)), ("lse", (zero, zero, one))):
        grad, = torch.autograd.grad(getattr(ada.token_logprobs(x, t.to(dev)), pick).sum(), x)
        assert (grad.cpu().double() - _grad64(z, t, *ups)).abs().max().item() <= 2e-6
        assert (grad[1] == 0).all() == (pick == "logprobs")
    r = ada.token_logprobs(x, t.to(dev), top_k=2)
    assert not r.top_logprobs.requires_grad and not r.top_tokens.requires_grad
    with torch.no_grad():
        assert not ada.token_logprobs(x, t.to(dev)).logprobs.requires_grad


def test_three_dimensional_gradient_of_a_shared_leaf(cuda_device):
    dev = cuda_device
    z, t = _make(12, 203, torch.bfloat16)
    x = z.view(3, 4, 203).to(dev).requires_grad_()
    r = ada.token_logprobs(x[:, :-1], t.view(3, 4)[:, 1:].to(dev))
    r.logprobs.sum().backward()
    zz, tt = z.view(3, 4, 203)[:, :-1].reshape(9, 203), t.view(3, 4)[:, 1:].reshape(9)
    want = _grad64(zz, tt, torch.ones(9), torch.zeros(9), torch.zeros(9)).view(3, 3, 203)
    got = x.grad.cpu().double()
    assert (got[:, -1] == 0).all()
    assert (got[:, :-1] - want).abs().max().item() <= 2.0 ** -9 + 1e-5


def test_captured_forward_and_gradient(cuda_device):
    """Two captured graphs and an eager call share nothing; a replay reads the new logits."""
    dev = cuda_device
    z, t = _make(8, 5000, torch.bfloat16)
    zd, td = z.to(dev), t.to(dev)
    ones = torch.ones(8, device=dev)

    def step():
        r = ada.token_logprobs(zd, td, top_k=4)
        # the gradient's own entry, as a step captured without autograd uses it
        m = zd.float().amax(-1)
        stats = torch.stack([m, r.lse - m], 1)
        return r, token_logprobs_backward(zd[None], td, stats, r.entropy, ones)

    want = step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = step()
        graphs.append((gr, got))
    z2, _ = _make(8, 5000, torch.bfloat16, seed=9)
    for src in (z, z2, z):
        zd.copy_(src)
        want = step()
        for gr, got in graphs:
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(got[0], want[0]):
                assert torch.equal(a, b)
            assert torch.equal(got[1], want[1])


def test_other_streams_repeat_the_bits(cuda_device):
    dev = cuda_device
    z, t = _make(20, 50257, torch.bfloat16)
    zd, td = z.to(dev), t.to(dev)
    a = ada.token_logprobs(zd, td, top_k=20)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        b = ada.token_logprobs(zd, td, top_k=20)
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_refusals(cuda_device):
    dev = cuda_device
    z, t = _make(4, 50, torch.float32)
    z, t = z.to(dev), t.to(dev)
    with pytest.raises(TypeError):
        ada.token_logprobs(z.double(), t)
    with pytest.raises(TypeError):
        ada.token_logprobs(z, t.float())
    with pytest.raises(ada.ShapeError):
        ada.token_logprobs(z, t[:3])
    with pytest.raises(ValueError):
        ada.token_logprobs(z, t, top_k=65)
    with pytest.raises(ValueError):
        ada.token_logprobs(z, t, top_k=51)
    with pytest.raises(RuntimeError):
        ada.token_logprobs(z.cpu(), t)
    with pytest.raises(RuntimeError):
        ada.token_logprobs(z, t.cpu())
    with pytest.raises(Exception):
        ada.token_logprobs(z[:, :0], t)


def _apart(z, t, dev, top):
    """token_logprobs against 64 bits by a bar on z - max alone: the kernel's
    sums hold exponents of x = z - max, and log p and H are differences of such.
    log p adds the roundings of z_t - max and of the log, 2^-23 of their size;
    only lse carries half a step of its own value."""
    got = ada.token_logprobs(z.to(dev), t.to(dev), top_k=top)
    zf = z.double()
    high = zf.amax(-1)
    lp, ent, lse, logp = _exact(zf - high[:, None], t)  # (64 bits hold 10^15 to 0.125 only)
    lse = lse + high
    x = (zf.amax(-1) - zf.amin(-1)).max().item()
    r = 2.0 ** -21 + min(x, 120.0) * 2.0 ** -23 + (z.shape[-1] / 256 + 40) * 2.0 ** -24
    bar = 2 * r + 2.0 ** -22 * (min(x, 200.0) + math.log(z.shape[1]))
    far = 2.0 ** -22 * lp.abs()  # a token far below the maximum
    assert ((got.logprobs.cpu().double() - lp).abs() <= bar + far).all()
    assert _off(got.entropy, ent) <= bar + 2 * r * (ent.max().item() + 1)
    assert ((got.lse.cpu().double() - lse).abs() <= bar + 2.0 ** -23 * lse.abs()).all()
    if top:
        ids = _top(z, top)
        assert torch.equal(got.top_tokens.cpu(), ids)
        want = logp.gather(1, ids)
        assert ((got.top_logprobs.cpu().double() - want).abs() <= bar + 2.0 ** -22 * want.abs()).all()
    return got, bar, r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [-3e4, -1e3, 1e3, 5e3, 3e4])
@pytest.mark.parametrize("rows,vocab", [(3, 50257), (300, 5003)])
def test_a_common_offset_costs_no_precision(rows, vocab, offset, dtype, cuda_device):
    """Logits around +-10^3 to 3 10^4: their differences are as exact as without the offset."""
    z, t = _make(rows, vocab, torch.float32)
    _apart((z + offset).to(dtype), t, cuda_device, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("level", [-1e4, 4e4, -1e6, -1e9, -1e10, 5e9, 1e15, -1e30, 1e38])
def test_rows_far_from_zero(level, dtype, cuda_device):
    """Constant rows, rows of two levels and rows that keep one large logit,
    at sizes where max * log2(e) has no bits left for the exponents; with their gradient."""
    dev = cuda_device
    vocab = 9000
    for rows in (4, 160):  # a cluster for each row, and a CTA
        z = torch.full((rows, vocab), level, dtype=dtype)
        z[1, 4000:] = level * (1 + 2.0 ** -7)  # another level, exactly held
        z[2] = torch.randn(vocab, generator=torch.Generator().manual_seed(5)).to(dtype)
        z[2, 77] = level
        t = torch.arange(rows) * 7 % vocab
        t[2] = 77
        x = z.to(dev).requires_grad_()
        got, bar, r = _apart(x.detach().cpu(), t, dev, 3)
        out = ada.token_logprobs(x, t.to(dev))
        for a, b in zip(out[:3], got[:3]):
            assert (a - b).abs().max().item() <= 2 * bar + 2.0 ** -21 * b.abs().max().item()
        g = torch.Generator().manual_seed(3)
        ups = [torch.randn(rows, generator=g) for _ in range(3)]
        grad, = torch.autograd.grad(out[:3], x, [u.to(dev) for u in ups])
        zs = z.double() - z.double().amax(-1, keepdim=True)
        want = _grad64(zs, t, *ups)
        _, ent, _, logp = _exact(zs, t)
        p = logp.exp()
        size = p * (sum(u.abs().double() for u in ups)[:, None]
                    * (1 + torch.where(p > 0, logp.abs(), torch.zeros_like(p)) + ent.abs()[:, None]))
        hit = torch.zeros_like(want)
        hit[torch.arange(rows), t] = ups[0].abs().double()
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        slack = want.abs() * torch.finfo(dtype).eps / 2 + 4 * r * (size + hit) + tiny
        assert ((grad.cpu().double() - want).abs() <= slack).all()


def test_hidden_logits_beside_low_maxima(cuda_device):
    """fp16 rows whose maximum is near the type's lowest value: what is -inf still has probability 0."""
    dev = cuda_device
    z = torch.full((2, 50000), -math.inf, dtype=torch.float16)
    z[0, 9], z[1, 9], z[1, 12] = -65472.0, -65472.0, -65504.0
    got = ada.token_logprobs(z.to(dev), torch.full((2,), 9, device=dev))
    # one logit: exactly 0; two, 32 apart: p = e^-32, H = log s + 32 p with s = 1 + e^-32, which fp32
    # rounds to 1: log s is 0 in place of e^-32, and the rest is off by fp32 roundings
    assert got.logprobs.tolist()[0] == 0 and got.entropy.tolist()[0] == 0
    p = math.exp(-32)
    assert abs(got.logprobs[1].item()) <= 1e-13 and abs(got.entropy[1].item() - 33 * p) <= p + 33 * p * 1e-5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(200, 6000, 3), (200, 6000, 40), (16, 50257, 3), (2, 131072, 20)])
def test_nan_comes_first_wherever_it_stands(rows, vocab, top, dtype, cuda_device):
    """One NaN a row, in a thread's first, middle or last round: it is the first alternative, the others follow in order."""
    z, _ = _make(rows, vocab, dtype, spread=1.0)
    at = torch.arange(rows) * 997 % vocab
    at[::3] = torch.arange(rows)[::3] % 64  # first rounds
    at[1::3] = vocab - 1 - torch.arange(rows)[1::3] % 64
    z[torch.arange(rows), at] = math.nan
    got = ada.token_logprobs(z.to(cuda_device), torch.zeros(rows, dtype=torch.int64, device=cuda_device), top_k=top)
    assert torch.equal(got.top_tokens[:, 0].cpu(), at)
    assert torch.equal(got.top_tokens[:, 1:].cpu(), _top(z.nan_to_num(nan=-math.inf), top - 1))
    assert torch.isnan(got.logprobs).all() and torch.isnan(got.top_logprobs).all()


def test_forward_mode_is_refused(cuda_device):
    """A dual tensor does not require grad; its tangent is not dropped without a word."""
    fwd = torch.autograd.forward_ad
    dev = cuda_device
    z, t = _make(4, 50, torch.float32)
    z, t = z.to(dev), t.to(dev)
    want = ada.token_logprobs(z, t)
    ones = torch.ones(4, device=dev)
    stats = torch.stack([z.amax(-1), want.lse - z.amax(-1)], 1)
    with fwd.dual_level():
        dual = fwd.make_dual(z, torch.ones_like(z))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ada.token_logprobs(dual, t)
        with pytest.raises(RuntimeError, match="forward-mode"):
            token_logprobs_backward(z[None], t, stats, want.entropy, fwd.make_dual(ones, ones))
        with pytest.raises(RuntimeError):
            ada.token_logprobs(fwd.make_dual(z.clone().requires_grad_(), torch.ones_like(z)), t)
        assert torch.equal(ada.token_logprobs(z, t).logprobs, want.logprobs)  # no tangent here
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: ada.token_logprobs(x, t).lse, (z,), (z,))


def test_gradient_takes_strided_statistics(cuda_device):
    """Statistics and entropies read through strides give the gradient of their values."""
    dev = cuda_device
    z, t = _make(6, 700, torch.float32)
    zd, td = z.to(dev), t.to(dev)
    r = ada.token_logprobs(zd, td)
    m = zd.amax(-1)
    ups = torch.randn(6, generator=torch.Generator().manual_seed(1)).to(dev)
    stats = torch.stack([m, r.lse - m], 1)
    want = token_logprobs_backward(zd[None], td, stats, r.entropy, ups)
    wide = torch.full((6, 4), math.nan, device=dev)
    wide[:, ::2] = stats
    ent = torch.stack([r.entropy, r.entropy * math.nan], 1)
    assert torch.equal(token_logprobs_backward(zd[None], td, wide[:, ::2], ent[:, 0], ups), want)


@pytest.mark.parametrize("lead", [(0, 2, 3), (2, 0, 3), (0, 5), (0,)])
def test_no_rows_of_any_leading_dimensions(lead, cuda_device):
    dev = cuda_device
    z = torch.zeros(*lead, 9, device=dev, requires_grad=True)
    r = ada.token_logprobs(z, torch.zeros(lead, dtype=torch.int64, device=dev), top_k=2)
    assert r.logprobs.shape == lead and r.top_tokens.shape == (*lead, 2)
    grad, = torch.autograd.grad((r.logprobs.sum(), r.entropy.sum()), z)
    assert grad.shape == z.shape


def test_outputs_are_tensors_of_their_own(cuda_device):
    """One may change in place while another waits for a backward pass, or take part in autograd itself."""
    dev = cuda_device
    z, t = _make(4, 300, torch.float32)
    z, t = z.to(dev), t.to(dev)
    want = ada.token_logprobs(z, t, top_k=2)
    w = torch.ones(4, device=dev, requires_grad=True)
    r = ada.token_logprobs(z, t, top_k=2)
    loss = (w * r.entropy).sum()
    r.logprobs.neg_()
    r.lse.zero_()
    g, = torch.autograd.grad(loss, w)
    assert torch.equal(g, want.entropy)
    r.lse.add_(w)
    assert r.lse.requires_grad and torch.equal(r.entropy, want.entropy) and torch.equal(r.logprobs, -want.logprobs)
    assert len({x.untyped_storage().data_ptr() for x in r}) == 5
    x = z.clone().requires_grad_()  # with autograd the same bits
    for a, b in zip(ada.token_logprobs(x, t, top_k=2), want):
        assert torch.equal(a, b)
