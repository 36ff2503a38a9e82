"""The router's balance loss, counts and gradient against 64-bit forms.

Bounds: the fast exponential is 4 units of 2^-24 off, a difference of logits and its product with log2 e one
unit each times its size (at most 2^-24 |x - max|, below 50 here where p matters: p < e^-50 is below
any bound), a softmax's sum and division at most 11 + 2 more steps: 128 2^-24 relative to p covers all. Sums over a warp's tokens (at most 64
here) add 64 2^-24 of the sum; the blocks are added in 64 bits. dlogits: p's bound twice, the dot
over at most 1024 experts in trees of 32 by at most 32 steps, and half a step of the type.
"""
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from layer_util import HALF_STEP, SUBNORMAL, mut, ref, status_clean, tdt

pytestmark = pytest.mark.gpu
REL = 200 * 2.0 ** -24


@pytest.fixture(autouse=True)
def _status():
    yield
    status_clean()


def router(seed, tokens, experts, top, dtype, padding=0, ids64=False):
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(tokens, experts, generator=gen, device="cuda") * 2).to(tdt(dtype))
    ids = torch.topk(x.float(), top, dim=1)[1]
    if padding:
        ids[torch.randperm(tokens, generator=gen, device="cuda")[:padding]] = -1
    return x, ids if ids64 else ids.to(torch.int32)


def want_of(x, ids, coef=1.0, dloss=1.0):
    torch = torch_cuda()
    e = x.shape[1]
    live = (ids >= 0).any(1)
    counts = torch.bincount(ids[ids >= 0].long().reshape(-1), minlength=e)
    none = (x == float("-inf")).all(1)
    p = torch.softmax(x.double(), 1)
    p = torch.where(none[:, None], 0.0, p) * live[:, None]
    t, n = max(1, int(live.sum())), max(1, int(counts.sum()))
    f = counts.double() / n
    rates = coef * e * f / t
    loss = (rates * p.sum(0)).sum()
    g = dloss * p * (rates - (p @ rates)[:, None])
    mag = abs(dloss) * p * (rates + (p @ rates)[:, None])
    return loss, counts, rates, g, mag


def check(x, ids, dtype, coef=1.0, dloss=0.5, dst=None):
    torch = torch_cuda()
    b = gk.moe_balance(ref(x), ids, coef=coef)
    loss, counts, rates, g, mag = want_of(x, ids, coef, dloss)
    assert torch.equal(b.counts.long(), counts)
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    assert torch.equal(b.offsets.long(), off)
    assert abs(float(b.loss) - float(loss)) <= REL * abs(float(loss))
    assert bool(((b.rates.double() - rates).abs() <= 2.0 ** -23 * rates).all())
    d = torch.full_like(x, 9.0) if dst is None else dst
    scale = torch.tensor([dloss], device="cuda")
    gk.moe_balance_backward(ref(x), ids, b, scale, mut(d))
    tol = REL * mag + HALF_STEP[dtype] * g.abs() + SUBNORMAL[dtype] + 2.0 ** -126
    assert bool(((d.double() - g).abs() <= tol).all())
    return b, d


@pytest.mark.parametrize("tokens", [1, 5, 64, 65, 1000, 9001])
@pytest.mark.parametrize("experts,top", [(1, 1), (2, 1), (8, 2), (33, 5), (128, 8), (256, 8), (260, 33),
                                         (1000, 3), (1024, 2), (999, 4)])
def test_balance(tokens, experts, top):
    dtype = ["f32", "bf16", "f16"][(tokens + experts) % 3]
    x, ids = router(tokens + experts, tokens, experts, top, dtype, tokens // 5, (tokens + top) % 2 == 0)
    check(x, ids, dtype, coef=0.25)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["columns", "odd", "wide", "shifted"])
def test_strides(dtype, layout):
    torch = torch_cuda()
    tokens, experts = 200, 64
    x, ids = router(3, tokens, experts, 4, dtype)
    if layout == "columns":
        v, d = x.t().contiguous().t(), torch.zeros_like(x).t().contiguous().t()
    else:
        pitch, lead = {"odd": (65, 0), "wide": (128, 0), "shifted": (68, 1)}[layout]
        v, d = (torch.zeros(tokens * pitch + lead, dtype=tdt(dtype), device="cuda")[lead:]
                .view(tokens, pitch)[:, :experts] for _ in range(2))
        v.copy_(x)
    check(v, ids, dtype, dst=d)


def test_nothing_live_and_no_tokens():
    torch = torch_cuda()
    for tokens in (0, 3, 500):
        x = torch.randn(tokens, 8, device="cuda")
        ids = torch.full((tokens, 2), -1, dtype=torch.int32, device="cuda")
        v = gk.MatRef(x.reshape(-1), tokens, 8, 8, 1)
        b = gk.moe_balance(v, ids)
        assert not b.loss.any() and not b.counts.any() and not b.offsets.any() and not b.rates.any()
        d = torch.ones(tokens, 8, device="cuda")
        gk.moe_balance_backward(v, ids, b, torch.ones(1, device="cuda"),
                                gk.MatMut(d.reshape(-1), tokens, 8, 8, 1))
        assert not d.any()


def test_masked_logits():
    """Minus infinity: probability 0, a whole row of them adds nothing; NaN and infinity reach the loss."""
    torch = torch_cuda()
    x, ids = router(5, 300, 40, 3, "f32", 20)
    x[:, 7] = float("-inf")
    x[11] = float("-inf")
    x[12, 1:] = float("-inf")
    ids[11], ids[12] = torch.tensor([0, 1, 2], device="cuda"), torch.tensor([0, 1, 1], device="cuda")
    lowest = torch.finfo(torch.float32).min
    x[13], x[14, 3:] = lowest, lowest
    check(x, ids, "f32")
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[100, 3] = bad
        ids[100] = 1
        assert gk.moe_balance(ref(y), ids).loss.isnan().all()
        ids[100] = -1  # in a padded row it does not count
        b = gk.moe_balance(ref(y), ids)
        assert b.loss.isfinite().all()
        d = torch.empty_like(y)
        gk.moe_balance_backward(ref(y), ids, b, torch.ones(1, device="cuda"), mut(d))
        assert d.isfinite().all() and not d[100].any()


def test_bad_ids_are_reported():
    torch = torch_cuda()
    x, ids = router(7, 100, 16, 2, "bf16", ids64=True)
    good = ids.clone()
    ids[3, 1], ids[50, 0], ids[60] = 16, 1 << 40, 99
    good[3, 1] = good[50, 0] = -1
    good[60] = -1
    b = gk.moe_balance(ref(x), ids)
    assert gk.device_status(0) == 1 << 5
    w = gk.moe_balance(ref(x), good)
    assert torch.equal(b.counts, w.counts) and torch.equal(b.loss, w.loss)


def test_in_place_repeats_and_capture():
    torch = torch_cuda()
    x, ids = router(9, 5000, 256, 8, "f32", 100)
    b, d = check(x, ids, "f32", dloss=1.0)
    one = torch.ones(1, device="cuda")
    y = x.clone()
    gk.moe_balance_backward(ref(y), ids, b, one, mut(y))
    assert torch.equal(y, d)
    b2 = gk.moe_balance(ref(x), ids)
    assert torch.equal(b2.loss, b.loss) and torch.equal(b2.rates, b.rates)
    graphs, outs = [], []
    for _ in range(2):
        o, dd = gk.MoeBalance.empty(256), torch.empty_like(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gk.moe_balance(ref(x), ids, out=o, sync=False)
            gk.moe_balance_backward(ref(x), ids, o, one, mut(dd), sync=False)
        graphs.append(g), outs.append((o, dd))
    s = torch.cuda.Stream()
    graphs[0].replay()
    with torch.cuda.stream(s):
        graphs[1].replay()
    torch.cuda.synchronize()
    for o, dd in outs:
        assert torch.equal(o.loss, b.loss) and torch.equal(o.offsets, b.offsets) and torch.equal(dd, d)


def test_gradient_against_differences():
    torch = torch_cuda()
    x, ids = router(13, 12, 6, 2, "f32", 2)
    b = gk.moe_balance(ref(x), ids)
    d = torch.empty_like(x)
    gk.moe_balance_backward(ref(x), ids, b, torch.ones(1, device="cuda"), mut(d))
    h = 2.0 ** -7
    for t in range(12):
        for e in range(6):
            v = []
            for s in (h, -h):
                y = x.clone()
                y[t, e] += s
                v.append(float(gk.moe_balance(ref(y), ids).loss))
            # loss < 6 to 2^-20 relative, its third derivative by a logit below 6 / 10
            assert abs((v[0] - v[1]) / (2 * h) - float(d[t, e])) < 6 * 2.0 ** -20 / h + h * h / 10
