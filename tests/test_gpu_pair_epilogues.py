"""The CTA-pair kernels' accumulating epilogues: beta != 0 (f32 and 16-bit C), and normal data against
f64, for both grouped products and the 4-bit product, at sizes that those kernels take (at least 74
tiles of 256 x 256, more than 128 rows a group).

Integer and grid data: products, sums, alpha * acc and beta * C are exact in f32 (fewer than 24
significant bits), so C is the exact value rounded once to its type. Normal data: the tolerances of
the small cases (see test_gpu_grouped.py and test_gpu_fp4.py). Every call runs twice: no sum depends
on which block gets where first, so the bits are the same."""
import numpy as np
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from test_gpu_fp4 import FMTS, grid_operand, mat, product, values
from test_gpu_grouped import (HALF_STEP, check_near, data, offsets_of, run_fwd, run_wgrad, tdt,
                              want_fwd, want_wgrad)

pytestmark = pytest.mark.gpu

SIZES = [900, 0, 1, 700, 515]
OUTS = [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")]
FACTORS = [(1.0, 1.0), (-0.5, 0.25), (2.0, 1.0)]


@pytest.fixture(autouse=True)
def _status():
    yield
    assert gk.device_status(0) == 0


def twice(c0, call):
    """call(c) on two copies of c0: the first result, after both have the same bits."""
    torch = torch_cuda()
    cs = [c0.clone(memory_format=torch.preserve_format) for _ in range(2)]
    for c in cs:
        call(c)
    torch.cuda.synchronize()
    assert torch.equal(*cs)
    return cs[0]


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("alpha,beta", FACTORS)
@pytest.mark.parametrize("k,n,major", [(200, 2304, "n"), (136, 2305, "k"), (1032, 2312, "k")])
@pytest.mark.parametrize("lead,tail", [(0, 0), (3, 2)])
def test_forward_accumulates_exactly(dtype, out, alpha, beta, k, n, major, lead, tail):
    torch = torch_cuda()
    rows, off = lead + sum(SIZES) + tail, offsets_of(SIZES, lead)
    a = data(1, (rows, k), dtype)
    b = data(2, (len(SIZES), n, k), dtype).transpose(1, 2) if major == "k" else \
        data(2, (len(SIZES), k, n), dtype)
    a[:lead] = float("nan")
    a[rows - tail:] = float("inf")
    c0 = data(3, (rows, n), out)
    c = twice(c0, lambda c: run_fwd(a, b, off, c, dtype, alpha, beta))
    want, _ = want_fwd(a, b, off, c0, alpha, beta)
    assert torch.equal(c, want.to(tdt(out)))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("alpha,beta", FACTORS)
@pytest.mark.parametrize("m,n", [(1032, 2304), (1100, 1513)])
def test_wgrad_accumulates_exactly(dtype, out, alpha, beta, m, n):
    """With an empty group (beta * C) and a group of one row."""
    torch = torch_cuda()
    rows, off = sum(SIZES) + 3, offsets_of(SIZES, 2)
    a, b = data(1, (rows, m), dtype), data(2, (rows, n), dtype)
    for t in (a, b):
        t[:2] = float("nan")
        t[rows - 1:] = float("inf")
    c0 = data(3, (len(SIZES), m, n), out)
    c = twice(c0, lambda c: run_wgrad(a, b, off, c, dtype, alpha, beta))
    want, _ = want_wgrad(a, b, off, c0, alpha, beta)
    assert torch.equal(c, want.to(tdt(out)))


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (1.0, 1.0), (-0.5, 0.25)])
def test_forward_near_large(dtype, out, alpha, beta):
    """beta == 0 with 16-bit C: the 512-column tiles."""
    k, n, off = 1032, 2312, offsets_of(SIZES)
    a = data(3, (sum(SIZES), k), dtype, ints=False)
    b = data(4, (len(SIZES), k, n), dtype, ints=False)
    c0 = data(5, (sum(SIZES), n), out, ints=False)
    c = twice(c0, lambda c: run_fwd(a, b, off, c, dtype, alpha, beta))
    want, mag = want_fwd(a, b, off, c0, alpha, beta)
    check_near(c, want, mag, k, out)


@pytest.mark.parametrize("dtype,out", OUTS)
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (1.0, 1.0), (-0.5, 0.25)])
def test_wgrad_near_large(dtype, out, alpha, beta):
    m, n, off = 1032, 2312, offsets_of(SIZES)
    a = data(3, (sum(SIZES), m), dtype, ints=False)
    b = data(4, (sum(SIZES), n), dtype, ints=False)
    c0 = data(5, (len(SIZES), m, n), out, ints=False)
    c = twice(c0, lambda c: run_wgrad(a, b, off, c, dtype, alpha, beta))
    want, mag = want_wgrad(a, b, off, c0, alpha, beta)
    check_near(c, want, mag, max(SIZES), out)


def expert_products(av, bv, n, c0, alpha, beta):
    """(f64 result, f64 sum of magnitudes) of the 4-bit product by expert over SIZES."""
    o = np.cumsum([0] + SIZES).tolist()
    want, mag = c0.double().clone(), c0.double().abs()
    for e in range(len(SIZES)):
        s, w = slice(o[e], o[e + 1]), bv[e * n:(e + 1) * n].double()
        x = av[s].double()
        want[s] = alpha * (x @ w.T) + beta * c0[s].double()
        mag[s] = abs(alpha) * (x.abs() @ w.abs().T) + abs(beta) * c0[s].double().abs()
    return want, mag


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("alpha,beta", FACTORS)
@pytest.mark.parametrize("k,n", [(320, 2304), (1000, 2305)])
def test_fp4_accumulates_exactly(fmt, out, alpha, beta, k, n):
    torch = torch_cuda()
    off = torch.tensor(np.cumsum([0] + SIZES), dtype=torch.int32, device="cuda")
    a, av = grid_operand(1, sum(SIZES), k, fmt, offsets=off)
    b, bv = grid_operand(2, len(SIZES) * n, k, fmt, groups=len(SIZES))
    c0 = data(3, (sum(SIZES), n), out)
    c = twice(c0, lambda c: product(a, b, c, alpha, beta))
    want, _ = expert_products(av, bv, n, c0, alpha, beta)
    assert torch.equal(c, want.to(tdt(out)))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (1.0, 1.0), (-0.5, 0.25)])
def test_fp4_near_large(fmt, out, alpha, beta):
    torch = torch_cuda()
    k, n = 1056, 2312
    sa, sb = (1.0, 1.0) if fmt == gk.FP4_MX else (0.01, 0.003)
    off = torch.tensor(np.cumsum([0] + SIZES), dtype=torch.int32, device="cuda")
    x = data(1, (sum(SIZES), k), "bf16", ints=False)
    w = data(2, (len(SIZES) * n, k), "f32", ints=False)
    a = gk.quantize_fp4(mat(x), fmt, scale=sa, offsets=off)
    b = gk.quantize_fp4(gk.MatRef(w.view(-1), n, k, k, 1), fmt, scale=sb, groups=len(SIZES), x_gs=n * k)
    c0 = data(3, (sum(SIZES), n), out, ints=False)
    c = twice(c0, lambda c: product(a, b, c, alpha, beta))
    want, mag = expert_products(values(a), values(b), n, c0, alpha, beta)
    # values() rounds code * scale * s once (2^-24 each side); the kernel applies s at the end
    tol = (k + 32 + 8) * 2.0 ** -23 * mag + HALF_STEP[out] * want.abs() + 1e-30
    if out == "f16":
        tol = tol + 2.0 ** -25
    err = (c.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
