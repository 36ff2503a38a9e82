"""Element offsets past 2^31: every store and every read by element of the grouped and the 4-bit
kernels, over operands and results whose rows or groups lie far apart. Integer and grid data, compared
for equality.

The wide views lie in one 11-GB buffer; only their elements are written and read."""
import numpy as np
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from test_gpu_fp4 import FMTS, grid_operand, grid_parts
from test_gpu_grouped import data, offsets_of, run_fwd, run_wgrad, tdt, want_fwd, want_wgrad

pytestmark = pytest.mark.gpu

PAST = 2 ** 31 + 2 ** 28  # the last row or group starts beyond this element


@pytest.fixture(scope="module")
def memory():
    torch = torch_cuda()
    buf = torch.empty(11 << 30, dtype=torch.uint8, device="cuda")
    yield buf
    del buf
    torch.cuda.empty_cache()


@pytest.fixture(autouse=True)
def _status():
    yield
    assert gk.device_status(0) == 0


def wide(memory, shape, dtype, odd=0, last=1, fill=None):
    """A view of `shape` whose first dimension's steps carry it past element PAST; the step is a multiple
    of 8 plus `odd`, the last dimension's stride `last`; filled with `fill` (a tensor or a number)."""
    torch = torch_cuda()
    flat = memory.view(tdt(dtype))
    step = -(-PAST // (shape[0] - 1)) // 8 * 8 + 8 + odd
    inner = [last]
    for s in shape[:0:-1][:-1]:
        inner.insert(0, inner[0] * s)
    t = torch.as_strided(flat, shape, (step, *inner))
    assert (shape[0] - 1) * step >= PAST and (shape[0] - 1) * step + shape[1] * inner[0] <= flat.numel()
    t.copy_(fill) if torch.is_tensor(fill) else t.fill_(fill)
    return t


# (rows of each group, n): one CTA's tiles, CTA pairs
PLANS = [([30, 0, 70], 136), ([900, 0, 1, 700, 515], 2304)]


@pytest.mark.parametrize("sizes,n", PLANS)
@pytest.mark.parametrize("out,odd,last", [("f32", 0, 1), ("f32", 1, 2), ("bf16", 0, 1), ("bf16", 1, 1)])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_forward_wide_c(memory, sizes, n, out, odd, last, beta):
    torch = torch_cuda()
    k, off = 72, offsets_of(sizes)
    a, b = data(1, (sum(sizes), k), "bf16"), data(2, (len(sizes), k, n), "bf16")
    c0 = data(3, (sum(sizes), n), out)
    c = wide(memory, c0.shape, out, odd, last, c0)
    run_fwd(a, b, off, c, "bf16", 1.0, beta)
    want, _ = want_fwd(a, b, off, c0, 1.0, beta)
    assert torch.equal(c, want.to(tdt(out)))


@pytest.mark.parametrize("sizes,m,n", [([30, 0, 70], 40, 136), ([5, 300, 0, 70], 1032, 2304)])
@pytest.mark.parametrize("out,odd", [("f32", 0), ("bf16", 0), ("bf16", 1)])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_wgrad_wide_groups_of_c(memory, sizes, m, n, out, odd, beta):
    torch = torch_cuda()
    off = offsets_of(sizes)
    a, b = data(1, (sum(sizes), m), "bf16"), data(2, (sum(sizes), n), "bf16")
    c0 = data(3, (len(sizes), m, n), out)
    c = wide(memory, c0.shape, out, odd, 1, c0)
    run_wgrad(a, b, off, c, "bf16", 1.0, beta)
    want, _ = want_wgrad(a, b, off, c0, 1.0, beta)
    assert torch.equal(c, want.to(tdt(out)))


@pytest.mark.parametrize("odd,last", [(0, 1), (1, 1), (1, 2)])  # in place, realigned by lines, by tiles
def test_wide_operands(memory, odd, last):
    torch = torch_cuda()
    sizes, k, n = [30, 0, 70], 136, 264
    off = offsets_of(sizes)
    a0, b0 = data(1, (100, k), "bf16"), data(2, (3, k, n), "bf16")
    dy = data(3, (100, n), "bf16")
    wf, _ = want_fwd(a0, b0, off, torch.zeros((100, n), device="cuda"), 1.0, 0.0)
    ww, _ = want_wgrad(a0, dy, off, torch.zeros((3, k, n), device="cuda"), 1.0, 0.0)
    c, w = torch.zeros((100, n), device="cuda"), torch.zeros((3, k, n), device="cuda")
    a = wide(memory, a0.shape, "bf16", odd, last, a0)
    run_fwd(a, b0, off, c, "bf16")
    run_wgrad(a, dy, off, w, "bf16")
    assert torch.equal(c.double(), wf) and torch.equal(w.double(), ww)
    b = wide(memory, b0.shape, "bf16", odd, last, b0)
    c.zero_()
    run_fwd(a0, b, off, c, "bf16")
    assert torch.equal(c.double(), wf)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype,odd,last", [("f32", 0, 1), ("f32", 1, 2), ("bf16", 0, 1), ("bf16", 1, 1)])
@pytest.mark.parametrize("rows", [70, 4800])  # 4800 rows of 4 stages: four stages a warp
def test_quantize_and_back_wide(memory, fmt, dtype, odd, last, rows):
    """Grid values (exact in 4 bits) through wide inputs, and back into wide outputs."""
    torch = torch_cuda()
    k = 1024
    _, _, val = grid_parts(1, rows, k, fmt)
    val[:, ::8] = 6.0  # the largest of every block
    x = wide(memory, val.shape, dtype, odd, last, val.clamp(-6, 6))
    near = gk.quantize_fp4(gk.MatRef.from_row_major(x.contiguous(), rows, k), fmt)
    q = gk.quantize_fp4(view(x), fmt)
    assert torch.equal(q.data, near.data) and torch.equal(values_of(q), values_of(near))
    if dtype == "f32":
        y = wide(memory, (rows, k), "f32", odd, last, 7.0)
        gk.dequantize_fp4(q, view(y, gk.MatMut))
        assert torch.equal(y, values_of(near))


def values_of(q):
    torch = torch_cuda()
    out = torch.full((q.rows, q.cols), 7.0, device="cuda")
    gk.dequantize_fp4(q, gk.MatMut.from_row_major(out, q.rows, q.cols))
    return out


def view(t, kind=gk.MatRef):
    torch = torch_cuda()
    r, c = t.shape
    rs, cs = t.stride()
    return kind(torch.as_strided(t, ((r - 1) * rs + (c - 1) * cs + 1,), (1,)), r, c, rs, cs)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_wide_stack(memory, fmt):
    """The groups of a stack lie far apart."""
    torch = torch_cuda()
    x0 = data(4, (3, 50, 264), "bf16")
    x = wide(memory, x0.shape, "bf16", 0, 1, x0)
    flat = torch.as_strided(x, (2 * x.stride(0) + 50 * 264,), (1,))
    q = gk.quantize_fp4(gk.MatRef(flat, 50, 264, 264, 1), fmt, groups=3, x_gs=x.stride(0))
    near = gk.quantize_fp4(gk.MatRef(x0.view(-1), 50, 264, 264, 1), fmt, groups=3, x_gs=50 * 264)
    assert torch.equal(q.data, near.data) and torch.equal(values_of(q), values_of(near))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sizes,n", PLANS)
@pytest.mark.parametrize("out,odd,last", [("f32", 0, 1), ("f32", 1, 2), ("bf16", 0, 1), ("bf16", 1, 1)])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_fp4_wide_c(memory, fmt, sizes, n, out, odd, last, beta):
    torch = torch_cuda()
    k, rows, g = 96, sum(sizes), len(sizes)
    o = np.cumsum([0] + sizes).tolist()
    a, av = grid_operand(1, rows, k, fmt, offsets=torch.tensor(o, dtype=torch.int32, device="cuda"))
    b, bv = grid_operand(2, g * n, k, fmt, groups=g)
    c0 = data(3, (rows, n), out)
    c = wide(memory, c0.shape, out, odd, last, c0)
    gk.gemm_fp4(1.0, a, b, beta, view(c, gk.MatMut))
    want = torch.cat([av[o[e]:o[e + 1]] @ bv[e * n:(e + 1) * n].T for e in range(g)]) + \
        beta * c0.double()
    assert torch.equal(c, want.to(tdt(out)))


@pytest.mark.parametrize("entry", ["forward", "wgrad"])
def test_longest_contraction(entry):
    """A contraction at the engine's limit (2^30 - 1) in one tile takes about 5 seconds: none of the
    kernel's bounded waits may give up meanwhile. Zeros but for integers at the two ends, in the middle
    and at random places: every sum is exact."""
    torch = torch_cuda()
    k, m, n = (2 ** 30 - 8 if entry == "forward" else 2 ** 30 - 1), 8, 8
    rng = np.random.default_rng(3)
    at = np.unique(np.concatenate([rng.integers(0, k, 3000), [0, 1, k // 2, k - 17, k - 2, k - 1]]))
    x, y = data(1, (len(at), m), "bf16"), data(2, (len(at), n), "bf16")
    at = torch.from_numpy(at).cuda()
    want = x.double().T @ y.double()
    shape = (lambda w: (w, k)) if entry == "forward" else (lambda w: (k, w))
    a, b = (torch.zeros(shape(w), dtype=torch.bfloat16, device="cuda") for w in (m, n))
    c = torch.full((m, n), 7.0, device="cuda")
    if entry == "forward":
        a[:, at], b[:, at] = x.T, y.T
        run_fwd(a, b.t()[None], offsets_of([m]), c, "bf16")
    else:
        a[at], b[at] = x, y
        run_wgrad(a, b, offsets_of([k]), c[None], "bf16")
    assert torch.equal(c.double(), want)
    del a, b
    torch.cuda.empty_cache()
