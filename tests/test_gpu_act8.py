"""Activations in 8 bits: the format exactly, and the weight gradient from it.

The gradient multiplies the checkpoint's values, which are exact in the operands' type: the bound is that of
the product of 16-bit operands (k + 36 steps of 2^-23 of the sum of magnitudes, half a step of the type).
"""
import numpy as np
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from layer_util import (HALF_STEP, SUBNORMAL, act8_values, mut, numbers, offsets_of, ref, spans,
                        status_clean, tdt)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    status_clean()


def quantized(x):
    """(codes, exponent bytes) by the definition, numpy f64."""
    rows, cols = x.shape
    nb = (cols + 31) // 32
    v = np.zeros((rows, nb * 32))
    v[:, :cols] = x
    v = v.reshape(rows, nb, 32)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    top = np.abs(v).max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1, -127)
    e = np.maximum(e, -127)
    q = np.clip(np.rint(np.ldexp(v, 6 - e[..., None])), -127, 127)
    return q.reshape(rows, nb * 32)[:, :cols].astype(np.int8), np.where(bad, 255, e + 127).astype(np.uint8)


SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 1000), (1, 4096), (129, 257), (64, 2049), (333, 4099)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_codes(rows, cols, dtype):
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    # magnitudes over the type's range, block by block
    span = {"bf16": 120, "f16": 14, "f32": 120}[dtype]
    scale = torch.randint(-span, span, (rows, (cols + 31) // 32), generator=gen, device="cuda")
    x = torch.ldexp(x.clamp(-3.9, 3.9), scale.repeat_interleave(32, 1)[:, :cols]).to(tdt(dtype))
    q = gk.quantize_act8(ref(x))
    codes, exps = quantized(x.double().cpu().numpy())
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(q.exponents.cpu().numpy(), exps)
    outs = ["f32", "bf16"] + (["f16"] if dtype == "f16" else [])
    for out in outs:  # exact
        y = torch.empty(rows, cols, dtype=tdt(out), device="cuda")
        gk.dequantize_act8(q, mut(y))
        assert torch.equal(y.double(), act8_values(q))


def test_borders_and_ties():
    """Values on and beside the rounding borders of every code, and the clamp at 127."""
    torch = torch_cuda()
    half = np.arange(-255, 256) / 2.0
    rows = []
    for eps in (-2.0 ** -15, 0.0, 2.0 ** -15):
        v = half * (1 + eps)
        v = np.concatenate([v, np.zeros(-len(v) % 31)]).reshape(-1, 31)
        rows.append(np.concatenate([v, np.full((len(v), 1), 127.9)], 1))  # the block's unit is 1
    x = np.concatenate(rows).astype(np.float32)
    for shift in (0, -100, 90, -140):
        y = np.ldexp(x, shift).astype(np.float32)
        q = gk.quantize_act8(ref(torch.from_numpy(y).cuda()))
        codes, exps = quantized(y.astype(np.float64))
        assert np.array_equal(q.codes.cpu().numpy(), codes)
        assert np.array_equal(q.exponents.cpu().numpy(), exps)


def test_special_blocks():
    """A block with an infinity or a NaN is NaN, its neighbours are not; zeros, subnormals, the largest."""
    torch = torch_cuda()
    x = torch.ones(6, 96, device="cuda")
    x[0, 40], x[1, 33], x[2, 63] = float("inf"), float("nan"), float("-inf")
    x[3] = 0.0
    x[4] = 2.0 ** -149
    x[5] = torch.finfo(torch.float32).max
    q = gk.quantize_act8(ref(x))
    y = torch.empty(6, 96, device="cuda")
    gk.dequantize_act8(q, mut(y))
    assert y[:3, 32:64].isnan().all() and torch.equal(y[:3, :32], x[:3, :32])
    assert torch.equal(y[:3, 64:], x[:3, 64:]) and not y[3:5].any()
    assert torch.equal(y[5], torch.full_like(y[5], 127 * 2.0 ** 121))
    bf = torch.empty(6, 96, dtype=torch.bfloat16, device="cuda")
    gk.dequantize_act8(q, mut(bf))
    assert torch.equal(bf.float().nan_to_num(9.0), y.nan_to_num(9.0))


@pytest.mark.parametrize("layout", ["columns", "odd", "shifted", "wide"])
def test_views(layout):
    torch = torch_cuda()
    rows, cols = 37, 100
    x = numbers(5, (rows, cols), "bf16", False)
    if layout == "columns":
        v = x.t().contiguous().t()
    else:
        pitch, lead = {"odd": (101, 0), "shifted": (104, 1), "wide": (160, 0)}[layout]
        v = torch.full((rows * pitch + lead,), float("nan"), dtype=torch.bfloat16, device="cuda")
        v = v[lead:].view(rows, pitch)[:, :cols]
        v.copy_(x)
    q = gk.quantize_act8(ref(v))
    codes, exps = quantized(x.double().cpu().numpy())
    assert np.array_equal(q.codes.cpu().numpy(), codes) and np.array_equal(q.exponents.cpu().numpy(), exps)
    keep = v._base.clone() if v._base is not None else None
    v.zero_()
    gk.dequantize_act8(q, mut(v))
    assert torch.equal(v.double(), act8_values(q))
    if layout in ("odd", "shifted", "wide"):  # nothing beside the view is written
        a, b = v._base.clone(), keep
        for t in (a, b):
            t.as_strided(v.shape, v.stride(), v.storage_offset()).zero_()
        assert torch.equal(a.nan_to_num(3.0), b.nan_to_num(3.0))


def test_rows_and_caller_memory():
    """Runs of rows, and codes with pitches of the caller's; bytes past a row's last block stay."""
    torch = torch_cuda()
    x = numbers(6, (50, 70), "f16", False)
    whole = gk.quantize_act8(ref(x))
    part = whole.rows_of(7, 31)
    y = torch.empty(24, 70, dtype=torch.float16, device="cuda")
    gk.dequantize_act8(part, mut(y))
    assert torch.equal(y.double(), act8_values(whole)[7:31])
    buf = torch.full((50, 160), 77, dtype=torch.int8, device="cuda")
    exps = torch.full((50, 5), 9, dtype=torch.uint8, device="cuda")
    q = gk.Act8Matrix(50, 70, buf[:, :70], exps[:, :3])
    gk.quantize_act8(ref(x), out=q)
    assert torch.equal(buf[:, :70], whole.codes) and torch.equal(exps[:, :3], whole.exponents)
    assert not buf[:, 70:96].any() and bool((buf[:, 96:] == 77).all()) and bool((exps[:, 3:] == 9).all())


def wgrad(q, b, off, c, dtype, alpha=1.0, beta=0.0, **kw):
    g, m, n = c.shape
    gs, rs, cs = c.stride()
    ln = (g - 1) * gs + (m - 1) * rs + (n - 1) * cs + 1
    cv = gk.MatMut(c.as_strided((ln,), (1,)), m, n, rs, cs)
    gk.gemm_act8_wgrad(alpha, q, ref(b), beta, cv, offsets=off, c_gs=gs, is_f16=dtype == "f16", **kw)


SIZES = [(None, 1), (None, 75), (None, 1000), ([1], 1), ([0, 1, 0], 1), ([5, 0, 37, 2], 51),
         ([130, 0, 1, 255], 388), ([0, 0], 5), ([3] * 70, 210), ([64, 128, 65], 260)]


@pytest.mark.parametrize("sizes,rows", SIZES)
@pytest.mark.parametrize("m,n", [(64, 128), (16, 8), (200, 136), (33, 65), (1, 1), (264, 72), (520, 264)])
@pytest.mark.parametrize("layout", ["mn", "nm"])
def test_wgrad_exact(sizes, rows, m, n, layout):
    """Integers: every partial sum is exact, the result one rounding. Rows of no group hold NaN."""
    torch = torch_cuda()
    dtype = "bf16" if (m + n) % 3 else "f16"
    off = None if sizes is None else offsets_of(sizes, 3 if rows > sum(sizes) + 3 else 0)
    groups = 1 if sizes is None else len(sizes)
    x, b = numbers(11, (rows, m), dtype), numbers(12, (rows, n), dtype)
    live = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for _, s in spans(off, rows):
        live[s] = True
    x[~live], b[~live] = float("nan"), float("inf")
    q = gk.quantize_act8(ref(x))
    c = torch.full((groups, m, n), 3.0, dtype=tdt(dtype), device="cuda")
    if layout == "nm":
        c = torch.full((groups, n, m), 3.0, dtype=tdt(dtype), device="cuda").transpose(1, 2)
    want = torch.stack([x[s].double().T @ b[s].double() for _, s in spans(off, rows)])
    wgrad(q, b, off, c, dtype)
    assert torch.equal(c.double(), want.to(tdt(dtype)).double())
    f = torch.full((groups, m, n), 3.0, device="cuda")
    wgrad(q, b, off, f, dtype, alpha=0.5, beta=2.0)
    assert torch.equal(f.double(), 0.5 * want + 6.0)


@pytest.mark.parametrize("rows,m,n,sizes,layout", [
    (2000, 1024, 4096, None, "mn"), (2047, 1000, 4104, None, "nm"), (1500, 512, 1024, 13, "mn"),
    (700, 1037, 4096, None, "mn")])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_wgrad_large(rows, m, n, sizes, layout, dtype):
    torch = torch_cuda()
    off = None
    if sizes:
        cut = np.sort(np.random.default_rng(3).integers(0, rows, sizes - 1))
        off = torch.tensor(np.concatenate([[0], cut, [rows]]), dtype=torch.int32, device="cuda")
    x, b = numbers(21, (rows, m), dtype, False), numbers(22, (rows, n), dtype, False)
    q = gk.quantize_act8(ref(x))
    v = act8_values(q)
    groups = sizes or 1
    shape = (groups, m, n) if layout == "mn" else (groups, n, m)
    c = torch.empty(shape, dtype=tdt(dtype), device="cuda")
    c = c if layout == "mn" else c.transpose(1, 2)
    wgrad(q, b, off, c, dtype)
    for g, s in spans(off, rows):
        want = v[s].T @ b[s].double()
        mag = v[s].abs().T @ b[s].double().abs()
        tol = (s.stop - s.start + 36) * 2.0 ** -23 * mag + HALF_STEP[dtype] * want.abs() + SUBNORMAL[dtype]
        assert bool(((c[g].double() - want).abs() <= tol).all())


def test_wgrad_nan_block_stays_in_its_columns():
    torch = torch_cuda()
    x, b = numbers(31, (70, 96), "bf16"), numbers(32, (70, 40), "bf16")
    x[17, 40] = float("inf")
    c = torch.empty(1, 96, 40, dtype=torch.bfloat16, device="cuda")
    wgrad(gk.quantize_act8(ref(x)), b, None, c, "bf16")
    assert c[0, 32:64].isnan().all() and c[0, :32].isfinite().all() and c[0, 64:].isfinite().all()


def test_wgrad_of_a_run_of_rows():
    torch = torch_cuda()
    x, b = numbers(41, (300, 64), "bf16"), numbers(42, (300, 128), "bf16")
    q = gk.quantize_act8(ref(x))
    c = torch.empty(1, 64, 128, device="cuda")
    wgrad(q.rows_of(33, 211), b[33:211], None, c, "bf16")
    assert torch.equal(c[0].double(), x[33:211].double().T @ b[33:211].double())


def test_captured():
    torch = torch_cuda()
    x, b = numbers(51, (260, 96), "bf16"), numbers(52, (260, 128), "bf16")
    q = gk.Act8Matrix.empty(260, 96)
    c = torch.empty(1, 96, 128, device="cuda")
    gk.quantize_act8(ref(x), out=q)
    wgrad(q, b, None, c, "bf16")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gk.quantize_act8(ref(x), out=q, sync=False)
        wgrad(q, b, None, c, "bf16", sync=False)
    for seed in (53, 54):
        x.copy_(numbers(seed, (260, 96), "bf16"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c[0].double(), x.double().T @ b.double())
