"""Microscaled 4-bit floats: quantisation and the values back (exact, against decisions made by
exact comparisons in f64), and the products, dense and by expert, against f64 products of the values.

Products. Grid data (codes with block scales of a few powers of two): every product is a multiple of
1/16 and every partial sum below 2^24 of those units, so f32 accumulation in any order is exact and
f32 results are compared for equality. Normal data: a product of two scaled elements is exact in f32
(4 + 8 significant bits), an accumulation step loses at most one unit of 2^-23 of the sum of
magnitudes, at most k + 32 steps; alpha (with the matrix scales) and beta add roundings of 2^-24, the
output type half a step.
"""
import numpy as np
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] +
                [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 0.0}
FMTS = [gk.FP4_MX, gk.FP4_NV]


@pytest.fixture(autouse=True)
def _status():
    yield
    assert gk.device_status(0) == 0


def tdt(name):
    torch = torch_cuda()
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def block(fmt):
    return 32 if fmt == gk.FP4_MX else 16


def nearest(x, unit, grid):
    """Index into `grid` of x / unit, ties to the even index, saturating: |x| is compared with
    border * unit (exact in f64 for these widths)."""
    mid = (grid[1:] + grid[:-1]) / 2
    idx = np.zeros(x.shape, int)
    for i, m in enumerate(mid):
        b = m * unit
        idx += (x > b) | ((x == b) & (i % 2 == 1))
    return idx


def reference(x, fmt, s=1.0):
    """f64 array -> the f32 values that its 4-bit form stands for."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    bs = block(fmt)
    out = np.zeros((rows, k), np.float32)
    for c in range(0, k, bs):
        v = x[:, c:c + bs]
        bad = ~np.isfinite(v).all(1)
        amax = np.where(bad, 0.0, np.abs(np.where(np.isfinite(v), v, 0)).max(1))
        if fmt == gk.FP4_MX:
            e = np.where(amax > 0, np.frexp(np.where(amax > 0, amax, 1))[1] - 1 - 2, -127)
            unit = np.ldexp(1.0, np.clip(e, -127, 127))
            post = 1.0
        else:
            sb = E4M3[nearest(amax, 6.0 * np.float64(np.float32(s)), E4M3)]
            unit, post = sb * np.float64(np.float32(s)), None
        with np.errstate(invalid="ignore"):
            code = nearest(np.abs(v), unit[:, None], GRID)
        val = GRID[code] * (unit[:, None] if post else sb[:, None])
        if fmt == gk.FP4_NV:
            val = np.where(sb[:, None] > 0, val, 0.0)
            val = (val.astype(np.float32) * np.float32(s)).astype(np.float64)
        val = np.where(bad[:, None], np.nan, val * np.where(np.signbit(v), -1, 1))
        out[:, c:c + bs] = val.astype(np.float32)
    return out


def mat(t, kind=gk.MatRef):
    """A view of a 2-D tensor with any strides, typed by a flat tensor over its storage."""
    torch = torch_cuda()
    r, c = t.shape
    rs, cs = t.stride()
    n = (r - 1) * rs + (c - 1) * cs + 1 if t.numel() else 0
    return kind(torch.as_strided(t, (n,), (1,)), r, c, rs, cs)


def values(q):
    torch = torch_cuda()
    out = torch.full((q.rows, q.cols), 7.0, device="cuda")
    gk.dequantize_fp4(q, gk.MatMut.from_row_major(out, q.rows, q.cols))
    return out


def same(got, want):
    assert np.array_equal(np.asarray(got.cpu()), want, equal_nan=True)


def sample(seed, rows, k, dtype, spread=3.0):
    """Values over many magnitudes, a third of them near the borders of the 4-bit grid."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)) * spread)
    edge = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], (rows, k)) * \
        rng.choice([-1, 1], (rows, k)) * 2.0 ** rng.integers(-3, 4, (rows, 1))
    x = np.where(rng.random((rows, k)) < 0.33, edge, x)
    torch = torch_cuda()
    return torch.tensor(x, dtype=torch.float64, device="cuda").to(tdt(dtype))


# ---- quantisation ----------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 16), (3, 17), (130, 32), (7, 33), (64, 100),
                                    (129, 256), (5, 257), (300, 1000), (2, 4099)])
def test_quantize_exact(fmt, dtype, rows, k):
    x = sample(rows * k, rows, k, dtype)
    for s in ([1.0] if fmt == gk.FP4_MX else [1.0, 0.0123, 37.5]):
        q = gk.quantize_fp4(mat(x), fmt, scale=s)
        same(values(q), reference(x.double().cpu().numpy(), fmt, s))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_extremes(fmt):
    """Zeros, subnormals, the largest values, saturation, infinities and NaN."""
    torch = torch_cuda()
    x = torch.zeros(12, 96, device="cuda")
    x[1] = 1e-45
    x[2] = 1.1754944e-38
    x[3] = torch.finfo(torch.float32).max
    x[4, ::3] = torch.finfo(torch.float32).min
    x[5, 40] = float("nan")
    x[6, 0] = float("inf")
    x[7, 95] = -float("inf")
    x[8] = torch.linspace(-1e-40, 1e-40, 96)
    x[9, 7] = 1e30
    x[9, 8:] = 1e-30
    x[10] = torch.arange(96) - 48.0
    x[11] = -0.0
    for s in ([1.0] if fmt == gk.FP4_MX else [1.0, 2.0 ** -100, 2.0 ** 100, 1e-20]):
        q = gk.quantize_fp4(mat(x), fmt, scale=s)
        same(values(q), reference(x.double().cpu().numpy(), fmt, s))


def test_quantize_every_border():
    """nv: all quotients of small integers by odd scales, where f32 division alone would decide some
    borders wrongly; mx: every bf16 mantissa in every place of the exponent."""
    torch = torch_cuda()
    a = torch.arange(1, 4097, dtype=torch.float32, device="cuda").view(-1, 16)
    for s in (1.0 / 3.0, 0.1, 7.0 / 48.0, 1.0):
        q = gk.quantize_fp4(mat(a), gk.FP4_NV, scale=float(np.float32(s)))
        same(values(q), reference(a.double().cpu().numpy(), gk.FP4_NV, float(np.float32(s))))
    bits = torch.arange(0, 65536, dtype=torch.int32, device="cuda").to(torch.uint16)
    x = bits.view(torch.bfloat16).view(-1, 32)  # every bf16, NaN and infinities among them
    q = gk.quantize_fp4(mat(x), gk.FP4_MX)
    same(values(q), reference(x.double().cpu().numpy(), gk.FP4_MX))
    mixed = x.t().contiguous()  # blocks of very different magnitudes
    mixed = mixed.nan_to_num(1.0, 2.0, -2.0)
    q = gk.quantize_fp4(mat(mixed), gk.FP4_MX)
    same(values(q), reference(mixed.double().cpu().numpy(), gk.FP4_MX))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("layout", ["col_major", "padded", "offset", "every_other"])
def test_quantize_strides(fmt, layout):
    rows, k = 70, 200
    x = sample(5, rows, k, "bf16")
    if layout == "col_major":
        x = sample(5, k, rows, "bf16").t()
    elif layout == "padded":
        x = sample(5, rows, k + 24, "bf16")[:, :k]
    elif layout == "offset":
        x = sample(5, rows, k + 3, "bf16")[:, 1:1 + k]
    elif layout == "every_other":
        x = sample(5, rows, 2 * k, "bf16")[:, ::2]
    q = gk.quantize_fp4(mat(x), fmt, scale=1.0)
    same(values(q), reference(x.double().cpu().numpy(), fmt))


@pytest.mark.parametrize("fmt", FMTS)
def test_groups_and_rows_outside(fmt):
    """Ragged groups: rows outside keep their codes; a stack: groups x_gs apart."""
    torch = torch_cuda()
    rows, k = 300, 80
    x = sample(6, rows, k, "f32")
    off = torch.tensor([4, 4, 150, 151, 290], dtype=torch.int32, device="cuda")
    x[:4] = float("nan")
    q = gk.quantize_fp4(mat(x), fmt, offsets=off)
    got = values(q)
    same(got[4:290], reference(x[4:290].double().cpu().numpy(), fmt))
    assert bool((got[:4] == 7).all()) and bool((got[290:] == 7).all())
    w = sample(7, 3 * 50, k + 2, "f16").view(3, 50, k + 2)[:, :, :k]  # a stack with a pitch
    q = gk.quantize_fp4(gk.MatRef(w._base.reshape(-1) if w._base is not None else w, 50, k, k + 2, 1),
                        fmt, groups=3, x_gs=50 * (k + 2))
    assert q.rows == 150 and q.groups == 3
    same(values(q), reference(w.reshape(150, k).double().cpu().numpy(), fmt))
    wt = sample(8, 3 * k, 50, "bf16").view(3, k, 50)  # stored k x n: quantised along k
    q = gk.quantize_fp4(gk.MatRef(wt.reshape(-1), 50, k, 1, 50), fmt, groups=3, x_gs=50 * k)
    same(values(q), reference(wt.transpose(1, 2).reshape(150, k).double().cpu().numpy(), fmt))


def grid_parts(seed, rows, k, fmt):
    """Random codes and block scales (a few powers of two) as a checkpoint holds them, and values."""
    torch = torch_cuda()
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, k), dtype=np.uint8)
    nb = -(-k // block(fmt))
    p = rng.integers(-1, 2, (rows, nb))
    byte = (127 + p) if fmt == gk.FP4_MX else (7 + p) * 8  # e8m0 / e4m3 of 2^p
    val = GRID[codes & 7] * np.where(codes >= 8, -1, 1) * \
        np.repeat(2.0 ** p, block(fmt), 1)[:, :k]
    padded = np.pad(codes, ((0, 0), (0, k % 2)), constant_values=15)  # a stray last nibble
    packed = padded[:, 0::2] | (padded[:, 1::2] << 4)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a.astype(np.uint8))).cuda()  # noqa: E731
    return dev(packed), dev(byte), torch.from_numpy(val).cuda()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (130, 64), (257, 515)])
def test_from_codes(fmt, rows, k):
    torch = torch_cuda()
    codes, scales, val = grid_parts(rows + k, rows, k, fmt)
    q = gk.Fp4Matrix.from_codes(codes, scales, rows, k, fmt)
    assert torch.equal(values(q).double(), val)


# ---- the product -----------------------------------------------------------------------------------

def grid_operand(seed, rows, k, fmt, **kw):
    """A matrix of grid data whose unowned bytes (the scales past a group's last row) are NaN."""
    import ctypes as C
    from gemmkit_b200 import _lib
    codes, scales, val = grid_parts(seed, rows, k, fmt)
    q = gk.Fp4Matrix.empty(rows, k, fmt, **kw)
    q.data.fill_(255)
    q.scales.fill_(255)
    gk._check(_lib.load().gk_fp4_import(codes.data_ptr(), codes.numel(), codes.stride(0),
                                        scales.data_ptr(), scales.numel(), scales.stride(0),
                                        C.byref(q.c), gk._stream(None)))
    return q, val


def product(a, b, c, alpha=1.0, beta=0.0, **kw):
    gk.gemm_fp4(alpha, a, b, beta, mat(c, gk.MatMut), **kw)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 5, 16, 33, 64, 65, 128, 200, 513])
@pytest.mark.parametrize("k,n", [(256, 128), (64, 40), (1, 1), (100, 300), (257, 129), (1000, 72)])
def test_product_exact(fmt, m, k, n):
    torch = torch_cuda()
    a, av = grid_operand(m + k, m, k, fmt)
    b, bv = grid_operand(n + k + 1, n, k, fmt)
    c = torch.full((m, n), float("nan"), device="cuda")  # beta == 0 never reads C
    product(a, b, c)
    assert torch.equal(c.double(), av @ bv.T)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (-0.5, 1.0), (0.0, 2.0)])
@pytest.mark.parametrize("m", [3, 150, 300])
def test_quantized_product_near(fmt, out, alpha, beta, m):
    torch = torch_cuda()
    k, n = 1056, 200
    sa, sb = (1.0, 1.0) if fmt == gk.FP4_MX else (0.01, 0.003)
    gen = torch.Generator(device="cuda").manual_seed(3)
    a = gk.quantize_fp4(mat(torch.randn(m, k, generator=gen, device="cuda").bfloat16()), fmt, scale=sa)
    b = gk.quantize_fp4(mat(torch.randn(n, k, generator=gen, device="cuda")), fmt, scale=sb)
    c0 = torch.randn(m, n, generator=gen, device="cuda").to(tdt(out))
    c = c0.clone()
    product(a, b, c, alpha, beta)
    av, bv = values(a).double(), values(b).double()
    want = alpha * (av @ bv.T) + beta * c0.double()
    mag = abs(alpha) * (av.abs() @ bv.abs().T) + abs(beta) * c0.double().abs()
    # values() rounds code * scale * s once (2^-24 each side); the kernel applies s at the end
    tol = (k + 32 + 8) * 2.0 ** -23 * mag + HALF_STEP[out] * want.abs() + 1e-30
    if out == "f16":
        tol = tol + 2.0 ** -25
    err = (c.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("layout", ["padded", "col_major", "strided"])
def test_product_output_layouts(layout):
    torch = torch_cuda()
    m, k, n, fmt = 150, 256, 136, gk.FP4_MX
    a, av = grid_operand(1, m, k, fmt)
    b, bv = grid_operand(2, n, k, fmt)
    buf = torch.full((2 * m, 2 * n + 1), 7.0, device="cuda")
    c = {"padded": buf[:m, 1:1 + n], "col_major": buf.view(-1)[:n * m].view(n, m).t(),
         "strided": buf[::2, :2 * n:2]}[layout]
    mask = torch.zeros_like(buf, dtype=torch.bool)
    {"padded": mask[:m, 1:1 + n], "col_major": mask.view(-1)[:n * m].view(n, m).t(),
     "strided": mask[::2, :2 * n:2]}[layout].fill_(True)
    product(a, b, c)
    assert torch.equal(c.double(), av @ bv.T)
    assert bool((buf[~mask] == 7).all())


SIZES = [([1], 0, 0), ([0, 1, 0], 0, 0), ([5, 0, 37, 2], 3, 4), ([33, 64, 31], 0, 0),
         ([130, 0, 1, 255], 0, 2), ([300, 513], 1, 0), ([0, 0], 2, 3), ([3] * 70, 0, 0)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sizes,lead,tail", SIZES)
@pytest.mark.parametrize("k,n", [(256, 128), (100, 72), (515, 200)])
def test_product_by_expert(fmt, sizes, lead, tail, k, n):
    torch = torch_cuda()
    rows, g = lead + sum(sizes) + tail, len(sizes)
    off = torch.tensor(np.cumsum([lead] + sizes), dtype=torch.int32, device="cuda")
    a, av = grid_operand(1, rows, k, fmt, offsets=off)
    b, bv = grid_operand(2, g * n, k, fmt, groups=g)
    c = torch.full((rows, n), 7.0, device="cuda")
    product(a, b, c)
    want = torch.full_like(c, 7.0).double()
    o = off.tolist()
    for e in range(g):
        want[o[e]:o[e + 1]] = av[o[e]:o[e + 1]] @ bv[e * n:(e + 1) * n].T
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("fmt", FMTS)
def test_equal_groups(fmt):
    """A batch: A a stack too, its groups not multiples of the tile."""
    torch = torch_cuda()
    g, m, k, n = 5, 37, 160, 100
    a, av = grid_operand(1, g * m, k, fmt, groups=g)
    b, bv = grid_operand(2, g * n, k, fmt, groups=g)
    c = torch.full((g * m, n), 7.0, device="cuda")
    product(a, b, c)
    want = torch.bmm(av.view(g, m, k), bv.view(g, n, k).transpose(1, 2)).view(g * m, n)
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("fmt", FMTS)
def test_nan_blocks(fmt):
    """A NaN or an infinity makes its row of A, or its column of the result, NaN and nothing else."""
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(140, 256, generator=gen, device="cuda")
    w = torch.randn(150, 256, generator=gen, device="cuda")
    x[131, 200] = float("inf")
    w[77, 3] = float("nan")
    a, b = gk.quantize_fp4(mat(x), fmt), gk.quantize_fp4(mat(w), fmt)
    c = torch.zeros(140, 150, device="cuda")
    product(a, b, c)
    want = torch.zeros(140, 150, dtype=torch.bool, device="cuda")
    want[131] = True
    want[:, 77] = True
    assert torch.equal(c.isnan(), want)


def test_bad_offsets_stay_inside_and_are_reported():
    torch = torch_cuda()
    rows, k, n, fmt = 64, 96, 136, gk.FP4_MX
    codes, scales, av = grid_parts(1, rows, k, fmt)
    b, bv = grid_operand(2, 3 * n, k, fmt, groups=3)
    for raw in ([0, 40, 20, 64], [-5, 10, 30, 200], [9, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 7]):
        off = torch.tensor(raw, dtype=torch.int32, device="cuda")
        safe = np.maximum.accumulate(np.clip(raw, 0, rows))
        a = gk.Fp4Matrix.from_codes(codes, scales, rows, k, fmt, offsets=off)
        c = torch.full((rows, n), 7.0, device="cuda")
        product(a, b, c)
        assert gk.device_status(0) == 1 << 5
        want = torch.full_like(c, 7.0).double()
        for e in range(3):
            i, j = int(safe[e]), int(safe[e + 1])
            want[i:j] = av[i:j] @ bv[e * n:(e + 1) * n].T
        assert torch.equal(c.double(), want)


def test_captured_layer_follows_its_inputs():
    """Quantise and multiply in a graph, with offsets and rows that change between replays; the same
    weights in two graphs on two streams."""
    torch = torch_cuda()
    rows, k, n, g, fmt = 180, 320, 264, 4, gk.FP4_NV
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, k, generator=gen, device="cuda").bfloat16()
    w = gk.quantize_fp4(gk.MatRef.from_row_major(torch.randn(g * n, k, generator=gen, device="cuda"),
                                                 n, k), fmt, scale=0.01, groups=g, x_gs=n * k)
    off = torch.tensor([0, 45, 90, 135, 180], dtype=torch.int32, device="cuda")
    runs = []
    for i in range(2):
        q = gk.Fp4Matrix.empty(rows, k, fmt, 0.02, offsets=off)
        c = torch.zeros(rows, n, device="cuda")
        s = torch.cuda.Stream()
        gr = torch.cuda.CUDAGraph()

        def step():
            gk.quantize_fp4(gk.MatRef.from_row_major(x, rows, k), fmt, out=q, sync=False)
            gk.gemm_fp4(float(i + 1), q, w, 0.0, gk.MatMut.from_row_major(c, rows, n), sync=False)
        step()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=s):
            step()
        runs.append((gr, s, c))
    wv = values(w).double()
    for o in ([0, 45, 90, 135, 180], [0, 180, 180, 180, 180], [3, 3, 4, 100, 177]):
        off.copy_(torch.tensor(o, dtype=torch.int32))
        x.copy_(torch.randn(rows, k, generator=gen, device="cuda"))
        for _, _, c in runs:
            c.fill_(7.0)
        torch.cuda.synchronize()
        for gr, s, _ in runs:
            with torch.cuda.stream(s):
                gr.replay()
                gr.replay()
        torch.cuda.synchronize()
        xv = torch.from_numpy(reference(x.double().cpu().numpy(), fmt, 0.02)).cuda().double()
        for i, (_, _, c) in enumerate(runs):
            want, mag = torch.full_like(c, 7.0).double(), torch.zeros_like(c).double()
            for e in range(g):
                s_ = slice(o[e], o[e + 1])
                we = wv[e * n:(e + 1) * n]
                want[s_] = (i + 1) * (xv[s_] @ we.T)
                mag[s_] = (i + 1) * (xv[s_].abs() @ we.abs().T)
            err = (c.double() - want).abs()
            assert bool((err <= (k + 40) * 2.0 ** -23 * mag).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_experts_layer(fmt):
    """The serving layer: routed rows quantised, first product, ReLU, quantised again, second
    product -- against the same steps on values (the first product's result is taken from the
    engine, since a border of the second quantisation may lie inside its rounding)."""
    torch = torch_cuda()
    sizes, d, h, g = [70, 0, 1, 33], 160, 288, 4
    rows = sum(sizes)
    off = torch.tensor(np.cumsum([0] + sizes), dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    s = 1.0 if fmt == gk.FP4_MX else 0.01
    x = torch.randn(rows, d, generator=gen, device="cuda").bfloat16()
    w1 = torch.randn(g, d, h, generator=gen, device="cuda").bfloat16()  # stored k x n
    w2 = torch.randn(g, d, h, generator=gen, device="cuda").bfloat16()  # stored n x k
    q1 = gk.quantize_fp4(gk.MatRef(w1, h, d, 1, h), fmt, scale=s, groups=g, x_gs=d * h)
    q2 = gk.quantize_fp4(gk.MatRef.from_row_major(w2, d, h), fmt, scale=s, groups=g, x_gs=d * h)

    def by_expert(a, w, n):
        o = off.tolist()
        wv = values(w).double().view(g, n, -1)
        av = values(a).double()
        want = torch.cat([av[o[e]:o[e + 1]] @ wv[e].T for e in range(g)])
        mag = torch.cat([av[o[e]:o[e + 1]].abs() @ wv[e].abs().T for e in range(g)])
        return want, (a.cols + 40) * 2.0 ** -23 * mag

    a1 = gk.quantize_fp4(mat(x), fmt, scale=s, offsets=off)
    h1 = torch.zeros(rows, h, device="cuda", dtype=torch.bfloat16)
    product(a1, q1, h1)
    want, tol = by_expert(a1, q1, h)
    assert bool(((h1.double() - want).abs() <= tol + 2.0 ** -8 * want.abs()).all())
    a2 = gk.quantize_fp4(mat(h1.relu()), fmt, scale=s, offsets=off)
    same(values(a2), reference(h1.relu().double().cpu().numpy(), fmt, s))
    y = torch.zeros(rows, d, device="cuda")
    product(a2, q2, y)
    want, tol = by_expert(a2, q2, d)
    assert bool(((y.double() - want).abs() <= tol).all())


def test_long_matrix_passes_32_bits():
    """Codes, scales and outputs past 2^31 elements."""
    torch = torch_cuda()
    rows, k, n, fmt = 530_000, 8192, 8, gk.FP4_MX  # 2.2 GB of codes, 4.3e9 elements
    q = gk.Fp4Matrix.empty(rows, k, fmt)
    q.data.zero_()
    q.scales.fill_(127)
    tail, tv = grid_parts(1, 300, k, fmt)[:2], grid_parts(1, 300, k, fmt)[2]
    t = gk.Fp4Matrix.from_codes(tail[0], tail[1], 300, k, fmt)
    # the last 300 rows as the last three scale blocks hold them (base = 4138 * 128)
    base = rows - 336
    q.data.view(rows, -1)[base:base + 300] = t.data.view(300, -1)
    nb = q.scales.numel() // -(-rows // 128)
    q.scales.view(-1, nb)[base // 128:base // 128 + 3] = t.scales.view(-1, nb)
    assert base % 128 == 0
    b, bv = grid_operand(2, n, k, fmt)
    c = torch.full((rows, n), 7.0, device="cuda")
    product(q, b, c)
    assert torch.equal(c[base:base + 300].double(), tv @ bv.T)
    assert not bool(c[:base].any())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k,n", [(2560, 320, 2560), (1300, 1000, 5000), (4097, 64, 1288),
                                   (300, 2304, 19000)])
def test_product_exact_large(fmt, m, k, n):
    """Sizes that the CTA-pair kernel takes: whole and cut tiles, short and long contractions."""
    torch = torch_cuda()
    a, av = grid_operand(m + k, m, k, fmt)
    b, bv = grid_operand(n + k + 1, n, k, fmt)
    c = torch.full((m, n), float("nan"), device="cuda")
    product(a, b, c)
    assert torch.equal(c.double(), av @ bv.T)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sizes,lead,tail", [([1000, 0, 700, 255, 257, 1, 2083], 2, 5),
                                             ([31, 4000, 33], 0, 1), ([300, 129, 160, 513], 0, 0)])
@pytest.mark.parametrize("k,n", [(320, 2600), (1000, 4224)])
def test_product_by_expert_large(fmt, sizes, lead, tail, k, n):
    test_product_by_expert(fmt, sizes, lead, tail, k, n)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,lead,tail,k,n", [([5, 0, 37, 2], 3, 4, 64, 136), ([20], 0, 0, 96, 40),
                                                 ([130, 0, 1, 255], 0, 2, 72, 264),
                                                 ([1000, 0, 700, 257], 2, 5, 320, 2600)])
def test_product_exact_16_bit(fmt, out, sizes, lead, tail, k, n):
    """16-bit C (whole 16-byte pieces, and rows that are not): the exact value rounded once."""
    torch = torch_cuda()
    rows, g = lead + sum(sizes) + tail, len(sizes)
    off = torch.tensor(np.cumsum([lead] + sizes), dtype=torch.int32, device="cuda")
    a, av = grid_operand(1, rows, k, fmt, offsets=off)
    b, bv = grid_operand(2, g * n, k, fmt, groups=g)
    buf = torch.full((rows, n + 16), 7.0, device="cuda", dtype=tdt(out))
    for c in (buf[:, 8:8 + n], buf[:, 3:3 + n]):
        buf.fill_(7.0)
        product(a, b, c, alpha=0.125)
        want = torch.full((rows, n), 7.0, device="cuda", dtype=torch.float64)
        o = off.tolist()
        for e in range(g):
            want[o[e]:o[e + 1]] = 0.125 * (av[o[e]:o[e + 1]] @ bv[e * n:(e + 1) * n].T)
        assert torch.equal(c, want.to(tdt(out)))
        at = c.storage_offset()
        assert bool((buf[:, :at] == 7).all()) and bool((buf[:, at + n:] == 7).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_empty_contractions_and_inputs(fmt):
    """k == 0: C <- beta * C on the groups' rows; no rows: nothing."""
    torch = torch_cuda()
    off = torch.tensor([1, 4, 4, 8], dtype=torch.int32, device="cuda")
    a = gk.Fp4Matrix.empty(9, 0, fmt, offsets=off)
    b = gk.Fp4Matrix.empty(3 * 24, 0, fmt, groups=3)
    for beta in (0.0, 0.5):
        for out in (torch.float32, torch.bfloat16):
            c = torch.full((9, 24), 8.0, device="cuda", dtype=out)
            product(a, b, c, beta=beta)
            want = torch.full_like(c, 8.0)
            want[1:8] *= beta
            assert torch.equal(c, want)
    x = torch.zeros(0, 64, device="cuda")
    q = gk.quantize_fp4(gk.MatRef(x, 0, 64, 64, 1), fmt)
    w = gk.quantize_fp4(mat(torch.zeros(24, 64, device="cuda")), fmt)
    product(q, w, torch.zeros(0, 24, device="cuda"))
    assert q.rows == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_most_groups(fmt):
    torch = torch_cuda()
    sizes = [(i * 7) % 5 if i % 3 == 0 else 0 for i in range(1024)]
    rows = sum(sizes)
    off = torch.tensor(np.cumsum([0] + sizes), dtype=torch.int32, device="cuda")
    a, av = grid_operand(1, rows, 96, fmt, offsets=off)
    b, bv = grid_operand(2, 1024 * 24, 96, fmt, groups=1024)
    c = torch.full((rows, 24), 7.0, device="cuda")
    product(a, b, c)
    o = off.tolist()
    want = torch.cat([av[o[e]:o[e + 1]] @ bv[e * 24:(e + 1) * 24].T for e in range(1024)])
    assert torch.equal(c.double(), want)


def test_extreme_matrix_scales():
    """Matrix scales at the ends of their range whose product is 1."""
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(40, 96, generator=gen, device="cuda")
    w = torch.randn(56, 96, generator=gen, device="cuda")
    one = [gk.quantize_fp4(mat(t), gk.FP4_NV) for t in (x, w)]
    far = [gk.quantize_fp4(mat(t * s), gk.FP4_NV, scale=s)
           for t, s in ((x, 2.0 ** 100), (w, 2.0 ** -100))]
    c = [torch.zeros(40, 56, device="cuda") for _ in range(2)]
    product(*one, c[0])
    product(*far, c[1])
    assert torch.equal(c[0], c[1])


@pytest.mark.parametrize("fmt", FMTS)
def test_chain_without_synchronisation(fmt):
    """A chain of quantise, product by expert, 16-bit grouped product and back, every call reading
    what the one before wrote and writing buffers that earlier calls read, with nothing waited for:
    the same bits as with a synchronisation after every call."""
    torch = torch_cuda()
    rows, d, h, g = 700, 512, 384, 3
    gen = torch.Generator(device="cuda").manual_seed(5)
    off = torch.tensor([0, 300, 301, 700], dtype=torch.int32, device="cuda")
    s = 1.0 if fmt == gk.FP4_MX else 0.002
    w4 = gk.quantize_fp4(gk.MatRef.from_row_major(
        torch.randn(g * h, d, generator=gen, device="cuda") * d ** -0.5, h, d), fmt, scale=s, groups=g,
        x_gs=h * d)
    w2 = (torch.randn(g, h, d, generator=gen, device="cuda") * h ** -0.5).bfloat16()
    x0 = torch.randn(rows, d, generator=gen, device="cuda").bfloat16()

    def chain(sync):
        x, y = x0.clone(), torch.zeros(rows, h, device="cuda", dtype=torch.bfloat16)
        q = gk.Fp4Matrix.empty(rows, d, fmt, s, offsets=off)
        for _ in range(30):
            gk.quantize_fp4(gk.MatRef.from_row_major(x, rows, d), fmt, out=q, sync=sync)
            gk.gemm_fp4(1.0, q, w4, 0.0, gk.MatMut.from_row_major(y, rows, h), sync=sync)
            gk.gemm_half_grouped(1.0, gk.MatRef.from_row_major(y, rows, h),
                                 gk.MatRef.from_row_major(w2, h, d), h * d, off, 0.0,
                                 gk.MatMut.from_row_major(x, rows, d), sync=sync)
        torch.cuda.synchronize()
        return x

    want = chain(True)
    assert bool(want.isfinite().all()) and float(want.abs().max()) > 0
    for _ in range(5):
        assert torch.equal(chain(False), want)


def test_result_memory_belongs_to_the_call_s_stream():
    """A matrix that quantize_fp4 makes for another stream does not lie where the current stream may
    still be writing: a buffer freed behind a delayed fill."""
    torch = torch_cuda()
    rows, k = 4096, 4096
    x = torch.randn(rows, k, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    X = gk.MatRef.from_row_major(x, rows, k)
    want = gk.quantize_fp4(X, gk.FP4_MX)
    size = want._data.numel()
    other = torch.cuda.Stream()
    torch.zeros(8, dtype=torch.uint8, device="cuda").fill_(1)  # a kernel's first use waits
    torch.cuda.synchronize()
    held = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(40_000_000)  # some 20 milliseconds on the current stream
    held.fill_(0x55)
    del held
    q = gk.quantize_fp4(X, gk.FP4_MX, stream=other.cuda_stream, sync=False)
    torch.cuda.synchronize()
    assert torch.equal(q._data, want._data)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [9, 50, 2048])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("alpha", [float("inf"), float("nan")])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_product_without_contraction_ignores_alpha(fmt, rows, out, alpha, beta):
    """k == 0: C <- beta * C on the groups' rows whatever alpha is."""
    torch = torch_cuda()
    off = torch.tensor([1, 4, 4, rows - 1], dtype=torch.int32, device="cuda")
    a = gk.Fp4Matrix.empty(rows, 0, fmt, offsets=off)
    b = gk.Fp4Matrix.empty(3 * 24, 0, fmt, groups=3)
    c = torch.full((rows, 24), 8.0, device="cuda", dtype=tdt(out))
    product(a, b, c, alpha, beta)
    want = torch.full_like(c, 8.0)
    want[1:rows - 1] = 8.0 * beta
    assert torch.equal(c, want)
