"""A feed-forward layer's products with their epilogues and their backward pass, against 64-bit forms.

Bounds. The accumulators: products of 16-bit floats are exact in f32, a step of the sum loses at most
2^-23 of the sum of magnitudes, at most k + 32 steps; alpha and the bias add a rounding of 2^-24 each
(counted as 4 steps). Activations and derivatives: |act'| < 1.13, |act''| < 1.2; their own evaluation in
f32 is at most 2^-20 |z| off for values (Phi to 7.5e-8, half of the 1.5e-7 that formula 7.1.26 of Abramowitz
and Stegun leaves, and a few roundings; sigma to 2^-21 relative, and sigma (1 - sigma) |t| < 0.23 for the
error of its argument) and 2^-18 for derivatives, which add two such terms of |z| phi(z) and z sigma
(1 - sigma) 2 u' < 0.6. R adds one rounding; the type half a step.
Small integers make the accumulators exact, and the piecewise linear activations then leave one rounding.
Column sums: each value's bound, and 2^-24 of the sum of magnitudes for each of at most 256 + 16 steps.
"""
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from layer_util import (ACTS, HALF_STEP, SUBNORMAL, act64, act8_values, act_of, mut, numbers, offsets_of,
                        ref, slope64, spans, status_clean, tdt)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    status_clean()


def stack_ref(b):
    """(group 0's view inside the stack's slice, group stride) of a groups x k x n tensor view."""
    g, k, n = b.shape
    gs, rs, cs = b.stride()
    m = (g - 1) * gs + (k - 1) * rs + (n - 1) * cs + 1
    return gk.MatRef(b.as_strided((m,), (1,)), k, n, rs, cs), gs


def product64(a, b, off):
    """(sum, sum of magnitudes) of each row with its group's matrix; rows of no group are 0."""
    torch = torch_cuda()
    z = torch.zeros(a.shape[0], b.shape[2], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(z)
    for g, s in spans(off, a.shape[0]):
        z[s] = a[s].double() @ b[g].double()
        mag[s] = a[s].double().abs() @ b[g].double().abs()
    return z, mag


def bias64(bias, off, like):
    torch = torch_cuda()
    out = torch.zeros_like(like)
    if bias is not None:
        for g, s in spans(off, like.shape[0]):
            out[s] = bias[g].double()
    return out


def in_groups(off, rows):
    torch = torch_cuda()
    m = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for _, s in spans(off, rows):
        m[s] = True
    return m


def near(got, want, tol, dtype):
    torch = torch_cuda()
    tol = tol + HALF_STEP[dtype] * want.abs() + SUBNORMAL[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def forward(a, b, off, dtype, act, bias=None, r=None, c=None, z=None, alpha=1.0, **kw):
    bv, gs = stack_ref(b)
    gk.gemm_half_epilogue(alpha, ref(a), bv, mut(c), bias=bias, act=act_of(act),
                          residual=None if r is None else ref(r), z=None if z is None else mut(z),
                          offsets=off, b_gs=gs, is_f16=dtype == "f16", **kw)


def check_forward(a, b, off, dtype, act, bias, r, c, z, c0, z0, alpha=1.0, out=None, exact=False):
    torch = torch_cuda()
    out = out or dtype
    k = a.shape[1]
    s, mag = product64(a, b, off)
    s, mag = alpha * s, abs(alpha) * mag
    bv = bias64(bias, off, s)
    zw = s + bv
    cw = act64(zw, act)
    if r is not None:
        cw = cw + r.double()
    live = in_groups(off, a.shape[0])
    if exact:
        assert torch.equal(c[live].double(), cw[live].to(tdt(out)).double())
        if z is not None:
            assert torch.equal(z[live].double(), zw[live].to(tdt(dtype)).double())
    else:
        ez = (k + 36) * 2.0 ** -23 * (mag + bv.abs())
        ec = 1.13 * ez + 2.0 ** -20 * zw.abs() + 2.0 ** -24 * (cw.abs() + act64(zw, act).abs())
        near(c[live], cw[live], ec[live], out)
        if z is not None:
            near(z[live], zw[live], ez[live], dtype)
    assert torch.equal(c[~live], c0[~live])
    if z is not None:
        assert torch.equal(z[~live], z0[~live])


SIZES = [
    (None, 1), (None, 37), (None, 300),
    ([1], 1), ([0, 1, 0], 1), ([5, 0, 37, 2], 51), ([130, 0, 1, 255], 388), ([0, 0], 5), ([3] * 70, 210),
]
WIDTHS = [(64, 128), (16, 8), (200, 136), (33, 65), (1, 1), (72, 302)]


def problem(sizes, rows, k, n, dtype, major, seed=0, ints=True):
    """a, b, offsets; rows of no group hold values that would show anywhere."""
    off = None if sizes is None else offsets_of(sizes, 3 if rows > sum(sizes) + 3 else 0)
    groups = 1 if sizes is None else len(sizes)
    std = 1.0 if ints else k ** -0.5
    a = numbers(seed + 1, (rows, k), dtype, ints)
    b = numbers(seed + 2, (groups, n, k), dtype, ints, std).transpose(1, 2) if major == "k" else \
        numbers(seed + 2, (groups, k, n), dtype, ints, std)
    a[~in_groups(off, rows)] = float("nan")
    return a, b, off, groups


@pytest.mark.parametrize("sizes,rows", SIZES)
@pytest.mark.parametrize("k,n", WIDTHS)
@pytest.mark.parametrize("major", ["k", "n"])
def test_forward_exact(sizes, rows, k, n, major):
    """Integers through the piecewise linear activations: one rounding, compared for equality."""
    torch = torch_cuda()
    dtype = "bf16" if (k + n) % 3 else "f16"
    act = ["none", "relu", "leaky"][(rows + n) % 3]
    a, b, off, groups = problem(sizes, rows, k, n, dtype, major)
    bias = numbers(3, (groups, n), dtype)
    r = numbers(4, (rows, n), dtype)
    c0 = torch.full((rows, n), 7.0, dtype=tdt(dtype), device="cuda")
    for with_r, with_z, with_b in ((True, True, True), (False, False, True), (False, True, False)):
        c, z = c0.clone(), c0.clone()
        forward(a, b, off, dtype, act, bias if with_b else None, r if with_r else None, c,
                z if with_z else None)
        check_forward(a, b, off, dtype, act, bias if with_b else None, r if with_r else None, c,
                      z if with_z else None, c0, c0, exact=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
def test_forward_activations(act, dtype, out):
    torch = torch_cuda()
    a, b, off, groups = problem([100, 0, 31], 140, 200, 264, dtype, "k", 10, ints=False)
    a = a * 2
    bias = numbers(13, (groups, 264), "f32" if out == "f32" else dtype, False)
    r = numbers(14, (140, 264), out, False)
    c0 = torch.full((140, 264), 7.0, dtype=tdt(out), device="cuda")
    z0 = c0.to(tdt(dtype))
    c, z = c0.clone(), z0.clone()
    forward(a, b, off, dtype, act, bias, r, c, z, alpha=0.75)
    check_forward(a, b, off, dtype, act, bias, r, c, z, c0, z0, alpha=0.75, out=out)


# the CTA-pair kernels: tall tiles (even widths), square ones (f32, odd widths), ragged groups
LARGE = [(None, 2047, 128, 4096, "bf16"), (None, 2048, 200, 4098, "f16"),
         ([700, 0, 1500, 257, 600], 3060, 96, 4096, "bf16"), (None, 2049, 64, 4097, "f32")]


@pytest.mark.parametrize("sizes,rows,k,n,out", LARGE)
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_forward_pairs(sizes, rows, k, n, out, act):
    torch = torch_cuda()
    dtype = "bf16" if out == "f32" else out
    exact = act != "gelu"
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "k" if act == "none" else "n", 20, exact)
    bias = numbers(23, (groups, n), dtype, exact)
    r = numbers(24, (rows, n), out, exact)
    c0 = torch.full((rows, n), 7.0, dtype=tdt(out), device="cuda")
    z0 = c0.to(tdt(dtype))
    c, z = c0.clone(), z0.clone()
    forward(a, b, off, dtype, act, bias, r, c, z)
    check_forward(a, b, off, dtype, act, bias, r, c, z, c0, z0, out=out, exact=exact)
    again = c0.clone()
    forward(a, b, off, dtype, act, bias, r, again, z)
    assert torch.equal(c, again)


# long contractions: tall tiles, whole and ragged
TALL = [(None, 2047, 4096, "bf16"), ([700, 0, 1500, 257], 2460, 4098, "f16"), (None, 2048, 4102, "bf16")]


@pytest.mark.parametrize("sizes,rows,n,dtype", TALL)
@pytest.mark.parametrize("act", ["none", "leaky", "silu"])
def test_forward_tall(sizes, rows, n, dtype, act):
    torch = torch_cuda()
    k, exact = 4168, act != "silu"
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "k" if act == "none" else "n", 26, exact)
    bias = numbers(27, (groups, n), dtype, exact)
    r = numbers(28, (rows, n), dtype, exact)
    c0 = torch.full((rows, n), 7.0, dtype=tdt(dtype), device="cuda")
    c, z = c0.clone(), c0.clone()
    forward(a, b, off, dtype, act, bias, r, c, z)
    check_forward(a, b, off, dtype, act, bias, r, c, z, c0, c0, exact=exact)
    onto = r.clone()  # C is the residual itself
    forward(a, b, off, dtype, act, bias, onto, onto)
    live = in_groups(off, rows)
    assert torch.equal(onto[live], c[live]) and torch.equal(onto[~live], r[~live])


# few tiles and a long contraction: clusters that share a tile, of 8, 4 and 2 CTAs
SHARED = [(None, 1, 4096, 300), (None, 17, 1000, 264), (None, 33, 2050, 512), (None, 100, 600, 1100),
          (None, 128, 4100, 7000), ([3, 0, 20, 9], 40, 777, 250), ([70, 58], 128, 1030, 1024)]


@pytest.mark.parametrize("sizes,rows,k,n", SHARED)
@pytest.mark.parametrize("act,out", [("relu", "bf16"), ("leaky", "f32"), ("gelu", "f16")])
def test_forward_shared_tiles(sizes, rows, k, n, act, out):
    torch = torch_cuda()
    dtype, exact = ("f16" if out == "f16" else "bf16"), act != "gelu"
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "k" if n % 8 else "n", 25, exact)
    bias = numbers(28, (groups, n), dtype, exact)
    r = numbers(29, (rows, n), out, exact)
    c0 = torch.full((rows, n), 7.0, dtype=tdt(out), device="cuda")
    z0 = c0.to(tdt(dtype))
    c, z = c0.clone(), z0.clone()
    forward(a, b, off, dtype, act, bias, r, c, z)
    check_forward(a, b, off, dtype, act, bias, r, c, z, c0, z0, out=out, exact=exact)
    again = c0.clone()
    forward(a, b, off, dtype, act, bias, r, again)
    assert torch.equal(c, again)


@pytest.mark.parametrize("rows,k,n", [(3, 40, 24), (150, 64, 130), (2048, 64, 4096)])
def test_forward_onto_the_residual(rows, k, n):
    """C is the residual itself."""
    torch = torch_cuda()
    a, b, _, _ = problem(None, rows, k, n, "bf16", "k", 30)
    c = numbers(33, (rows, n), "bf16")
    r = c.clone()
    forward(a, b, None, "bf16", "relu", None, c, c)
    check_forward(a, b, None, "bf16", "relu", None, r, c, None, r, None, exact=True)


@pytest.mark.parametrize("layout", ["columns", "wide", "odd", "shifted"])
def test_forward_strides(layout):
    torch = torch_cuda()
    rows, k, n = 70, 48, 66
    a, b, _, _ = problem(None, rows, k, n, "f16", "k", 40)
    bias = numbers(43, (1, n), "f16")

    def make(seed):
        x = numbers(seed, (rows, n), "f16")
        if layout == "columns":
            return x.t().contiguous().t()
        pitch, lead = {"wide": (160, 0), "odd": (77, 0), "shifted": (80, 1)}[layout]
        buf = torch.full((rows * pitch + lead,), 9.0, dtype=tdt("f16"), device="cuda")
        v = buf[lead:].view(rows, pitch)[:, :n]
        v.copy_(x)
        return v

    r, c, z = make(44), make(45), make(46)
    buf = c._base
    outside = None
    if layout != "columns":
        keep = buf.clone()
        keep.as_strided(c.shape, c.stride(), c.storage_offset()).zero_()
        outside = keep
    forward(a, b, None, "f16", "leaky", bias, r, c, z)
    check_forward(a, b, None, "f16", "leaky", bias, r, c, z, c, z, exact=True)
    if outside is not None:  # nothing beside the views is written
        now = buf.clone()
        now.as_strided(c.shape, c.stride(), c.storage_offset()).zero_()
        assert torch.equal(now, outside)


@pytest.mark.parametrize("k,alpha", [(0, 1.0), (24, 0.0), (0, float("nan"))])
def test_forward_without_a_product(k, alpha):
    """k == 0 or alpha == 0: C <- act(bias) + R, whatever A and B hold."""
    torch = torch_cuda()
    rows, n = 40, 34
    a = torch.full((rows, k), float("nan"), dtype=torch.bfloat16, device="cuda")
    b = torch.full((2, k, n), float("inf"), dtype=torch.bfloat16, device="cuda")
    off = offsets_of([10, 25])
    bias, r = numbers(51, (2, n), "bf16"), numbers(52, (rows, n), "bf16")
    c0 = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
    c, z = c0.clone(), c0.clone()
    gk.gemm_half_epilogue(alpha, gk.MatRef(a.reshape(-1), rows, k, max(k, 1), 1),
                          gk.MatRef(b.reshape(-1), k, n, n, 1), mut(c), bias=bias,
                          act=act_of("relu"), residual=ref(r), z=mut(z), offsets=off, b_gs=k * n)
    want = bias64(bias, off, c.double())
    assert torch.equal(z[:35].double(), want[:35])
    assert torch.equal(c[:35].double(), want[:35].clamp(min=0) + r[:35].double())
    assert torch.equal(c[35:], c0[35:]) and torch.equal(z[35:], c0[35:])


def test_forward_special_values():
    """Infinities and NaN through each activation: limits, and the engine's rule for ReLU."""
    torch = torch_cuda()
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([inf, -inf, nan, 0.0, -200.0, 200.0, -1e30, 1e30], dtype=torch.bfloat16,
                     device="cuda")
    n = x.numel()
    a = torch.zeros(2, 8, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(1, 8, n, dtype=torch.bfloat16, device="cuda")
    big = float(x[7])
    want = {"none": [inf, -inf, nan, 0, -200, 200, -big, big], "relu": [inf, 0, 0, 0, 0, 200, 0, big],
            "leaky": [inf, -inf, 0, 0, -25, 200, -big / 8, big],
            "gelu": [inf, 0, nan, 0, 0, 200, 0, big], "gelu_tanh": [inf, 0, nan, 0, 0, 200, 0, big],
            "silu": [inf, 0, nan, 0, 0, 200, 0, big]}
    for act, w in want.items():
        c = torch.empty(2, n, dtype=torch.float32, device="cuda")
        forward(a, b, None, "bf16", act, x.view(1, n), None, c)
        w = torch.tensor(w, device="cuda").expand(2, n)
        assert torch.equal(c.isnan(), w.isnan()), act
        ok = ~w.isnan()
        assert torch.equal(c[ok], w[ok]), act


def backward(a, b, off, dtype, z, act, c, dbias=None, alpha=1.0, **kw):
    bv, gs = stack_ref(b)
    gk.gemm_half_dact(alpha, ref(a), bv, z if z is None or isinstance(z, gk.Act8Matrix) else ref(z),
                      act_of(act), mut(c), dbias=dbias, offsets=off, b_gs=gs, is_f16=dtype == "f16", **kw)


def check_backward(d, ed, z, off, dtype, act, c, c0, dbias, out=None, exact=False):
    """d: what reaches the activation, 64 bits, off by at most ed; z: the activation's input, 64 bits."""
    torch = torch_cuda()
    out = out or dtype
    rows = d.shape[0]
    g = slope64(z, act) if z is not None else torch.ones_like(d)
    want = d * g
    live = in_groups(off, rows)
    ec = 1.13 * ed + 2.0 ** -18 * d.abs() if act not in ("none", "relu", "leaky") else ed
    ec = ec + 2.0 ** -23 * want.abs()
    if c is not None:
        if exact:
            assert torch.equal(c[live].double(), want[live].to(tdt(out)).double())
        else:
            near(c[live], want[live], ec[live], out)
        assert torch.equal(c[~live], c0[~live])
    if dbias is not None:
        bt = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[dbias.dtype]
        for g_, s in spans(off, rows):
            w = want[s].sum(0)
            if exact:  # integers: sums are exact below 2^24
                assert torch.equal(dbias[g_].double(), w.to(dbias.dtype).double())
            else:
                near(dbias[g_], w, ec[s].sum(0) + 272 * 2.0 ** -24 * want[s].abs().sum(0), bt)


@pytest.mark.parametrize("sizes,rows", SIZES)
@pytest.mark.parametrize("k,n", WIDTHS)
@pytest.mark.parametrize("zform", ["half", "act8"])
def test_backward_exact(sizes, rows, k, n, zform):
    torch = torch_cuda()
    dtype = "bf16" if (k + n) % 3 else "f16"
    act = ["none", "relu", "leaky"][(rows + n) % 3]
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "n" if n % 2 else "k", 60)
    z = numbers(63, (rows, n), dtype)
    q = gk.quantize_act8(ref(z)) if zform == "act8" else z
    c0 = torch.full((rows, n), 7.0, dtype=tdt(dtype), device="cuda")
    c = c0.clone()
    dbias = torch.full((groups, n), 5.0, dtype=torch.float32, device="cuda")
    backward(a, b, off, dtype, q, act, c, dbias, alpha=0.5)
    d, mag = product64(a, b, off)
    check_backward(0.5 * d, 0 * mag, z.double(), off, dtype, act, c, c0, dbias, exact=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,out,zform", [("bf16", "bf16", "act8"), ("f16", "f16", "half"),
                                             ("bf16", "f32", "half"), ("f16", "f32", "act8")])
def test_backward_activations(act, dtype, out, zform):
    torch = torch_cuda()
    a, b, off, groups = problem([100, 0, 31], 140, 200, 264, dtype, "n", 70, ints=False)
    z = numbers(73, (140, 264), dtype, False, 2.0)
    q = gk.quantize_act8(ref(z)) if zform == "act8" else z
    z64 = act8_values(q) if zform == "act8" else z.double()
    c0 = torch.full((140, 264), 7.0, dtype=tdt(out), device="cuda")
    c = c0.clone()
    dbias = torch.empty(groups, 264, dtype=tdt(out), device="cuda")
    backward(a, b, off, dtype, q, act, c, dbias)
    d, mag = product64(a, b, off)
    check_backward(d, 236 * 2.0 ** -23 * mag, z64, off, dtype, act, c, c0, dbias, out)


@pytest.mark.parametrize("sizes,rows,k,n,out", LARGE)
@pytest.mark.parametrize("act,zform", [("none", None), ("relu", "act8"), ("gelu", "half"), ("silu", "act8")])
def test_backward_pairs(sizes, rows, k, n, out, act, zform):
    torch = torch_cuda()
    dtype = "bf16" if out == "f32" else out
    exact = act in ("none", "relu")
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "k" if act == "relu" else "n", 80, exact)
    z = numbers(83, (rows, n), dtype, exact, 2.0)
    q = {"act8": lambda: gk.quantize_act8(ref(z)), "half": lambda: z, None: lambda: None}[zform]()
    z64 = act8_values(q) if zform == "act8" else z.double()
    c0 = torch.full((rows, n), 7.0, dtype=tdt(out), device="cuda")
    c = c0.clone()
    dbias = torch.empty(groups, n, dtype=torch.float32, device="cuda")
    backward(a, b, off, dtype, q, act, c, dbias)
    d, mag = product64(a, b, off)
    check_backward(d, (k + 36) * 2.0 ** -23 * mag, z64, off, dtype, act, c, c0, dbias, out, exact)
    again = torch.empty_like(dbias)
    backward(a, b, off, dtype, q, act, c, again)
    assert torch.equal(dbias, again)


@pytest.mark.parametrize("sizes,rows,n,dtype", TALL)
@pytest.mark.parametrize("act,zform", [("none", None), ("relu", "act8"), ("gelu", "half"), ("gelu_tanh", "act8")])
def test_backward_tall(sizes, rows, n, dtype, act, zform):
    torch = torch_cuda()
    k, exact = 8200, act in ("none", "relu")
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "k" if act == "relu" else "n", 86, exact)
    if exact:  # sums over k and the rows stay below 2^24
        a = a.clamp(-1, 1)
    z = numbers(87, (rows, n), dtype, exact, 2.0)
    q = {"act8": lambda: gk.quantize_act8(ref(z)), "half": lambda: z, None: lambda: None}[zform]()
    z64 = act8_values(q) if zform == "act8" else z.double()
    c0 = torch.full((rows, n), 7.0, dtype=tdt(dtype), device="cuda")
    c = c0.clone()
    dbias = torch.empty(groups, n, dtype=torch.float32, device="cuda")
    backward(a, b, off, dtype, q, act, c, dbias)
    d, mag = product64(a, b, off)
    check_backward(d, (k + 36) * 2.0 ** -23 * mag, z64, off, dtype, act, c, c0, dbias, exact=exact)
    again = torch.empty_like(dbias)
    backward(a, b, off, dtype, q, act, c, again)
    assert torch.equal(dbias, again)


@pytest.mark.parametrize("sizes,rows,k,n", SHARED)
@pytest.mark.parametrize("act,zform,out", [("relu", "act8", "bf16"), ("leaky", "half", "f32"),
                                           ("silu", "act8", "f16")])
def test_backward_shared_tiles(sizes, rows, k, n, act, zform, out):
    torch = torch_cuda()
    dtype, exact = ("f16" if out == "f16" else "bf16"), act != "silu"
    a, b, off, groups = problem(sizes, rows, k, n, dtype, "k" if n % 8 else "n", 85, exact)
    z = numbers(88, (rows, n), dtype, exact, 2.0)
    q = gk.quantize_act8(ref(z)) if zform == "act8" else z
    z64 = act8_values(q) if zform == "act8" else z.double()
    c0 = torch.full((rows, n), 7.0, dtype=tdt(out), device="cuda")
    c = c0.clone()
    dbias = torch.empty(groups, n, dtype=torch.float32, device="cuda")
    backward(a, b, off, dtype, q, act, c, dbias)
    d, mag = product64(a, b, off)
    check_backward(d, (k + 36) * 2.0 ** -23 * mag, z64, off, dtype, act, c, c0, dbias, out, exact)
    again = torch.empty_like(dbias)
    backward(a, b, off, dtype, q, act, c, again)
    assert torch.equal(dbias, again)


def test_backward_onto_z():
    """C is z itself, in small and in tall tiles."""
    torch = torch_cuda()
    for rows, k, n in ((5, 24, 40), (2048, 64, 4096)):
        a, b, _, _ = problem(None, rows, k, n, "bf16", "k", 90)
        z = numbers(93, (rows, n), "bf16")
        c = z.clone()
        backward(a, b, None, "bf16", c, "relu", c)
        d, mag = product64(a, b, None)
        check_backward(d, 0 * mag, z.double(), None, "bf16", "relu", c, c, None, exact=True)


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 4096), (65, 264), (777, 33), (2000, 520)])
@pytest.mark.parametrize("sizes", [None, "groups"])
@pytest.mark.parametrize("zform,act", [("half", "silu"), ("act8", "gelu"), (None, "none"), ("half", "relu")])
def test_act_backward(rows, n, sizes, zform, act):
    torch = torch_cuda()
    dtype, exact = ("f16", True) if act in ("none", "relu") else ("bf16", False)
    sizes = None if sizes is None else [rows // 3, 0, rows - rows // 3 - (1 if rows > 2 else 0)]
    off = None if sizes is None else offsets_of(sizes)
    groups = 1 if sizes is None else 3
    dy, z = numbers(101, (rows, n), dtype, exact), numbers(102, (rows, n), dtype, exact, 2.0)
    dy[~in_groups(off, rows)] = float("nan")
    q = {"act8": lambda: gk.quantize_act8(ref(z)), "half": lambda: z, None: lambda: None}[zform]()
    z64 = act8_values(q) if zform == "act8" else z.double()
    for out in (dtype, "f32"):
        c0 = torch.full((rows, n), 7.0, dtype=tdt(out), device="cuda")
        c = c0.clone()
        dbias = torch.full((groups, n), 3.0, device="cuda")
        args = (ref(dy), q if zform != "half" else ref(q), act_of(act))
        gk.act_backward(*args, mut(c), dbias=dbias, offsets=off, is_f16=dtype == "f16")
        d = torch.where(in_groups(off, rows)[:, None], dy.double(), 0.0)
        check_backward(d, 0 * d, z64, off, dtype, act, c, c0, dbias, out, exact)
        only = torch.full((groups, n), 3.0, device="cuda")
        gk.act_backward(*args, None, dbias=only, offsets=off, is_f16=dtype == "f16")
        assert torch.equal(only, dbias)
        c2 = c0.clone()
        gk.act_backward(*args, mut(c2), offsets=off, is_f16=dtype == "f16")
        assert torch.equal(c2, c)


def test_act_backward_strides_and_places():
    """Column-major operands, and dz in the place of dy."""
    torch = torch_cuda()
    rows, n = 130, 70
    dy, z = numbers(111, (rows, n), "bf16"), numbers(112, (rows, n), "bf16")
    want = torch.where(z > 0, dy, torch.zeros_like(dy))
    cm = dy.t().contiguous().t()
    c = torch.empty(n, rows, dtype=torch.bfloat16, device="cuda").t()
    gk.act_backward(ref(cm), ref(z), act_of("relu"), mut(c))
    assert torch.equal(c, want)
    gk.act_backward(ref(cm), ref(z), act_of("relu"), mut(cm))
    assert torch.equal(cm, want)
    odd = torch.zeros(rows, n + 1, dtype=torch.bfloat16, device="cuda")[:, 1:]
    odd.copy_(dy)
    gk.act_backward(ref(odd), ref(z), act_of("relu"), mut(odd))
    assert torch.equal(odd, want)


def test_broadcast_rows():
    """R, z and dY whose rows are all the same memory (row stride 0), as a sum's gradient arrives."""
    torch = torch_cuda()
    for rows, k, n in ((70, 48, 66), (2048, 64, 4096)):
        a, b, _, _ = problem(None, rows, k, n, "bf16", "n", 35)
        one = numbers(38, (1, n), "bf16")
        many = one.expand(rows, n)
        row = gk.MatRef(one.reshape(-1), rows, n, 0, 1)
        c0 = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        c = c0.clone()
        bv, gs = stack_ref(b)
        gk.gemm_half_epilogue(1.0, ref(a), bv, mut(c), act=act_of("relu"), residual=row)
        check_forward(a, b, None, "bf16", "relu", None, many, c, None, c0, None, exact=True)
        gk.gemm_half_dact(1.0, ref(a), bv, row, act_of("relu"), mut(c))
        d, mag = product64(a, b, None)
        check_backward(d, 0 * mag, many.double(), None, "bf16", "relu", c, c0, None, exact=True)
        dbias = torch.empty(n, device="cuda")
        gk.act_backward(row, ref(c), None, None, dbias=dbias)
        assert torch.equal(dbias.double(), rows * one[0].double())


def test_derivatives_at_special_values():
    torch = torch_cuda()
    inf = float("inf")
    z = torch.tensor([[inf, -inf, 0.0, 3e38, -3e38]], dtype=torch.bfloat16, device="cuda")
    dy = torch.ones_like(z)
    want = {"relu": [1, 0, 0, 1, 0], "leaky": [1, .125, .125, 1, .125], "gelu": [1, 0, .5, 1, 0],
            "gelu_tanh": [1, 0, .5, 1, 0], "silu": [1, 0, .5, 1, 0]}
    for act, w in want.items():
        dz = torch.empty(1, 5, device="cuda")
        gk.act_backward(ref(dy), ref(z), act_of(act), mut(dz))
        assert torch.equal(dz, torch.tensor([w], device="cuda", dtype=torch.float32)), act


def test_no_rows_leave_zero_sums():
    torch = torch_cuda()
    n = 33
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in ("dact", "act"):
        dbias = torch.full((3, n), 3.0, device="cuda")
        none = torch.empty(0, n, dtype=torch.bfloat16, device="cuda")
        b = numbers(1, (3, 8, n), "bf16")
        if call == "dact":
            gk.gemm_half_dact(1.0, gk.MatRef(torch.empty(0, dtype=torch.bfloat16, device="cuda"), 0, 8, 8, 1),
                              stack_ref(b)[0], None, None, gk.MatMut(none.reshape(-1), 0, n, n, 1),
                              dbias=dbias, offsets=off, b_gs=8 * n)
        else:
            gk.act_backward(gk.MatRef(none.reshape(-1), 0, n, n, 1), None, None, None, dbias=dbias,
                            offsets=off)
        assert not dbias.any()


def test_gradients_against_differences():
    """dZ and dbias against differences of the forward pass: L = sum(G * C), C = act(A B + bias)."""
    torch = torch_cuda()
    rows, k, n = 6, 16, 10
    for act in ("gelu", "gelu_tanh", "silu"):
        a, b, _, _ = problem(None, rows, k, n, "f16", "k", 120, ints=False)
        bias = numbers(123, (1, n), "f32", False)
        g = numbers(124, (rows, n), "f16", False)

        def loss(bb):
            c = torch.empty(rows, n, device="cuda")
            z = torch.empty(rows, n, dtype=torch.float16, device="cuda")
            forward(a, b, None, "f16", act, bb, None, c, z)
            return c.double() * g.double(), z
        _, z = loss(bias)
        dbias = torch.empty(1, n, device="cuda")
        gk.act_backward(ref(g), ref(z), act_of(act), None, dbias=dbias, is_f16=True)
        h = 2.0 ** -6
        up, down = loss(bias + h)[0].sum(0), loss(bias - h)[0].sum(0)
        # differences: h^2 / 6 |act'''| < h^2 / 2, f32 values to 2^-18; z in 16 bits: 2^-11 |z| 1.2
        lim = g.double().abs().sum(0) * (h * h / 2 + 2.0 ** -18 / h) + \
            (g.double().abs() * z.double().abs()).sum(0) * 2.0 ** -11 * 1.2
        assert bool(((up - down) / (2 * h) - dbias[0].double()).abs().le(lim).all()), act


def test_captured_and_on_two_streams():
    """Calls captured into two graphs and replayed in turn, beside eager calls on other streams."""
    torch = torch_cuda()
    rows, k, n = 300, 96, 200
    cases = []
    for seed in (130, 140):
        a, b, off, groups = problem([100, 150, 50], rows, k, n, "bf16", "k", seed)
        z = numbers(seed + 5, (rows, n), "bf16")
        c = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        db = torch.empty(groups, n, device="cuda")
        cases.append((a, b, off, z, c, db))

    def call(x, **kw):
        a, b, off, z, c, db = x
        backward(a, b, off, "bf16", z, "relu", c, db, **kw)

    call(cases[0])
    graphs = []
    for x in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(x, sync=False)
        graphs.append(g)
    s = torch.cuda.Stream()
    for _ in range(3):
        for x in cases:
            x[4].zero_(), x[5].zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(s):
            graphs[1].replay()
        torch.cuda.synchronize()
        for a, b, off, z, c, db in cases:
            d, mag = product64(a, b, off)
            check_backward(d, 0 * mag, z.double(), off, "bf16", "relu", c, c, db, exact=True)
    # an explicit stream
    for x in cases:
        x[4].zero_(), x[5].zero_()
    torch.cuda.synchronize()
    call(cases[0], stream=s.cuda_stream, sync=False)
    call(cases[1], sync=False)
    torch.cuda.synchronize()
    for a, b, off, z, c, db in cases:
        d, mag = product64(a, b, off)
        check_backward(d, 0 * mag, z.double(), off, "bf16", "relu", c, c, db, exact=True)
