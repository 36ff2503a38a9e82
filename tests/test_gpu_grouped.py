"""The products of rows grouped by expert, and their weight gradients, against f64 products.

Two kinds of data. Small integers: every product and partial sum is an integer below 2^24, so f32
accumulation in any order is exact and results are compared for equality (16-bit outputs with the
f64 value rounded once). Normal data: products of 16-bit floats are exact in f32 (at most 22
significant bits); an accumulation step loses at most one unit of 2^-23 of the sum of magnitudes,
there are at most k + 32 of them, alpha and beta add two roundings of 2^-24 each, and the output type
half a step (2^-8 bf16, 2^-11 f16, 0 beyond the above for f32).
"""
import numpy as np
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 0.0}


@pytest.fixture(autouse=True)
def _status():
    yield
    assert gk.device_status(0) == 0


def tdt(name):
    torch = torch_cuda()
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def offsets_of(sizes, lead=0):
    torch = torch_cuda()
    return torch.tensor(np.cumsum([lead] + list(sizes)), dtype=torch.int32, device="cuda")


def data(seed, shape, dtype, ints=True):
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if ints:
        x = torch.randint(-4, 5, shape, generator=gen, device="cuda").float()
    else:
        x = torch.randn(shape, generator=gen, device="cuda")
    return x.to(tdt(dtype))


def view(t2, kind=gk.MatRef):
    """A MatRef / MatMut of a 2-D tensor view (its storage from its first element on)."""
    r, c = t2.shape
    rs, cs = t2.stride()
    n = (r - 1) * rs + (c - 1) * cs + 1 if t2.numel() else 0
    return kind((t2.data_ptr(), n), r, c, rs, cs)


def stack(t3, kind=gk.MatRef):
    """(view of group 0 in the slice of all groups, group stride) of a 3-D tensor view."""
    g, r, c = t3.shape
    gs, rs, cs = t3.stride()
    n = (g - 1) * gs + (r - 1) * rs + (c - 1) * cs + 1
    return kind((t3.data_ptr(), n), r, c, rs, cs), gs


def run_fwd(a, b, off, c, dtype, alpha=1.0, beta=0.0, stream=None, sync=True):
    """One grouped product through the C ABI; a, b, c are tensor views of any strides."""
    import ctypes as C
    from gemmkit_b200 import _lib
    bv, gs = stack(b)
    out = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}[str(c.dtype)]
    rc = _lib.load().gk_gemm_half_grouped(
        int(dtype == "f16"), off.numel() - 1, C.c_void_p(off.data_ptr()), alpha, view(a).c(),
        bv.c(), gs, beta, view(c, gk.MatMut).c(), out, gk.SERIAL.c(), gk._stream(stream))
    gk._check(rc)
    if sync:
        torch_cuda().cuda.synchronize()


def run_wgrad(a, b, off, c, dtype, alpha=1.0, beta=0.0):
    run_wgrad_async(a, b, off, c, dtype, alpha, beta)
    torch_cuda().cuda.synchronize()


def run_wgrad_async(a, b, off, c, dtype, alpha=1.0, beta=0.0):
    import ctypes as C
    from gemmkit_b200 import _lib
    cv, gs = stack(c, gk.MatMut)
    out = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}[str(c.dtype)]
    rc = _lib.load().gk_gemm_half_grouped_wgrad(
        int(dtype == "f16"), off.numel() - 1, C.c_void_p(off.data_ptr()), alpha, view(a).c(),
        view(b).c(), beta, cv.c(), gs, out, gk.SERIAL.c(), gk._stream(None))
    gk._check(rc)


def want_fwd(a, b, off, c0, alpha, beta):
    """(f64 result, f64 sum of magnitudes); rows outside the groups keep c0."""
    want, mag = c0.double().clone(), c0.double().abs()
    o = off.tolist()
    for g in range(len(o) - 1):
        s = slice(o[g], o[g + 1])
        x, w = a[s].double(), b[g].double()
        base = beta * c0[s].double() if beta else 0.0
        want[s] = alpha * (x @ w) + base
        mag[s] = abs(alpha) * (x.abs() @ w.abs()) + (abs(beta) * c0[s].double().abs() if beta else 0)
    return want, mag


def want_wgrad(a, b, off, c0, alpha, beta):
    o = off.tolist()
    w, m = [], []
    for g in range(len(o) - 1):
        s = slice(o[g], o[g + 1])
        base = beta * c0[g].double() if beta else 0.0
        w.append(alpha * (a[s].double().T @ b[s].double()) + base)
        m.append(abs(alpha) * (a[s].double().abs().T @ b[s].double().abs())
                 + (abs(beta) * c0[g].double().abs() if beta else 0.0))
    torch = torch_cuda()
    return torch.stack(w), torch.stack(m)


def check_near(got, want, mag, k, out):
    tol = (k + 32 + 4) * 2.0 ** -23 * mag + HALF_STEP[out] * want.abs() + 1e-30
    if out == "f16":
        tol = tol + 2.0 ** -25  # half a step of f16's subnormals
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


SIZES = [
    ([1], 0, 0),                       # one token, one expert
    ([0, 1, 0], 0, 0),                 # empty groups around one row
    ([5, 0, 37, 2], 3, 4),             # rows before the first and after the last group
    ([33, 64, 31], 0, 0),
    ([130, 0, 1, 255], 0, 2),
    ([300, 513], 1, 0),
    ([0, 0], 2, 3),                    # nothing at all
    ([3] * 70, 0, 0),                  # more groups than a warp
]
WIDTHS = [(64, 128), (16, 8), (200, 136), (1000, 72), (33, 65), (1, 1), (72, 300)]


@pytest.mark.parametrize("sizes,lead,tail", SIZES)
@pytest.mark.parametrize("k,n", WIDTHS)
@pytest.mark.parametrize("major", ["k", "n"])
def test_forward_exact(sizes, lead, tail, k, n, major):
    torch = torch_cuda()
    dtype = "bf16" if (k + n) % 3 else "f16"
    rows = lead + sum(sizes) + tail
    off = offsets_of(sizes, lead)
    a = data(1, (rows, k), dtype)
    b = data(2, (len(sizes), n, k), dtype).transpose(1, 2) if major == "k" else \
        data(2, (len(sizes), k, n), dtype)
    # rows that belong to no group hold values that would show anywhere
    a[:lead] = float("nan")
    a[rows - tail:] = float("inf")
    c = torch.full((rows, n), 7.0, device="cuda")
    run_fwd(a, b, off, c, dtype)
    want, _ = want_fwd(a, b, off, torch.full_like(c, 7.0), 1.0, 0.0)
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("sizes,lead,tail", SIZES)
@pytest.mark.parametrize("m,n", [(64, 128), (16, 8), (200, 136), (33, 65), (1, 1), (264, 72)])
def test_wgrad_exact(sizes, lead, tail, m, n):
    torch = torch_cuda()
    dtype = "bf16" if (m + n) % 3 else "f16"
    rows = lead + sum(sizes) + tail
    off = offsets_of(sizes, lead)
    a, b = data(1, (rows, m), dtype), data(2, (rows, n), dtype)
    for t in (a, b):
        t[:lead] = float("nan")
        t[rows - tail:] = float("inf")
    c = torch.full((len(sizes), m, n), 7.0, device="cuda")
    run_wgrad(a, b, off, c, dtype)
    want, _ = want_wgrad(a, b, off, c, 1.0, 0.0)
    assert torch.equal(c.double(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("out", ["half", "f32"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (-0.5, 1.0), (0.0, 2.0), (2.0, 0.25)])
@pytest.mark.parametrize("sizes", [[17, 0, 50], [700, 300]])
def test_forward_near(dtype, out, alpha, beta, sizes):
    torch = torch_cuda()
    out = dtype if out == "half" else out
    rows, k, n = sum(sizes), 1032, 392
    off = offsets_of(sizes)
    a = data(3, (rows, k), dtype, ints=False)
    b = data(4, (len(sizes), k, n), dtype, ints=False)
    c0 = data(5, (rows, n), out, ints=False)
    c = c0.clone()
    if beta == 0.0:
        c.fill_(float("nan"))  # beta == 0 never reads C
    if alpha == 0.0:
        a.fill_(float("nan"))  # alpha == 0 reads neither operand
    run_fwd(a, b, off, c, dtype, alpha, beta)
    want, mag = want_fwd(a.nan_to_num(), b, off, c0, alpha, beta)
    check_near(c, want, mag, k, out)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("out", ["half", "f32"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (-0.5, 1.0), (0.0, 2.0)])
def test_wgrad_near(dtype, out, alpha, beta):
    torch = torch_cuda()
    out = dtype if out == "half" else out
    sizes, m, n = [517, 0, 90, 1], 392, 264
    off = offsets_of(sizes)
    a = data(3, (sum(sizes), m), dtype, ints=False)
    b = data(4, (sum(sizes), n), dtype, ints=False)
    c0 = data(5, (len(sizes), m, n), out, ints=False)
    c = c0.clone()
    if beta == 0.0:
        c.fill_(float("nan"))
    run_wgrad(a, b, off, c, dtype, alpha, beta)
    want, mag = want_wgrad(a, b, off, c0, alpha, beta)
    check_near(c, want, mag, max(sizes), out)


@pytest.mark.parametrize("layout", ["padded", "odd_pitch", "offset", "a_col_major", "c_col_major",
                                    "b_strided", "shared_b", "one_col"])
def test_forward_strides(layout):
    """Pitches, misaligned bases and orders; what lies between the elements of C stays."""
    torch = torch_cuda()
    sizes, k, n, dtype = [40, 0, 91], 136, 200, "bf16"
    rows, g = sum(sizes), len(sizes)
    off = offsets_of(sizes)
    a, b = data(1, (rows, k), dtype), data(2, (g, k, n), dtype)
    cbuf = torch.full((rows, n), 7.0, device="cuda")
    c = cbuf
    if layout == "padded":
        a = data(1, (rows, k + 24), dtype)[:, :k]
        b = data(2, (g, k + 1, n + 8), dtype)[:, :k, :n]
        cbuf = torch.full((rows, n + 5), 7.0, device="cuda")
        c = cbuf[:, 2:2 + n]
    elif layout == "odd_pitch":
        a = data(1, (rows, k + 3), dtype)[:, :k]
        b = data(2, (g, n, k + 1), dtype)[:, :, :k].transpose(1, 2)
    elif layout == "offset":
        a = data(1, (rows, k + 8), dtype)[:, 1:1 + k]
        b = data(2, (g, k, n + 8), dtype)[:, :, 3:3 + n]
    elif layout == "a_col_major":
        a = data(1, (k, rows), dtype).t()
    elif layout == "c_col_major":
        cbuf = torch.full((n, rows), 7.0, device="cuda")
        c = cbuf.t()
    elif layout == "b_strided":
        b = data(2, (g, k, 2 * n), dtype)[:, :, ::2]
    elif layout == "shared_b":
        b = data(2, (1, k, n), dtype).expand(g, k, n)
    elif layout == "one_col":
        b, cbuf = b[:, :, :1], torch.full((rows, 1), 7.0, device="cuda")
        c = cbuf
    run_fwd(a, b, off, c, dtype)
    want, _ = want_fwd(a, b, off, c, 1.0, 0.0)
    assert torch.equal(c.double(), want)
    if layout == "padded":
        assert bool((cbuf[:, :2] == 7).all()) and bool((cbuf[:, 2 + n:] == 7).all())


@pytest.mark.parametrize("layout", ["padded", "odd_pitch", "offset", "a_col_major", "c_col_major"])
def test_wgrad_strides(layout):
    torch = torch_cuda()
    sizes, m, n, dtype = [40, 0, 91, 3], 136, 200, "f16"
    rows, g = sum(sizes), len(sizes)
    off = offsets_of(sizes)
    a, b = data(1, (rows, m), dtype), data(2, (rows, n), dtype)
    cbuf = torch.full((g, m + 1, n + 3), 7.0, device="cuda")
    c = cbuf[:, :m, :n]
    if layout == "padded":
        a, b = data(1, (rows, m + 24), dtype)[:, :m], data(2, (rows, n + 8), dtype)[:, :n]
    elif layout == "odd_pitch":
        a, b = data(1, (rows, m + 3), dtype)[:, :m], data(2, (rows, n + 1), dtype)[:, :n]
    elif layout == "offset":
        a, b = data(1, (rows, m + 8), dtype)[:, 1:1 + m], data(2, (rows, n + 8), dtype)[:, 3:3 + n]
    elif layout == "a_col_major":
        a = data(1, (m, rows), dtype).t()
    elif layout == "c_col_major":
        c = torch.full((g, n, m), 7.0, device="cuda").transpose(1, 2)
        cbuf = None
    run_wgrad(a, b, off, c, dtype)
    want, _ = want_wgrad(a, b, off, c, 1.0, 0.0)
    assert torch.equal(c.double(), want)
    if cbuf is not None:
        assert bool((cbuf[:, m:] == 7).all()) and bool((cbuf[:, :, n:] == 7).all())


def test_nan_stays_in_its_row_and_group():
    """A NaN in one row of A reaches that row of C only; in one group's rows, that group's weight
    gradient only."""
    torch = torch_cuda()
    sizes, k, n, dtype = [70, 50, 9], 128, 136, "bf16"
    off = offsets_of(sizes)
    a, b = data(1, (129, k), dtype), data(2, (3, k, n), dtype)
    a[75, 5] = float("nan")
    c = torch.zeros((129, n), device="cuda")
    run_fwd(a, b, off, c, dtype)
    bad = c.isnan().any(1)
    assert bad.nonzero().flatten().tolist() == [75] and bool(c[75].isnan().all())
    d = data(3, (129, n), dtype)
    w = torch.zeros((3, k, n), device="cuda")
    run_wgrad(a, d, off, w, dtype)
    assert bool(w[1, 5].isnan().all()) and int(w.isnan().sum()) == n
    want, _ = want_wgrad(a, d, off, w, 1.0, 0.0)
    assert torch.equal(w[0].double(), want[0]) and torch.equal(w[2].double(), want[2])


@pytest.mark.parametrize("raw", [[0, 40, 20, 64], [-5, 10, 30, 200], [9, 0, 0, 0],
                                 [2 ** 31 - 1, -2 ** 31, 5, 7], [70, 71, 72, 73]])
def test_bad_offsets_stay_inside_and_are_reported(raw):
    """Offsets that do not ascend inside the rows: the running maximum clamped to the rows."""
    torch = torch_cuda()
    rows, k, n, dtype = 64, 72, 136, "bf16"
    off = torch.tensor(raw, dtype=torch.int32, device="cuda")
    safe = np.maximum.accumulate(np.clip(raw, 0, rows))
    a, b = data(1, (rows, k), dtype), data(2, (3, k, n), dtype)
    c = torch.full((rows, n), 7.0, device="cuda")
    run_fwd(a, b, off, c, dtype)
    assert gk.device_status(0) == 1 << 5
    soff = torch.tensor(safe, dtype=torch.int32, device="cuda")
    want, _ = want_fwd(a, b, soff, torch.full_like(c, 7.0), 1.0, 0.0)
    assert torch.equal(c.double(), want)
    d = data(3, (rows, n), dtype)
    w = torch.full((3, k, n), 7.0, device="cuda")
    run_wgrad(a, d, off, w, dtype)
    assert gk.device_status(0) == 1 << 5
    want, _ = want_wgrad(a, d, soff, w, 1.0, 0.0)
    assert torch.equal(w.double(), want)


def test_gradients_against_differences():
    """loss = sum(G * C): the input and weight gradients equal differences of the forward product
    (integers: exact), through the Python entries."""
    torch = torch_cuda()
    sizes, k, n = [6, 0, 11], 24, 40
    rows, off = sum(sizes), offsets_of(sizes)
    a, w = data(1, (rows, k), "bf16"), data(2, (3, k, n), "bf16")
    g = data(3, (rows, n), "bf16")

    def loss(a, w):
        c = torch.zeros(rows, n, device="cuda")
        gk.gemm_half_grouped(1.0, gk.MatRef.from_row_major(a, rows, k),
                             gk.MatRef.from_row_major(w, k, n), k * n, off, 0.0,
                             gk.MatMut.from_row_major(c, rows, n))
        return float((c.double() * g.double()).sum())

    da = torch.zeros(rows, k, device="cuda")
    gk.gemm_half_grouped(1.0, gk.MatRef.from_row_major(g, rows, n),
                         gk.MatRef.from_col_major(w, n, k), k * n, off, 0.0,
                         gk.MatMut.from_row_major(da, rows, k))
    dw = torch.zeros(3, k, n, device="cuda")
    gk.gemm_half_grouped_wgrad(1.0, gk.MatRef.from_row_major(a, rows, k),
                               gk.MatRef.from_row_major(g, rows, n), off, 0.0,
                               gk.MatMut.from_row_major(dw, k, n), k * n)
    base = loss(a, w)
    for i, p in [(0, 0), (5, 23), (6, 1), (16, 12)]:
        a2 = a.clone()
        a2[i, p] += 1
        assert loss(a2, w) - base == float(da[i, p])
    for e, p, j in [(0, 0, 0), (1, 3, 4), (2, 23, 39), (2, 7, 11)]:
        w2 = w.clone()
        w2[e, p, j] += 1
        assert loss(a, w2) - base == float(dw[e, p, j])


def test_offsets_written_on_the_stream_and_graph_replay():
    """The offsets are read when the kernel runs: a captured call follows offsets and operands that
    change between replays; two graphs replayed on two streams do not disturb each other."""
    torch = torch_cuda()
    rows, k, n, dtype = 200, 136, 264, "bf16"
    a, b = data(1, (rows, k), dtype), data(2, (4, k, n), dtype)
    off = offsets_of([50, 50, 50, 50])
    cs, graphs = [], []
    for i in range(2):
        c = torch.zeros((rows, n), device="cuda")
        run_fwd(a, b, off, c, dtype)  # first use before the capture
        s = torch.cuda.Stream()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            run_fwd(a, b, off, c, dtype, alpha=float(i + 1), sync=False)
            run_fwd(a, b, off, c, dtype, alpha=float(i + 1), beta=1.0, sync=False)
        cs.append(c)
        graphs.append((gr, s))
    for sizes in ([50] * 4, [200, 0, 0, 0], [1, 2, 3, 194], [0, 0, 7, 0]):
        off.copy_(offsets_of(sizes))
        a.copy_(data(sizes[0] + 9, (rows, k), dtype))
        for c in cs:
            c.fill_(7.0)
        torch.cuda.synchronize()
        for gr, s in graphs:
            with torch.cuda.stream(s):
                for _ in range(3):
                    gr.replay()
        torch.cuda.synchronize()
        for i, c in enumerate(cs):
            want, _ = want_fwd(a, b, off, torch.full_like(c, 7.0), 2.0 * (i + 1), 0.0)
            assert torch.equal(c.double(), want)


def test_experts_layer_forward_and_backward():
    """The entries as a training step uses them: two expert products with a ReLU between, all four
    gradients, against the same layer in f64 (integer data, small enough to stay exact)."""
    torch = torch_cuda()
    sizes, d, h = [21, 0, 90, 17], 32, 48
    rows, off, g = sum(sizes), offsets_of(sizes), 4
    gen = torch.Generator(device="cuda").manual_seed(8)

    def small(*shape):
        return torch.randint(-1, 2, shape, generator=gen, device="cuda").to(torch.bfloat16)

    x, w1, w2, gy = small(rows, d), small(g, d, h), small(g, h, d), small(rows, d)
    M, U = gk.MatRef, gk.MatMut
    h1 = torch.zeros(rows, h, device="cuda", dtype=torch.bfloat16)
    gk.gemm_half_grouped(1.0, M.from_row_major(x, rows, d), M.from_row_major(w1, d, h), d * h, off,
                         0.0, U.from_row_major(h1, rows, h))
    r = h1.relu()
    y = torch.zeros(rows, d, device="cuda")
    gk.gemm_half_grouped(1.0, M.from_row_major(r, rows, h), M.from_row_major(w2, h, d), h * d, off,
                         0.0, U.from_row_major(y, rows, d))
    dr = torch.zeros(rows, h, device="cuda", dtype=torch.bfloat16)
    gk.gemm_half_grouped(1.0, M.from_row_major(gy, rows, d), M.from_col_major(w2, d, h), h * d, off,
                         0.0, U.from_row_major(dr, rows, h))
    dh = dr * (h1 > 0)
    dw2, dw1 = torch.zeros(g, h, d, device="cuda"), torch.zeros(g, d, h, device="cuda")
    gk.gemm_half_grouped_wgrad(1.0, M.from_row_major(r, rows, h), M.from_row_major(gy, rows, d), off,
                               0.0, U.from_row_major(dw2, h, d), h * d)
    gk.gemm_half_grouped_wgrad(1.0, M.from_row_major(x, rows, d), M.from_row_major(dh, rows, h), off,
                               0.0, U.from_row_major(dw1, d, h), d * h)
    dx = torch.zeros(rows, d, device="cuda")
    gk.gemm_half_grouped(1.0, M.from_row_major(dh, rows, h), M.from_col_major(w1, h, d), d * h, off,
                         0.0, U.from_row_major(dx, rows, d))
    X, W1, W2 = (t.double().requires_grad_() for t in (x, w1, w2))
    o = off.tolist()
    Y = torch.cat([(X[o[e]:o[e + 1]] @ W1[e]).relu() @ W2[e] for e in range(g)])
    Y.backward(gy.double())
    for got, want in ((y, Y), (dx, X.grad), (dw1, W1.grad), (dw2, W2.grad)):
        assert torch.equal(got.double(), want.detach())


def test_wide_rows_pass_32_bits():
    """Element offsets of A and C past 2^31: a group's rows at the end of a 4.3-GB matrix."""
    torch = torch_cuda()
    rows, k, n = 33_600, 64_000, 8
    a = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    a[-3:] = data(1, (3, k), "bf16")
    b = data(2, (1, k, n), "bf16")
    off = torch.tensor([rows - 3, rows], dtype=torch.int32, device="cuda")
    big = torch.zeros((rows, n), device="cuda")
    run_fwd(a, b, off, big, "bf16")
    want = a[-3:].double() @ b[0].double()
    assert torch.equal(big[-3:].double(), want) and not bool(big[:-3].any())


PAIR_SIZES = [([1000, 0, 700, 255, 257, 1, 2083], 2, 5), ([4096], 0, 0), ([31, 4000, 33], 0, 1)]


@pytest.mark.parametrize("sizes,lead,tail", PAIR_SIZES)
@pytest.mark.parametrize("k,n,major", [(136, 1512, "k"), (72, 2048, "n"), (1, 4096, "n"),
                                       (520, 1288, "n")])
def test_forward_exact_large(sizes, lead, tail, k, n, major):
    """Sizes that the CTA-pair kernel takes: whole and cut tiles on both sides."""
    test_forward_exact(sizes, lead, tail, k, n, major)


@pytest.mark.parametrize("sizes,lead,tail", PAIR_SIZES + [([16, 1, 0, 15, 17, 64, 63, 65], 0, 3)])
@pytest.mark.parametrize("m,n", [(1032, 1512), (2048, 2304), (264, 4104)])
def test_wgrad_exact_large(sizes, lead, tail, m, n):
    test_wgrad_exact(sizes, lead, tail, m, n)


HALF_SHAPES = [([5, 0, 37, 2], 3, 4, 64, 136), ([130, 0, 1, 255], 0, 2, 72, 264),
               ([3] * 70, 0, 0, 40, 8), ([64, 200, 16], 1, 0, 33, 72),
               ([1000, 0, 700, 255, 257, 1, 2083], 2, 5, 72, 1512), ([31, 4000, 33], 0, 1, 24, 2056)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,lead,tail,k,n", HALF_SHAPES)
def test_forward_exact_16_bit(dtype, sizes, lead, tail, k, n):
    """16-bit C (whole 16-byte pieces): the f64 value rounded once; rows outside the groups stay."""
    torch = torch_cuda()
    rows, off = lead + sum(sizes) + tail, offsets_of(sizes, lead)
    a, b = data(1, (rows, k), dtype), data(2, (len(sizes), k, n), dtype)
    buf = torch.full((rows, n + 16), 7.0, device="cuda", dtype=tdt(dtype))
    for c in (buf[:, 8:8 + n], buf[:, 3:3 + n]):  # aligned pieces, and not
        buf.fill_(7.0)
        run_fwd(a, b, off, c, dtype, alpha=0.5)
        want, _ = want_fwd(a, b, off, torch.full((rows, n), 7.0, device="cuda"), 0.5, 0.0)
        assert torch.equal(c, want.to(tdt(dtype)))
        at = c.storage_offset()
        assert bool((buf[:, :at] == 7).all()) and bool((buf[:, at + n:] == 7).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,m,n", [([5, 0, 37, 2], 40, 136), ([130, 0, 1, 255], 264, 72),
                                       ([1000, 0, 700, 17], 1032, 1512)])
def test_wgrad_exact_16_bit(dtype, sizes, m, n):
    torch = torch_cuda()
    off = offsets_of(sizes)
    a, b = data(1, (sum(sizes), m), dtype), data(2, (sum(sizes), n), dtype)
    c = torch.full((len(sizes), m + 1, n + 8), 7.0, device="cuda", dtype=tdt(dtype))
    run_wgrad(a, b, off, c[:, :m, :n], dtype, alpha=0.25)
    want, _ = want_wgrad(a, b, off, c, 0.25, 0.0)
    assert torch.equal(c[:, :m, :n], want.to(tdt(dtype)))
    assert bool((c[:, m:] == 7).all()) and bool((c[:, :, n:] == 7).all())


# Many full tiles and 16-bit C in whole pieces: tiles of 512 columns of C. Odd numbers of
# 256-column blocks, a last block of 8, contractions of one stage, of a few and of many.
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("major", ["k", "n"])
@pytest.mark.parametrize("sizes,lead,tail,n", [([1301, 0, 2, 2150], 3, 4, 4360),
                                               ([8192], 0, 0, 1288), ([2000, 3000, 257], 0, 1, 2304),
                                               ([1024] * 9, 0, 0, 1032)])
@pytest.mark.parametrize("k", [8, 72, 200, 1000])
def test_forward_exact_tall_tiles(dtype, major, sizes, lead, tail, n, k):
    torch = torch_cuda()
    rows, off = lead + sum(sizes) + tail, offsets_of(sizes, lead)
    a = data(1, (rows, k), dtype)
    b = data(2, (len(sizes), n, k), dtype).transpose(1, 2) if major == "k" else \
        data(2, (len(sizes), k, n), dtype)
    a[:lead] = float("nan")
    a[rows - tail:] = float("inf")
    c = torch.full((rows, n + 8), 7.0, device="cuda", dtype=tdt(dtype))
    run_fwd(a, b, off, c[:, :n], dtype)
    want, _ = want_fwd(a, b, off, torch.full((rows, n), 7.0, device="cuda"), 1.0, 0.0)
    assert torch.equal(c[:, :n], want.to(tdt(dtype)))
    assert bool((c[:, n:] == 7).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,lead,tail", [([1000, 0, 705, 17, 64, 1], 2, 5), ([2049, 190], 0, 1),
                                             ([0, 0, 130], 0, 0), ([3, 5, 0, 200, 257, 31], 1, 0)])
@pytest.mark.parametrize("m,n", [(2048, 2304), (1032, 4360), (4100, 2056)])
def test_wgrad_exact_tall_tiles(dtype, sizes, lead, tail, m, n):
    torch = torch_cuda()
    rows, off = lead + sum(sizes) + tail, offsets_of(sizes, lead)
    a, b = data(1, (rows, m), dtype), data(2, (rows, n), dtype)
    for t in (a, b):
        t[:lead] = float("nan")
        t[rows - tail:] = float("inf")
    c = torch.full((len(sizes), m + 1, n), 7.0, device="cuda", dtype=tdt(dtype))
    run_wgrad(a, b, off, c[:, :m], dtype)
    want, _ = want_wgrad(a, b, off, c, 1.0, 0.0)
    assert torch.equal(c[:, :m], want.to(tdt(dtype)))
    assert bool((c[:, m:] == 7).all())


def test_realigned_operands_in_graphs_and_on_two_streams():
    """Operands that are copied to aligned scratch first (odd pitches, no unit stride): captured calls
    replayed on two streams at once, and eager calls on two streams, each with its own scratch."""
    torch = torch_cuda()
    rows, k, n, dtype = 300, 133, 259, "bf16"
    off = offsets_of([100, 0, 150, 50])
    a = data(1, (rows, k), dtype)
    bs = [data(2 + i, (4, k, 2 * n), dtype)[:, :, ::2] for i in range(2)]  # no unit stride
    cs = [torch.zeros((rows, n), device="cuda") for _ in range(2)]
    ws = [torch.zeros((4, k, n), device="cuda") for _ in range(2)]
    dy = data(9, (rows, n), dtype)
    streams = [torch.cuda.Stream() for _ in range(2)]
    wants = [want_fwd(a, b, off, torch.zeros_like(cs[0]), 1.0, 0.0)[0] for b in bs]
    wgrad = want_wgrad(a, dy, off, ws[0], 1.0, 0.0)[0]
    torch.cuda.synchronize()

    def calls(i):
        run_fwd(a, bs[i], off, cs[i], dtype, sync=False)
        run_wgrad_async(a, dy, off, ws[i], dtype)

    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                calls(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(cs[i].double(), wants[i]) and torch.equal(ws[i].double(), wgrad)
    graphs = []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            calls(i)
            calls(i)
        graphs.append(g)
        cs[i].zero_()
        ws[i].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(cs[i].double(), wants[i]) and torch.equal(ws[i].double(), wgrad)


@pytest.mark.parametrize("seed", range(6))
def test_random_shapes_and_strides(seed):
    """Small random problems with random pitches, offsets of the base and orders."""
    torch = torch_cuda()
    rng = np.random.default_rng(seed)
    for _ in range(12):
        g = int(rng.integers(1, 6))
        sizes = [int(x) for x in rng.integers(0, 90, g)]
        lead, tail = int(rng.integers(0, 3)), int(rng.integers(0, 3))
        rows, k, n = lead + sum(sizes) + tail, int(rng.integers(1, 300)), int(rng.integers(1, 300))
        if rows == 0:
            continue
        off = offsets_of(sizes, lead)

        def mat(r, c):
            pad, at = int(rng.integers(0, 9)), int(rng.integers(0, 9))
            if rng.random() < 0.5:
                return data(int(rng.integers(1 << 30)), (r, c + pad + at), "bf16")[:, at:at + c]
            return data(int(rng.integers(1 << 30)), (c, r + pad + at), "bf16")[:, at:at + r].t()

        a = mat(rows, k)
        b = mat(g * k, n) if rng.random() < 0.5 else mat(n, g * k).t()
        b = torch.as_strided(b, (g, k, n), (k * b.stride(0), *b.stride()), b.storage_offset())
        c = torch.full((rows, n), 7.0, device="cuda")
        run_fwd(a, b, off, c, "bf16")
        want, _ = want_fwd(a, b, off, torch.full_like(c, 7.0), 1.0, 0.0)
        assert torch.equal(c.double(), want)
        y = mat(rows, n)
        w = torch.full((g, k, n), 7.0, device="cuda")
        run_wgrad(a, y, off, w, "bf16")
        want, _ = want_wgrad(a, y, off, w, 1.0, 0.0)
        assert torch.equal(w.double(), want)


def test_empty_contractions_and_inputs():
    """k == 0 and no rows at all: C <- beta * C on the groups' rows, on every group of a weight
    gradient."""
    torch = torch_cuda()
    off = offsets_of([3, 0, 4], 1)
    for beta in (0.0, 0.5):
        c = torch.full((9, 24), 8.0, device="cuda")
        run_fwd(torch.zeros((9, 0), device="cuda", dtype=torch.bfloat16),
                torch.zeros((3, 0, 24), device="cuda", dtype=torch.bfloat16), off, c, "bf16", beta=beta)
        want = torch.full_like(c, 8.0)
        want[1:8] *= beta
        assert torch.equal(c, want)
        for out in (torch.float32, torch.bfloat16):
            w = torch.full((3, 40, 24), 8.0, device="cuda", dtype=out)
            run_wgrad(torch.zeros((0, 40), device="cuda", dtype=torch.bfloat16),
                      torch.zeros((0, 24), device="cuda", dtype=torch.bfloat16), offsets_of([0, 0, 0]),
                      w, "bf16", beta=beta)
            assert torch.equal(w, torch.full_like(w, 8.0 * beta))


def test_most_groups():
    """1024 groups, most of them empty."""
    torch = torch_cuda()
    sizes = [(i * 7) % 5 if i % 3 == 0 else 0 for i in range(1024)]
    off, rows = offsets_of(sizes), sum(sizes)
    a, b = data(1, (rows, 40), "bf16"), data(2, (1024, 40, 24), "bf16")
    c = torch.full((rows, 24), 7.0, device="cuda")
    run_fwd(a, b, off, c, "bf16")
    assert torch.equal(c.double(), want_fwd(a, b, off, c, 1.0, 0.0)[0])
    y = data(3, (rows, 24), "bf16")
    w = torch.full((1024, 40, 24), 7.0, device="cuda")
    run_wgrad(a, y, off, w, "bf16")
    assert torch.equal(w.double(), want_wgrad(a, y, off, w, 1.0, 0.0)[0])


def test_first_call_inside_a_capture():
    """A process whose first calls are captured (aligned operands, then operands that need scratch)."""
    import os
    import subprocess
    import sys
    code = """
import torch, gemmkit_b200 as gk
off = torch.tensor([0, 30, 50], dtype=torch.int32, device="cuda")
for k, n in ((64, 72), (33, 71)):
    a = torch.randint(-4, 5, (50, k), device="cuda").bfloat16()
    b = torch.randint(-4, 5, (2, k, n), device="cuda").bfloat16()
    c = torch.zeros(50, n, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gk.gemm_half_grouped(1.0, gk.MatRef.from_row_major(a, 50, k), gk.MatRef.from_row_major(b, k, n),
                             k * n, off, 0.0, gk.MatMut.from_row_major(c, 50, n), sync=False)
    g.replay()
    torch.cuda.synchronize()
    want = torch.cat([a[:30].double() @ b[0].double(), a[30:].double() @ b[1].double()])
    assert torch.equal(c.double(), want), (k, n)
print("ok")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "ok" in out.stdout, out.stderr[-2000:]


# Sizes for each tile plan of the weight gradient: one CTA with 64, 128 and 256 rows of the Q side,
# CTA pairs with 256 columns (f32 C) and with 512 (16-bit C).
@pytest.mark.parametrize("sizes,m,n,out", [([3, 0, 20], 40, 24, "f32"), ([3, 0, 20], 40, 24, "bf16"),
                                           ([70, 0, 1], 100, 72, "f32"),
                                           ([70, 0, 1], 200, 136, "bf16"),
                                           ([5, 0, 100], 1032, 2304, "f32"),
                                           ([5, 0, 100], 1032, 2304, "bf16")])
@pytest.mark.parametrize("alpha", [float("inf"), -float("inf"), float("nan"), -3.0])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_empty_group_gradient_ignores_alpha(sizes, m, n, out, alpha, beta):
    """An empty group's C[g] becomes beta * C[g], with an infinite or NaN alpha too; the other groups
    get alpha times their product (integers: exact before that product)."""
    torch = torch_cuda()
    off = offsets_of(sizes)
    a, b = data(1, (sum(sizes), m), "bf16"), data(2, (sum(sizes), n), "bf16")
    c = torch.full((len(sizes), m, n), 8.0, device="cuda", dtype=tdt(out))
    run_wgrad(a, b, off, c, "bf16", alpha, beta)
    acc, _ = want_wgrad(a, b, off, c, 1.0, 0.0)
    want = (alpha * acc + beta * 8.0).to(tdt(out))
    want[1] = beta * 8.0
    assert bool(((c == want) | (c.isnan() & want.isnan())).all())


@pytest.mark.parametrize("rows,n", [(9, 24), (200, 136), (2048, 2304)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("alpha", [float("inf"), float("nan")])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_forward_without_contraction_ignores_alpha(rows, n, out, alpha, beta):
    """k == 0: C <- beta * C on the groups' rows whatever alpha is."""
    torch = torch_cuda()
    off = offsets_of([rows - 4, 0, 2], 1)
    c = torch.full((rows, n), 8.0, device="cuda", dtype=tdt(out))
    run_fwd(torch.zeros((rows, 0), device="cuda", dtype=torch.bfloat16),
            torch.zeros((3, 0, n), device="cuda", dtype=torch.bfloat16), off, c, "bf16", alpha, beta)
    want = torch.full_like(c, 8.0)
    want[1:rows - 1] = 8.0 * beta
    assert torch.equal(c, want)


def test_scratch_is_given_back():
    """Operands that are copied to scratch: past a synchronisation the engine keeps at most 1/64 of
    the device's memory, and nothing after scratch_release; calls go on working."""
    torch = torch_cuda()
    rows, k, n, g = 16, 8192, 8192, 27
    off = torch.tensor([0, 4] + [8] * (g - 2) + [rows], dtype=torch.int32, device="cuda")
    b = torch.zeros((g, n, k + 1), device="cuda", dtype=torch.bfloat16)
    b[0], b[1], b[-1] = data(2, (3, n, k + 1), "bf16")
    b = b[:, :, :k].transpose(1, 2)  # an odd pitch: 3.6 GB of scratch
    a = data(1, (rows, k), "bf16")
    c = torch.zeros((rows, n), device="cuda")
    small = data(3, (1, 72, 65), "bf16")  # the process's first use of the pool and the kernels
    run_fwd(data(4, (3, 72), "bf16"), small, offsets_of([3]), torch.zeros((3, 65), device="cuda"), "bf16")
    want, _ = want_fwd(a, b, off, c, 1.0, 0.0)
    gk.scratch_release()
    for release in (False, True, False, True):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        free, total = torch.cuda.mem_get_info()
        c.fill_(7.0)
        run_fwd(a, b, off, c, "bf16")
        torch.cuda.synchronize()
        assert torch.equal(c.double(), want)
        if release:
            gk.scratch_release()
        assert free - torch.cuda.mem_get_info()[0] <= (0 if release else total // 64)
