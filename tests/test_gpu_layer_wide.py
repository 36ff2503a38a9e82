"""Element offsets past 2^31 in the feed-forward layers' operators: rows that lie far apart in C, R, z, dY, dZ,
8-bit codes and logits. Integer data, compared for equality; and first calls from several threads."""
import os
import subprocess
import sys

import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from layer_util import act8_values, act_of, mut, numbers, offsets_of, ref, status_clean, tdt
from test_gpu_linear import backward, check_backward, check_forward, forward, problem, product64

pytestmark = pytest.mark.gpu

PAST = 2 ** 31 + 2 ** 28  # the last row starts beyond this element
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def _status():
    yield
    status_clean()
    torch_cuda().cuda.empty_cache()


def wide(rows, n, dtype, odd, fill):
    """rows x n whose rows lie so far apart, in memory of its own (only its elements are written)."""
    torch = torch_cuda()
    step = -(-PAST // (rows - 1)) // 8 * 8 + 8 + odd
    t = torch.empty((rows - 1) * step + n, dtype=tdt(dtype), device="cuda").as_strided((rows, n), (step, 1))
    t.copy_(fill) if torch.is_tensor(fill) else t.fill_(fill)
    return t


PLANS = [([30, 0, 70], 136), ([900, 0, 1, 700, 515], 2304)]


@pytest.mark.parametrize("sizes,n", PLANS)
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_forward(sizes, n, odd, out):
    torch = torch_cuda()
    rows = sum(sizes)
    a, b, off, groups = problem(sizes, rows, 72, n, "bf16", "n", 1)
    bias, r = numbers(4, (groups, n), "bf16"), numbers(5, (rows, n), out)
    c0 = torch.full((rows, n), 7.0, dtype=tdt(out), device="cuda")
    c, z, rr = wide(rows, n, out, odd, 7.0), wide(rows, n, "bf16", odd, 7.0), wide(rows, n, out, odd, r)
    forward(a, b, off, "bf16", "relu", bias, rr, c, z)
    check_forward(a, b, off, "bf16", "relu", bias, r, c, z, c0, c0, out=out, exact=True)


@pytest.mark.parametrize("sizes,n", PLANS)
@pytest.mark.parametrize("odd,zform", [(0, "half"), (1, "half"), (0, "act8")])
def test_backward(sizes, n, odd, zform):
    torch = torch_cuda()
    rows = sum(sizes)
    a, b, off, groups = problem(sizes, rows, 72, n, "f16", "k", 11)
    z = numbers(14, (rows, n), "f16")
    if zform == "half":
        zz = wide(rows, n, "f16", odd, z)
    else:
        nb = (n + 31) // 32
        step = -(-PAST // (rows - 1)) // 32 * 32 + 32
        codes = torch.empty((rows - 1) * step + nb * 32, dtype=torch.int8, device="cuda")
        zz = gk.Act8Matrix(rows, n, codes.as_strided((rows, n), (step, 1)),
                           torch.empty(rows, nb, dtype=torch.uint8, device="cuda"))
        gk.quantize_act8(ref(z), out=zz)
        assert torch.equal(act8_values(zz), z.double())
        y = torch.empty(rows, n, dtype=torch.float16, device="cuda")
        gk.dequantize_act8(zz, mut(y))
        assert torch.equal(y, z)
    c = wide(rows, n, "f16", odd, 7.0)
    dbias = torch.empty(groups, n, device="cuda")
    backward(a, b, off, "f16", zz, "relu", c, dbias)
    d, mag = product64(a, b, off)
    check_backward(d, 0 * mag, z.double(), off, "f16", "relu", c, c, dbias, exact=True)
    dy = wide(rows, n, "f16", odd, numbers(15, (rows, n), "f16"))
    again = torch.empty_like(dbias)
    gk.act_backward(ref(dy), zz if zform == "act8" else ref(zz), act_of("relu"), mut(c), dbias=again,
                    offsets=off, is_f16=True)
    check_backward(dy.double(), 0 * mag, z.double(), off, "f16", "relu", c, c, again, exact=True)


def test_act8_of_far_rows():
    torch = torch_cuda()
    x = numbers(21, (50, 200), "bf16", False)
    far = wide(50, 200, "bf16", 0, x)
    q = gk.quantize_act8(ref(far))
    near = gk.quantize_act8(ref(x))
    assert torch.equal(q.codes, near.codes) and torch.equal(q.exponents, near.exponents)
    far.zero_()
    gk.dequantize_act8(q, mut(far))
    assert torch.equal(far.double(), act8_values(q))


@pytest.mark.parametrize("experts,odd", [(64, 0), (33, 1)])
def test_balance_of_far_rows(experts, odd):
    torch = torch_cuda()
    x = numbers(31, (500, experts), "f32", False)
    ids = torch.topk(x, 4, dim=1)[1].to(torch.int32)
    far, d = wide(500, experts, "f32", odd, x), wide(500, experts, "f32", odd, 9.0)
    one = torch.ones(1, device="cuda")
    b, bf = gk.moe_balance(ref(x), ids), gk.moe_balance(ref(far), ids)
    g = torch.empty_like(x)
    gk.moe_balance_backward(ref(x), ids, b, one, mut(g))
    gk.moe_balance_backward(ref(far), ids, bf, one, mut(d))
    assert torch.equal(b.counts, bf.counts)
    # the two may take their tokens by other lanes: both are within the gradient's bound
    assert bool((d - g).abs().le(2 * 200 * 2.0 ** -24 * (g.abs() + 2 * b.rates.max())).all())


THREADS = """
import threading, torch, gemmkit_b200 as gk
M, U = gk.MatRef.from_row_major, gk.MatMut.from_row_major
gen = torch.Generator(device="cuda").manual_seed(1)
def ints(*shape):
    return torch.randint(-4, 5, shape, generator=gen, device="cuda").bfloat16()
args = [(300, 133, 258), (16, 4096, 256), (2048, 64, 4096), (65, 64, 72)]
data = [(ints(r, k), ints(n, k), ints(n), ints(r, n)) for r, k, n in args]
torch.cuda.synchronize()
streams = [torch.cuda.Stream() for _ in args]
gate, errors = threading.Barrier(len(args)), []
def work(i):
    try:
        r, k, n = args[i]
        a, b, bias, z = data[i]
        with torch.cuda.stream(streams[i]):
            gate.wait()
            c, dz = torch.empty(r, n, device="cuda"), torch.empty(r, n, device="cuda")
            db, dw = torch.empty(n, device="cuda"), torch.empty(k, n, device="cuda")
            logits = a.float()[:, :32].contiguous()
            ids = torch.topk(logits, 2, dim=1)[1]
            for _ in range(20):
                gk.gemm_half_epilogue(1.0, M(a, r, k), gk.MatRef.from_col_major(b, k, n), U(c, r, n),
                                      bias=bias, act=gk.Activation.Relu(), sync=False)
                q = gk.quantize_act8(M(z, r, n), sync=False)
                gk.gemm_half_dact(1.0, M(a, r, k), gk.MatRef.from_col_major(b, k, n), q,
                                  gk.Activation.Relu(), U(dz, r, n), dbias=db, sync=False)
                x = gk.quantize_act8(M(a, r, k), sync=False)
                gk.gemm_act8_wgrad(1.0, x, M(z, r, n), 0.0, U(dw, k, n), sync=False)
                bal = gk.moe_balance(M(logits, r, 32), ids, sync=False)
            p = a.double() @ b.double().T
            assert torch.equal(c.double(), (p + bias.double()).clamp(min=0)), "forward"
            w = p * (z > 0)
            assert torch.equal(dz.double(), w) and torch.equal(db.double(), w.sum(0)), "backward"
            assert torch.equal(dw.double(), a.double().T @ z.double()), "gradient"
            assert torch.equal(bal.counts.long(), torch.bincount(ids.reshape(-1), minlength=32)), "counts"
    except BaseException as e:
        errors.append((i, repr(e)))
threads = [threading.Thread(target=work, args=(i,)) for i in range(len(args))]
for t in threads: t.start()
for t in threads: t.join()
assert not errors, errors
assert gk.device_status(0) == 0
print("ok")
"""


def test_first_calls_from_several_threads():
    out = subprocess.run([sys.executable, "-c", THREADS], cwd=ROOT, capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "ok" in out.stdout, out.stderr[-2000:]
