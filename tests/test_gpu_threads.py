"""Entries called from several threads at once, each on a stream of its own, in a process whose first
calls these are."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import threading, torch, gemmkit_b200 as gk
M, U = gk.MatRef.from_row_major, gk.MatMut.from_row_major
gen = torch.Generator(device="cuda").manual_seed(1)
def ints(*shape):
    return torch.randint(-4, 5, shape, generator=gen, device="cuda").bfloat16()
args = [(300, 133, 259), (512, 128, 256), (2048, 256, 2304), (65, 64, 72)]
data = []
for rows, k, n in args:
    a, b = ints(rows, k), ints(2, k, n)
    off = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    w = ints(n, k)
    data.append((a, b, off, w))
torch.cuda.synchronize()
streams = [torch.cuda.Stream() for _ in args]
gate, errors = threading.Barrier(len(args)), []
def work(i):
    try:
        rows, k, n = args[i]
        a, b, off, w = data[i]
        with torch.cuda.stream(streams[i]):
            gate.wait()
            c = torch.full((rows, n), 7.0, device="cuda")
            g = torch.full((2, k, n), 7.0, device="cuda")
            y = torch.full((rows, n), 7.0, device="cuda")
            z = torch.full((rows, n), 7.0, device="cuda")
            for _ in range(20):
                gk.gemm_half_grouped(1.0, M(a, rows, k), M(b, k, n), k * n, off, 0.0, U(c, rows, n),
                                     sync=False)
                gk.gemm_half_grouped_wgrad(1.0, M(a, rows, k), M(c.bfloat16(), rows, n), off, 0.0,
                                           U(g, k, n), k * n, sync=False)
                x4 = gk.quantize_fp4(M(a, rows, k), gk.FP4_MX, sync=False)
                w4 = gk.quantize_fp4(M(w, n, k), gk.FP4_MX, sync=False)
                gk.gemm_fp4(1.0, x4, w4, 0.0, U(y, rows, n), sync=False)
                gk.gemm_half_f32(1.0, M(a, rows, k), M(b, k, n), 0.0, U(z, rows, n), sync=False)
            cut = rows // 3
            want = torch.cat([a[:cut].double() @ b[0].double(), a[cut:].double() @ b[1].double()])
            assert torch.equal(c.double(), want), "forward"
            h = c.bfloat16().double()
            want = torch.stack([a[:cut].double().T @ h[:cut], a[cut:].double().T @ h[cut:]])
            mag = torch.stack([a[:cut].double().abs().T @ h[:cut].abs(),
                               a[cut:].double().abs().T @ h[cut:].abs()])
            assert bool(((g.double() - want).abs() <= (rows + 36) * 2.0 ** -23 * mag).all()), "gradient"
            assert torch.equal(z.double(), a.double() @ b[0].double()), "dense"
            xa, wa = torch.empty(rows, k, device="cuda"), torch.empty(n, k, device="cuda")
            gk.dequantize_fp4(x4, U(xa, rows, k), sync=False)
            gk.dequantize_fp4(w4, U(wa, n, k), sync=False)
            assert torch.equal(xa.double(), a.double()) and torch.equal(wa.double(), w.double())
            assert torch.equal(y.double(), a.double() @ w.double().T), "4-bit"
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
    out = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "ok" in out.stdout, out.stderr[-2000:]
