"""A training step of a mixture of experts' feed-forward layer, its operators one after the other as they are
used: router, up-projection, checkpoints, down-projection, and the whole backward pass. Every stage is
checked against the 64-bit form of what it was given (bounds as in the stages' own tests); the step is run
eagerly without a synchronisation and captured into a graph, with the same bits."""
import pytest

import gemmkit_b200 as gk
from gpu_util import torch_cuda
from layer_util import act8_values, act_of, mut, numbers, ref, spans, status_clean
from test_gpu_act8 import quantized
from test_gpu_linear import check_backward, check_forward, near, product64, stack_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    status_clean()


class Layer:
    def __init__(self, seed, tokens, experts, top, d, hidden, act):
        torch = torch_cuda()
        self.act, self.top = act, top
        self.x = numbers(seed, (tokens, d), "bf16", False)
        self.logits = numbers(seed + 1, (tokens, experts), "f32", False)
        self.w1 = numbers(seed + 2, (experts, hidden, d), "bf16", False, d ** -0.5)
        self.w2 = numbers(seed + 3, (experts, d, hidden), "bf16", False, hidden ** -0.5)
        self.b1 = numbers(seed + 4, (experts, hidden), "bf16", False, 0.3)
        self.b2 = numbers(seed + 5, (experts, d), "bf16", False, 0.3)
        rows = tokens * top
        self.dy = numbers(seed + 6, (rows, d), "bf16", False, 0.05)
        self.one = torch.full((1,), 0.01, device="cuda")
        self.ids = torch.topk(self.logits, top, dim=1)[1]
        self.ids[3] = -1  # a padded token: its rows lie behind the last expert's

        def make(*shape, dtype=torch.bfloat16):
            return torch.full(shape, 7.0, dtype=dtype, device="cuda")
        self.z, self.h = make(rows, hidden), make(rows, hidden)
        self.y, self.dz, self.dx = make(rows, d), make(rows, hidden), make(rows, d)
        self.dw1, self.dw2 = make(experts, hidden, d), make(experts, d, hidden)
        self.db1 = make(experts, hidden, dtype=torch.float32)
        self.db2 = make(experts, d, dtype=torch.float32)
        self.dlogits = torch.full_like(self.logits, 7.0)
        self.q = [gk.Act8Matrix.empty(rows, n) for n in (d, hidden, hidden)]  # of x, z and h
        self.bal = gk.MoeBalance.empty(experts)
        self.xs = make(rows, d)

    def step(self):
        torch = torch_cuda()
        gk.moe_balance(ref(self.logits), self.ids, out=self.bal, sync=False)
        off = self.bal.offsets
        # rows by expert, padding last
        flat = self.ids.reshape(-1)
        order = torch.sort(flat.masked_fill(flat < 0, 1 << 20), stable=True)[1]
        torch.index_select(self.x, 0, order // self.top, out=self.xs)
        b1, g1 = stack_ref(self.w1.transpose(1, 2))
        b2, g2 = stack_ref(self.w2.transpose(1, 2))
        gk.gemm_half_epilogue(1.0, ref(self.xs), b1, mut(self.h), bias=self.b1, act=act_of(self.act),
                              z=mut(self.z), offsets=off, b_gs=g1, sync=False)
        for q, t in zip(self.q, (self.xs, self.z, self.h)):
            gk.quantize_act8(ref(t), out=q, sync=False)
        gk.gemm_half_epilogue(1.0, ref(self.h), b2, mut(self.y), bias=self.b2, residual=ref(self.xs),
                              offsets=off, b_gs=g2, sync=False)
        # backward: the biases, the activation's input, the weights, the input, the router
        gk.act_backward(ref(self.dy), None, None, None, dbias=self.db2, offsets=off, sync=False)
        w2, gs = stack_ref(self.w2)
        gk.gemm_half_dact(1.0, ref(self.dy), w2, self.q[1], act_of(self.act), mut(self.dz), dbias=self.db1,
                          offsets=off, b_gs=gs, sync=False)
        for q, d, dw in ((self.q[2], self.dy, self.dw2), (self.q[0], self.dz, self.dw1)):
            g, n, k = dw.shape
            gk.gemm_act8_wgrad(1.0, q, ref(d), 0.0, gk.MatMut(dw.reshape(-1), k, n, 1, k), offsets=off,
                               c_gs=n * k, sync=False)
        w1, gs = stack_ref(self.w1)
        gk.gemm_half_grouped(1.0, ref(self.dz), w1, gs, off, 0.0, mut(self.dx), sync=False)
        gk.moe_balance_backward(ref(self.logits), self.ids, self.bal, self.one, mut(self.dlogits), sync=False)

    def outputs(self):
        return {k: getattr(self, k) for k in ("z", "h", "y", "dz", "dx", "dw1", "dw2", "db1", "db2", "dlogits")}


@pytest.mark.parametrize("tokens,experts,top,d,hidden,act", [
    (70, 8, 2, 96, 200, "gelu"), (1500, 4, 2, 512, 1024, "silu"), (5, 16, 1, 64, 64, "relu")])
def test_training_step(tokens, experts, top, d, hidden, act):
    torch = torch_cuda()
    m = Layer(11, tokens, experts, top, d, hidden, act)
    m.step()
    torch.cuda.synchronize()
    off, rows = m.bal.offsets, tokens * top
    assert int(off[-1]) == rows - top
    full = torch.full((rows, max(d, hidden)), 7.0, dtype=torch.bfloat16, device="cuda")
    f = {n: full[:, :n].contiguous() for n in (d, hidden)}
    check_forward(m.xs, m.w1.transpose(1, 2), off, "bf16", act, m.b1, None, m.h, m.z, f[hidden], f[hidden])
    check_forward(m.h, m.w2.transpose(1, 2), off, "bf16", "none", m.b2, m.xs, m.y, None, f[d], None)
    for q, t in zip(m.q, (m.xs, m.z, m.h)):
        codes, exps = quantized(t.double().cpu().numpy())
        assert (q.codes.cpu().numpy() == codes).all() and (q.exponents.cpu().numpy() == exps).all()
    g, mag = product64(m.dy, m.w2, off)
    check_backward(g, (d + 36) * 2.0 ** -23 * mag, act8_values(m.q[1]), off, "bf16", act, m.dz, f[hidden],
                   m.db1)
    check_backward(m.dy.double(), 0 * m.dy.double(), None, off, "bf16", "none", None, None, m.db2)
    for q, dd, dw in ((m.q[2], m.dy, m.dw2), (m.q[0], m.dz, m.dw1)):
        v = act8_values(q)
        for e, s in spans(off, rows):
            want, mg = dd[s].double().T @ v[s], dd[s].double().abs().T @ v[s].abs()
            near(dw[e], want, (s.stop - s.start + 36) * 2.0 ** -23 * mg, "bf16")
    want, mg = product64(m.dz, m.w1, off)
    near(m.dx[:rows - top], want[:rows - top], (hidden + 36) * 2.0 ** -23 * mg[:rows - top], "bf16")
    assert torch.equal(m.dx[rows - top:], f[d][rows - top:])
    assert not m.dlogits[3].any() and m.dlogits.isfinite().all()

    first = {k: v.clone() for k, v in m.outputs().items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step()
    for v in m.outputs().values():
        v.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    for k, v in m.outputs().items():
        assert torch.equal(v, first[k]), k


def test_two_layers_at_once():
    """Two steps interleaved on two streams give what each gives alone."""
    torch = torch_cuda()
    layers = [Layer(s, 300, 8, 2, 128, 264, "gelu") for s in (21, 31)]
    want = []
    for m in layers:
        m.step()
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in m.outputs().items()})
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(3):
        for m, s in zip(layers, streams):
            with torch.cuda.stream(s):
                m.step()
    torch.cuda.synchronize()
    for m, w in zip(layers, want):
        for k, v in m.outputs().items():
            assert torch.equal(v, w[k]), k
