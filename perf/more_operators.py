"""Operators of a transformer's feed-forward layers, dense or by expert, as they are measured: the
product with bias, activation and residual in its epilogue, its backward pass, activation
checkpoints in 8 bits with their use in the backward pass, and the router's balance loss.

The cases take their widths from the engine's own workloads: 4096 x 14336, 8192, 4096, 1024, 512.

Formulas (rows i of group g are offsets[g] <= i < offsets[g + 1]; without offsets g is 0):
  linear       z = A . B[g] + bias[g];  C = act(z) + R                          (z on demand)
  dact         dZ = (dY . B[g]) * act'(z);  dbias[g] = sum of dZ over g's rows  (z in 16 or 8 bits)
  act_grad     dZ = dY * act'(z);  dbias[g] likewise                            (no product)
  act8         q = round(x / 2^(e - 6)), e = floor(log2 max|x|) per 32 consecutive elements of a
               row, q in [-127, 127]; returned as the values q 2^(e - 6)
  act8_wgrad   dW[g] = X8_g^T . dZ_g, X8 an 8-bit checkpoint
  balance      p = softmax(logits), f_e = routed_e / routed, P_e = mean of p_te over the live
               tokens, loss = experts * sum_e f_e P_e;  its gradient by the logits, the counts
               routed_e and their running sums (the offsets of the experts' products)
"""
import math

import torch

own = False

BLOCK = 32
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token through a layer while serving: the weights are read for one row
        {"name": "linear-token", "op": "linear", "groups": 0, "rows": 1, "k": 4096, "n": 14336,
         "act": "silu", "residual": False, "save_z": False, "dtype": "bf16", "b_major": "k"},
        # the up-projection of a training batch: its input to the activation is kept for backward
        {"name": "linear-up", "op": "linear", "groups": 0, "rows": 8192, "k": 4096, "n": 14336,
         "act": "gelu", "residual": False, "save_z": True, "dtype": "bf16", "b_major": "k"},
        # the down-projection onto the residual stream, a ragged number of rows
        {"name": "linear-down", "op": "linear", "groups": 0, "rows": 2047, "k": 14336, "n": 4096,
         "act": "none", "residual": True, "save_z": False, "dtype": "f16", "b_major": "k"},
        # many small experts with biases, weights stored k x n
        {"name": "linear-experts", "op": "linear", "groups": 64, "rows": 4099, "k": 1024, "n": 512,
         "act": "gelu_tanh", "residual": False, "save_z": True, "dtype": "bf16", "b_major": "n"},
        # the down-projection's input gradient, through the activation whose input is held in 8 bits
        {"name": "dact-down", "op": "dact", "groups": 0, "rows": 8192, "k": 4096, "n": 14336,
         "act": "gelu", "z": "act8", "dtype": "bf16", "b_major": "n"},
        # the gradient that reaches a layer whose output went through the activation last
        {"name": "act-grad", "op": "act_grad", "groups": 8, "rows": 8192, "n": 4096,
         "act": "silu", "z": "half", "dtype": "bf16"},
        # a layer's input into its checkpoint, and back
        {"name": "act8", "op": "act8", "rows": 8192, "k": 8192, "dtype": "bf16"},
        # a ragged f32 matrix, the last block of each row cut
        {"name": "act8-odd", "op": "act8", "rows": 333, "k": 4099, "dtype": "f32"},
        # the weights' gradient of the up-projection from its input's checkpoint
        {"name": "wgrad8", "op": "act8_wgrad", "groups": 0, "rows": 8192, "k": 4096, "n": 14336,
         "layout": "kn", "dtype": "bf16"},
        # the same for many small experts, weights stored n x k
        {"name": "wgrad8-experts", "op": "act8_wgrad", "groups": 64, "rows": 4099, "k": 1024,
         "n": 512, "layout": "nk", "dtype": "f16"},
        # the router of one decode step
        {"name": "balance-small", "op": "balance", "rows": 16, "experts": 8, "top": 2,
         "padding": 0, "dtype": "bf16"},
        # the router of a training batch, padded rows among its tokens
        {"name": "balance-large", "op": "balance", "rows": 65536, "experts": 256, "top": 8,
         "padding": 1000, "dtype": "f32"},
    ]


def draw(rng):
    def size(lo, hi, step=1):  # spread over the logarithm, odd ones among them
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, v // step * step if v >= step else v))

    op = rng.choice(["linear", "linear", "dact", "act_grad", "act8", "act8_wgrad", "balance"])
    step = rng.choice([1, 8, 8, 64])  # odd widths too, most of them whole 16-byte rows
    dtype = rng.choice(["bf16", "f16"])
    act = rng.choice(["none", "relu", "leaky", "gelu", "gelu_tanh", "silu"])
    groups = rng.choice([0, 0, size(1, 64)])
    wide = 4096 if groups <= 8 else 2048  # a stack of weights no larger than the listed ones
    if op == "linear":
        return {"op": op, "groups": groups, "rows": size(1, 4096), "k": size(64, wide, step),
                "n": size(64, wide, step), "act": act, "residual": rng.random() < 0.5,
                "save_z": rng.random() < 0.5, "dtype": dtype, "b_major": rng.choice("kn")}
    if op == "dact":
        return {"op": op, "groups": groups, "rows": size(1, 4096), "k": size(64, wide, step),
                "n": size(64, wide, step), "act": act, "z": rng.choice(["half", "act8"]),
                "dtype": dtype, "b_major": rng.choice("kn")}
    if op == "act_grad":
        return {"op": op, "groups": groups, "rows": size(1, 8192), "n": size(64, 8192, step),
                "act": act, "z": rng.choice(["half", "act8"]), "dtype": dtype}
    if op == "act8":
        return {"op": op, "rows": size(1, 8192), "k": size(16, 8192, step),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "act8_wgrad":
        return {"op": op, "groups": groups, "rows": size(1, 8192), "k": size(64, wide, step),
                "n": size(64, wide, step), "layout": rng.choice(["kn", "nk"]), "dtype": dtype}
    rows, experts = size(1, 65536), size(2, 256)
    return {"op": op, "rows": rows, "experts": experts, "top": size(1, min(8, experts)),
            "padding": rng.choice([0, rows // 7]), "dtype": rng.choice(["bf16", "f16", "f32"])}


def group_sizes(groups, rows):
    """Rows of each expert: a skewed load (the largest share first), the last of four or more
    experts without any."""
    live = groups - 1 if groups >= 4 else groups
    share = [1.0 / (i + 3) for i in range(live)]
    total = sum(share)
    sizes = [int(rows * s / total) for s in share]
    for i in range(rows - sum(sizes)):
        sizes[i % live] += 1
    return sizes + [0] * (groups - live)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(std)

    def activations(rows, k):
        # a few channels much larger than the rest, as in a transformer's residual stream
        x = normal(rows, k)
        x[:, ::97] *= 8.0
        return x

    def weights(groups, a, b, k):
        w = torch.empty(groups, a, b, dtype=dt, device=dev)
        for g in range(groups):
            w[g] = normal(a, b, std=k ** -0.5)
        return w

    s = dict(case)
    op, rows = case["op"], case["rows"]
    groups = max(1, case.get("groups", 0))
    s["offsets"], s["cap"] = None, rows
    if case.get("groups", 0):
        sizes = group_sizes(groups, rows)
        order = torch.randperm(groups, generator=gen, device=dev)
        sizes = torch.tensor(sizes, device=dev)[order]
        s["cap"] = max(1, int(sizes.max()))  # the rows that the largest expert gets
        s["offsets"] = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)
    if op == "linear":
        k, n = case["k"], case["n"]
        s["a"] = activations(rows, k).to(dt)
        s["b"] = weights(groups, n, k, k) if case["b_major"] == "k" else weights(groups, k, n, k)
        s["bias"] = normal(groups, n, std=0.5).to(dt)
        s["r"] = activations(rows, n).to(dt) if case["residual"] else None
        s["c"] = torch.empty(rows, n, dtype=dt, device=dev)
        s["zout"] = torch.empty(rows, n, dtype=dt, device=dev) if case["save_z"] else None
    elif op in ("dact", "act_grad"):
        n = case["n"]
        if op == "dact":
            k = case["k"]
            s["a"] = normal(rows, k, std=0.05).to(dt)
            s["b"] = weights(groups, n, k, n) if case["b_major"] == "k" else \
                weights(groups, k, n, n)
        else:
            s["a"] = normal(rows, n, std=0.05).to(dt)
        z = normal(rows, n, std=1.5)
        if case["z"] == "act8":
            hold(s, z)
        else:
            s["z16"] = z.to(dt)
        s["dz"] = torch.empty(rows, n, dtype=dt, device=dev)
        s["dbias"] = torch.empty(groups, n, dtype=dt, device=dev)
    elif op == "act8":
        s["x"] = activations(rows, case["k"]).to(dt)
        s["c"] = torch.empty(rows, case["k"], dtype=dt, device=dev)
    elif op == "act8_wgrad":
        k, n = case["k"], case["n"]
        hold(s, activations(rows, k))
        s["b"] = normal(rows, n, std=0.05).to(dt)
        shape = (groups, k, n) if case["layout"] == "kn" else (groups, n, k)
        s["c"] = torch.empty(shape, dtype=dt, device=dev)
    else:
        experts, top = case["experts"], case["top"]
        # some experts are liked more than others
        s["logits"] = (normal(rows, experts, std=1.5) + normal(1, experts)).to(dt)
        ids = torch.topk(s["logits"].float(), top, dim=1)[1]
        if case["padding"]:
            pad = torch.randperm(rows, generator=gen, device=dev)[:case["padding"]]
            ids[pad] = -1
        s["ids"] = ids.to(torch.int32)
        s["dloss"] = torch.full((1,), 0.01, device=dev)
        s["dlogits"] = torch.empty_like(s["logits"])
    return s


def hold(s, x):
    """The 8-bit checkpoint of x (of its values in the operands' type) that the forward pass left."""
    codes, scales = quantize_plain(x.to(DT[s["dtype"]]))
    rows, k = x.shape
    s["codes"], s["scales"] = codes, scales
    if own:
        import gemmkit_b200 as gk
        q = gk.Act8Matrix.empty(rows, k)
        q.codes.copy_(codes)
        q.exponents.copy_(scales)
        s["q"] = q


# ---- the plain forms ---------------------------------------------------------------------------

def quantize_plain(x):
    """(codes int8, exponent bytes) of a matrix, a byte for each 32 elements of a row."""
    rows, k = x.shape
    nb = -(-k // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - k)).view(rows, nb, BLOCK)
    amax = v.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 1, -127).clamp(min=-127)
    q = torch.round(torch.ldexp(v.double(), (6 - e)[..., None])).clamp(-127, 127)
    return q.view(rows, nb * BLOCK)[:, :k].to(torch.int8), (e + 127).to(torch.uint8)


def values(codes, scales):
    """The values that codes and exponent bytes stand for, in 32 bits (exact)."""
    e = scales.int().repeat_interleave(BLOCK, 1)[:, :codes.shape[1]] - 127
    return torch.ldexp(codes.double(), e - 6).float()


def by_group(s, x):
    """(group of each row, its place there, the rows of x padded to [groups, cap, k])."""
    i = torch.arange(x.shape[0], device=x.device)
    if s["offsets"] is None:
        return torch.zeros_like(i), i, x[None]
    off = s["offsets"].long()
    g = torch.searchsorted(off[1:], i, right=True)
    pos = i - off[g]
    padded = torch.zeros(max(1, s["groups"]), s["cap"], x.shape[1], device=x.device, dtype=x.dtype)
    padded[g, pos] = x
    return g, pos, padded


def act_plain(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "leaky":
        return torch.where(z > 0, z, 0.125 * z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def slope_plain(z, act):
    """The activation's derivative."""
    if act == "relu":
        return (z > 0).float()
    if act == "leaky":
        return torch.where(z > 0, 1.0, 0.125)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    return torch.ones_like(z)


def product_plain(s, a):
    """Rows of a (f32) by their group's matrix."""
    g, pos, padded = by_group(s, a)
    b = s["b"].float()
    c = torch.bmm(padded, b.transpose(1, 2) if s["b_major"] == "k" else b)
    return c[g, pos], g


def run_plain(s):
    op = s["op"]
    dt = DT[s["dtype"]]
    if op == "linear":
        z, g = product_plain(s, s["a"].float())
        z = z + s["bias"].float()[g]
        c = act_plain(z, s["act"])
        if s["r"] is not None:
            c = c + s["r"].float()
        return {"c": c.to(dt), "z": z.to(dt)} if s["save_z"] else {"c": c.to(dt)}
    if op in ("dact", "act_grad"):
        dh = product_plain(s, s["a"].float())[0] if op == "dact" else s["a"].float()
        z = values(s["codes"], s["scales"]) if s["z"] == "act8" else s["z16"].float()
        dz = dh * slope_plain(z, s["act"])
        return {"dz": dz.to(dt), "dbias": by_group(s, dz)[2].sum(1, dtype=torch.float64).to(dt)}
    if op == "act8":
        return values(*quantize_plain(s["x"])).to(dt)
    if op == "act8_wgrad":
        x = by_group(s, values(s["codes"], s["scales"]))[2]
        d = by_group(s, s["b"].float())[2]
        dw = torch.bmm(x.transpose(1, 2), d) if s["layout"] == "kn" else \
            torch.bmm(d.transpose(1, 2), x)
        return dw.to(dt)
    x, ids, experts = s["logits"].float(), s["ids"].long(), s["experts"]
    e = torch.exp(x - x.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    live = (ids >= 0).any(1)
    counts = torch.bincount(ids[ids >= 0].view(-1), minlength=experts)
    f = counts.double() / counts.sum().clamp(min=1)
    tokens = live.sum().clamp(min=1)
    mean = torch.where(live[:, None], p, 0.0).sum(0, dtype=torch.float64) / tokens
    loss = experts * (f * mean).sum()
    rate = (s["dloss"] * experts / tokens).double() * f
    dx = p * (rate.float() - (p.double() @ rate).float()[:, None])
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return {"loss": loss.float().view(1), "counts": counts.to(torch.int32),
            "offsets": offsets.to(torch.int32),
            "dlogits": torch.where(live[:, None], dx, 0.0).to(dt)}


# ---- the engine's calls --------------------------------------------------------------------------

def activation(gk, act):
    return {"none": lambda: None, "relu": gk.Activation.Relu,
            "leaky": lambda: gk.Activation.LeakyRelu(0.125), "gelu": gk.Activation.Gelu,
            "gelu_tanh": gk.Activation.GeluTanh, "silu": gk.Activation.Silu}[act]()


def run_own(s):
    import gemmkit_b200 as gk
    op, rows, f16 = s["op"], s["rows"], s["dtype"] == "f16"

    def mat(t, m, n):
        return gk.MatRef.from_row_major(t, m, n)

    def out(t, m, n):
        return gk.MatMut.from_row_major(t, m, n)

    if op in ("linear", "dact"):
        k, n = s["k"], s["n"]
        b = gk.MatRef.from_col_major(s["b"], k, n) if s["b_major"] == "k" else mat(s["b"], k, n)
    if op == "linear":
        gk.gemm_half_epilogue(
            1.0, mat(s["a"], rows, k), b, out(s["c"], rows, n), bias=s["bias"],
            act=activation(gk, s["act"]),
            residual=None if s["r"] is None else mat(s["r"], rows, n),
            z=None if s["zout"] is None else out(s["zout"], rows, n),
            offsets=s["offsets"], b_gs=k * n, is_f16=f16, sync=False)
        return {"c": s["c"], "z": s["zout"]} if s["save_z"] else {"c": s["c"]}
    if op in ("dact", "act_grad"):
        n = s["n"]
        z = s["q"] if s["z"] == "act8" else mat(s["z16"], rows, n)
        dz = out(s["dz"], rows, n)
        if op == "dact":
            gk.gemm_half_dact(1.0, mat(s["a"], rows, k), b, z, activation(gk, s["act"]), dz,
                              dbias=s["dbias"], offsets=s["offsets"], b_gs=k * n, is_f16=f16,
                              sync=False)
        else:
            gk.act_backward(mat(s["a"], rows, n), z, activation(gk, s["act"]), dz,
                            dbias=s["dbias"], offsets=s["offsets"], is_f16=f16, sync=False)
        return {"dz": s["dz"], "dbias": s["dbias"]}
    if op == "act8":
        q = gk.quantize_act8(mat(s["x"], rows, s["k"]), sync=False)
        gk.dequantize_act8(q, out(s["c"], rows, s["k"]), sync=False)
        return s["c"]
    if op == "act8_wgrad":
        k, n = s["k"], s["n"]
        c = out(s["c"], k, n) if s["layout"] == "kn" else gk.MatMut.from_col_major(s["c"], k, n)
        gk.gemm_act8_wgrad(1.0, s["q"], mat(s["b"], rows, n), 0.0, c, offsets=s["offsets"],
                           c_gs=k * n, is_f16=f16, sync=False)
        return s["c"]
    logits = mat(s["logits"], rows, s["experts"])
    bal = gk.moe_balance(logits, s["ids"], sync=False)
    gk.moe_balance_backward(logits, s["ids"], bal, s["dloss"],
                            out(s["dlogits"], rows, s["experts"]), sync=False)
    return {"loss": bal.loss, "counts": bal.counts, "offsets": bal.offsets,
            "dlogits": s["dlogits"]}


def run(state):
    return run_own(state) if own else run_plain(state)


# ---- bytes and operations --------------------------------------------------------------------------

def work(case):
    op, rows = case["op"], case["rows"]
    es = 4 if case["dtype"] == "f32" else 2
    groups = max(1, case.get("groups", 0))
    live = sum(1 for x in group_sizes(groups, rows) if x) if case.get("groups", 0) else 1

    def act8_bytes(m, n):
        return m * (n + -(-n // BLOCK))

    if op == "linear":
        k, n = case["k"], case["n"]
        wide = 1 + case["residual"] + case["save_z"]  # C, and R and z
        return {"bytes": es * (rows * k + live * (k * n + n) + wide * rows * n),
                "flops": 2 * rows * k * n}
    if op in ("dact", "act_grad"):
        n = case["n"]
        z = act8_bytes(rows, n) if case["z"] == "act8" else es * rows * n
        if op == "act_grad":
            return {"bytes": es * (2 * rows * n + groups * n) + z, "flops": 10 * rows * n}
        k = case["k"]
        return {"bytes": es * (rows * k + live * k * n + rows * n + groups * n) + z,
                "flops": 2 * rows * k * n}
    if op == "act8":
        # read, written in 8 bits, read again and the values written
        n = case["k"]
        return {"bytes": 2 * es * rows * n + 2 * act8_bytes(rows, n), "flops": 4 * rows * n}
    if op == "act8_wgrad":
        k, n = case["k"], case["n"]
        return {"bytes": act8_bytes(rows, k) + es * (rows * n + groups * k * n),
                "flops": 2 * rows * k * n}
    experts = case["experts"]
    # the logits are read in the forward and in the backward pass
    return {"bytes": 3 * es * rows * experts + 8 * rows * case["top"] + 8 * experts,
            "flops": 12 * rows * experts}


# ---- the definition in 64 bits ------------------------------------------------------------------------

def stored(codes, scales):
    """What a checkpoint holds, in 64 bits."""
    at = torch.arange(codes.shape[1], device=codes.device) // BLOCK
    return codes.double() * torch.exp2(scales.double() - 133.0)[:, at]


def exact(case, seed):
    s = prepare(case, seed)
    op, act = case["op"], case.get("act")
    spans = [(0, case["rows"])]
    if s["offsets"] is not None:
        off = s["offsets"].tolist()
        spans = list(zip(off[:-1], off[1:]))

    def phi(t):  # the normal distribution's
        return torch.special.ndtr(t)

    def f(t):
        if act == "relu":
            return t.clamp(min=0)
        if act == "leaky":
            return t.clamp(min=0) + 0.125 * t.clamp(max=0)
        if act == "gelu":
            return t * phi(t)
        if act == "gelu_tanh":
            return t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3))
        if act == "silu":
            return t * torch.sigmoid(t)
        return t

    def df(t):
        if act == "relu":
            return t.gt(0).double()
        if act == "leaky":
            return 0.125 + 0.875 * t.gt(0).double()
        if act == "gelu":
            return phi(t) + t * torch.exp(-t ** 2 / 2) / math.sqrt(2 * math.pi)
        if act == "gelu_tanh":
            c = 2 * math.sqrt(2 / math.pi)
            h = torch.sigmoid(c * (t + 0.044715 * t ** 3))
            return h + t * h * (1 - h) * c * (1 + 0.134145 * t ** 2)
        if act == "silu":
            h = torch.sigmoid(t)
            return h + t * h * (1 - h)
        return torch.ones_like(t)

    def product(rows_of):
        c = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for g, (i, j) in enumerate(spans):
            w = s["b"][g].double()
            c[i:j] = rows_of[i:j].double() @ (w.T if case["b_major"] == "k" else w)
        return c

    if op == "linear":
        z = product(s["a"])
        for g, (i, j) in enumerate(spans):
            z[i:j] += s["bias"][g].double()
        c = f(z)
        if s["r"] is not None:
            c += s["r"].double()
        return {"c": c, "z": z} if case["save_z"] else {"c": c}
    if op in ("dact", "act_grad"):
        d = product(s["a"]) if op == "dact" else s["a"].double()
        d = d * df(stored(s["codes"], s["scales"]) if case["z"] == "act8" else s["z16"].double())
        return {"dz": d, "dbias": torch.stack([d[i:j].sum(0) for i, j in spans])}
    if op == "act8":
        x = s["x"].double()
        out = torch.empty_like(x)
        for j in range(0, x.shape[1], BLOCK):
            v = x[:, j:j + BLOCK]
            top = v.abs().amax(1, keepdim=True).clamp(min=2.0 ** -127)
            e = torch.floor(torch.log2(top))
            e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double()
            unit = torch.exp2(e - 6)
            out[:, j:j + BLOCK] = torch.round(v / unit).clamp(-127, 127) * unit
        return out
    if op == "act8_wgrad":
        x = stored(s["codes"], s["scales"])
        dw = torch.stack([x[i:j].T @ s["b"][i:j].double() for i, j in spans])
        return dw if case["layout"] == "kn" else dw.transpose(1, 2)
    ids, experts = s["ids"].long(), case["experts"]
    live = ids.amax(1) >= 0
    p = torch.softmax(s["logits"].double(), 1) * live[:, None]
    hits = torch.stack([(ids == e).sum() for e in range(experts)]).double()
    share = hits / hits.sum().clamp(min=1)
    tokens = float(max(1, int(live.sum())))
    loss = experts * torch.dot(share, p.sum(0) / tokens)
    inner = p @ share
    scale = float(s["dloss"]) * experts / tokens
    return {"loss": loss.view(1), "counts": None, "offsets": None,
            "dlogits": scale * (p * share - p * inner[:, None])}
