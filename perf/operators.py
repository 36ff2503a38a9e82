"""Operators of large language models on this engine, as they are measured: the products of a
mixture of experts (rows grouped by expert, with both gradients) and the microscaled 4-bit
floating-point path (quantisation, product, product by expert).

The cases take their widths from the engine's own workloads: 4096 x 14336 (the decode GEMV),
8192 (the half-precision product), 4096 and 1024 (the integer products), 512 (the batch).

Formulas (rows i of group g are offsets[g] <= i < offsets[g + 1]):
  grouped         C[i, :] = A[i, :] . B[g]                          (forward and input gradient)
  grouped_wgrad   C[g]    = A_g^T . B_g                             (weight gradient)
  quantize        q = e2m1(x / (s_block * s)), s_block per 32 (mx: a power of two) or 16 (nv: e4m3)
                  consecutive elements of a row; returned as the values that q stands for
  fp4             C = deq(quantize(A)) . deq(B)^T, A quantised in the call, B held in 4 bits
  fp4_grouped     the same by expert
"""
import math

import torch

own = False

MX, NV = 0, 1                      # the engine's FP4_MX, FP4_NV
BLOCK = {MX: 32, NV: 16}
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of e2m1, by code


def listed():
    return [
        # one decode step of 8 experts, 16 routed rows: every expert's weights are read for a few rows
        {"name": "experts-decode", "op": "grouped", "groups": 8, "rows": 16, "k": 4096, "n": 14336,
         "dtype": "bf16", "b_major": "k"},
        # a prefill or training batch through the same experts' up-projection
        {"name": "experts-prefill", "op": "grouped", "groups": 8, "rows": 8192, "k": 4096,
         "n": 14336, "dtype": "bf16", "b_major": "k"},
        # many small experts, weights stored k x n
        {"name": "experts-fine", "op": "grouped", "groups": 64, "rows": 4099, "k": 1024, "n": 512,
         "dtype": "f16", "b_major": "n"},
        # the gradient of the up-projection's input: the same weights, contracted over their rows
        {"name": "experts-dgrad", "op": "grouped", "groups": 8, "rows": 4096, "k": 14336, "n": 4096,
         "dtype": "bf16", "b_major": "n"},
        # the weights' gradients: contraction over each expert's rows
        {"name": "experts-wgrad", "op": "grouped_wgrad", "groups": 8, "rows": 8192, "m": 4096,
         "n": 4096, "dtype": "bf16"},
        {"name": "experts-wgrad-fine", "op": "grouped_wgrad", "groups": 64, "rows": 4099, "m": 1024,
         "n": 512, "dtype": "f16"},
        # activations of a prefill into 4 bits
        {"name": "quantize-mx", "op": "quantize", "rows": 4096, "k": 4096, "fmt": MX,
         "dtype": "bf16"},
        # a ragged f32 matrix, its last block of each row cut
        {"name": "quantize-nv-odd", "op": "quantize", "rows": 333, "k": 4099, "fmt": NV,
         "dtype": "f32"},
        # one token through a 4-bit layer
        {"name": "fp4-decode", "op": "fp4", "m": 1, "k": 4096, "n": 14336, "fmt": NV,
         "dtype": "bf16"},
        # a long prefill through a 4-bit layer
        {"name": "fp4-prefill", "op": "fp4", "m": 8192, "k": 8192, "n": 8192, "fmt": MX,
         "dtype": "bf16"},
        # 4-bit experts: a decode step and a prefill
        {"name": "fp4-experts-decode", "op": "fp4_grouped", "groups": 8, "rows": 16, "k": 4096,
         "n": 14336, "fmt": MX, "dtype": "bf16"},
        {"name": "fp4-experts-prefill", "op": "fp4_grouped", "groups": 8, "rows": 8192, "k": 4096,
         "n": 14336, "fmt": NV, "dtype": "bf16"},
    ]


def draw(rng):
    def size(lo, hi, step=1):  # spread over the logarithm, odd ones among them
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, v // step * step if v >= step else v))

    op = rng.choice(["grouped", "grouped", "grouped_wgrad", "quantize", "fp4", "fp4_grouped"])
    step = rng.choice([1, 8, 8, 64])  # odd widths too, most of them whole 16-byte rows
    dtype = rng.choice(["bf16", "f16"])
    fmt = rng.choice([MX, NV])
    if op == "grouped":
        return {"op": op, "groups": size(1, 64), "rows": size(1, 4096), "k": size(64, 4096, step),
                "n": size(64, 4096, step), "dtype": dtype, "b_major": rng.choice("kn")}
    if op == "grouped_wgrad":
        return {"op": op, "groups": size(1, 64), "rows": size(1, 8192), "m": size(64, 2048, step),
                "n": size(64, 4096, step), "dtype": dtype}
    if op == "quantize":
        return {"op": op, "rows": size(1, 4096), "k": size(16, 8192, step), "fmt": fmt,
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "fp4":
        return {"op": op, "m": size(1, 8192), "k": size(64, 8192, step), "n": size(64, 8192, step),
                "fmt": fmt, "dtype": dtype}
    return {"op": op, "groups": size(1, 32), "rows": size(1, 4096), "k": size(64, 4096, step),
            "n": size(64, 4096, step), "fmt": fmt, "dtype": dtype}


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

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(std)

    def activations(rows, k, dtype):
        # a few channels much larger than the rest, as in a transformer's residual stream
        x = normal(rows, k)
        x[:, ::97] *= 8.0
        return x.to(DT[dtype])

    def weights(groups, a, b, dtype):
        w = torch.empty(groups, a, b, dtype=DT[dtype], device=dev)
        for g in range(groups):
            w[g] = normal(a, b, std=b ** -0.5)
        return w

    s = dict(case)
    op = case["op"]
    if "groups" in case:
        sizes = group_sizes(case["groups"], case["rows"])
        order = torch.randperm(case["groups"], generator=gen, device=dev)
        sizes = torch.tensor(sizes, device=dev)[order]
        s["cap"] = max(1, int(sizes.max()))  # the rows that the largest expert gets
        s["offsets"] = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)
    if op == "grouped":
        k, n = case["k"], case["n"]
        s["a"] = activations(case["rows"], k, case["dtype"])
        if case["b_major"] == "k":  # stored [groups, n, k]
            s["b"] = weights(case["groups"], n, k, case["dtype"])
        else:                       # stored [groups, k, n]
            s["b"] = weights(case["groups"], k, n, case["dtype"])
        s["c"] = torch.empty(case["rows"], n, dtype=DT[case["dtype"]], device=dev)
    elif op == "grouped_wgrad":
        s["a"] = activations(case["rows"], case["m"], case["dtype"])
        s["b"] = normal(case["rows"], case["n"], std=0.05).to(DT[case["dtype"]])
        s["c"] = torch.empty(case["groups"], case["m"], case["n"], dtype=DT[case["dtype"]],
                             device=dev)
    elif op == "quantize":
        s["x"] = activations(case["rows"], case["k"], case["dtype"])
        s["scale"] = tensor_scale(case["fmt"], 32.0)
        s["c"] = torch.empty(case["rows"], case["k"], device=dev)
    else:
        rows = case["m"] if op == "fp4" else case["rows"]
        groups = case.get("groups", 1)
        k, n, fmt = case["k"], case["n"], case["fmt"]
        s["x"] = activations(rows, k, case["dtype"])
        s["scale"] = tensor_scale(fmt, 32.0)
        # the layer's weights as a 4-bit checkpoint holds them: two codes a byte and the blocks'
        # scales, row after row
        s["w_scale"] = tensor_scale(fmt, 6.0 * k ** -0.5)
        parts = []
        for g in range(groups):
            parts.append(quantize_plain(normal(n, k, std=k ** -0.5), fmt, s["w_scale"]))
        s["w_codes"] = torch.cat([pack_codes(p[0]) for p in parts])
        s["w_scales"] = torch.cat([p[1] for p in parts])
        del parts
        s["c"] = torch.empty(rows, n, dtype=DT[case["dtype"]], device=dev)
        if own:
            import gemmkit_b200 as gk
            s["w"] = gk.Fp4Matrix.from_codes(s["w_codes"], s["w_scales"], groups * n, k, fmt,
                                             scale=s["w_scale"], groups=groups)
    return s


def tensor_scale(fmt, largest):
    """The per-tensor scale of the nv format: its largest value at the top of both grids."""
    return 1.0 if fmt == MX else float(torch.tensor(largest / (6.0 * 448.0), dtype=torch.float32))


# ---- the plain forms ---------------------------------------------------------------------------

def quantize_plain(x, fmt, scale):
    """(codes, scales) of a matrix: a code (0..15) for each element and a byte for each block of a
    row. In 64 bits: the grid's borders decide which code a value gets."""
    rows, k = x.shape
    bs = BLOCK[fmt]
    nb = -(-k // bs)
    v = torch.nn.functional.pad(x.double(), (0, nb * bs - k)).view(rows, nb, bs)
    amax = v.abs().amax(-1)
    if fmt == MX:
        exp = torch.frexp(amax)[1] - 1 - 2  # floor(log2(amax)) - 2: amax lands in [4, 8)
        exp = torch.where(amax > 0, exp, -127).clamp(-127, 127)
        scales = (exp + 127).to(torch.uint8)
        div = torch.ldexp(torch.ones_like(amax), exp)
    else:
        block = (amax / (6.0 * scale)).clamp(max=448.0)
        # to e4m3 from 64 bits in one rounding: its step at this magnitude, ties to even
        step = torch.ldexp(torch.ones_like(block), torch.frexp(block)[1].clamp(min=-5) - 4)
        scales = (torch.round(block / step) * step).float().to(torch.float8_e4m3fn)
        div = scales.double() * scale
        scales = scales.view(torch.uint8)
    mag = torch.where(div[..., None] > 0, v.abs() / div[..., None], 0.0).clamp(max=6.0)
    step = torch.where(mag < 2.0, 0.5, torch.where(mag < 4.0, 1.0, 2.0))
    mag = torch.round(mag / step) * step
    codes = torch.where(mag <= 2.0, mag * 2, torch.where(mag <= 4.0, mag + 2, mag / 2 + 4))
    codes = codes.to(torch.uint8) + 8 * (v < 0).to(torch.uint8)
    return codes.view(rows, nb * bs)[:, :k], scales


def pack_codes(codes):
    codes = torch.nn.functional.pad(codes, (0, codes.shape[1] % 2))
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack_codes(packed, k):
    return torch.stack([packed & 15, packed >> 4], -1).view(packed.shape[0], -1)[:, :k]


def values(codes, scales, fmt, scale):
    """The f32 values that codes and scales stand for."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    bs = BLOCK[fmt]
    if fmt == MX:
        s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    else:
        s = scales.view(torch.float8_e4m3fn).double() * scale
    v = grid[codes.int()].double() * s.repeat_interleave(bs, 1)[:, :codes.shape[1]]
    return v.float()


def by_group(s, x):
    """(group of each row, its place there, the rows of x padded to [groups, cap, k] in f32)."""
    off = s["offsets"].long()
    i = torch.arange(x.shape[0], device=x.device)
    g = torch.searchsorted(off[1:], i, right=True)
    pos = i - off[g]
    padded = torch.zeros(s["groups"], s["cap"], x.shape[1], device=x.device)
    padded[g, pos] = x.float()
    return g, pos, padded


def run_plain(s):
    op = s["op"]
    if op == "grouped":
        g, pos, a = by_group(s, s["a"])
        b = s["b"].float()
        c = torch.bmm(a, b.transpose(1, 2) if s["b_major"] == "k" else b)
        return c[g, pos].to(s["c"].dtype)
    if op == "grouped_wgrad":
        a = by_group(s, s["a"])[2]
        b = by_group(s, s["b"])[2]
        return torch.bmm(a.transpose(1, 2), b).to(s["c"].dtype)
    q = values(*quantize_plain(s["x"], s["fmt"], s["scale"]), s["fmt"], s["scale"])
    if op == "quantize":
        return q
    w = values(unpack_codes(s["w_codes"], s["k"]), s["w_scales"], s["fmt"], s["w_scale"])
    if op == "fp4":
        return (q @ w.t()).to(s["c"].dtype)
    g, pos, a = by_group(s, q)
    c = torch.bmm(a, w.view(s["groups"], s["n"], s["k"]).transpose(1, 2))
    return c[g, pos].to(s["c"].dtype)


# ---- the engine's calls --------------------------------------------------------------------------

def run_own(s):
    import gemmkit_b200 as gk
    op, c = s["op"], s["c"]
    if op == "grouped":
        rows, k, n = s["rows"], s["k"], s["n"]
        a = gk.MatRef.from_row_major(s["a"], rows, k)
        if s["b_major"] == "k":
            b = gk.MatRef.from_col_major(s["b"], k, n)
        else:
            b = gk.MatRef.from_row_major(s["b"], k, n)
        gk.gemm_half_grouped(1.0, a, b, k * n, s["offsets"], 0.0,
                             gk.MatMut.from_row_major(c, rows, n), is_f16=s["dtype"] == "f16",
                             sync=False)
        return c
    if op == "grouped_wgrad":
        rows, m, n = s["rows"], s["m"], s["n"]
        gk.gemm_half_grouped_wgrad(1.0, gk.MatRef.from_row_major(s["a"], rows, m),
                                   gk.MatRef.from_row_major(s["b"], rows, n), s["offsets"], 0.0,
                                   gk.MatMut.from_row_major(c, m, n), m * n,
                                   is_f16=s["dtype"] == "f16", sync=False)
        return c
    x = s["x"]
    rows, k = x.shape
    q = gk.quantize_fp4(gk.MatRef.from_row_major(x, rows, k), s["fmt"], scale=s["scale"],
                        offsets=s.get("offsets"), sync=False)
    if op == "quantize":
        gk.dequantize_fp4(q, gk.MatMut.from_row_major(c, rows, k), sync=False)
    else:
        gk.gemm_fp4(1.0, q, s["w"], 0.0, gk.MatMut.from_row_major(c, rows, s["n"]), sync=False)
    return c


def run(state):
    return run_own(state) if own else run_plain(state)


# ---- bytes and operations --------------------------------------------------------------------------

def work(case):
    op = case["op"]
    es = 4 if case["dtype"] == "f32" else 2

    def fp4_bytes(rows, k):
        return rows * (-(-k // 2) + -(-k // BLOCK[case["fmt"]]))

    if op == "grouped":
        rows, k, n = case["rows"], case["k"], case["n"]
        live = sum(1 for x in group_sizes(case["groups"], rows) if x)
        return {"bytes": es * (rows * k + live * k * n + rows * n), "flops": 2 * rows * k * n}
    if op == "grouped_wgrad":
        rows, m, n = case["rows"], case["m"], case["n"]
        return {"bytes": es * (rows * (m + n) + case["groups"] * m * n), "flops": 2 * rows * m * n}
    if op == "quantize":
        # read, written in 4 bits, and the values it stands for written in f32
        n = case["rows"] * case["k"]
        return {"bytes": es * n + 2 * fp4_bytes(case["rows"], case["k"]) + 4 * n, "flops": 4 * n}
    rows = case["m"] if op == "fp4" else case["rows"]
    live = 1 if op == "fp4" else sum(1 for x in group_sizes(case["groups"], rows) if x)
    k, n = case["k"], case["n"]
    return {"bytes": es * rows * (k + n) + live * fp4_bytes(n, k), "flops": 2 * rows * k * n}


# ---- the definition in 64 bits ------------------------------------------------------------------------

def nearest(x, grid):
    """Each value of x (64 bits, not negative) to the nearest of an ascending grid, ties to the
    entry of even index, past the end to the last."""
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    lo = torch.bucketize(x, mid)               # entries whose lower border lies below x
    hi = torch.bucketize(x, mid, right=True)   # ... or at x
    return grid[torch.where(lo % 2 == 0, lo, hi)]


def quantized_values(x, fmt, scale):
    """The values that the 4-bit form of x stands for, from the formats' definition."""
    k, bs = x.shape[1], BLOCK[fmt]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    whole = k // bs * bs
    for part in (slice(0, whole), slice(whole, k)):
        if part.start == part.stop:
            continue
        v = x[:, part].to(torch.float64).reshape(x.shape[0], -1, min(bs, part.stop - part.start))
        top = v.abs().max(dim=2, keepdim=True).values
        if fmt == MX:
            e = torch.floor(torch.log2(top.clamp(min=2.0 ** -130)))
            e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double()
            unit = torch.exp2((e - 2).clamp(-127, 127))
        else:
            e4m3 = [m * 2.0 ** -9 for m in range(8)]
            e4m3 += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
            unit = nearest(top / (6.0 * scale), e4m3) * scale
        ratio = torch.where(unit > 0, v.abs() / unit, torch.zeros_like(v))
        out[:, part] = (nearest(ratio, GRID) * unit * v.sign()).reshape(x.shape[0], -1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if "groups" in case:
        off = s["offsets"].tolist()
        spans = list(zip(off[:-1], off[1:]))
    if op == "grouped":
        c = torch.empty(s["c"].shape, dtype=torch.float64, device=s["c"].device)
        for g, (i, j) in enumerate(spans):
            w = s["b"][g].double()
            c[i:j] = s["a"][i:j].double() @ (w.T if case["b_major"] == "k" else w)
        return c
    if op == "grouped_wgrad":
        return torch.stack([s["a"][i:j].double().T @ s["b"][i:j].double() for i, j in spans])
    q = quantized_values(s["x"], case["fmt"], s["scale"])
    if op == "quantize":
        return q
    k, n, fmt = case["k"], case["n"], case["fmt"]
    table = torch.tensor(GRID, dtype=torch.float64, device=q.device)

    def layer(g):
        codes = s["w_codes"][g * n:(g + 1) * n]
        sc = s["w_scales"][g * n:(g + 1) * n]
        w = torch.empty(n, codes.shape[1] * 2, dtype=torch.float64, device=q.device)
        for half, c4 in enumerate((codes % 16, codes // 16)):
            w[:, half::2] = table[(c4 % 8).long()] * (1.0 - 2.0 * (c4 >= 8).double())
        if fmt == MX:
            unit = torch.exp2(sc.double() - 127)
        else:
            unit = sc.view(torch.float8_e4m3fn).double() * s["w_scale"]
        at = torch.arange(k, device=q.device) // BLOCK[fmt]
        return w[:, :k] * unit[:, at]

    if op == "fp4":
        return q @ layer(0).T
    c = torch.empty(s["c"].shape, dtype=torch.float64, device=q.device)
    for g, (i, j) in enumerate(spans):
        c[i:j] = q[i:j] @ layer(g).T
    return c
