"""What the tests of the feed-forward layers' operators share: views of tensors, and the plain forms in
64 bits."""
import math

import numpy as np

import gemmkit_b200 as gk
from gpu_util import torch_cuda

HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
SUBNORMAL = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}
ACTS = ["none", "relu", "leaky", "gelu", "gelu_tanh", "silu"]
SLOPE = 0.125


def tdt(name):
    torch = torch_cuda()
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def ref(t2, kind=gk.MatRef):
    """A MatRef / MatMut of a 2-D tensor view, of its own storage from its first element on."""
    r, c = t2.shape
    rs, cs = t2.stride()
    n = (r - 1) * rs + (c - 1) * cs + 1 if t2.numel() else 0
    return kind(t2.as_strided((n,), (1,)) if n else t2.reshape(-1), r, c, rs, cs)


def mut(t2):
    return ref(t2, gk.MatMut)


def act_of(name):
    a = gk.Activation
    return {"none": lambda: None, "relu": a.Relu, "leaky": lambda: a.LeakyRelu(SLOPE), "gelu": a.Gelu,
            "gelu_tanh": a.GeluTanh, "silu": a.Silu}[name]()


def act64(z, name):
    torch = torch_cuda()
    if name == "relu":
        return z.clamp(min=0)
    if name == "leaky":
        return z.clamp(min=0) + SLOPE * z.clamp(max=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, name):
    """act', by 64-bit differentiation of act64 (ReLU and LeakyReLU: the value at 0 is the left one)."""
    torch = torch_cuda()
    if name == "relu":
        return (z > 0).double()
    if name == "leaky":
        return torch.where(z > 0, 1.0, SLOPE).double()
    if name == "none":
        return torch.ones_like(z)
    x = z.detach().clone().requires_grad_(True)
    return torch.autograd.grad(act64(x, name).sum(), x)[0]


def numbers(seed, shape, dtype, ints=True, std=1.0):
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if ints:
        x = torch.randint(-4, 5, shape, generator=gen, device="cuda").float()
    else:
        x = torch.randn(shape, generator=gen, device="cuda") * std
    return x.to(tdt(dtype))


def offsets_of(sizes, lead=0):
    torch = torch_cuda()
    return torch.tensor(np.cumsum([lead] + list(sizes)), dtype=torch.int32, device="cuda")


def spans(off, rows):
    """(group, its rows) as slices; one group of all rows without offsets."""
    if off is None:
        return [(0, slice(0, rows))]
    o = off.tolist()
    return [(g, slice(o[g], o[g + 1])) for g in range(len(o) - 1)]


def act8_values(q):
    """What an Act8Matrix stands for, in 64 bits, by the format's definition."""
    torch = torch_cuda()
    e = q.exponents.double()
    unit = torch.where(e == 255, float("nan"), torch.exp2(e - 133))
    return q.codes.double() * unit.repeat_interleave(32, 1)[:, :q.cols]


def status_clean():
    assert gk.device_status(0) == 0
