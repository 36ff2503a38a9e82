"""What the feed-forward layers' entries refuse, all before any device work (no GPU needed)."""
import ctypes as C

import pytest

import gemmkit_b200 as gk
from gemmkit_b200 import _lib


def refused(call, text):
    with pytest.raises(gk.GemmkitError) as e:
        call()
    assert e.value.code == gk.GK_EINVAL and text in str(e.value), str(e.value)


def at(page, n):
    """A (pointer, length) pair: no memory is touched before a refusal."""
    return page << 20, n


def mat(page, rows, cols, rs=None, cs=1, n=None, kind=gk.MatRef):
    rs = cols if rs is None else rs
    return kind(at(page, (rows - 1) * rs + (cols - 1) * cs + 1 if n is None else n), rows, cols, rs, cs)


def out(page, rows, cols, **kw):
    return mat(page, rows, cols, kind=gk.MatMut, **kw)


A, B, Cm = mat(1, 4, 8), mat(2, 8, 6), out(3, 4, 6)


def forward(a=A, b=B, c=Cm, **kw):
    return lambda: gk.gemm_half_epilogue(1.0, a, b, c, sync=False, **kw)


def test_epilogue_refusals():
    refused(forward(a=mat(1, 4, 7)), "A.cols (7) != B.rows (8)")
    refused(forward(c=out(3, 5, 6)), "A.rows (4) != C.rows (5)")
    refused(forward(c=out(3, 4, 6, rs=0)), "aliases itself")
    refused(forward(c=out(1, 4, 6)), "C aliases A or B")
    refused(forward(a=mat(1, 4, 8, rs=-8)), "negative strides")
    refused(forward(c=gk.MatMut(((3 << 20) + 1, 24), 4, 6, 6, 1)), "not aligned")
    refused(forward(offsets=(4096, 1)), "1 to 1024 groups")
    refused(forward(offsets=(4096, 3), b_gs=47), "does not fit its slice")
    refused(forward(offsets=(4096, 3), b_gs=-1), "must not be negative")
    two = mat(2, 8, 6, n=96)
    refused(forward(b=two, offsets=(4096, 3), b_gs=48, bias=at(4, 11)), "bias holds 11 elements, 2 groups of 6 need 12")
    refused(forward(b=two, offsets=(4096, 3), b_gs=48, bias=at(4, 12), bias_gs=-6), "bad group stride -6 of bias")
    refused(forward(bias=at(4, 5)), "bias holds 5 elements")
    refused(forward(bias=((4 << 20) + 1, 6)), "bias is not aligned")
    refused(forward(bias=at(3, 6)), "C aliases another operand")
    refused(forward(residual=mat(4, 4, 5)), "the residual is 4x5, the output is 4x6")
    refused(forward(residual=mat(4, 4, 6, n=23)), "view of 4x6")
    refused(forward(residual=gk.MatRef(((3 << 20) + 12, 24), 4, 6, 6, 1)), "C aliases the residual")
    refused(forward(residual=mat(3, 4, 6, rs=7)), "C aliases the residual")
    refused(forward(z=out(4, 3, 6)), "z is 3x6, the output is 4x6")
    refused(forward(z=out(4, 4, 6, rs=0)), "z view aliases itself")
    for page in (1, 2, 3):
        refused(forward(z=out(page, 4, 6)), "z aliases another operand")
    refused(forward(z=out(4, 4, 6), residual=mat(4, 4, 6)), "z aliases another operand")
    refused(forward(z=out(4, 4, 6), bias=at(4, 6)), "z aliases another operand")
    refused(forward(act=gk.Activation(6)), "unknown activation 6")
    refused(forward(act=gk.Activation(-1)), "unknown activation -1")
    refused(forward(a=mat(0, 4, 8)), "null A or B")
    refused(forward(c=out(0, 4, 6)), "null C")
    lib = _lib.load()
    args = (0, 1, None, 1.0, A.c(), B.c(), 0)
    assert lib.gk_gemm_half_epilogue(*args, None, Cm.c(), 2, gk.SERIAL.c(), None) == gk.GK_EINVAL
    e = _lib.EpilogueC()
    for bad in (1, 7, -1):  # f16 C of bf16 operands, unknown types
        assert lib.gk_gemm_half_epilogue(*args, C.byref(e), Cm.c(), bad, gk.SERIAL.c(), None) == gk.GK_EINVAL
    e.bias, e.bias_len, e.bias_type = 4 << 20, 6, 1
    assert lib.gk_gemm_half_epilogue(*args, C.byref(e), Cm.c(), 2, gk.SERIAL.c(), None) == gk.GK_EINVAL
    assert b"bias must hold f32 or the operands" in lib.gk_last_error()
    # several groups need offsets
    assert lib.gk_gemm_half_epilogue(0, 2, None, 1.0, A.c(), B.c(), 0, C.byref(e), Cm.c(), 2, gk.SERIAL.c(),
                                     None) == gk.GK_EINVAL
    # nothing to do is accepted without a device
    gk.gemm_half_epilogue(1.0, mat(1, 0, 8, n=0), B, out(3, 0, 6, n=0), sync=False)


def act8(rows, cols, page=8, epage=9, codes_len=None, ld=None, exps_len=None, eld=None):
    q = gk.Act8Matrix.__new__(gk.Act8Matrix)
    nb = (cols + 31) // 32
    ld, eld = nb * 32 if ld is None else ld, nb if eld is None else eld
    q.rows, q.cols, q._where = rows, cols, None
    q.c = _lib.Act8MatrixC(rows, cols, page << 20, rows * ld if codes_len is None else codes_len, ld,
                           epage << 20, rows * eld if exps_len is None else exps_len, eld)
    return q


def test_backward_refusals():
    z, silu = mat(4, 4, 6), gk.Activation.Silu()

    def dact(a=A, b=B, z=z, act=silu, c=Cm, **kw):
        return lambda: gk.gemm_half_dact(1.0, a, b, z, act, c, sync=False, **kw)
    refused(dact(a=mat(1, 4, 7)), "A.cols (7) != B.rows (8)")
    refused(dact(z=None), "null z")
    refused(dact(z=mat(4, 4, 5)), "z is 4x5, the output is 4x6")
    refused(dact(z=act8(4, 5)), "z is 4x5, the output is 4x6")
    refused(dact(z=gk.MatRef(((3 << 20) + 12, 24), 4, 6, 6, 1)), "C aliases z")
    refused(dact(z=act8(4, 6, page=3)), "C aliases z")
    refused(dact(z=act8(4, 6, epage=3)), "C aliases z")
    refused(dact(z=act8(4, 6, ld=48)), "must be a multiple of 32")
    refused(dact(z=act8(4, 40, ld=32), c=out(3, 4, 40), b=mat(2, 8, 40)), "must be a multiple of 32")
    refused(dact(z=act8(4, 6, codes_len=127)), "needs 128 bytes of codes (has 127)")
    refused(dact(z=act8(4, 6, exps_len=3)), "4 of exponents (has 3)")
    refused(dact(dbias=at(5, 5)), "dbias holds 5 elements")
    refused(dact(dbias=at(3, 6)), "dbias aliases another operand")
    refused(dact(dbias=at(1, 6)), "dbias aliases another operand")
    refused(dact(dbias=at(4, 6)), "dbias aliases another operand")
    refused(dact(b=mat(2, 8, 6, n=96), offsets=(4096, 3), b_gs=48, dbias=at(5, 12), dbias_gs=5),
            "bad group stride 5 of dbias")
    refused(dact(act=gk.Activation(9)), "unknown activation 9")

    dy, dz = mat(1, 4, 6), out(3, 4, 6)

    def grad(dy=dy, z=z, act=silu, dz=dz, **kw):
        return lambda: gk.act_backward(dy, z, act, dz, sync=False, **kw)
    refused(grad(dz=out(3, 4, 5)), "dZ is 4x5, dY is 4x6")
    refused(grad(dz=out(3, 4, 6, rs=0)), "dZ view aliases itself")
    refused(grad(dz=gk.MatMut(((1 << 20) + 4, 24), 4, 6, 6, 1)), "dZ aliases dY")
    refused(grad(dz=None), "neither dZ nor dbias")
    refused(grad(dz=None, dbias=at(1, 6)), "dbias aliases another operand")
    refused(grad(z=None), "null z")
    refused(grad(offsets=(4096, 1026)), "1 to 1024 groups")
    refused(grad(dy=mat(0, 4, 6), dz=None, dbias=at(5, 6)), "null dY")


def test_act8_refusals():
    def quant(x=mat(1, 4, 40), q=None, t=_lib.DT_BF16):
        return lambda: gk.quantize_act8(x, out=q or act8(4, 40), x_type=t, sync=False)
    refused(quant(t=7), "unknown element type 7")
    refused(quant(x=mat(1, 4, 39)), "the source is 4x39, the 8-bit matrix holds 4x40")
    refused(quant(x=mat(1, 4, 40, n=10)), "X view of 4x40")
    refused(quant(x=mat(8, 4, 40)), "aliases its source or itself")
    refused(quant(q=act8(4, 40, epage=8)), "aliases its source or itself")
    refused(quant(q=act8(4, 40, ld=63)), "must be a multiple of 32")
    refused(quant(q=act8(4, 40, eld=1)), "must hold 2 blocks")
    refused(quant(q=act8(4, 40, page=0)), "null codes or exponents")
    refused(quant(x=mat(0, 4, 40)), "null X")
    odd = act8(4, 40)
    odd.c.codes += 8
    refused(quant(q=odd), "16-byte aligned")

    def deq(q=None, c=out(3, 4, 40), t=_lib.DT_BF16):
        return lambda: gk.dequantize_act8(q or act8(4, 40), c, out_type=t, sync=False)
    refused(deq(t=-1), "unknown element type -1")
    refused(deq(c=out(3, 4, 39)), "the 8-bit matrix holds 4x40, the output is 4x39")
    refused(deq(c=out(8, 4, 40)), "C aliases the 8-bit matrix")
    refused(deq(c=out(3, 4, 40, rs=0)), "aliases itself")
    refused(deq(c=out(0, 4, 40)), "null C")

    def wgrad(q=None, b=mat(2, 4, 6), c=out(3, 40, 6), **kw):
        return lambda: gk.gemm_act8_wgrad(1.0, q or act8(4, 40), b, 0.0, c, sync=False, **kw)
    refused(wgrad(b=mat(2, 5, 6)), "A.cols (4) != B.rows (5)")
    refused(wgrad(c=out(3, 39, 6)), "A.rows (40) != C.rows (39)")
    refused(wgrad(c=out(8, 40, 6)), "C aliases A or B")
    refused(wgrad(c=out(2, 40, 6)), "C aliases A or B")
    refused(wgrad(c=out(3, 40, 6, n=480), offsets=(4096, 3), c_gs=239), "the groups of C overlap")
    refused(wgrad(c=out(3, 40, 6, n=479), offsets=(4096, 3), c_gs=240), "does not fit its slice")
    refused(wgrad(b=mat(0, 4, 6)), "null A or B")
    refused(wgrad(q=act8(4, 40, codes_len=1)), "bytes of codes (has 1)")
    refused(lambda: gk.gemm_act8_wgrad(1.0, act8(4, 40), mat(2, 4, 6), 0.0, out(3, 40, 6),
                                       offsets=(4096, 1), sync=False), "1 to 1024 groups")


def test_act8_matrix_of_tensors():
    torch = pytest.importorskip("torch")
    codes, exps = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    refused(lambda: gk.Act8Matrix(4, 40, codes, exps), "codes must be 4x40 int8")
    refused(lambda: gk.Act8Matrix(4, 64, codes, exps[:, :1]), "exponents must be 4x2 uint8")
    refused(lambda: gk.Act8Matrix(4, 64, codes.to(torch.uint8), exps), "codes must be")
    refused(lambda: gk.Act8Matrix(4, 64, codes, exps), "not in device memory")


def test_balance_refusals():
    lib = _lib.load()
    x = mat(1, 4, 8)

    def call(x=x, t=0, ids=2 << 20, n=8, top=2, loss=3 << 20, counts=4 << 20, offsets=5 << 20, rates=6 << 20):
        return lib.gk_moe_balance(x.c(), t, ids, n, top, 0, 1.0, loss, counts, offsets, rates, None)

    def bad(text, **kw):
        assert call(**kw) == gk.GK_EINVAL
        assert text.encode() in lib.gk_last_error(), lib.gk_last_error()
    bad("unknown element type 5", t=5)
    bad("1 to 1024 experts (has 0)", x=mat(1, 4, 0, n=0))
    bad("1 to 1024 experts (has 1025)", x=mat(1, 4, 1025))
    bad("dimensions exceed", top=0)
    bad("need as many ids (has 7)", n=7)
    bad("null logits or ids", ids=None)
    bad("null logits or ids", x=mat(0, 4, 8))
    bad("null output", loss=None)
    bad("not aligned", ids=(2 << 20) + 2)
    bad("not aligned", rates=(6 << 20) + 1)
    bad("alias each other or the inputs", counts=(5 << 20) + 4)
    bad("alias each other or the inputs", loss=1 << 20)
    bad("alias each other or the inputs", rates=(2 << 20) + 28)
    bad("view of 4x8", x=mat(1, 4, 8, n=31))

    def back(d=out(7, 4, 8), rates=6 << 20, dloss=3 << 20, x=x):
        return lib.gk_moe_balance_backward(x.c(), 0, 2 << 20, 8, 2, 0, rates, dloss, d.c(), None)

    def bad2(text, **kw):
        assert back(**kw) == gk.GK_EINVAL
        assert text.encode() in lib.gk_last_error(), lib.gk_last_error()
    bad2("the gradient is 4x7, the logits are 4x8", d=out(7, 4, 7))
    bad2("dlogits view aliases itself", d=out(7, 4, 8, rs=0))
    bad2("null rates or dloss", rates=None)
    bad2("null dlogits", d=out(0, 4, 8))
    bad2("alias another operand", d=gk.MatMut(((1 << 20) + 16, 32), 4, 8, 8, 1))
    bad2("alias another operand", d=out(6, 4, 8))
    bad2("alias another operand", d=out(2, 4, 8))
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        refused(lambda: gk.moe_balance(mat(1, 4, 8), torch.zeros(4, 2, dtype=torch.int32), x_type=0),
                "not in device memory")


def test_the_older_epilogues_keep_their_activations():
    a, b, c = mat(1, 4, 8), mat(2, 8, 6), out(3, 4, 6)
    for act in (gk.Activation.Gelu(), gk.Activation.GeluTanh(), gk.Activation.Silu()):
        refused(lambda: gk.gemm_half_f32_fused(1.0, a, b, 0.0, c, act=act, sync=False),
                f"unknown activation {act.kind}")
