"""CPU: the MXFP4 and residual-norm entry points refuse what their documentation rules out, before anything touches the device (the
context handed in is a block of zeros: a call that got as far as reading it would find no stream), and calls without rows do nothing."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import mxfp4_ref as R

OK, INVALID, SHAPE = 0, 1, 4
F32, BF16, F16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib(flux2mi):
    return flux2mi.lib()


@pytest.fixture(scope="module")
def ctx():
    buf = C.create_string_buffer(1 << 16)
    yield C.addressof(buf)


A = lambda i: 0x10000000 * (i + 1)  # noqa: E731  addresses far apart that nothing reads


def test_sizes(lib):
    for cols in (1, 31, 32, 33, 127, 128, 129, 4096, 5119):
        assert lib.flux2mi_mxfp4_code_bytes(3, cols) == 3 * R.padded(cols) // 2
        assert lib.flux2mi_mxfp4_scale_bytes(3, cols) == 3 * R.padded(cols) // 32
    assert lib.flux2mi_mxfp4_code_bytes(0, 32) == 0
    for rows, cols in ((-1, 32), (3, 0), (3, -5), (3, 1 << 31)):
        assert lib.flux2mi_mxfp4_code_bytes(rows, cols) == 0 and lib.flux2mi_mxfp4_scale_bytes(rows, cols) == 0
    assert lib.flux2mi_mxfp4_code_bytes(1 << 33, 4096) == (1 << 33) * 2048   # past 32 bits


@pytest.mark.parametrize("rows,cols", [((1 << 40) - 1, 1 << 30), (1 << 40, 1 << 30), (1 << 40, 1 << 26), (1 << 36, 1 << 28), ((1 << 33) + 1, 1 << 30), (1 << 33, 1 << 30)])
def test_sizes_past_64_bits(lib, ctx, rows, cols):
    """Sizes that do not fit 63 bits are 0, the largest that fit are right; a matrix of either reaches over every other buffer and is refused."""
    for size, per_byte in ((lib.flux2mi_mxfp4_code_bytes, 2), (lib.flux2mi_mxfp4_scale_bytes, 32)):
        want = rows * (cols // per_byte)
        assert size(rows, cols) == (want if want < 1 << 63 else 0)
    for x, codes, scales in ((A(0), A(1), A(2)), (A(2), A(1), A(0)), (A(1), A(0), A(2))):
        refuses(lib, lib.flux2mi_op_quantize_mxfp4(ctx, x, F32, cols, rows, cols, codes, scales), INVALID, "overlap")
        refuses(lib, lib.flux2mi_op_dequantize_mxfp4(ctx, codes, scales, rows, cols, x, BF16, cols), INVALID, "overlap")


def refuses(lib, code, status, *words):
    assert code == status, (code, lib.flux2mi_last_error())
    if status != OK:
        message = lib.flux2mi_last_error().decode()
        assert message and all(w in message for w in words), message


@pytest.mark.parametrize("change,status,word", [
    ({}, None, ""), ({"ctx": None}, INVALID, "ctx"), ({"dtype": 3}, INVALID, "dtype"), ({"dtype": -1}, INVALID, "dtype"), ({"rows": -1}, SHAPE, "rows"),
    ({"cols": 0}, SHAPE, "cols"), ({"ld": 63}, SHAPE, "stride"), ({"x": None}, INVALID, "NULL"), ({"x": A(0) + 1}, INVALID, "aligned"),
    ({"codes": None}, INVALID, "NULL"), ({"scales": None}, INVALID, "NULL"), ({"codes": A(1) + 8}, INVALID, "aligned"),
    ({"scales": A(2) + 2}, INVALID, "aligned"), ({"codes": A(0) + 16}, INVALID, "overlap"), ({"scales": A(0) + 512}, INVALID, "overlap"),
    ({"rows": 0}, OK, ""), ({"rows": 0, "x": None, "codes": None, "scales": None}, OK, "")])
def test_quantize_and_dequantize(lib, ctx, change, status, word):
    if status is None:
        return   # the valid call itself needs a device
    v = {"ctx": ctx, "x": A(0), "dtype": BF16, "ld": 64, "rows": 5, "cols": 64, "codes": A(1), "scales": A(2), **change}
    refuses(lib, lib.flux2mi_op_quantize_mxfp4(v["ctx"], v["x"], v["dtype"], v["ld"], v["rows"], v["cols"], v["codes"], v["scales"]), status, word)
    refuses(lib, lib.flux2mi_op_dequantize_mxfp4(v["ctx"], v["codes"], v["scales"], v["rows"], v["cols"], v["x"], v["dtype"], v["ld"]), status, word)


def test_quantize_result_buffers_overlap(lib, ctx):
    refuses(lib, lib.flux2mi_op_quantize_mxfp4(ctx, A(0), F32, 64, 5, 64, A(1), A(1) + 64), INVALID, "overlap")


@pytest.mark.parametrize("change,status,word", [
    ({"ctx": None}, INVALID, "ctx"), ({"m": -1}, SHAPE, "M -1"), ({"n": -1}, SHAPE, "N -1"), ({"k": 0}, SHAPE, "K 0"), ({"odt": F16}, INVALID, "out_dtype"),
    ({"odt": BF16, "resid": A(6)}, INVALID, "residual"), ({"w": None}, INVALID, "W"), ({"ws": None}, INVALID, "W"), ({"w": A(2) + 4}, INVALID, "aligned"),
    ({"ws": A(3) + 1}, INVALID, "aligned"), ({"out": None}, INVALID, "NULL"), ({"ldo": 39}, SHAPE, "stride"), ({"resid": A(6), "ldr": 8}, SHAPE, "stride"),
    ({"out": A(7) + 2}, INVALID, "aligned"), ({"bias": A(4) + 2}, INVALID, "aligned"), ({"gate": A(5) + 1}, INVALID, "aligned"),
    ({"out": A(0)}, INVALID, "overlap"), ({"out": A(2) + 64}, INVALID, "overlap"), ({"out": A(4), "bias": A(4)}, INVALID, "overlap"),
    ({"resid": A(7), "ldr": 48}, INVALID, "overlap"), ({"resid": A(7) + 4, "ldr": 40}, INVALID, "overlap"),
    ({"m": 0}, OK, ""), ({"n": 0}, OK, ""), ({"m": 0, "a": None, "as": None, "w": None, "ws": None, "out": None}, OK, "")])
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_products(lib, ctx, kind, change, status, word):
    v = {"ctx": ctx, "a": A(0), "as": A(1), "w": A(2), "ws": A(3), "bias": None, "gate": None, "resid": None, "ldr": 40, "out": A(7), "odt": F32, "ldo": 40,
         "m": 9, "n": 40, "k": 70, **change}
    tail = (v["w"], v["ws"], v["bias"], v["gate"], v["resid"], v["ldr"], v["out"], v["odt"], v["ldo"], v["m"], v["n"], v["k"])
    if kind == "mxfp4":
        refuses(lib, lib.flux2mi_op_gemm_mxfp4(v["ctx"], v["a"], v["as"], *tail), status, word)
    else:
        refuses(lib, lib.flux2mi_op_gemm_bf16_mxfp4(v["ctx"], v["a"], 70, *tail), status, word)


def test_column_slices_that_share_a_column(lib, ctx):
    """Rows of 100 f32: out is 40 columns from 30 on (or wraps into the next row's first ones), resid the first 40."""
    call = lambda off: lib.flux2mi_op_gemm_bf16_mxfp4(ctx, A(0), 70, A(2), A(3), None, None, A(7) + 400, 100, A(7) + off, F32, 100, 9, 40, 70)  # noqa: E731
    for column in (30, 39, 70 - 100, 99 - 100, 130, 170, 830):
        refuses(lib, call(400 + 4 * column), INVALID, "overlap")


@pytest.mark.parametrize("ld", [1 << 40, 1 << 61, (1 << 63) - 1])
def test_row_strides_beyond_memory(flux2mi, lib, ctx, ld):
    """Sizes whose bytes do not fit 64 bits, or reach over the other operands."""
    refuses(lib, lib.flux2mi_op_quantize_mxfp4(ctx, A(0), F32, ld, 1 << 38, 64, A(1), A(2)), INVALID, "overlap")
    refuses(lib, lib.flux2mi_op_gemm_bf16_mxfp4(ctx, A(0), ld, A(2), A(3), None, None, None, 0, A(7), F32, 40, 1 << 30, 40, 70), INVALID, "overlap")


def test_products_first_operand(lib, ctx):
    tail = (A(2), A(3), None, None, None, 0, A(7), F32, 40, 9, 40, 70)
    refuses(lib, lib.flux2mi_op_gemm_mxfp4(ctx, None, A(1), *tail), INVALID, "A")
    refuses(lib, lib.flux2mi_op_gemm_mxfp4(ctx, A(0), None, *tail), INVALID, "A")
    refuses(lib, lib.flux2mi_op_gemm_mxfp4(ctx, A(0) + 8, A(1), *tail), INVALID, "aligned")
    refuses(lib, lib.flux2mi_op_gemm_bf16_mxfp4(ctx, None, 70, *tail), INVALID, "NULL")
    refuses(lib, lib.flux2mi_op_gemm_bf16_mxfp4(ctx, A(0), 69, *tail), SHAPE, "stride")
    refuses(lib, lib.flux2mi_op_gemm_bf16_mxfp4(ctx, A(0) + 1, 70, *tail), INVALID, "aligned")


@pytest.mark.parametrize("change,status,word", [
    ({"rows": -1}, SHAPE, "rows"), ({"rows": 1 << 24}, SHAPE, "rows"), ({"dim": 0}, SHAPE, "dim"), ({"dim": 16385}, SHAPE, "dim"), ({"post_norm": 3}, INVALID, "norm"),
    ({"norm": -1}, INVALID, "norm"), ({"y_dtype": F16}, INVALID, "y_dtype"), ({"out_dtype": F16}, INVALID, "out_dtype"), ({"eps": -1.0}, INVALID, "eps"),
    ({"post_eps": float("nan")}, INVALID, "eps"), ({"y": None}, INVALID, "without y"), ({"out": None}, INVALID, "without out"), ({"x": None}, INVALID, "NULL"),
    ({"x_out": None, "out": None, "norm": 0}, INVALID, "NULL"), ({"ldx": 63}, SHAPE, "stride"), ({"ldy": 63}, SHAPE, "stride"), ({"ldx_out": 63}, SHAPE, "stride"),
    ({"ldo": 63}, SHAPE, "stride"), ({"x": A(0) + 2}, INVALID, "aligned"), ({"y": A(1) + 1}, INVALID, "aligned"), ({"out": A(3) + 1}, INVALID, "aligned"),
    ({"weight": A(4) + 1}, INVALID, "aligned"), ({"x_out": A(0) + 256}, INVALID, "x_out"), ({"x_out": A(0), "ldx_out": 128}, INVALID, "x_out"),
    ({"out": A(0)}, INVALID, "overlap"), ({"out": A(1)}, INVALID, "overlap"), ({"x_out": A(3)}, INVALID, "overlap"), ({"weight": A(3)}, INVALID, "overlap"),
    ({"rows": 0}, OK, ""), ({"rows": 0, "x": None, "y": None, "x_out": None, "out": None}, OK, "")])
def test_residual_norm(flux2mi, lib, ctx, change, status, word):
    from flux2mi import _lib as L
    v = {"rows": 7, "dim": 64, "split": 2, "post_norm": 1, "norm": 2, "post_eps": 1e-6, "eps": 1e-6, "resid_scale": 1.0, "x": A(0), "ldx": 64, "y": A(1), "y_dtype": BF16,
         "ldy": 64, "x_out": A(2), "ldx_out": 64, "out": A(3), "out_dtype": BF16, "ldo": 64, **change}
    refuses(lib, lib.flux2mi_op_residual_norm(ctx, C.byref(L.ResidualNorm(**v))), status, word)
    refuses(lib, lib.flux2mi_op_residual_norm(None, C.byref(L.ResidualNorm(**v))), INVALID, "NULL")
    refuses(lib, lib.flux2mi_op_residual_norm(ctx, None), INVALID, "NULL")


def test_the_definition_itself():
    """The float64 reference of the GPU tests on values whose codes are known by hand."""
    x = torch.zeros((1, 32))
    x[0, :16] = torch.tensor([0, 0.25, 0.2500001, 0.75, 1.25, 1.2500001, 1.75, 2.5, 2.5000002, 3.5, 5.0, 5.0000005, 7.9, -0.75, -7.0, 6.0])
    codes, scales = R.quantize(x)
    assert scales.tolist() == [[127, 0, 0, 0]] and codes.shape == (1, 64)
    flat = np.stack([codes & 15, codes >> 4], 2).reshape(-1)
    assert flat[:16].tolist() == [0, 0, 1, 2, 2, 3, 4, 4, 5, 6, 6, 7, 7, 10, 15, 7] and not flat[16:].any()
    assert R.dequantize(codes, scales, 32)[0, :16].tolist() == [0, 0, 0.5, 1, 1, 1.5, 2, 2, 3, 4, 4, 6, 6, -1, -6, 6]
    for v, byte in ((0.0, 0), (2.0 ** -149, 0), (2.0 ** -126, 0), (2.0 ** -124, 1), (1.0, 125), (3.9, 126), (4.0, 127), (3.4e38, 252), (float("inf"), 255), (float("nan"), 255)):
        assert int(R.quantize(torch.full((1, 1), v))[1][0, 0]) == byte, v
