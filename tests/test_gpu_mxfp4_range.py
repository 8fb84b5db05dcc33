"""-m gpu: the products over the whole range of scale bytes, one product of two values per output, hence exact up to the rounding to float32
(subnormals included).  A W element of 2^128 or more is infinity for the product with A in bfloat16, as documented; not for MXFP4 x MXFP4."""
import math

import pytest
import torch

from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu


def one_value(flux2mi, scale_bytes, code, cols, at):
    """MXFP4 with one code per row, at column `at`, under the row's scale byte."""
    from flux2mi.api import MXFP4
    rows, p = len(scale_bytes), R.padded(cols)
    codes, scales = torch.zeros((rows, p // 2), dtype=torch.uint8), torch.zeros((rows, p // 32), dtype=torch.uint8)
    codes[:, at // 2] = code << (4 * (at & 1))
    scales[:, at // 32] = torch.tensor(scale_bytes, dtype=torch.uint8)
    return MXFP4(codes.cuda(), scales.cuda(), cols)


def powers(scale_bytes):
    return torch.ldexp(torch.ones(len(scale_bytes), dtype=torch.float64), torch.tensor(scale_bytes) - 127)


def spread(n):   # n scale bytes over 0 ... 254
    return [round(i * 254 / (n - 1)) for i in range(n)] if n < 255 else [i % 255 for i in range(n)]


@pytest.mark.parametrize("code", [1, 2, 7, 14])
@pytest.mark.parametrize("m,n,k,at", [(16, 255, 128, 3), (16, 4080, 1000, 500), (64, 4080, 2048, 2047), (255, 4080, 640, 0), (1020, 4080, 1100, 1000)])
def test_mxfp4_product(ctx, flux2mi, m, n, k, at, code):
    a, w = spread(m), spread(n)
    want = (powers(a)[:, None] * powers(w)[None] * R.E2M1[code & 7] ** 2).float()
    got = ctx.op_gemm_mxfp4(one_value(flux2mi, a, code, k, at), one_value(flux2mi, w, code, k, at), dtype=torch.float32)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("code", [1, 2, 4, 7, 15])
@pytest.mark.parametrize("m,n,k,at", [(4, 255, 128, 3), (23, 255, 128, 3), (64, 4080, 2048, 2047), (40, 510, 1101, 1000), (255, 4080, 640, 0), (512, 4080, 1100, 1000)])
def test_bf16_product(ctx, flux2mi, m, n, k, at, code):
    w = spread(n)
    value = torch.ldexp(torch.ones(m, dtype=torch.float64), torch.tensor([-133 + round(i * 260 / (m - 1)) for i in range(m)]))   # every bf16 binade
    value[m // 2] = 0
    a = torch.zeros((m, k), dtype=torch.bfloat16)
    a[:, at] = value.bfloat16()
    elements = powers(w) * R.E2M1[code & 7] * (-1 if code & 8 else 1)
    elements = torch.where(elements.abs() >= 2.0 ** 128, elements * math.inf, elements)
    want = (value[:, None] * elements[None]).float()
    got = ctx.op_gemm_bf16_mxfp4(a.cuda(), one_value(flux2mi, w, code, k, at), dtype=torch.float32).cpu()
    nan = torch.isnan(want)
    assert bool(nan.any()) == (code in (4, 7, 15))   # 0 x infinity; 2, 6 and -6 reach 2^128
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])


def test_read_back_beyond_float32(ctx, flux2mi):
    m = one_value(flux2mi, [252, 253, 253, 254, 254], 6, 64, 40)   # 4 x 2^125 ...
    for dtype in (torch.float32, torch.bfloat16):
        assert ctx.op_dequantize_mxfp4(m, dtype)[:, 40].tolist() == [2.0 ** 127, math.inf, math.inf, math.inf, math.inf]
