"""-m gpu: MXFP4 quantisation, reading back and the two products, against their definition in float64 (tests/mxfp4_ref.py).
Codes, scales and read-back values are compared bit for bit; products within the bound that float32 sums and one rounding of the result allow."""
import math

import numpy as np
import pytest
import torch

from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # relative: half a step


def gen(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 31))


def same_bytes(m, x):
    codes, scales = R.quantize(x)
    assert m.cols == x.shape[1] and m.codes.shape == codes.shape and m.scales.shape == scales.shape
    assert np.array_equal(m.scales.cpu().numpy(), scales)
    assert np.array_equal(m.codes.cpu().numpy(), codes)


# ------------------------------------------------------------------------------------------------------------ quantise
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 127), (2, 128), (4, 129), (130, 257), (1, 4099), (67, 2560), (3, 8200)])
def test_quantize(ctx, rows, cols, dtype):
    g = gen(rows, cols)
    x = torch.randn((rows, cols), generator=g) * torch.exp(torch.randn((rows, 1), generator=g) * 3)
    x[:, ::7] = 0
    same_bytes(ctx.op_quantize_mxfp4(x.to(dtype).cuda()), x.to(dtype))


def test_quantize_every_bfloat16(ctx):
    """All 65536 bf16 values, NaN and infinities among them: alone in a block, and beside every power of two."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    v = bits.view(torch.bfloat16)
    alone = torch.zeros((65536, 32), dtype=torch.bfloat16)
    alone[:, 5] = v
    same_bytes(ctx.op_quantize_mxfp4(alone.cuda()), alone)
    finite = v[torch.isfinite(v.float())]
    dense = finite[torch.randperm(len(finite), generator=gen(1))][: len(finite) // 4096 * 4096].view(-1, 4096)
    same_bytes(ctx.op_quantize_mxfp4(dense.cuda()), dense)
    order = finite[torch.argsort(finite.float().abs())][: len(finite) // 32 * 32].view(-1, 32)   # neighbours in size: every code, ties
    same_bytes(ctx.op_quantize_mxfp4(order.cuda()), order)


def test_quantize_ties_and_subnormals(ctx):
    base = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.99, .5, 1, 1.5, 2, 3, 4])
    rows = []
    for e in (-149, -140, -127, -126, -125, -124, -1, 0, 60, 124):
        for nudge in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24):
            rows.append(torch.nn.functional.pad((base.double() * nudge * 2.0 ** e).float(), (0, 32 - len(base))))
    x = torch.stack(rows)
    x = torch.cat([x, -x, x.flip(1)])
    same_bytes(ctx.op_quantize_mxfp4(x.cuda()), x)


def test_quantize_not_finite(ctx):
    x = torch.randn((6, 96), generator=gen(2))
    x[1, 40], x[2, 0], x[3, 95], x[4, 33] = math.nan, math.inf, -math.inf, math.nan
    m = ctx.op_quantize_mxfp4(x.cuda())
    same_bytes(m, x)
    back = ctx.op_dequantize_mxfp4(m, torch.float32).cpu()
    bad = torch.isnan(back)
    assert bad[1, 32:64].all() and bad[2, :32].all() and bad[3, 64:].all() and bad[4, 32:64].all() and bad.sum() == 128


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_strides_and_alignment(ctx, dtype):
    """Rows inside wider ones, from an unaligned column on; transposed input is copied; reading back into such rows leaves the rest alone."""
    wide = torch.randn((40, 300), generator=gen(3)).to(dtype)
    dev = wide.cuda()
    for c0, c1 in ((0, 300), (8, 264), (1, 258), (3, 4), (17, 300)):
        same_bytes(ctx.op_quantize_mxfp4(dev[:, c0:c1]), wide[:, c0:c1])
    same_bytes(ctx.op_quantize_mxfp4(dev[::3, 5:200]), wide[::3, 5:200])
    same_bytes(ctx.op_quantize_mxfp4(dev.t()), wide.t())
    same_bytes(ctx.op_quantize_mxfp4(dev[:1].expand(4, 300)), wide[:1].expand(4, 300))
    m = ctx.op_quantize_mxfp4(dev[:, 1:258])
    out = torch.full((42, 300), 77.0, dtype=dtype, device="cuda")
    ctx.op_dequantize_mxfp4(m, dtype, out=out[1:41, 1:258])
    want = torch.full((42, 300), 77.0, dtype=dtype)
    want[1:41, 1:258] = R.dequantize(m.codes, m.scales, 257).to(dtype)
    assert torch.equal(out.cpu(), want)


def test_rows_of_other_memory_stay(ctx, flux2mi):
    """Nothing is written in front of the first or behind the last row of codes and scales (the C entry, on buffers with a margin)."""
    from flux2mi.api import check, lib
    x = torch.randn((9, 130), generator=gen(4)).cuda()
    codes, scales = torch.full((11, 128), 201, dtype=torch.uint8, device="cuda"), torch.full((11, 8), 202, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    check(lib().flux2mi_op_quantize_mxfp4(ctx.handle, x.data_ptr(), 0, 130, 9, 130, codes[1].data_ptr(), scales[1].data_ptr()))
    ctx.sync()
    want, want_s = R.quantize(x)
    assert np.array_equal(codes[1:10].cpu().numpy(), want) and np.array_equal(scales[1:10].cpu().numpy(), want_s)
    assert (codes[0] == 201).all() and (codes[10] == 201).all() and (scales[0] == 202).all() and (scales[10] == 202).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_read_back_every_scale_and_code(ctx, flux2mi, dtype):
    from flux2mi.api import MXFP4
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).repeat(256, 1)[:, :256].contiguous()     # 512 columns: every byte
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None].repeat(1, 16).contiguous()
    got = ctx.op_dequantize_mxfp4(MXFP4(codes.cuda(), scales.cuda(), 512), dtype).cpu()
    want = R.dequantize(codes, scales, 512)
    if dtype == torch.float16:
        want = want.to(torch.float32).to(dtype)    # exact in float32, one rounding to float16
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.double()[~torch.isnan(want)], want.to(dtype).double()[~torch.isnan(want)])


def test_no_rows(ctx, flux2mi):
    from flux2mi.api import MXFP4
    m = ctx.op_quantize_mxfp4(torch.empty((0, 40), device="cuda"))
    assert m.codes.shape == (0, 64) and m.scales.shape == (0, 4) and ctx.op_dequantize_mxfp4(m).shape == (0, 40)
    w = ctx.op_quantize_mxfp4(torch.randn((5, 40), generator=gen(5)).cuda())
    assert ctx.op_gemm_mxfp4(m, w).shape == (0, 5) and ctx.op_gemm_mxfp4(w, m).shape == (5, 0)
    assert ctx.op_gemm_bf16_mxfp4(torch.empty((0, 40), dtype=torch.bfloat16, device="cuda"), w).shape == (0, 5)


def test_quantize_past_32_bits(ctx):
    """More than 2^31 elements and codes offsets past 2^30: the last rows are where they belong."""
    rows, cols = 263000, 8200
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    at = [0, 1, 131071, 131072, 261123, 261124, rows - 2, rows - 1]
    for i in at:
        x[i] = torch.randn((cols,), generator=gen(6, i)).to(torch.bfloat16)
    m = ctx.op_quantize_mxfp4(x)
    codes, scales = R.quantize(x[at])
    assert np.array_equal(m.codes[at].cpu().numpy(), codes) and np.array_equal(m.scales[at].cpu().numpy(), scales)
    back = ctx.op_dequantize_mxfp4(m, torch.bfloat16, out=x)
    assert torch.equal(back[at].double().cpu(), R.dequantize(codes, scales, cols))


# ------------------------------------------------------------------------------------------------------------ products
def operands(ctx, kind, m, n, k, key=0):
    g = gen(m, n, k, key)
    a, w = torch.randn((m, k), generator=g), torch.randn((n, k), generator=g) * 0.1
    a[:, ::11] *= 12
    if m > 4:
        a[m // 2] = 0
    w4 = ctx.op_quantize_mxfp4(w.cuda())
    w64 = R.dequantize(*R.quantize(w), k)
    if kind == "mxfp4":
        return ctx.op_quantize_mxfp4(a.cuda()), w4, R.dequantize(*R.quantize(a), k), w64
    a = a.bfloat16()
    return a.cuda(), w4, a.double(), w64


def product(ctx, kind, a, w, **more):
    return ctx.op_gemm_mxfp4(a, w, **more) if kind == "mxfp4" else ctx.op_gemm_bf16_mxfp4(a, w, **more)


def near(got, want, bound, dtype):
    assert got.dtype == dtype
    err, allowed = (got.double().cpu() - want).abs(), bound + (want.abs() + bound) * HALF_STEP[dtype]
    assert (err <= allowed).all(), f"off by up to {float((err / allowed.clamp(min=1e-300)).max()):.3g} of what is allowed at {divmod(int((err / allowed.clamp(min=1e-300)).argmax()), got.shape[1])}"


SIZES = [(1, 1, 1), (1, 16, 128), (1, 300, 4100), (2, 17, 33), (3, 65, 129), (5, 130, 640), (16, 64, 256), (17, 48, 257), (31, 257, 96), (33, 100, 1000),
         (64, 128, 384), (65, 129, 260), (127, 300, 200), (128, 256, 512), (130, 64, 1100), (140, 200, 128), (140, 200, 300), (140, 200, 900), (200, 520, 320), (256, 256, 128), (257, 511, 384), (300, 770, 129),
         (513, 1025, 640), (700, 512, 2048), (1, 9731, 200), (1100, 260, 130), (1093, 12113, 388), (4100, 3300, 640),
         (4, 200, 5000), (5, 300, 1000), (13, 17000, 136), (20, 200, 5000), (29, 9000, 264), (40, 300, 1032), (48, 12300, 136), (60, 4100, 264), (66, 9000, 900), (100, 12288, 264), (520, 3900, 520),
         (1030, 4096, 264), (1100, 12288, 392),
         (7, 100, 2), (9, 100, 5), (9, 100, 6), (9, 100, 10), (40, 130, 12), (40, 130, 262), (70, 130, 390), (70, 130, 396), (70, 130, 255), (600, 4096, 1001), (1030, 4096, 258), (1100, 12288, 271)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_product(ctx, kind, m, n, k):
    a, w, a64, w64 = operands(ctx, kind, m, n, k)
    want, bound = R.gemm(a64, w64)
    near(product(ctx, kind, a, w, dtype=torch.float32), want, bound, torch.float32)
    near(product(ctx, kind, a, w), want, bound, torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 33, 200), (19, 130, 260), (140, 264, 512), (530, 300, 384), (600, 516, 640)])
@pytest.mark.parametrize("bias,gate,resid", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)])
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_epilogue(ctx, kind, m, n, k, bias, gate, resid):
    a, w, a64, w64 = operands(ctx, kind, m, n, k)
    g = gen(m, n, 9)
    b = torch.randn((n,), generator=g) if bias else None
    s = torch.randn((n,), generator=g) if gate else None
    x = torch.randn((m, n), generator=g) if resid else None
    want, bound = R.gemm(a64, w64, b, s, x)
    dev = {k_: v.cuda() for k_, v in (("bias", b), ("gate", s), ("resid", x)) if v is not None}
    near(product(ctx, kind, a, w, dtype=torch.float32, **dev), want, bound, torch.float32)
    if resid:
        near(product(ctx, kind, a, w, out=dev["resid"], **dev), want, bound, torch.float32)
        near(dev["resid"], want, bound, torch.float32)
    else:
        near(product(ctx, kind, a, w, **dev), want, bound, torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 4112, 128), (13, 4200, 129), (16, 5003, 2600), (30, 1000, 300), (40, 200, 4200), (100, 5120, 1100), (128, 4096, 700), (33, 12290, 520),
                                   (190, 4100, 2050), (250, 3000, 4480), (64, 64, 16000), (20, 12290, 4098), (90, 4090, 2562), (200, 5000, 1030), (129, 4096, 1412)])
@pytest.mark.parametrize("every", [False, True])
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_product_of_few_rows(ctx, kind, m, n, k, every):
    """Sizes where k is split over groups of waves: steps that do not fill a stage, ragged tiles, each epilogue."""
    a, w, a64, w64 = operands(ctx, kind, m, n, k)
    g = gen(m, n, k, 9)
    bias, gate, resid = (torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn((m, n), generator=g)) if every else (None, None, None)
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    want, bound = R.gemm(a64, w64, bias, gate, resid)
    near(product(ctx, kind, a, w, bias=cuda(bias), gate=cuda(gate), resid=cuda(resid), dtype=torch.float32), want, bound, torch.float32)
    want, bound = R.gemm(a64, w64, bias, gate)
    near(product(ctx, kind, a, w, bias=cuda(bias), gate=cuda(gate)), want, bound, torch.bfloat16)


@pytest.mark.parametrize("n,dtype", [(4100, torch.float32), (4104, torch.bfloat16)])
def test_epilogue_over_both_tile_sizes(ctx, n, dtype):
    """A product whose last columns go to the smaller tiles (18 x 17 large tiles are 1.2 rounds): every operand of the epilogue moves along."""
    m, k = 4500, 260
    a, w, a64, w64 = operands(ctx, "mxfp4", m, n, k)
    g = gen(n)
    b, s = torch.randn((n,), generator=g), torch.randn((n,), generator=g)
    x = torch.randn((m, n), generator=g) if dtype == torch.float32 else None
    want, bound = R.gemm(a64, w64, b, s, x)
    near(ctx.op_gemm_mxfp4(a, w, bias=b.cuda(), gate=s.cuda(), resid=None if x is None else x.cuda(), dtype=dtype), want, bound, dtype)


@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_product_is_not_transposed(ctx, kind):
    """The identity against a matrix of distinct code values: every element where it belongs, exactly."""
    n = 160
    w = ((torch.arange(n * n).view(n, n) * 7) % 15 - 7).clamp(-6, 6).float()
    w = torch.where(w.abs() == 5, torch.full_like(w, 4.0), w)
    eye = torch.eye(n)
    w4 = ctx.op_quantize_mxfp4(w.cuda())
    a = ctx.op_quantize_mxfp4(eye.cuda()) if kind == "mxfp4" else eye.bfloat16().cuda()
    assert torch.equal(product(ctx, kind, a, w4, dtype=torch.float32).cpu(), w.t().contiguous())


@pytest.mark.parametrize("m,n", [(3, 40), (150, 300), (400, 520)])
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_values_that_are_not_finite(ctx, kind, m, n):
    """A NaN of A reaches its own output row, one of W its own column, and nothing else."""
    k = 200
    g = gen(m, n)
    a, w = torch.randn((m, k), generator=g), torch.randn((n, k), generator=g)
    a[1, 77], w[n - 2, 140] = math.nan, math.inf
    w4 = ctx.op_quantize_mxfp4(w.cuda())
    a4 = ctx.op_quantize_mxfp4(a.cuda()) if kind == "mxfp4" else a.bfloat16().cuda()
    bad = torch.isnan(product(ctx, kind, a4, w4, dtype=torch.float32).cpu())
    want = torch.zeros((m, n), dtype=torch.bool)
    want[1], want[:, n - 2] = True, True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
@pytest.mark.parametrize("m,n,k", [(5, 70, 200), (160, 132, 300), (520, 388, 256)])
def test_product_strides(ctx, kind, m, n, k):
    """An output inside wider rows (vector and scalar stores), a residual of another stride, A inside wider rows from an odd column on."""
    a, w, a64, w64 = operands(ctx, kind, m, n, k)
    x = torch.randn((m + 2, n + 9), generator=gen(m))
    want, bound = R.gemm(a64, w64, resid=x[1:-1, 4:4 + n])
    if kind == "bf16":
        wide = torch.full((m, k + 19), 1e30, dtype=torch.bfloat16, device="cuda")
        wide[:, 11:11 + k] = a
        a = wide[:, 11:11 + k]
    for c0 in (0, 4, 5):
        out = torch.full((m + 2, n + 12), 55.0, device="cuda")
        got = product(ctx, kind, a, w, resid=x.cuda()[1:-1, 4:4 + n], out=out[1:-1, c0:c0 + n])
        near(got, want, bound, torch.float32)
        out[1:-1, c0:c0 + n] = 55.0
        assert (out == 55.0).all()
    xd = x.cuda()
    near(product(ctx, kind, a, w, resid=xd[1:-1, 4:4 + n], out=xd[1:-1, 4:4 + n]), want, bound, torch.float32)


def test_bf16_rows_past_their_end_are_not_read_into_the_product(ctx):
    """K that is no multiple of 128: what lies behind a row of A (the next row, NaN here) does not reach the sums."""
    for k in (1, 7, 33, 100, 129, 250):
        a, w, a64, w64 = operands(ctx, "bf16", 37, 50, k)
        wide = torch.full((37, 384), math.nan, dtype=torch.bfloat16, device="cuda")
        wide[:, :k] = a
        want, bound = R.gemm(a64, w64)
        near(ctx.op_gemm_bf16_mxfp4(wide[:, :k], w, dtype=torch.float32), want, bound, torch.float32)


@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_output_past_32_bits(ctx, kind):
    """A row stride that carries the output past 2^32 bytes."""
    m, n, k, ld = 70, 260, 256, 1 << 24
    a, w, a64, w64 = operands(ctx, kind, m, n, k)
    want, bound = R.gemm(a64, w64)
    out = torch.empty(((m - 1) * ld + n,), dtype=torch.float32, device="cuda").as_strided((m, n), (ld, 1))
    near(product(ctx, kind, a, w, dtype=torch.float32, out=out), want, bound, torch.float32)


@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
@pytest.mark.parametrize("m,n", [(1, (1 << 26) + 17), ((1 << 26) + 17, 1), (33000, 33100)])
def test_more_outputs_than_a_launch_holds(ctx, flux2mi, kind, m, n):
    """One column, so that an output is one product, exact in f32."""
    g = torch.Generator("cuda").manual_seed(m)
    a = torch.randint(-6, 7, (m, 1), generator=g, device="cuda").bfloat16()
    w = ctx.op_quantize_mxfp4(torch.randint(1, 7, (n, 1), generator=g, device="cuda").float())
    wv = ctx.op_dequantize_mxfp4(w, torch.float32)
    if kind == "mxfp4":
        a4 = ctx.op_quantize_mxfp4(a)
        av = ctx.op_dequantize_mxfp4(a4, torch.float32)
        out = ctx.op_gemm_mxfp4(a4, w, dtype=torch.float32)
    else:
        av = a.float()
        out = ctx.op_gemm_bf16_mxfp4(a, w, dtype=torch.float32)
    assert torch.equal(out, av * wv[:, 0])


@pytest.mark.parametrize("m,n,k", [(24, 12290, 131), (48, 2560, 261), (164, 1024, 3879), (100, 4100, 519), (300, 4200, 129), (600, 8000, 391)])
def test_rows_of_odd_length(ctx, m, n, k):
    """A in bf16 whose rows start in the middle of a dword, at every tile size."""
    a, w, a64, w64 = operands(ctx, "bf16", m, n, k)
    want, bound = R.gemm(a64, w64)
    near(product(ctx, "bf16", a, w, dtype=torch.float32), want, bound, torch.float32)
    near(product(ctx, "bf16", a, w), want, bound, torch.bfloat16)


def test_column_slices_of_one_buffer(ctx):
    """Operands and results beside each other in the rows of one buffer share no element."""
    m, n, k = 37, 96, 160
    a, w, a64, w64 = operands(ctx, "bf16", m, n, k)
    f = torch.zeros((m, 300), device="cuda")
    f[:, 5:5 + n] = 1.5
    ctx.op_gemm_bf16_mxfp4(a, w, resid=f[:, 5:5 + n], out=f[:, 5 + n:5 + 2 * n])
    want, bound = R.gemm(a64, w64, resid=torch.full((m, n), 1.5))
    near(f[:, 5 + n:5 + 2 * n], want, bound, torch.float32)
    assert (f[:, 5:5 + n] == 1.5).all() and not f[:, :5].any() and not f[:, 5 + 2 * n:].any()
    h = torch.zeros((m, k + n), dtype=torch.bfloat16, device="cuda")
    h[:, n:] = a
    ctx.op_gemm_bf16_mxfp4(h[:, n:], w, out=h[:, :n])
    want, bound = R.gemm(a64, w64)
    near(h[:, :n], want, bound, torch.bfloat16)
    assert torch.equal(h[:, n:], a)


@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_same_result_every_time(ctx, kind):
    for m, n, k in ((1, 500, 3000), (40, 300, 3000), (300, 700, 1000)):
        a, w, _, _ = operands(ctx, kind, m, n, k)
        first = product(ctx, kind, a, w, dtype=torch.float32)
        for _ in range(3):
            assert torch.equal(first, product(ctx, kind, a, w, dtype=torch.float32))


def test_two_products_of_one_context_and_another_stream(ctx, flux2mi):
    """Calls from a side stream of torch, two contexts at once: each in order with its caller's stream."""
    from flux2mi.api import Context
    other = Context(0)
    try:
        side = torch.cuda.Stream()
        a, w, a64, w64 = operands(ctx, "mxfp4", 300, 400, 512)
        want, bound = R.gemm(a64, w64)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            big = torch.randn((4000, 4000), device="cuda") @ torch.randn((4000, 4000), device="cuda")
            x = R.dequantize(*R.quantize(torch.zeros(1, 1)), 1)  # host work beside it
            m = ctx.op_quantize_mxfp4(big)
            first = ctx.op_gemm_mxfp4(a, w, dtype=torch.float32)
        second = other.op_gemm_mxfp4(a, w, dtype=torch.float32)
        torch.cuda.synchronize()
        assert x is not None
        same_bytes(m, big.cpu())
        near(first, want, bound, torch.float32)
        assert torch.equal(first, second)
    finally:
        other.close()


# ------------------------------------------------------------------------------------------------------------ as they are used together
def chain(ctx, x, y, w_in, w_out, gate, pw, nw):
    x1, h = ctx.op_residual_norm(x, y, x_out=torch.empty_like(x), post_norm="rms", post_weight=pw, gate=gate, norm="rms", weight=nw)
    u = ctx.op_gemm_mxfp4(ctx.op_quantize_mxfp4(h), w_in)
    return ctx.op_gemm_bf16_mxfp4(u, w_out, gate=gate, resid=x1), h, u


def chain_inputs(ctx, rows, d, f):
    g = gen(rows, d, f)
    x, y = torch.randn((rows, d), generator=g).cuda(), torch.randn((rows, d), generator=g).bfloat16().cuda()
    w_in = ctx.op_quantize_mxfp4((torch.randn((f, d), generator=g) * 0.05).cuda())
    w_out = ctx.op_quantize_mxfp4((torch.randn((d, f), generator=g) * 0.05).cuda())
    gate = torch.randn((d,), generator=g).cuda()
    pw, nw = (1 + 0.1 * torch.randn((2, d), generator=g)).bfloat16().cuda()
    return x, y, w_in, w_out, gate, pw, nw


@pytest.mark.parametrize("rows", [1, 13, 300])
def test_block_in_four_bits(ctx, rows):
    """residual norm -> quantise -> product -> product with gate and residual, each link against the definition on the link's own input."""
    d, f = 384, 1000
    x, y, w_in, w_out, gate, pw, nw = chain_inputs(ctx, rows, d, f)
    out, h, u = chain(ctx, x, y, w_in, w_out, gate, pw, nw)
    x1, x1_err, h_want, h_err = R.residual_norm(x, y, post_norm="rms", post_weight=pw, gate=gate, norm="rms", weight=nw)
    near(h, h_want, h_err, torch.bfloat16)
    want, bound = R.gemm(R.dequantize(*R.quantize(h), d), R.dequantize(w_in.codes, w_in.scales, d))
    near(u, want, bound, torch.bfloat16)
    want, bound = R.gemm(u, R.dequantize(w_out.codes, w_out.scales, f), gate=gate, resid=x1)
    near(out, want, bound + x1_err, torch.float32)


def test_captured_and_replayed(ctx):
    """The same run in two graphs, replayed in turn with eager work between: every replay equals the eager result of its inputs."""
    graphs = []
    for rows in (3, 290):
        args = chain_inputs(ctx, rows, 384, 1000)
        chain(ctx, *args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(ctx, *args)
        graphs.append((g, args, out))
    for turn in range(3):
        for g, args, out in graphs:
            args[0].copy_(torch.randn(args[0].shape, generator=gen(turn, args[0].shape[0])))
            g.replay()
            torch.cuda.synchronize()
            eager = chain(ctx, *args)
            torch.cuda.synchronize()
            for got, want in zip(out, eager):
                assert torch.equal(got, want)


def test_refused_tensors(ctx, flux2mi):
    """What the Python layer refuses before the C entry."""
    from flux2mi.api import MXFP4
    E = flux2mi.Flux2Error
    x = torch.randn((4, 64)).cuda()
    m = ctx.op_quantize_mxfp4(x)
    w = ctx.op_quantize_mxfp4(torch.randn((8, 96)).cuda())
    for call in (lambda: ctx.op_quantize_mxfp4(x.cpu()), lambda: ctx.op_quantize_mxfp4(x.double()), lambda: ctx.op_quantize_mxfp4(x[0]),
                 lambda: ctx.op_quantize_mxfp4(x[:, :0]), lambda: ctx.op_dequantize_mxfp4(MXFP4(m.codes, m.scales, 200)),
                 lambda: ctx.op_dequantize_mxfp4(MXFP4(m.codes, m.scales[:3], 64)), lambda: ctx.op_dequantize_mxfp4(m, torch.float64),
                 lambda: ctx.op_dequantize_mxfp4(m, torch.float32, out=torch.empty((4, 63), device="cuda")),
                 lambda: ctx.op_dequantize_mxfp4(m, torch.float32, out=torch.empty((64, 4), device="cuda").t()),
                 lambda: ctx.op_gemm_mxfp4(m, w), lambda: ctx.op_gemm_bf16_mxfp4(x, w), lambda: ctx.op_gemm_mxfp4(m, m, dtype=torch.float16),
                 lambda: ctx.op_gemm_mxfp4(m, m, bias=torch.zeros(3).cuda()), lambda: ctx.op_gemm_mxfp4(m, m, gate=torch.zeros(4, dtype=torch.bfloat16).cuda()),
                 lambda: ctx.op_gemm_mxfp4(m, m, resid=torch.zeros((4, 4)).cuda(), dtype=torch.bfloat16),
                 lambda: ctx.op_gemm_mxfp4(m, m, resid=torch.zeros((4, 5)).cuda()),
                 lambda: ctx.op_residual_norm(x.bfloat16()), lambda: ctx.op_residual_norm(x, x[:3]), lambda: ctx.op_residual_norm(x, norm="max"),
                 lambda: ctx.op_residual_norm(x, x.clone(), gate=(torch.zeros(64).cuda(),)), lambda: ctx.op_residual_norm(x, dtype=torch.float16),
                 lambda: ctx.op_residual_norm(x, x), lambda: ctx.op_residual_norm(x.t())):
        with pytest.raises(E):
            call()
