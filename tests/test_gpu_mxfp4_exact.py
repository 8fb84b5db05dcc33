"""-m gpu: the two products on operands whose sums are exact in float32 (tests/mxfp4_ref.py, exact_operands): float32 results are the definition's
bit for bit, bfloat16 results its one rounding.  Nothing of a sum can be lost, taken twice, scaled by another block's power of two or rounded on
the way without showing.  Sizes are chosen by the kernel that the launch rules send them to, named beside them; the K are long enough for the
steady state of each loop (16 scale bytes a row are 4 steps of 128, a ring's scales 16 steps)."""
import pytest
import torch

from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu


def check(ctx, flux2mi, kind, m, n, k, lda=None, first_column=0):
    """Plain and with the whole epilogue, both output types."""
    from flux2mi.api import MXFP4
    a, w = R.exact_operands(m, n, k, seed=m * 31 + n * 7 + k)
    a64, w64 = R.dequantize(*a, k), R.dequantize(*w, k)
    dev = lambda pair: MXFP4(torch.from_numpy(pair[0]).cuda(), torch.from_numpy(pair[1]).cuda(), k)  # noqa: E731
    w4 = dev(w)
    if kind == "mxfp4":
        a4 = dev(a)
        call = lambda **more: ctx.op_gemm_mxfp4(a4, w4, **more).cpu()  # noqa: E731
    else:
        if lda is None:
            ab = a64.bfloat16().cuda()
        else:   # inside wider rows, NaN around
            ab = torch.full((m * lda + first_column,), float("nan"), dtype=torch.bfloat16, device="cuda").as_strided((m, k), (lda, 1), first_column)
            ab.copy_(a64.bfloat16())
        call = lambda **more: ctx.op_gemm_bf16_mxfp4(ab, w4, **more).cpu()  # noqa: E731
    bias, gate, resid = R.exact_epilogue(m, n, m + n)
    want = R.exact_gemm(a64, w64)
    assert torch.equal(call(dtype=torch.float32).double(), want)
    assert torch.equal(call(dtype=torch.bfloat16), want.float().bfloat16())
    want = (want + bias.double()) * gate.double()
    assert torch.equal(call(bias=bias.cuda(), gate=gate.cuda(), dtype=torch.bfloat16), want.float().bfloat16())
    assert torch.equal(call(bias=bias.cuda(), gate=gate.cuda(), resid=resid.cuda()).double(), want + resid.double())


@pytest.mark.parametrize("m,n", [(1100, 12288), (700, 2500)])   # 256 x 256 tiles, 128 x 128 tiles
@pytest.mark.parametrize("k", [2049, 2200, 2400, 2560])         # 17, 18, 19 and 20 steps: every remainder of a last group of four
def test_mxfp4_tiles_in_their_steady_state(ctx, flux2mi, m, n, k):
    check(ctx, flux2mi, "mxfp4", m, n, k)


@pytest.mark.parametrize("m,n,k", [(4500, 4100, 1700), (4500, 4104, 2047), (4500, 4100, 2300), (4500, 4104, 2420)])   # 14, 16, 18 and 19 steps
def test_mxfp4_columns_split_over_two_launches(ctx, flux2mi, m, n, k):
    """18 x 17 large tiles are 1.2 rounds of 256: 14 columns of them are launched as they are, the others as 128 x 128 tiles, and w, its scales, bias, gate,
    resid and out move along (4104 columns: 16-byte rows of bfloat16 as well).  The first launch alone would cost two rounds, the second alone 2.3."""
    check(ctx, flux2mi, "mxfp4", m, n, k)


@pytest.mark.parametrize("m,n,k", [(7, 4000, 2570), (4, 9000, 3001),                                  # 16-row workgroups
                                   (13, 5003, 6660), (64, 4096, 4226), (40, 2500, 16000),             # 16 x 64 tiles, four k groups
                                   (30, 12290, 4300), (128, 4096, 5000),                              # 32 x 64
                                   (100, 5120, 4400), (250, 3000, 4480), (190, 4100, 2050)])          # 32 x 128
def test_mxfp4_few_rows(ctx, flux2mi, m, n, k):
    check(ctx, flux2mi, "mxfp4", m, n, k)


@pytest.mark.parametrize("m,n,k", [(1, 300, 3000), (5, 300, 4400), (23, 5121, 5120), (48, 2560, 2600), (40, 2500, 16000),   # A whole in LDS; 16 x 32 tiles
                                   (64, 4096, 2100), (100, 4100, 2600),                               # 16 x 64
                                   (30, 12290, 4300), (128, 4096, 2562),                              # 32 x 64
                                   (100, 5120, 4400), (256, 4096, 2560),                              # 32 x 128
                                   (250, 6000, 2600), (512, 4096, 2700),                              # 64 x 128
                                   (300, 12288, 1030), (4500, 4100, 1700),                            # 64 x 256
                                   (600, 8000, 1300), (1100, 12288, 1300),                            # 128 x 256
                                   (48, 2560, 2601), (164, 1024, 3879), (24, 12290, 2049), (24, 5120, 2049),   # rows of odd length: 16 x 32, 16 x 64
                                   (300, 4200, 1029), (700, 2500, 2049), (600, 8000, 1291)])          # 32 x 128, 128 x 256
def test_bf16_tiles(ctx, flux2mi, m, n, k):
    check(ctx, flux2mi, "bf16", m, n, k)


@pytest.mark.parametrize("m,n,k", [(4, 200, 9000), (4, 200, 8192), (4, 200, 8193), (4, 37, 20001), (3, 200, 12001), (3, 200, 10242), (2, 200, 17000), (2, 33, 16385), (1, 40, 33000)])
def test_bf16_rows_in_several_chunks(ctx, flux2mi, m, n, k):
    """Up to 4 rows: 64 KB of A in LDS at a time (8192 k of 4 rows, 10240 of 3, 16384 of 2, 32768 of one), staged anew while W streams on; the rows of
    odd length are staged through shifted dwords."""
    check(ctx, flux2mi, "bf16", m, n, k)


@pytest.mark.parametrize("lda,first_column", [(1 << 24, 0), (1 << 24, 8), ((1 << 24) + 8, 3), ((1 << 24) + 1, 0), ((1 << 24) - 8, 8), ((1 << 24) - 1, 1)])
@pytest.mark.parametrize("m,n,k", [(5, 70, 200), (40, 300, 2300), (33, 130, 1001)])
def test_bf16_rows_far_apart(ctx, flux2mi, m, n, k, lda, first_column):
    """Rows of A 2^24 elements apart leave the 32-bit offsets of the tiles: 16 rows a workgroup, A in 64 KB chunks, whole and from an odd column on; just
    below that stride the tiles take them."""
    check(ctx, flux2mi, "bf16", m, n, k, lda=lda, first_column=first_column)


@pytest.mark.parametrize("k", [(1 << 24) - 2, 1 << 24, (1 << 24) + 130])
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
def test_k_past_the_tiles_offsets(ctx, flux2mi, kind, k):
    """K on both sides of 2^24, more rows than a 16-row workgroup has: operands that are zero but for some columns, the first and the last among them."""
    from flux2mi.api import MXFP4
    m, n = 21, 35
    at = torch.tensor([0, 1, 127, 128, 8191, 8192, 65537, 1 << 20, (1 << 23) + 77, k - 129, k - 2, k - 1])
    g = torch.Generator().manual_seed(k)
    codes = lambda rows: torch.randint(0, 16, (rows, len(at)), generator=g)  # noqa: E731
    ac, wc, p = codes(m), codes(n), R.padded(k)

    def matrix(c):
        q, s = torch.zeros((len(c), p // 2), dtype=torch.uint8, device="cuda"), torch.zeros((len(c), p // 32), dtype=torch.uint8, device="cuda")
        for j, column in enumerate(at.tolist()):
            q[:, column // 2] |= (c[:, j] << (4 * (column & 1))).to(torch.uint8).cuda()
            s[:, column // 32] = 126 + column % 3
        return MXFP4(q, s, k)

    table = torch.from_numpy(R.E2M1)
    value = lambda c: torch.where(c >= 8, -1.0, 1.0) * table[c & 7]  # noqa: E731
    scale = {}   # columns of one block share the last one's
    for column in at.tolist():
        scale[column // 32] = 2.0 ** (column % 3 - 1)
    scale = torch.tensor([scale[column // 32] for column in at.tolist()], dtype=torch.float64)
    a64, w64 = value(ac) * scale, value(wc) * scale
    w4 = matrix(wc)
    if kind == "mxfp4":
        got = ctx.op_gemm_mxfp4(matrix(ac), w4, dtype=torch.float32)
    else:
        a = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
        a[:, at.cuda()] = a64.bfloat16().cuda()
        got = ctx.op_gemm_bf16_mxfp4(a, w4, dtype=torch.float32)
    assert torch.equal(got.double().cpu(), a64 @ w64.t())   # multiples of 2^-4 below 2^14: exact in float32
