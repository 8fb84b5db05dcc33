"""-m gpu: the residual norm (norms behind and in front of a block with its gate and residual scale) against its definition in float64."""
import math

import pytest
import torch

from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def near(got, want, bound, dtype):
    assert got.dtype == dtype
    err, allowed = (got.double().cpu() - want).abs(), bound + (want.abs() + bound) * HALF_STEP[dtype]
    worst = float((err / allowed.clamp(min=1e-300)).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"off by up to {worst:.3g} of what is allowed"


def case(rows, dim, seed=0, y_dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(rows * 100003 + dim + seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, y = r(rows, dim) + 0.3 * r(rows, 1), (r(rows, dim) * 0.7 + 0.2).to(y_dtype)
    pair = lambda spread: (r(dim) * spread, r(dim) * spread)  # noqa: E731
    return x, y, {"gate": pair(0.5), "shift": pair(0.2), "scale": pair(0.2)}, (1 + 0.1 * r(dim)).bfloat16(), (1 + 0.1 * r(dim)).bfloat16()


def dev(v):
    return tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() if isinstance(v, torch.Tensor) else v


def check(ctx, x, y, dtype=torch.bfloat16, **kw):
    xs, xerr, out, oerr = R.residual_norm(x, y, **kw)
    got_x, got = ctx.op_residual_norm(x.cuda(), None if y is None else y.cuda(), x_out=torch.empty(x.shape, device="cuda"), dtype=dtype,
                                      **{k: dev(v) for k, v in kw.items()})
    near(got_x, xs, xerr, torch.float32)
    near(got, out, oerr, dtype)


DIMS = [1, 3, 4, 63, 64, 65, 255, 256, 257, 511, 512, 516, 1000, 1024, 1028, 2047, 2048, 2560, 4096, 4100, 5119, 6144, 8192, 8193, 12000, 16383, 16384]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 7])
def test_every_width(ctx, rows, dim):
    x, y, mod, pw, w = case(rows, dim)
    check(ctx, x, y, split=3, post_norm="rms", post_weight=pw, resid_scale=0.9, norm="layer", weight=w, **mod)
    check(ctx, x, y, split=1, post_norm="layer", norm="rms", dtype=torch.float32, **mod)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("y_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
def test_every_form(ctx, post, norm, y_dtype, dtype):
    for rows, dim in ((5, 300), (130, 1024), (33, 2570)):
        x, y, mod, pw, w = case(rows, dim, y_dtype=y_dtype)
        check(ctx, x, y, dtype, split=rows // 2, post_norm=post, post_weight=pw, resid_scale=1.1, norm=norm, weight=w, **mod)
        check(ctx, x, y, dtype, post_norm=post, norm=norm)
        check(ctx, x, y, dtype, post_norm=post, norm=norm, gate=mod["gate"][0], shift=mod["shift"][1])


def test_without_y(ctx):
    for rows, dim in ((1, 2560), (40, 515), (9, 200)):
        x, _, mod, _, w = case(rows, dim)
        check(ctx, x, None, norm="rms", weight=w)
        check(ctx, x, None, norm="layer", resid_scale=0.5, split=3, scale=mod["scale"], shift=mod["shift"])


@pytest.mark.parametrize("split", [-5, 0, 1, 9, 10, 400])
def test_split(ctx, split):
    x, y, mod, _, _ = case(10, 640)
    check(ctx, x, y, split=split, **mod)


def test_in_place_and_without_out(ctx):
    for dim in (200, 1536, 1537):
        x, y, mod, pw, _ = case(21, dim)
        xs, xerr, out, oerr = R.residual_norm(x, y, post_norm="rms", post_weight=pw, gate=mod["gate"][0])
        xd = x.cuda()
        same, got = ctx.op_residual_norm(xd, y.cuda(), post_norm="rms", post_weight=pw.cuda(), gate=mod["gate"][0].cuda())
        assert same.data_ptr() == xd.data_ptr()
        near(xd, xs, xerr, torch.float32)
        near(got, out, oerr, torch.bfloat16)
        xd = x.cuda()
        _, none = ctx.op_residual_norm(xd, y.cuda(), post_norm="rms", post_weight=pw.cuda(), gate=mod["gate"][0].cuda(), norm="none", want_out=False)
        assert none is None
        near(xd, xs, xerr, torch.float32)


def test_without_out_by_default_norm(ctx):
    """want_out=False with every other argument at its default: x' alone."""
    x, y, _, _, _ = case(9, 640)
    xs, xerr, _, _ = R.residual_norm(x, y)
    xd = x.cuda()
    _, none = ctx.op_residual_norm(xd, y.cuda(), want_out=False)
    assert none is None
    near(xd, xs, xerr, torch.float32)


def test_strides(ctx):
    """x, y and x_out inside wider rows, aligned for vectors and not; what lies beside them stays."""
    for dim, c0, width in ((512, 4, 520), (512, 3, 520), (1029, 1, 1031)):
        x, y, mod, pw, w = case(17, dim)
        kw = dict(split=4, post_norm="layer", post_weight=pw, norm="rms", weight=w, **mod)
        xs, xerr, out, oerr = R.residual_norm(x, y, **kw)
        xw, yw, ow = torch.full((19, width), 3.0).cuda(), torch.full((19, width + 8), 5.0, dtype=torch.bfloat16).cuda(), torch.full((19, width + 4), 7.0).cuda()
        xw[1:-1, c0:c0 + dim], yw[1:-1, c0:c0 + dim] = x.cuda(), y.cuda()
        view = ow[1:-1, c0:c0 + dim]
        _, got = ctx.op_residual_norm(xw[1:-1, c0:c0 + dim], yw[1:-1, c0:c0 + dim], x_out=view, **{k: dev(v) for k, v in kw.items()})
        near(view, xs, xerr, torch.float32)
        near(got, out, oerr, torch.bfloat16)
        view.fill_(7.0)
        assert (ow == 7.0).all()


def test_rows_that_are_zero_constant_or_not_finite(ctx):
    """A row of zeros gives zeros (eps holds the norm), a constant row's LayerNorm is zero, a NaN stays in its row."""
    dim = 1280
    x, y = torch.randn((6, dim), generator=torch.Generator().manual_seed(4)), torch.zeros((6, dim))
    x[1], x[2], x[4, 7] = 0, 3.0, math.nan
    for norm in ("rms", "layer"):
        xs, got = ctx.op_residual_norm(x.cuda(), y.cuda(), x_out=torch.empty((6, dim), device="cuda"), post_norm="rms", norm=norm, dtype=torch.float32)
        got = got.cpu()
        assert (got[1] == 0).all()
        assert torch.isnan(got[4]).all() and torch.isfinite(got[[0, 1, 2, 3, 5]]).all()
        assert torch.equal(torch.isnan(xs.cpu()), torch.isnan(x))
        if norm == "layer":
            assert (got[2] == 0).all()   # 1280 x 3.0 and its mean are exact


def test_no_rows(ctx):
    x, out = ctx.op_residual_norm(torch.empty((0, 64), device="cuda"), torch.empty((0, 64), device="cuda"), post_norm="rms")
    assert x.shape == (0, 64) and out.shape == (0, 64)


def test_many_rows_past_32_bits(ctx):
    """x at offsets past 2^32 bytes."""
    rows, dim, ld = 9, 2048, 1 << 28
    x, y, _, _, w = case(rows, dim)
    big = torch.empty(((rows - 1) * ld + dim,), dtype=torch.float32, device="cuda").as_strided((rows, dim), (ld, 1))
    big.copy_(x)
    xs, xerr, out, oerr = R.residual_norm(x, y, post_norm="rms", weight=w)
    _, got = ctx.op_residual_norm(big, y.cuda(), post_norm="rms", weight=w.cuda())
    near(big, xs, xerr, torch.float32)
    near(got, out, oerr, torch.bfloat16)


@pytest.mark.parametrize("rows,dim", [((1 << 24) - 1, 3), ((1 << 23) + 5, 2049)])
def test_more_rows_than_a_grid_dimension_holds(ctx, rows, dim):
    """Every row is updated once, in place."""
    x = torch.full((rows, dim), 3.0, device="cuda")
    gate = torch.arange(dim, device="cuda").float()
    y = torch.ones((rows, dim), dtype=torch.bfloat16, device="cuda")
    ctx.op_residual_norm(x, y, gate=gate, resid_scale=2.0, norm="none", want_out=False)
    del y
    want = 6.0 + gate
    for at in range(0, rows, 1 << 20):
        assert (x[at:at + (1 << 20)] == want).all(), at
