"""MXFP4 and the residual norm from their definitions, in float64 on the CPU (numpy / torch), one value at a time where that is clearer:
what the kernels are compared with.  Shares no code with the package."""
import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def padded(cols: int) -> int:
    return (cols + 127) // 128 * 128


def quantize(x: torch.Tensor):
    """x [rows, cols] (any float dtype) -> codes u8 [rows, P/2], scales u8 [rows, P/32] as numpy arrays."""
    v = x.detach().cpu().double().numpy()
    rows, cols = v.shape
    full = np.zeros((rows, padded(cols)))
    full[:, :cols] = v
    b = full.reshape(rows, -1, 32)
    finite = np.isfinite(b).all(axis=2)
    b = np.where(finite[..., None], b, 0.0)
    top = np.abs(b).max(axis=2)
    _, e = np.frexp(top)                                   # top = f 2^e, f in [0.5, 1): floor(log2 top) = e - 1
    byte = np.where(top > 0, np.maximum(e - 1 - 2 + 127, 0), 0).astype(np.int64)
    a = np.ldexp(np.abs(b), (127 - byte)[..., None])       # exact in float64 (|x| < 2^128, byte >= 0)
    d = np.abs(np.minimum(a, 6.0)[..., None] - E2M1)       # distance to every value; the first of two equal ones is the lower code
    lo = d.argmin(axis=-1)
    tie = (lo < 7) & (np.take_along_axis(d, lo[..., None], -1)[..., 0] == np.take_along_axis(d, np.minimum(lo + 1, 7)[..., None], -1)[..., 0])
    code = np.where(tie & (lo % 2 == 1), lo + 1, lo)       # ties go to the even code
    code = np.where(np.signbit(b), code + 8, code)
    code = np.where(finite[..., None], code, 0).astype(np.uint8).reshape(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), np.where(finite, byte, 255).astype(np.uint8)


def dequantize(codes, scales, cols: int) -> torch.Tensor:
    """float64 [rows, cols]"""
    codes, scales = (np.asarray(t.cpu()) if isinstance(t, torch.Tensor) else t for t in (codes, scales))
    c = np.empty((codes.shape[0], 2 * codes.shape[1]), np.uint8)
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    v = np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return torch.from_numpy((v.reshape(len(c), -1, 32) * s[..., None]).reshape(len(c), -1)[:, :cols])


def gemm(a: torch.Tensor, w: torch.Tensor, bias=None, gate=None, resid=None):
    """(out, bound): float64 out = resid + gate (a w^T + bias) and how far a float32 evaluation may be off.  The products of code values
    (and of bf16 with a code value) are exact in float32; n additions in any order cost at most n roundings of the running sum each, which
    is <= sum |a w|; 2^-23 covers an adder that truncates.  The epilogue's three operations add one rounding each of what they return."""
    a, w = a.double().cpu(), w.double().cpu()
    d = lambda t: t.double().cpu()  # noqa: E731
    s, mag = a @ w.t(), a.abs() @ w.abs().t()
    bound = mag * (a.shape[1] + 4) * 2.0 ** -23
    if bias is not None:
        s, mag = s + d(bias), mag + d(bias).abs()
    if gate is not None:
        s, mag, bound = s * d(gate), mag * d(gate).abs(), bound * d(gate).abs()
    if resid is not None:
        s, mag = s + d(resid), mag + d(resid).abs()
    return s, bound + 3 * 2.0 ** -24 * mag


def normal(v: torch.Tensor, kind: str, eps: float):
    """(norm(v), spread): float64; spread = mean |v| / sigma, what an error of the mean is worth in normalised units."""
    if kind == "none":
        return v, torch.zeros_like(v[:, :1])
    mu = v.mean(dim=1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    sigma = ((v - mu).square().mean(dim=1, keepdim=True) + eps).sqrt()
    return (v - mu) / sigma, v.abs().mean(dim=1, keepdim=True) / sigma


def by_row(pair, rows, split):
    pair = pair if isinstance(pair, (tuple, list)) else (pair, pair)
    return torch.where((torch.arange(rows) < split)[:, None], pair[0].double().cpu()[None], pair[1].double().cpu()[None])


# A row's sums run over at most 64 registers of a thread, then 6 + 2 halvings over lanes and waves: 72 roundings of partial sums that are at
# most the sum of magnitudes; the square root halves what the sum of squares is off; the remaining operations add a few roundings.
ROUNDINGS = 96


def residual_norm(x, y=None, split=0, post_norm="none", post_weight=None, post_eps=1e-6, gate=None, resid_scale=1.0, norm="rms", weight=None,
                  eps=1e-6, shift=None, scale=None):
    """-> (x', bound of x', out, bound of out), float64; the bounds without the output's own rounding to fewer bits."""
    x = x.double().cpu()
    rows = x.shape[0]
    rs = float(torch.tensor(resid_scale, dtype=torch.float32))   # the scale travels as a float
    u64 = 2.0 ** -24
    xs = rs * x
    if y is not None:
        u, spread = normal(y.double().cpu(), post_norm, float(torch.tensor(post_eps, dtype=torch.float32)))
        f = torch.ones((1, x.shape[1]), dtype=torch.float64)
        if post_weight is not None:
            f = f * post_weight.double().cpu()[None]
        if gate is not None:
            f = f * by_row(gate, rows, split)
        err = u64 * f.abs() * ((ROUNDINGS if post_norm != "none" else 4) * u.abs() + ROUNDINGS * spread * (post_norm == "layer"))
        xs, xerr = xs + f * u, err + 2 * u64 * ((rs * x).abs() + (f * u).abs())
    else:
        xerr = u64 * xs.abs()
    n, spread = normal(xs, norm, float(torch.tensor(eps, dtype=torch.float32)))
    f = torch.ones((1, x.shape[1]), dtype=torch.float64)
    if weight is not None:
        f = f * weight.double().cpu()[None]
    if scale is not None:
        f = f * (1 + by_row(scale, rows, split))
    out = f * n
    if shift is not None:
        out = out + by_row(shift, rows, split)
    # x' is off by xerr: in normalised units that is xerr / sigma for the value itself, and at most its mean over the row for mean and sigma
    if norm == "none":
        per = xerr
    else:
        mu = xs.mean(dim=1, keepdim=True) if norm == "layer" else 0.0
        sigma = ((xs - mu).square().mean(dim=1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))).sqrt()
        rms = xerr.square().mean(dim=1, keepdim=True).sqrt()
        per = (xerr + rms) / sigma + n.abs() * rms / sigma
    oerr = f.abs() * (per + u64 * ((ROUNDINGS if norm != "none" else 4) * n.abs() + ROUNDINGS * spread * (norm == "layer"))) + 4 * u64 * (out.abs() + (f * n).abs())
    return xs, xerr, out, oerr


def exact_operands(m: int, n: int, k: int, seed: int):
    """Operands whose sums are exact in float32 in whatever order they are taken: (a, w), each (codes, scales) as numpy arrays.  Codes are random,
    scales 2^-2 ... 2^1 and different in neighbouring blocks, so every product is a multiple of UNIT = (0.5 x 2^-2)^2 = 2^-6, and a sum of any of
    them is exact while sum |a w| < 2^24 UNIT (24-bit significands)."""
    rng = np.random.default_rng(seed)

    def matrix(rows):
        codes = rng.integers(0, 256, (rows, padded(k) // 2), dtype=np.uint8)
        codes[:, (k + 1) // 2:] = 0
        if k % 2:
            codes[:, k // 2] &= 15
        blocks = padded(k) // 32
        step = rng.integers(1, 4, (rows, blocks))
        step[:, 0] = rng.integers(0, 4, rows)
        scales = (125 + np.cumsum(step, axis=1) % 4).astype(np.uint8)
        scales[:, -(-k // 32):] = 0   # the padding
        return codes, scales

    return matrix(m), matrix(n)


UNIT = 2.0 ** -6


def exact_epilogue(m: int, n: int, seed: int):
    """(bias, gate, resid): multiples of UNIT and powers of two, so that the epilogue is exact as well."""
    g = torch.Generator().manual_seed(seed)
    bias = torch.randint(-4096, 4097, (n,), generator=g) * UNIT
    gate = torch.tensor([0.5, -1.0, 1.0, -0.5])[torch.randint(0, 4, (n,), generator=g)]
    return bias, gate, torch.randint(-4096, 4097, (m, n), generator=g) * UNIT


def exact_gemm(a64: torch.Tensor, w64: torch.Tensor, bias=None, gate=None, resid=None) -> torch.Tensor:
    """float64 resid + gate (a w^T + bias), which is also what float32 gives: sum |a w| <= ||a|| ||w|| (taken itself where that is too wide); bias and
    residual are at most 64 = 4096 UNIT, and a gate of 0.5 halves value and unit alike: (0.5 (sum + 64) + 64) / (UNIT / 2) = (sum + 192) / UNIT < 2^24."""
    fits = lambda top: float(top) + 192 < 2.0 ** 24 * UNIT  # noqa: E731
    assert fits(a64.norm(dim=1).max() * w64.norm(dim=1).max()) or fits((a64.abs() @ w64.abs().t()).max())
    s = a64 @ w64.t()
    if bias is not None:
        s = s + bias.double()
    if gate is not None:
        s = s * gate.double()
    if resid is not None:
        s = s + resid.double()
    assert torch.equal(s.float().double(), s)
    return s
