"""The microscaled 4-bit operators and the residual norm of flux2mi, as measurable cases: their inputs, their plain form in elementary
torch operations, the calls a user makes of the framework, and their definition in 64 bits.

Microscaled 4-bit floating point (MXFP4): a row is cut into blocks of 32 values; a block keeps one power of two 2^(byte - 127) and 32
codes of the format e2m1, whose values are +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}.  With a = max |x| over the block the exponent is
floor(log2 a) - 2 (at least -127, also for a = 0) and a code is x 2^-exponent rounded to the nearest value, ties to the even code, larger
ones to +-6.  A row's codes are padded with zeros to a multiple of 128 values; two codes lie in a byte, the first in its low half.

Kinds of case
  quantize        x -> blocks, and the blocks read back
  gemm_mxfp4      A W^T of two operands in blocks, with bias, gate and residual
  gemm_bf16_mxfp4 A W^T with A in bfloat16 (weights alone are in 4 bits), the same epilogue
  residual_norm   x' = resid_scale x + gate * norm(y), out = norm(x') * (1 + scale) + shift: the norms behind and in front of a block"""
import contextlib
import math

import torch

own = False
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # hidden states of a 512-token prompt (hidden 2560), on their way into a 4-bit product
        {"name": "quantize-prompt", "op": "quantize", "rows": 512, "cols": 2560, "dtype": "bfloat16"},
        # a whole fused weight (9 x 4096 rows) quantised as it is loaded from a float32 checkpoint
        {"name": "quantize-weight-f32", "op": "quantize", "rows": 36864, "cols": 4096, "dtype": "float32"},
        # the q | k | v projection of 4096 image + 512 text tokens, width 4096: the ordinary large product
        {"name": "mxfp4-qkv-1024px", "op": "gemm_mxfp4", "m": 4608, "n": 12288, "k": 4096, "out": "bfloat16", "bias": False, "gate": False},
        # a block's output projection on a short, ragged prompt, added to the float32 residual stream through its gate
        {"name": "mxfp4-out-ragged", "op": "gemm_mxfp4", "m": 333, "n": 6144, "k": 18432, "out": "float32", "bias": False, "gate": True},
        # one token's hidden state against a 4-bit matrix of odd sizes, with a bias
        {"name": "mxfp4-token-odd", "op": "gemm_mxfp4", "m": 1, "n": 9731, "k": 2590, "out": "float32", "bias": True, "gate": False},
        # the fused attention + MLP input projection at 1024 x 1024 pixels: the largest product
        {"name": "mxfp4-linear1-1024px", "op": "gemm_mxfp4", "m": 4608, "n": 36864, "k": 4096, "out": "bfloat16", "bias": False, "gate": False},
        # one token through the gate | up projection of a language model, weights alone in 4 bits
        {"name": "weight4-token", "op": "gemm_bf16_mxfp4", "m": 1, "n": 19456, "k": 2560, "out": "bfloat16", "bias": False, "gate": False},
        # a padded prompt of 512 tokens through a down projection, weights alone in 4 bits
        {"name": "weight4-prompt", "op": "gemm_bf16_mxfp4", "m": 512, "n": 4096, "k": 12288, "out": "float32", "bias": False, "gate": True},
        # a few sequences at once, ragged
        {"name": "weight4-batch-odd", "op": "gemm_bf16_mxfp4", "m": 23, "n": 5121, "k": 5120, "out": "bfloat16", "bias": True, "gate": False},
        # one token between two blocks: the call that latency decides
        {"name": "norm-token", "op": "residual_norm", "rows": 1, "dim": 2560, "split": 0, "y": "bfloat16", "post": "rms", "gate": False,
         "pre": "rms", "mod": False, "out": "bfloat16"},
        # a double block's text and image rows at 1024 x 1024 pixels, gated and modulated by two sets of vectors
        {"name": "norm-joint-1024px", "op": "residual_norm", "rows": 4608, "dim": 4096, "split": 512, "y": "bfloat16", "post": "rms",
         "gate": True, "pre": "layer", "mod": True, "out": "bfloat16"},
        # an odd width, float32 throughout
        {"name": "norm-odd-f32", "op": "residual_norm", "rows": 1031, "dim": 5119, "split": 77, "y": "float32", "post": "none", "gate": True,
         "pre": "rms", "mod": True, "out": "float32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _odd(rng, v, step):
    """Half of the sizes on a multiple of `step`, half wherever they fell."""
    return max(step, v // step * step) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["quantize", "gemm_mxfp4", "gemm_mxfp4", "gemm_bf16_mxfp4", "gemm_bf16_mxfp4", "residual_norm"])
    if op == "quantize":
        cols = _odd(rng, _log(rng, 33, 20000), 128)
        return {"op": op, "rows": _log(rng, 1, min(40000, 140_000_000 // cols)), "cols": cols, "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    if op == "residual_norm":
        dim = _odd(rng, _log(rng, 65, 12000), 64)
        rows = _log(rng, 1, min(20000, 40_000_000 // dim))
        return {"op": op, "rows": rows, "dim": dim, "split": rng.randint(0, rows), "y": rng.choice(["bfloat16", "float32"]),
                "post": rng.choice(["none", "rms", "layer"]), "gate": rng.random() < 0.5, "pre": rng.choice(["rms", "layer"]),
                "mod": rng.random() < 0.5, "out": rng.choice(["bfloat16", "float32"])}
    while True:
        n, k = _odd(rng, _log(rng, 300, 40000), 256), _odd(rng, _log(rng, 100, 20000), 128)
        m = _log(rng, 1, 5000 if op == "gemm_mxfp4" else 2500)
        if m * n * k <= 4608 * 36864 * 4096 and n * k <= 160_000_000:
            break
    gate = rng.random() < 0.4
    return {"op": op, "m": m, "n": n, "k": k, "out": "float32" if gate else rng.choice(["bfloat16", "float32"]), "bias": rng.random() < 0.4, "gate": gate}


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _activations(g, rows, cols):
    """Hidden states: normal values, a few channels many times larger, a share of rows that are padding (zeros)."""
    x = torch.randn((rows, cols), generator=g, device=DEV)
    x.mul_(torch.where(torch.rand((1, cols), generator=g, device=DEV) < 0.005, 20.0, 1.0))
    if rows > 8:
        x.mul_((torch.rand((rows, 1), generator=g, device=DEV) > 0.02).float())
    return x


def _pad128(n):
    return (n + 127) // 128 * 128


def _blocks(x):
    """float32 [rows, cols] -> (exponents int32 [rows, blocks], x 2^-exponent [rows, blocks, 32]), the columns padded with zeros."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, _pad128(cols) - cols)).view(rows, -1, 32)
    top = b.abs().amax(dim=2)
    _, e = torch.frexp(top)  # top = f 2^e, f in [0.5, 1): floor(log2 top) = e - 1
    e = torch.where(top > 0, e - 3, torch.full_like(e, -127)).clamp_(min=-127)
    return e, torch.ldexp(b, -e.unsqueeze(2))


def _nearest(v):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |v| as a code 0..7; a tie goes to the even code."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8)
    for at, ties_up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= at) if ties_up else (a > at)
    return c


def _values(codes):
    """e2m1 codes 0..15 -> float32"""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return table[codes.long()]


def _quantize(x):
    """-> packed codes u8 [rows, pad128(cols) / 2], scale bytes u8 [rows, pad128(cols) / 32]"""
    e, v = _blocks(x)
    c = (_nearest(v) + (torch.signbit(v).to(torch.uint8) << 3)).view(x.shape[0], -1)
    return c[:, 0::2] | (c[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _read_back(codes, scales, cols):
    """float32 [rows, cols]"""
    rows = codes.shape[0]
    c = torch.stack((codes & 15, codes >> 4), dim=2).view(rows, -1, 32)
    return torch.ldexp(_values(c), scales.int().unsqueeze(2) - 127).view(rows, -1)[:, :cols]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "quantize":
        x = _activations(g, case["rows"], case["cols"]) if case["dtype"] != "float32" else torch.randn((case["rows"], case["cols"]), generator=g, device=DEV) * 0.02
        s["x"] = x.to(getattr(torch, case["dtype"]))
    elif op == "residual_norm":
        r, d = case["rows"], case["dim"]
        s["x"] = _activations(g, r, d) + torch.randn((r, 1), generator=g, device=DEV) * 0.1
        s["y"] = (torch.randn((r, d), generator=g, device=DEV) * 0.7).to(getattr(torch, case["y"]))
        vec = lambda spread: torch.randn((d,), generator=g, device=DEV) * spread  # noqa: E731
        s["post_weight"] = (1 + vec(0.1)).bfloat16() if case["post"] != "none" else None
        s["weight"] = (1 + vec(0.1)).bfloat16() if case["pre"] == "rms" else None
        s["gate"] = (vec(0.5), vec(0.5)) if case["gate"] else None
        s["shift"], s["scale"] = ((vec(0.2), vec(0.2)), (vec(0.2), vec(0.2))) if case["mod"] else (None, None)
        s["resid_scale"] = 0.9
    else:
        m, n, k = case["m"], case["n"], case["k"]
        a = _activations(g, m, k).bfloat16()
        if op == "gemm_mxfp4":
            s["a"], s["a_scale"] = _quantize(a.float())
        else:
            s["a"] = a
        w = (torch.randn((n, k), generator=g, device=DEV) * (1 / math.sqrt(k))).bfloat16()
        s["w"], s["w_scale"] = _quantize(w.float())
        s["bias"] = torch.randn((n,), generator=g, device=DEV) * 0.3 if case["bias"] else None
        s["gate"] = torch.randn((n,), generator=g, device=DEV) * 0.5 if case["gate"] else None
        s["resid"] = torch.randn((m, n), generator=g, device=DEV) if case["gate"] else None
    return s


# ---------------------------------------------------------------------------------------------------------- a user's calls
_context = None


def _own_context():
    """The framework's context (one GPU, one stream), made at its first use as a program makes it at its start."""
    global _context
    if _context is None:
        from flux2mi.api import Context
        _context = Context(0)
    return _context


def _run_own(s):
    ctx = _own_context()
    with torch.cuda.stream(ctx.stream):  # as a program that works on the framework's stream
        return _calls(ctx, s["case"], s)


def _calls(ctx, c, s):
    from flux2mi.api import MXFP4
    if c["op"] == "quantize":
        q = ctx.op_quantize_mxfp4(s["x"])
        return {"values": ctx.op_dequantize_mxfp4(q, dtype=s["x"].dtype), "scales": q.scales}
    if c["op"] == "residual_norm":
        x, out = ctx.op_residual_norm(s["x"], s["y"], x_out=torch.empty_like(s["x"]), split=c["split"], post_norm=c["post"],
                                      post_weight=s["post_weight"], gate=s["gate"], resid_scale=s["resid_scale"], norm=c["pre"],
                                      weight=s["weight"], shift=s["shift"], scale=s["scale"], dtype=getattr(torch, c["out"]))
        return {"x": x, "out": out}
    w = MXFP4(s["w"], s["w_scale"], c["k"])
    more = {"bias": s["bias"], "gate": s["gate"], "resid": s["resid"], "dtype": getattr(torch, c["out"])}
    if c["op"] == "gemm_mxfp4":
        return ctx.op_gemm_mxfp4(MXFP4(s["a"], s["a_scale"], c["k"]), w, **more)
    return ctx.op_gemm_bf16_mxfp4(s["a"], w, **more)


# ------------------------------------------------------------------------------------------------------------- plain form
@contextlib.contextmanager
def _full_float32():
    """Products in float32 as float32: no shortened operands."""
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        yield
    finally:
        torch.backends.cuda.matmul.allow_tf32 = before


EPS = 1e-6


def _norm(v, kind):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    return v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS)


def _by_row(pair, rows, split):
    """Two vectors -> one row each: the first for rows below `split`."""
    first = torch.arange(rows, device=pair[0].device).unsqueeze(1) < split
    return torch.where(first, pair[0].unsqueeze(0), pair[1].unsqueeze(0))


def _plain_norm(s):
    c = s["case"]
    r, split = c["rows"], c["split"]
    u = _norm(s["y"].float(), c["post"])
    if s["post_weight"] is not None:
        u = u * s["post_weight"].float()
    if s["gate"] is not None:
        u = u * _by_row(s["gate"], r, split)
    x = s["resid_scale"] * s["x"] + u
    out = _norm(x, c["pre"])
    if s["weight"] is not None:
        out = out * s["weight"].float()
    if s["scale"] is not None:
        out = out * (1 + _by_row(s["scale"], r, split)) + _by_row(s["shift"], r, split)
    return {"x": x, "out": out.to(getattr(torch, c["out"]))}


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "quantize":
        codes, scales = _quantize(s["x"].float())
        return {"values": _read_back(codes, scales, c["cols"]).to(s["x"].dtype), "scales": scales}
    if c["op"] == "residual_norm":
        return _plain_norm(s)
    a = _read_back(s["a"], s["a_scale"], c["k"]) if c["op"] == "gemm_mxfp4" else s["a"].float()
    with _full_float32():
        out = a @ _read_back(s["w"], s["w_scale"], c["k"]).t()
    if s["bias"] is not None:
        out = out + s["bias"]
    if s["gate"] is not None:
        out = s["resid"] + s["gate"] * out
    return out.to(getattr(torch, c["out"]))


# ------------------------------------------------------------------------------------------------------------------- work
def _mx_bytes(rows, cols):
    return rows * _pad128(cols) * 17 / 32  # 16 bytes of codes and one of scale for 32 values


def work(case):
    size = {"bfloat16": 2, "float16": 2, "float32": 4}
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        # written in blocks, read back from them
        return {"bytes": 2 * n * size[case["dtype"]] + 2 * _mx_bytes(case["rows"], case["cols"]), "flops": 0}
    if case["op"] == "residual_norm":
        return {"bytes": case["rows"] * case["dim"] * (8 + size[case["y"]] + size[case["out"]]), "flops": 0}
    m, n, k = case["m"], case["n"], case["k"]
    a = _mx_bytes(m, k) if case["op"] == "gemm_mxfp4" else 2 * m * k
    out = m * n * (size[case["out"]] + (4 if case["gate"] else 0))
    return {"bytes": a + _mx_bytes(n, k) + out + 4 * n * (case["bias"] + case["gate"]), "flops": 2.0 * m * n * k}


# --------------------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_blocks(codes, scales, cols):
    """sign (-1)^s, a 2-bit exponent f and one fraction bit t: (2 + t) 2^(f - 2) for f > 0 and t / 2 for f = 0, times 2^(byte - 127)"""
    rows, half = codes.shape
    c = torch.empty((rows, 2 * half), dtype=torch.int16, device=codes.device)
    c[:, 0::2], c[:, 1::2] = (codes % 16).short(), (codes // 16).short()
    f, t = (c // 2) % 4, c % 2
    v = torch.where(f > 0, (2 + t).double() * torch.exp2(f.double() - 2), t.double() / 2)
    v *= 1 - 2 * (c // 8).double()
    v *= torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)
    return v[:, :cols]


def _exact_quantize(x):
    rows, cols = x.shape
    v = torch.zeros((rows, _pad128(cols)), dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, -1, 32)
    top = v.abs().amax(dim=2, keepdim=True)
    # floor(log2 top), exact at powers of two
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)))
    e = e - (torch.exp2(e) > top).double() + (torch.exp2(e + 1) <= top).double()
    unit = torch.exp2(torch.where(top > 0, (e - 2).clamp(min=-127), torch.full_like(e, -127)))
    a = v.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    a = (torch.round(a / step) * step).clamp(max=6)  # round() sends ties to the even multiple
    return (torch.copysign(a, v) * unit).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        parts = [_exact_quantize(p.double()) for p in s["x"].split(max(1, 50_000_000 // case["cols"]))]
        return {"values": torch.cat(parts), "scales": None}
    if case["op"] == "residual_norm":
        d = case["dim"]
        which = (torch.arange(case["rows"], device=DEV) >= case["split"]).long()
        y, x = s["y"].double(), s["x"].double()

        def normal(v, kind):
            if kind == "none":
                return v
            mu = v.sum(dim=1, keepdim=True) / d if kind == "layer" else 0.0
            return (v - mu) / ((v - mu).pow(2).sum(dim=1, keepdim=True) / d + EPS).sqrt()

        u = normal(y, case["post"])
        u = u if s["post_weight"] is None else u * s["post_weight"].double()
        u = u if s["gate"] is None else u * torch.stack(s["gate"]).double()[which]
        x = s["resid_scale"] * x + u
        o = normal(x, case["pre"])
        o = o if s["weight"] is None else o * s["weight"].double()
        o = o if s["scale"] is None else o * (1 + torch.stack(s["scale"]).double()[which]) + torch.stack(s["shift"]).double()[which]
        return {"x": x, "out": o}
    a = _exact_blocks(s["a"], s["a_scale"], case["k"]) if case["op"] == "gemm_mxfp4" else s["a"].double()
    out = torch.empty((case["m"], case["n"]), dtype=torch.float64, device=DEV)
    at = 0
    for w, ws in zip(s["w"].split(4096), s["w_scale"].split(4096)):
        out[:, at:at + w.shape[0]] = a @ _exact_blocks(w, ws, case["k"]).t().contiguous()
        at += w.shape[0]
    out = out if s["bias"] is None else out + s["bias"].double()
    return out if s["gate"] is None else s["resid"].double() + s["gate"].double() * out
