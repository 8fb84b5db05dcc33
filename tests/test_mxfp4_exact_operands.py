"""CPU: the operands of the exact product tests (tests/test_gpu_mxfp4_exact.py) notice what a wide tolerance would not: each mistake is planted
in the definition here and changes the result, at every size."""
import pytest
import torch

from tests import mxfp4_ref as R


def case(m, n, k):
    a, w = R.exact_operands(m, n, k, seed=m + n + k)
    return a, w, R.dequantize(*a, k), R.dequantize(*w, k)


SIZES = [(1, 64, 200), (5, 40, 1001), (64, 64, 4099), (23, 130, 9000), (64, 64, 16000)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_sums_are_exact_in_float32_in_any_order(m, n, k):
    _, _, a, w = case(m, n, k)
    want = R.exact_gemm(a, w)
    af, wf = a.float(), w.float()
    assert torch.equal((af @ wf.t()).double(), want)
    assert torch.equal((af.flip(1) @ wf.flip(1).t()).double(), want)
    groups = [af[:, at:at + 128] @ wf[:, at:at + 128].t() for at in range(0, k, 128)]
    assert torch.equal(torch.stack(groups[::-1]).cumsum(0)[-1].double(), want)
    bias, gate, resid = R.exact_epilogue(m, n, 3)
    assert torch.equal((resid + gate * (af @ wf.t() + bias)).double(), R.exact_gemm(a, w, bias, gate, resid))


@pytest.mark.parametrize("m,n,k", SIZES)
def test_planted_mistakes_show(m, n, k):
    (ac, asc), (wc, wsc), a, w = case(m, n, k)
    want = R.exact_gemm(a, w)
    a16 = a.bfloat16().double()
    assert torch.equal(a16, a)   # A is bfloat16 as it is
    steps = [a[:, at:at + 128] @ w[:, at:at + 128].t() for at in range(0, k, 128)]
    wrong = {"the sum in bfloat16": want.bfloat16().double(), "the last column lost": a[:, :-1] @ w[:, :-1].t(), "a step lost": want - steps[len(steps) // 2],
             "a step twice": want + steps[-1]}
    for bits, kind in (("bfloat16", torch.bfloat16), ("float16", torch.float16)):
        if k >= 1000:   # (shorter sums of four groups may fit 11 bits)
            wrong[f"four groups' sums in {bits}"] = sum(sum(steps[g::4]).to(kind).double() for g in range(4))
    for name, (c, s), other, first in (("A", (ac, asc), w, True), ("W", (wc, wsc), a, False)):
        for what, moved in (("the next block's", 1), ("the next step's", 4), ("the next group's", 16)):
            blocks = -(-k // 32)
            if blocks <= moved:
                continue
            t = s.copy()
            t[:, blocks - moved - 1] = s[:, blocks - 1]
            v = R.dequantize(c, t, k)
            if not (t == s).all():
                wrong[f"{what} scale in {name}"] = v @ other.t() if first else other @ v.t()
    for name, got in wrong.items():
        assert not torch.equal(got, want), name
