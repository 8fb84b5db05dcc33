"""CPU: what the Python wrappers of the MXFP4 operators and of the residual norm hand to the C entry points (the entry points themselves are
replaced: tensors in host memory, nothing is launched)."""
import types

import pytest
import torch


class Recorder:
    """In place of the library: keeps the arguments of every call."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def host(flux2mi, monkeypatch):
    """(context on host memory, recorder)"""
    from flux2mi import api
    ctx = api.Context.__new__(api.Context)
    ctx.device, ctx.handle = torch.device("cpu"), 0x1000
    ctx._enter = ctx._exit = lambda: None
    recorder = Recorder()
    monkeypatch.setattr(api, "lib", lambda: recorder)
    return types.SimpleNamespace(ctx=ctx, calls=recorder.calls)


@pytest.mark.parametrize("norm", [None, "none", "rms", "layer"])
def test_residual_norm_without_out(host, norm):
    """want_out=False alone is enough: without `out` there is nothing to normalise, whatever `norm` says (the C entry refuses a norm of a NULL out)."""
    x, y = torch.zeros((3, 64)), torch.zeros((3, 64), dtype=torch.bfloat16)
    kept, none = host.ctx.op_residual_norm(x, y, post_norm="rms", want_out=False, **({} if norm is None else {"norm": norm}))
    (name, args), = host.calls
    p = args[1]._obj
    assert name == "flux2mi_op_residual_norm" and none is None and kept is x
    assert not p.out and p.norm == 0 and p.post_norm == 1 and p.x == p.x_out == x.data_ptr()


@pytest.mark.parametrize("norm,kind", [("none", 0), ("rms", 1), ("layer", 2)])
def test_residual_norm_with_out(host, norm, kind):
    _, out = host.ctx.op_residual_norm(torch.zeros((3, 64)), None, norm=norm)
    p = host.calls[0][1][1]._obj
    assert p.norm == kind and p.out == out.data_ptr() and p.ldo == 64
