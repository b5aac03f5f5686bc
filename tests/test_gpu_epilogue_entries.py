"""Which C entry points the launchers of the fused epilogue call: a launcher that fell back to the plain product and
torch operations would give the same values."""
import pytest
import torch

import flydsl_amd as fly
from flydsl_amd import _lib
from test_gpu_epilogue import KINDS, OUT, compare, extras, launcher, operands, reference

pytestmark = pytest.mark.gpu


class Counting:
    """The library, with the calls of each entry point counted."""

    def __init__(self, lib):
        self.lib, self.calls = lib, {}

    def __getattr__(self, name):
        entry = getattr(self.lib, name)

        def call(*args):
            self.calls[name] = self.calls.get(name, 0) + 1
            return entry(*args)
        return call


@pytest.mark.parametrize("kind", KINDS)
def test_launchers_call_the_fused_entries(gpu, kind, monkeypatch):
    M, N, K = 19, 96, 256
    lib = Counting(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: lib)
    ops, av, bv = operands(kind, M, N, K, gpu)
    bias, res = extras(M, N, "bf16", gpu)
    want = reference(kind, av, bv, bias, res, "silu", "bf16")
    fn = launcher(kind, K, "bf16", "silu")
    name = {"fp4": "flygemm_mxfp4_epilogue", "fp8_block": "flygemm_blockscale_epilogue"}.get(kind, "flygemm_preshuffle_epilogue")
    lib.calls.clear()
    c = torch.full((M, N), float("nan"), dtype=OUT["bf16"], device=gpu)
    fn(c, *ops, bias, res, M, N, torch.cuda.current_stream())
    assert lib.calls == {name: 1}
    compare(c, *want)
    fast = fly.compile(fn, c, *ops, bias, res, M, N, torch.cuda.current_stream())
    lib.calls.clear()
    c.fill_(float("nan"))
    fast(c, *ops, bias, res, M, N, torch.cuda.current_stream())
    assert lib.calls == {name: 1}
    compare(c, *want)
