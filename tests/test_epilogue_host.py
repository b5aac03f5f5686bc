"""Refusals of the fused-epilogue products that need no GPU: the builders' checks, and the C entry points'
on made-up addresses (every one of them returns before a launch)."""
import pytest
import torch

from flydsl_amd import _lib
from flydsl_amd.kernels.blockscale_preshuffle_gemm import compile_blockscale_preshuffle_gemm_epilogue
from flydsl_amd.kernels.preshuffle_gemm import compile_preshuffle_gemm_epilogue

A, B, C, S, BIAS, RES = (0x10000000 * i for i in range(1, 7))
M, N, K = 8, 64, 128


def dense(c=C, a=A, b=B, sa=S, sb=S, bias=BIAS, res=RES, n=N, k=K, kind=1, out=0, bias_dtype=2, act=1, variant=-1):
    return _lib.load().flygemm_preshuffle_epilogue(c, a, b, sa, sb, bias, res, M, n, k, kind, out, bias_dtype, act, variant, 0)


@pytest.mark.parametrize("kw,why", [
    (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(bias_dtype=1), "bias"), (dict(out=2), "out_dtype"),
    (dict(c=C + 8), "misaligned"), (dict(bias=BIAS + 4), "misaligned"), (dict(res=RES + 2), "misaligned"),
    (dict(a=A + 4), "misaligned"), (dict(b=B + 8), "misaligned"), (dict(res=C + 16), "overlaps the residual"),
    (dict(res=C - 16), "overlaps the residual"), (dict(bias=C + M * N * 2 - 16), "overlaps"),
    (dict(a=C - 16), "overlaps"), (dict(b=C - N * K + 16), "overlaps"), (dict(kind=5), "in_dtype"), (dict(n=24), "multiple of 16"),
    (dict(k=96), "multiple of 64"), (dict(sa=0), "null scale"), (dict(c=0), "null tensor"), (dict(variant=999), "variant")])
def test_dense_entry_refuses(kw, why):
    assert dense(**kw) != 0
    assert why in _lib.load().flygemm_last_error().decode()


def test_other_entries_refuse():
    lib = _lib.load()
    block = dict(k=K, sbk=128, out=0, bd=2, act=0)
    for kw, why in ((dict(act=9), "activation"), (dict(sbk=64), "scale_block_k"), (dict(k=192), "multiple of"), (dict(bd=1), "bias")):
        v = {**block, **kw}
        assert lib.flygemm_blockscale_epilogue(C, A, B, S, S, BIAS, RES, M, N, v["k"], v["sbk"], v["out"], v["bd"], v["act"], -1, 0)
        assert why in lib.flygemm_last_error().decode()
    mx = dict(n=N, k=256, out=0, bd=2, act=0, res=RES)
    for kw, why in ((dict(act=9), "activation"), (dict(n=48), "multiple of 32"), (dict(k=128), "multiple of 256"),
                    (dict(out=2), "out_dtype"), (dict(res=C + 32), "overlaps the residual")):
        v = {**mx, **kw}
        assert lib.flygemm_mxfp4_epilogue(C, A, B, S, S, BIAS, v["res"], M, v["n"], v["k"], v["out"], v["bd"], v["act"], -1, 0)
        assert why in lib.flygemm_last_error().decode()


def test_builders_refuse():
    kw = dict(K=K, tile_m=64, tile_n=64, tile_k=64, in_dtype="int8", out_dtype="bf16")
    with pytest.raises(ValueError, match="activation"):
        compile_preshuffle_gemm_epilogue(activation="tanh", **kw)
    with pytest.raises(ValueError, match="out_dtype"):
        compile_preshuffle_gemm_epilogue(**{**kw, "out_dtype": "fp32"})
    with pytest.raises(ValueError, match="activation"):
        compile_blockscale_preshuffle_gemm_epilogue(activation="swish", K=K)
    launch = compile_preshuffle_gemm_epilogue(activation="relu", **kw)
    t = torch.zeros(M, N, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        launch(t, t, t, t, t, None, None, M, N)
    with pytest.raises(TypeError, match="stream"):
        launch(t, t, t, t, t, None, None, M, N, "stream")


@pytest.mark.parametrize("kind", ["int8", "fp8_block", "fp4"])
@pytest.mark.parametrize("out", ["bf16", "fp16"])
def test_bound_calls_refuse_types(kind, out):
    """flydsl_amd.compile's call: a bias that is neither fp32 nor the output's type would be read as the output's, and one of
    one-byte elements, or such a residual, past its end."""
    m, n, k = 4, 64, 256
    if kind == "fp8_block":
        launch = compile_blockscale_preshuffle_gemm_epilogue(K=k, out_dtype=out)
    else:
        launch = compile_preshuffle_gemm_epilogue(K=k, tile_m=64, tile_n=64, tile_k=256, in_dtype=kind, out_dtype=out)
    call = launch._bind()
    ot, other = (torch.bfloat16, torch.float16) if out == "bf16" else (torch.float16, torch.bfloat16)
    codes, scales = torch.zeros(n * k, dtype=torch.int8), torch.ones(32 * k)
    c, bias, res = torch.zeros(m, n, dtype=ot), torch.zeros(n), torch.zeros(m, n, dtype=ot)
    for t in (torch.float64, other, torch.int8, torch.int32):
        with pytest.raises(TypeError, match="bias is fp32 or"):
            call(c, codes, codes, scales, scales, bias.to(t), res, m, n)
    for t in (torch.float32, other, torch.uint8):
        with pytest.raises(TypeError, match="residual"):
            call(c, codes, codes, scales, scales, None, res.to(t), m, n)
        with pytest.raises(TypeError, match="residual"):
            call(c, codes, codes, scales, scales, bias.to(ot), res.to(t), m, n)


@pytest.mark.parametrize("kind", ["int8", "fp8_block"])
def test_bound_calls_refuse_layouts(kind):
    """An expanded bias or residual has as many elements as the call needs, but not as much memory."""
    m, n, k = 4, 64, 256
    if kind == "fp8_block":
        launch = compile_blockscale_preshuffle_gemm_epilogue(K=k, out_dtype="bf16")
    else:
        launch = compile_preshuffle_gemm_epilogue(K=k, tile_m=64, tile_n=64, tile_k=256, in_dtype=kind, out_dtype="bf16")
    call = launch._bind()
    codes, scales = torch.zeros(n * k, dtype=torch.int8), torch.ones(n * k)
    c = torch.zeros(m, n, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="contiguous"):
        call(c, codes, codes, scales, scales, torch.zeros(1).expand(n), c, m, n)
    for res in (c[:1].expand(m, n), torch.zeros(n, m, dtype=torch.bfloat16).t()):
        with pytest.raises(ValueError, match="contiguous"):
            call(c, codes, codes, scales, scales, None, res, m, n)
