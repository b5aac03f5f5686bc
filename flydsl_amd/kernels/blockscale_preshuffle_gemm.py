"""MI355X FP8 blockscale preshuffle GEMM: drop-in for the reference's
``kernels/blockscale_preshuffle_gemm.py``.

The reference snapshot lacks that file; its contract is the call site
``tests/kernels/test_blockscale_preshuffle_gemm.py:173-204`` and the torch oracle
``:86-109`` (the block-scale compute pattern also appears in
``kernels/moe_blockscale_2stage.py:677-777``)::

    exe = compile_blockscale_preshuffle_gemm(M=M, N=N, K=K, tile_m=.., tile_n=.., tile_k=..,
                                             scale_block_k=128, out_dtype="bf16")
    exe(c, x_fp8, b_preshuffled, x_scale_t, w_scale, M, N, stream)

computes ``c[m, n] = sum_kb (sum_{k in kb} x[m,k] w[n,k]) * x_scale[m, kb] * w_scale[n//128, kb]``
with ``x_scale_t`` = ``x_scale.T`` flattened ([K/128, M], K-block major) and ``w_scale``
[ceil(N/128), K/128] row-major.  Per 128-deep K block the kernel forms the fp32 MFMA partial
and folds it into the accumulator with one fused multiply-add by ``sa * sb``.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._launch import check_activation, device_ptr, epilogue_operands, same_device, stream_handle

_OUT_TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}


class BlockscaleGemm:
    def __init__(self, *, K, tile_m, tile_n, tile_k, scale_block_k, out_dtype, variant=-1, **hints):
        self.K = int(K)
        self.tile_m, self.tile_n, self.tile_k = int(tile_m), int(tile_n), int(tile_k)
        self.scale_block_k = int(scale_block_k)
        self.out_dtype = out_dtype
        self.variant = int(variant)
        self.hints = hints

    def __call__(self, arg_c, arg_a, arg_b, arg_scale_a, arg_scale_b, M, N, stream=None):
        h_stream = stream_handle(stream)
        ptrs, M, N = self._operands(arg_c, arg_a, arg_b, arg_scale_a, arg_scale_b, M, N)
        rc = _lib.load().flygemm_blockscale(*ptrs, M, N, self.K, self.scale_block_k,
                                            _lib.FLYGEMM_OUT[self.out_dtype], self.variant, h_stream)
        _lib.check(rc, "flygemm_blockscale")

    def _operands(self, arg_c, arg_a, arg_b, arg_scale_a, arg_scale_b, M, N):
        """Every check of the tensors: their pointers in the C order, and the sizes as ints."""
        M, N, K = int(M), int(N), self.K
        if M < 0 or N <= 0 or N % 16:
            raise ValueError(f"invalid M={M}, N={N} (N must be a positive multiple of 16)")
        sk = K // self.scale_block_k
        sn = (N + 127) // 128
        c = device_ptr(arg_c, "arg_c", M * N, dtypes=(_OUT_TORCH[self.out_dtype],))
        a = device_ptr(arg_a, "arg_a", M * K, elem_bytes=1)
        b = device_ptr(arg_b, "arg_b", N * K, elem_bytes=1)
        sa = device_ptr(arg_scale_a, "arg_scale_a", M * sk, dtypes=(torch.float32,))
        sb = device_ptr(arg_scale_b, "arg_scale_b", sn * sk, dtypes=(torch.float32,))
        return (c, a, b, sa, sb), M, N

    def _bind(self):
        """The launch with only its bounds checks, for ``flydsl_amd.compile`` (as
        ``PreshuffleGemm._bind``)."""
        fn = _lib.load().flygemm_blockscale
        K, sbk, out, var = self.K, self.scale_block_k, _lib.FLYGEMM_OUT[self.out_dtype], self.variant
        sk = K // sbk
        check = _lib.check

        last = [None] * 7

        def call(c, a, b, sa, sb, M, N, stream=None):
            s = 0 if stream is None else (stream if type(stream) is int else stream.cuda_stream)
            if not (c is last[0] and a is last[1] and b is last[2] and sa is last[3] and sb is last[4]
                    and M == last[5] and N == last[6]):
                if (c.numel() < M * N or a.numel() < M * K or b.numel() < N * K or sa.numel() < M * sk
                        or sb.numel() < (N + 127) // 128 * sk):
                    raise ValueError(f"a tensor is too small for M={M}, N={N}, K={K}")
                last[:] = (c, a, b, sa, sb, M, N)
            rc = fn(c.data_ptr(), a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), M, N, K, sbk, out, var, s)
            if rc:
                check(rc, "flygemm_blockscale")
        return call


def compile_blockscale_preshuffle_gemm(*, M: int = 0, N: int = 0, K: int, tile_m: int = 64, tile_n: int = 128,
                                       tile_k: int = 128, scale_block_k: int = 128, out_dtype: str = "bf16",
                                       use_async_copy: bool = False, variant: int = -1):
    if out_dtype not in _OUT_TORCH:
        raise ValueError(f"out_dtype must be 'fp16' or 'bf16', got {out_dtype!r}")
    if int(scale_block_k) != 128:
        raise ValueError(f"scale_block_k must be 128, got {scale_block_k}")
    if int(tile_k) % int(scale_block_k) != 0:
        raise ValueError(f"tile_k={tile_k} must be a multiple of scale_block_k={scale_block_k}")
    if int(K) % int(tile_k) != 0:
        raise ValueError(f"K={K} must be divisible by tile_k={tile_k}")
    if int(tile_m) * int(tile_k) // 256 < 16:
        raise ValueError(f"tile_m*tile_k/256 must be >= 16, got tile {tile_m}x{tile_k}")
    return BlockscaleGemm(K=K, tile_m=tile_m, tile_n=tile_n, tile_k=tile_k, scale_block_k=scale_block_k,
                          out_dtype=out_dtype, variant=variant, M=M, N=N, use_async_copy=use_async_copy)


class BlockscaleGemmEpilogue:
    """Launcher returned by :func:`compile_blockscale_preshuffle_gemm_epilogue`:
    ``(c, x, b_preshuffled, x_scale_t, w_scale, bias, residual, M, N, stream=None)``."""

    def __init__(self, gemm: BlockscaleGemm, activation: str):
        self.gemm = gemm
        self.activation = activation
        self._act = check_activation(activation)

    def __call__(self, arg_c, arg_a, arg_b, arg_scale_a, arg_scale_b, bias, residual, M, N, stream=None):
        g = self.gemm
        h_stream = stream_handle(stream)
        ptrs, M, N = g._operands(arg_c, arg_a, arg_b, arg_scale_a, arg_scale_b, M, N)
        bp, rp, bias_code = epilogue_operands(bias, residual, M, N, _OUT_TORCH[g.out_dtype])
        with same_device(arg_c, stream, arg_a=arg_a, arg_b=arg_b, arg_scale_a=arg_scale_a, arg_scale_b=arg_scale_b,
                         bias=bias, residual=residual):
            rc = _lib.load().flygemm_blockscale_epilogue(*ptrs, bp, rp, M, N, g.K, g.scale_block_k,
                                                         _lib.FLYGEMM_OUT[g.out_dtype], bias_code, self._act, g.variant,
                                                         h_stream)
        _lib.check(rc, "flygemm_blockscale_epilogue")

    def _bind(self):
        """The launch with only its bounds checks, for ``flydsl_amd.compile`` (as ``PreshuffleGemm._bind``), and
        the bias's and residual's types (the bias's chooses how it is read) and layouts (an expanded one has more
        elements than memory)."""
        g, act = self.gemm, self._act
        fn = _lib.load().flygemm_blockscale_epilogue
        K, sbk, out, var = g.K, g.scale_block_k, _lib.FLYGEMM_OUT[g.out_dtype], g.variant
        sk = K // sbk
        check, f32, out_t, code32 = _lib.check, torch.float32, _OUT_TORCH[g.out_dtype], _lib.FLYGEMM_OUT["fp32"]

        def call(c, a, b, sa, sb, bias, res, M, N, stream=None):
            s = 0 if stream is None else (stream if type(stream) is int else stream.cuda_stream)
            if (c.numel() < M * N or a.numel() < M * K or b.numel() < N * K or sa.numel() < M * sk
                    or sb.numel() < (N + 127) // 128 * sk or (bias is not None and bias.numel() < N)
                    or (res is not None and res.numel() < M * N)):
                raise ValueError(f"a tensor is too small for M={M}, N={N}, K={K}")
            if ((bias is not None and bias.dtype is not f32 and bias.dtype is not out_t)
                    or (res is not None and res.dtype is not out_t)):
                raise TypeError(f"bias is fp32 or {out_t}, residual {out_t}: got {bias if bias is None else bias.dtype} "
                                f"and {res if res is None else res.dtype}")
            if (bias is not None and not bias.is_contiguous()) or (res is not None and not res.is_contiguous()):
                raise ValueError("bias and residual must be contiguous")
            rc = fn(c.data_ptr(), a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(),
                    None if bias is None else bias.data_ptr(), None if res is None else res.data_ptr(), M, N, K, sbk, out,
                    code32 if bias is None or bias.dtype is f32 else out, act, var, s)
            if rc:
                check(rc, "flygemm_blockscale_epilogue")
        return call


def compile_blockscale_preshuffle_gemm_epilogue(*, activation: str = "none", **kwargs):
    """The product of :func:`compile_blockscale_preshuffle_gemm` (same arguments) with bias, activation and
    residual in its epilogue; the launcher and its rules are those of
    ``compile_preshuffle_gemm_epilogue``."""
    check_activation(activation)
    return BlockscaleGemmEpilogue(compile_blockscale_preshuffle_gemm(**kwargs), activation)


__all__ = ["compile_blockscale_preshuffle_gemm", "compile_blockscale_preshuffle_gemm_epilogue", "BlockscaleGemm",
           "BlockscaleGemmEpilogue"]
