"""Routing for the MoE 2-stage GEMM: ``moe_topk`` chooses each token's experts from the router's logits,
``moe_balance_loss`` says how evenly they are loaded, and ``moe_sorting`` groups the routes of a top-k
routing by expert and pads each expert's run to the GEMM's row block.

``moe_sorting``: same outputs as the reference harness's ``moe_sorting_torch_native``
(``tests/kernels/test_moe_gemm.py:97-160``), computed without a per-expert loop or a host
synchronisation, so it runs on the device tensors it is given:

* ``sorted_ids`` int32 ``[tokens*topk + E*block - topk]``: per expert in order, its routes in
  row-major order of ``topk_ids`` as ``(slot << 24) | token``, padded to a multiple of ``block``
  with ``(topk << 24) | tokens``;
* ``sorted_weights`` fp32, aligned with ``sorted_ids`` (0 in the padding);
* ``sorted_expert_ids`` int32 ``[ceil(len(sorted_ids) / block)]``: the expert of each block,
  -1 past the last;
* ``num_tokens_post_pad`` int32 ``[2]``: the padded row count and ``tokens``.

With ``expert_mask`` (0/1 per expert), routes to masked experts are dropped and the remaining
experts are renumbered consecutively, as in the reference.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._tensors import on_device, plain_cuda, raw_stream


def _sort_kernel(topk_ids, topk_weights, E, bs, expert_mask):
    """moe_sorting through flygemm_moe_sort (one or two launches, no synchronisation)."""
    dev = topk_ids.device
    M, topk = topk_ids.shape
    max_pad = M * topk + E * bs - topk
    ids = topk_ids if topk_ids.dtype in (torch.int32, torch.int64) else topk_ids.to(torch.int64)
    ids, w = ids.contiguous(), topk_weights.to(torch.float32).contiguous()
    mask = None if expert_mask is None else (expert_mask.reshape(-1)[:E].to(torch.int64) != 0).contiguous()
    sorted_ids = torch.empty(max_pad, dtype=torch.int32, device=dev)
    sorted_w = torch.empty(max_pad, dtype=torch.float32, device=dev)
    sorted_eids = torch.empty((max_pad + bs - 1) // bs, dtype=torch.int32, device=dev)
    post = torch.empty(2, dtype=torch.int32, device=dev)
    lib = _lib.load()
    n = lib.flygemm_moe_sort_scratch(M, topk, E)
    scratch = torch.empty(n, dtype=torch.int32, device=dev) if n else None
    rc = lib.flygemm_moe_sort(sorted_ids.data_ptr(), sorted_w.data_ptr(), sorted_eids.data_ptr(), post.data_ptr(),
                              scratch.data_ptr() if n else None, ids.data_ptr(), w.data_ptr(),
                              None if mask is None else mask.data_ptr(), M, topk, E, bs,
                              int(ids.dtype == torch.int64), torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, "flygemm_moe_sort")
    return sorted_ids, sorted_w, sorted_eids, post


def moe_sorting(topk_ids: torch.Tensor, topk_weights: torch.Tensor, num_experts: int, block_size: int,
                expert_mask: torch.Tensor | None = None):
    if topk_ids.dim() != 2 or topk_weights.shape != topk_ids.shape:
        raise ValueError(f"topk_ids / topk_weights must both be [tokens, topk], got {tuple(topk_ids.shape)} "
                         f"and {tuple(topk_weights.shape)}")
    E, bs = int(num_experts), int(block_size)
    if E <= 0 or bs <= 0:
        raise ValueError(f"num_experts={E} and block_size={bs} must be positive")
    dev = topk_ids.device
    M, topk = topk_ids.shape
    max_pad = M * topk + E * bs - topk
    # On the GPU: the counting-sort kernel (csrc/moe_sort.hip) in place of about 40 operators, two
    # of which (bincount, torch.tensor) wait for the device.  Measured on MI355X, calls back to
    # back: 8 tokens, 256 experts, top-8 16.5 us against 400; 8192 tokens, 128 experts, top-8 21 against 440-460.
    # More experts than the kernel's counters, a top-k above the experts (whose rows may not fit
    # the buffers), empty routings and masks shorter than the experts take the operators below.
    if (0 < topk <= E <= _lib.MOE_SORT_MAX_EXPERTS and M > 0 and max_pad < 2**31 - 2**16
            and (expert_mask is None or expert_mask.numel() >= E)
            and plain_cuda(*(t for t in (topk_ids, topk_weights, expert_mask) if t is not None))):
        with on_device(dev):
            return _sort_kernel(topk_ids, topk_weights, E, bs, expert_mask)
    max_blocks = (max_pad + bs - 1) // bs

    flat = topk_ids.reshape(-1).to(torch.int64)
    route = torch.arange(M * topk, device=dev, dtype=torch.int64)     # t * topk + s
    keep = (flat >= 0) & (flat < E)
    local = torch.arange(E, device=dev, dtype=torch.int64)
    if expert_mask is not None:
        m = expert_mask.to(device=dev).reshape(-1)[:E].to(torch.int64) != 0
        keep = keep & m[flat.clamp(0, E - 1)]
        local = torch.cumsum(m.to(torch.int64), 0) - 1                # renumbered id of kept experts
    key = torch.where(keep, flat, torch.full_like(flat, E))           # dropped routes sort last
    key_sorted, order = torch.sort(key, stable=True)
    counts = torch.bincount(key, minlength=E + 1)[:E]
    padded = (counts + bs - 1) // bs * bs
    start = torch.cumsum(padded, 0) - padded                          # first row of each expert
    first = torch.cumsum(counts, 0) - counts                          # first sorted route of each expert

    n_keep = M * topk  # routes past the kept ones carry key E and are discarded below
    j = torch.arange(n_keep, device=dev, dtype=torch.int64)
    valid = key_sorted < E
    e_of = key_sorted.clamp(max=E - 1)
    dest = torch.where(valid, start[e_of] + (j - first[e_of]), torch.full_like(j, max_pad))

    t = order // topk
    s = order % topk
    sorted_ids = torch.full((max_pad + 1,), (topk << 24) | M, device=dev, dtype=torch.int64)
    sorted_ids[dest] = (s << 24) | t
    sorted_w = torch.zeros(max_pad + 1, device=dev, dtype=torch.float32)
    sorted_w[dest] = topk_weights.reshape(-1).to(torch.float32)[order]

    # expert of each block: blocks [start_e / bs, (start_e + padded_e) / bs) belong to expert e
    blk_end = torch.cumsum(padded // bs, 0)                           # exclusive end block per expert
    b = torch.arange(max_blocks, device=dev, dtype=torch.int64)
    e_blk = torch.searchsorted(blk_end, b, right=True)
    sorted_eids = torch.where(e_blk < E, local[e_blk.clamp(max=E - 1)], torch.full_like(b, -1))

    post = torch.stack([padded.sum(), torch.tensor(M, device=dev, dtype=torch.int64)]).to(torch.int32)
    return sorted_ids[:max_pad].to(torch.int32), sorted_w[:max_pad], sorted_eids.to(torch.int32), post


_LOGITS = {torch.float16: _lib.QUANT_IN["fp16"], torch.bfloat16: _lib.QUANT_IN["bf16"],
           torch.float32: _lib.QUANT_IN["fp32"]}


def _check_logits(logits, scoring):
    """Type, device and size of a router's logits; (T, E)."""
    if type(logits) is not torch.Tensor and type(logits) is not torch.nn.Parameter:
        raise TypeError(f"logits must be a torch.Tensor, got {type(logits).__name__}")
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("torch.jit cannot trace the router's kernels")   # it would record their results as constants
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, experts], got {tuple(logits.shape)}")
    if logits.dtype not in _LOGITS:
        raise TypeError(f"logits dtype {logits.dtype} not supported (fp16, bf16, fp32)")
    if scoring not in _lib.SCORING:
        raise ValueError(f"scoring must be one of {tuple(_lib.SCORING)}, got {scoring!r}")
    T, E = logits.shape
    if not 0 < E <= _lib.MOE_SORT_MAX_EXPERTS:
        raise ValueError(f"{E} experts: the router's kernels take 1 to {_lib.MOE_SORT_MAX_EXPERTS}")
    if T > _lib.MOE_ROUTER_MAX_TOKENS:
        raise ValueError(f"{T} tokens: the router's kernels take at most {_lib.MOE_ROUTER_MAX_TOKENS}")
    if not logits.is_cuda or logits.layout is not torch.strided:
        raise ValueError(f"logits must be a dense GPU tensor, got {logits.layout} on {logits.device}")
    return T, E


def _rows(logits):
    """The logits with their values in memory and consecutive experts next to each other."""
    x = logits.resolve_neg() if logits.is_neg() else logits
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _differentiates(logits) -> bool:
    """Whether a call has to go through autograd (whose forward mode then refuses it)."""
    return logits.requires_grad and torch.is_grad_enabled() or torch.autograd.forward_ad._current_level >= 0


def _check_mask(token_mask, logits):
    if token_mask is None:
        return None
    if not isinstance(token_mask, torch.Tensor) or token_mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError("token_mask must be a bool or uint8 tensor")
    if token_mask.shape != logits.shape[:1] or token_mask.device != logits.device:
        raise ValueError(f"token_mask must be [{logits.shape[0]}] on {logits.device}, got {tuple(token_mask.shape)} "
                         f"on {token_mask.device}")
    return token_mask.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _topk_launch(logits, topk, kinds, bias, mask, groups):
    x = _rows(logits)
    dev = x.device
    (T, E), (scoring, renormalize, scale) = x.shape, kinds
    with on_device(dev):
        ids = torch.empty(T, topk, dtype=torch.int32, device=dev)
        w = torch.empty(T, topk, dtype=torch.float32, device=dev)
        rc = _lib.load().flygemm_moe_topk(ids.data_ptr(), w.data_ptr(), x.data_ptr(), x.stride(0), _ptr(bias), _ptr(mask),
                                          T, E, topk, *groups, _LOGITS[x.dtype], scoring, renormalize, scale,
                                          raw_stream(dev))
        _lib.check(rc, "flygemm_moe_topk")
    return ids, w


class _Topk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, kinds, bias, mask, groups):
        ids, w = _topk_launch(logits, topk, kinds, bias, mask, groups)
        ctx.save_for_backward(logits, ids)
        ctx.kinds = kinds
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, w

    @staticmethod
    @once_differentiable
    def backward(ctx, _, dw):
        if dw is None:
            return (None,) * 6
        logits, ids = ctx.saved_tensors
        x = _rows(logits)
        dev = x.device
        T, E = x.shape
        with on_device(dev):
            dw = (dw.resolve_neg() if dw.is_neg() else dw).contiguous()
            dx = torch.empty(T, E, dtype=x.dtype, device=dev)
            rc = _lib.load().flygemm_moe_topk_grad(dx.data_ptr(), dw.data_ptr(), ids.data_ptr(), x.data_ptr(), x.stride(0),
                                                   T, E, ids.shape[1], _LOGITS[x.dtype], *ctx.kinds,
                                                   raw_stream(dev))
            _lib.check(rc, "flygemm_moe_topk_grad")
        return dx, None, None, None, None, None


def moe_topk(logits: torch.Tensor, topk: int, *, scoring: str = "softmax", correction_bias: torch.Tensor | None = None,
             num_groups: int = 1, topk_groups: int = 1, renormalize: bool = True, route_scale: float = 1.0,
             token_mask: torch.Tensor | None = None):
    """Each token's experts, for :func:`moe_sorting`: ``(topk_ids int32, topk_weights fp32)``, both
    [tokens, topk], from the router's ``logits`` [tokens, experts] (fp32, bf16 or fp16, on the GPU).

    Scores are ``softmax`` over the experts or ``sigmoid``.  The ``topk`` experts with the largest logits are
    chosen, or with ``correction_bias`` ([experts], in fp32) those with the largest score + bias, compared in 64 bits;
    in descending order, the lower index first where they are equal.  With ``num_groups`` > 1 only the
    ``topk_groups`` best groups of consecutive experts take part, a group counting as its largest logit, or
    with a bias as the sum of its two largest scores + bias.  The weights are the chosen experts' scores
    (without the bias), divided by their sum with ``renormalize``, times ``route_scale``.

    Tokens with ``token_mask`` False get ids -1 and weights 0, and their logits are not read; an expert whose
    logit is -inf is never chosen, and a slot that finds no expert gets id -1 and weight 0 too
    (:func:`moe_sorting` drops those).  A NaN logit (or +inf under softmax) makes its row's weights NaN.

    The weights are differentiable with respect to the logits (once); the bias takes part in the choice only
    and has no gradient.  Work is queued on the current stream of the logits' device."""
    T, E = _check_logits(logits, scoring)
    topk, groups = int(topk), (int(num_groups), int(topk_groups))
    if not 1 <= topk <= min(E, 64):
        raise ValueError(f"topk={topk} must be in 1 .. {min(E, 64)}")
    if not 1 <= groups[0] <= 64 or E % groups[0] or not 1 <= groups[1] <= groups[0]:
        raise ValueError(f"num_groups={groups[0]} must divide the {E} experts and be at most 64, topk_groups={groups[1]} "
                         f"at most num_groups")
    if topk > E // groups[0] * groups[1]:
        raise ValueError(f"topk={topk} above the {E // groups[0] * groups[1]} experts of {groups[1]} groups")
    scale = float(route_scale)
    if not math.isfinite(scale):
        raise ValueError(f"route_scale={scale}")
    bias = None
    if correction_bias is not None:
        bias = correction_bias
        if not isinstance(bias, torch.Tensor) or not bias.is_floating_point():
            raise TypeError("correction_bias must be a floating point tensor")
        if bias.shape != (E,) or bias.device != logits.device:
            raise ValueError(f"correction_bias must be [{E}] on {logits.device}, got {tuple(bias.shape)} on {bias.device}")
        if bias.dtype != torch.float32 or bias.requires_grad or bias.is_neg() or not bias.is_contiguous():
            bias = bias.detach().to(torch.float32).resolve_neg().contiguous()
    args = (topk, (_lib.SCORING[scoring], int(bool(renormalize)), scale), bias, _check_mask(token_mask, logits), groups)
    if _differentiates(logits):
        return _Topk.apply(logits, *args)
    return _topk_launch(logits, *args)


def _balance_launch(logits, ids, scoring, mask, cu):
    x = _rows(logits)
    dev = x.device
    (T, E), B = x.shape, 1 if cu is None else cu.numel() - 1
    with on_device(dev):
        if T == 0:
            return (torch.zeros((), dtype=torch.float32, device=dev), torch.zeros(E, dtype=torch.int32, device=dev), None)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        counts = torch.empty(E, dtype=torch.int32, device=dev)
        aux = torch.empty(B * E + 1, dtype=torch.float32, device=dev)
        lib = _lib.load()
        scratch = torch.empty(lib.flygemm_moe_balance_scratch(T, E, B), dtype=torch.uint8, device=dev)
        rc = lib.flygemm_moe_balance(loss.data_ptr(), counts.data_ptr(), aux.data_ptr(), scratch.data_ptr(), x.data_ptr(),
                                     x.stride(0), ids.data_ptr(), _ptr(mask), _ptr(cu), T, E, ids.shape[1], B,
                                     _LOGITS[x.dtype], scoring, int(ids.dtype == torch.int64),
                                     raw_stream(dev))
        _lib.check(rc, "flygemm_moe_balance")
    return loss, counts, aux


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, scoring, mask, cu):
        loss, counts, aux = _balance_launch(logits, ids, scoring, mask, cu)
        ctx.save_for_backward(logits, aux, mask, cu)
        ctx.scoring = scoring
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        if dloss is None:
            return (None,) * 5
        logits, aux, mask, cu = ctx.saved_tensors
        x = _rows(logits)
        dev = x.device
        T, E = x.shape
        with on_device(dev):
            dx = torch.empty(T, E, dtype=x.dtype, device=dev)
            if T:
                dloss = dloss.resolve_neg() if dloss.is_neg() else dloss
                rc = _lib.load().flygemm_moe_balance_grad(dx.data_ptr(), dloss.data_ptr(), aux.data_ptr(), x.data_ptr(),
                                                          x.stride(0), _ptr(mask), _ptr(cu), T, E,
                                                          1 if cu is None else cu.numel() - 1, _LOGITS[x.dtype], ctx.scoring,
                                                          raw_stream(dev))
                _lib.check(rc, "flygemm_moe_balance_grad")
        return dx, None, None, None, None


def moe_balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, *, scoring: str = "softmax",
                     token_mask: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None):
    """How evenly a routing loads the experts: ``(loss fp32 [], counts int32 [experts])`` from the router's
    ``logits`` [tokens, experts] and its choice ``topk_ids`` [tokens, topk] (int32 or int64; ids outside
    [0, experts) count for no expert).

    With ``p`` a token's ``softmax``, or its ``sigmoid`` over their sum, ``n`` the tokens and ``count_e`` the
    routes to expert e: ``f_e = experts * count_e / (topk * n)``, ``P_e = mean_t p_te``, and the loss is
    ``sum_e f_e P_e`` -- 1 for an even load.  With ``cu_seqlens`` ([sequences + 1], int32 or int64,
    non-decreasing within [0, tokens]) it is computed per sequence and averaged over the sequences that have
    tokens.  Tokens before the first and behind the last sequence, with ``token_mask`` False, or without a
    logit above -inf count nowhere and get gradient 0, whatever their logits hold.

    The loss is differentiable with respect to the logits (once; the counts are constants to it).  Sums run
    in a fixed order: the same inputs give the same bits.  Work is queued on the current stream of the
    logits' device."""
    T, E = _check_logits(logits, scoring)
    if not isinstance(topk_ids, torch.Tensor) or topk_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("topk_ids must be an int32 or int64 tensor")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_ids.shape[1] < 1 or topk_ids.device != logits.device:
        raise ValueError(f"topk_ids must be [{T}, topk] on {logits.device}, got {tuple(topk_ids.shape)} on {topk_ids.device}")
    if topk_ids.shape[1] >= 2**31:
        raise ValueError(f"topk_ids has {topk_ids.shape[1]} ids a token, which do not fit 32 bits")
    cu = None
    if cu_seqlens is not None:
        cu = cu_seqlens
        if not isinstance(cu, torch.Tensor) or cu.dtype not in (torch.int32, torch.int64):
            raise TypeError("cu_seqlens must be an int32 or int64 tensor")
        if cu.dim() != 1 or cu.numel() < 2 or cu.device != logits.device:
            raise ValueError(f"cu_seqlens must be [sequences + 1] on {logits.device}, got {tuple(cu.shape)} on {cu.device}")
        if cu.numel() > 2**31:
            raise ValueError(f"cu_seqlens has {cu.numel()} entries: its sequences do not fit 32 bits")
        cu = cu.to(torch.int32).contiguous()
    args = (topk_ids.contiguous(), _lib.SCORING[scoring], _check_mask(token_mask, logits), cu)
    if _differentiates(logits):
        return _Balance.apply(logits, *args)
    return _balance_launch(logits, *args)[:2]
