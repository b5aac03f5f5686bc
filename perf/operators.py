"""The dense and routing operators of an MoE transformer block, as performance work measures them.

Three operators:

* ``linear``   a product with preshuffled weights whose epilogue adds a bias, applies an activation and adds a
  residual: ``c = T(act((a b^T) scales + bias) + residual)``;
* ``topk``     the router's choice of experts: ids and weights of the ``topk`` best experts of every token, from
  logits [T, E]; with ``grad`` also the logits' gradient;
* ``balance``  the router's balance loss and the experts' counts; with ``grad`` also the logits' gradient.

A case is a dict of plain values.  With ``own`` false, ``run`` computes in elementary torch operations in 32 bits
(64 for the keys of a choice that depends on rounded sums, and for sums over tokens), rounded once at the end;
with ``own`` true it calls the library.
"""
from __future__ import annotations

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
T16 = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a decode step of one sequence through a down projection that ends in the residual stream: all latency
        dict(name="linear_fp8_1", op="linear", kind="fp8", M=1, N=7168, K=2048, out="bf16", act="none", bias=False,
             residual=True),
        # a decode step of 16 sequences through an up projection: streams 235 MB of weights
        dict(name="linear_fp8_16", op="linear", kind="fp8", M=16, N=28672, K=8192, out="bf16", act="silu", bias=False,
             residual=False),
        # 4-bit weights at a large decode batch, the first layer of a feed-forward block with biases
        dict(name="linear_int4_256", op="linear", kind="int4", M=256, N=14336, K=4096, out="fp16", act="gelu_tanh",
             bias=True, residual=False),
        # a prefill chunk through a block-scaled output projection
        dict(name="linear_block_1024", op="linear", kind="fp8_block", M=1024, N=7168, K=7168, out="bf16", act="none",
             bias=False, residual=True),
        # a long prompt in INT8, everything in the epilogue
        dict(name="linear_int8_4096", op="linear", kind="int8", M=4096, N=4096, K=4096, out="bf16", act="relu",
             bias=True, residual=True),
        # an unquantized layer on a ragged batch of prompts: rows and K tiles that fill no tile, the largest product
        dict(name="linear_bf16_5133", op="linear", kind="bf16", M=5133, N=5120, K=8320, out="bf16", act="gelu",
             bias=True, residual=True),
        # a decode step of 8 sequences: grouped sigmoid routing with a correction bias, the smallest call
        dict(name="topk_8", op="topk", T=8, E=256, k=8, dtype="fp32", scoring="sigmoid", bias=True, groups=8,
             topk_groups=4, renorm=True, masked=False, grad=False),
        # a prefill batch, softmax routing of 16-bit logits (many ties), some rows padding
        dict(name="topk_8192", op="topk", T=8192, E=128, k=8, dtype="bf16", scoring="softmax", bias=False, groups=1,
             topk_groups=1, renorm=True, masked=True, grad=False),
        # a training step's tokens on one GPU: choice and gradient
        dict(name="topk_grad_32768", op="topk", T=32768, E=256, k=8, dtype="fp32", scoring="sigmoid", bias=True,
             groups=8, topk_groups=4, renorm=True, masked=False, grad=True),
        # odd sizes: 333 tokens, 17 experts, some of them padding; latency counts
        dict(name="balance_333", op="balance", T=333, E=17, k=9, dtype="fp32", scoring="softmax", sequences=0,
             masked=True, grad=True),
        # ragged sequences packed behind each other, one loss per sequence, rows behind the last one
        dict(name="balance_seq_8192", op="balance", T=8192, E=128, k=8, dtype="bf16", scoring="sigmoid", sequences=13,
             masked=False, grad=True),
        # a training step's tokens on one GPU as one batch
        dict(name="balance_32768", op="balance", T=32768, E=256, k=8, dtype="fp32", scoring="softmax", sequences=0,
             masked=False, grad=True),
    ]


MOST_FLOPS, MOST_BYTES = 2 * 5133 * 5120 * 8320, 7e8
EXPERTS = (8, 16, 17, 32, 60, 64, 72, 96, 128, 160, 256, 384, 512)


def _log(rng, lo, hi, step=1):
    """A multiple of step in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(-(-lo // step) * step, int(v) // step * step)


def draw(rng):
    while True:
        op = rng.choice(["linear", "topk", "balance"])
        if op == "linear":
            kind = rng.choice(["fp8", "int8", "int4", "bf16", "fp16", "mxfp4", "fp8_block"])
            n_step, k_step = {"mxfp4": (32, 256), "fp8": (16, 128), "fp8_block": (16, 128)}.get(kind, (16, 64))
            c = dict(op=op, kind=kind, M=_log(rng, 1, 8192), N=_log(rng, 256, 28672, n_step),
                     K=_log(rng, 256, 8320, k_step), out=rng.choice(["bf16", "bf16", "fp16"]),
                     act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.5,
                     residual=rng.random() < 0.5)
        else:
            E = rng.choice(EXPERTS)
            c = dict(op=op, T=_log(rng, 1, 32768), E=E, k=rng.randint(1, min(E, 10)),
                     dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), scoring=rng.choice(["softmax", "sigmoid"]),
                     masked=rng.random() < 0.4, grad=rng.random() < 0.6)
            if op == "topk":
                groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 2])
                need = -(-c["k"] // (E // groups))
                c.update(bias=rng.random() < 0.5, groups=groups, topk_groups=rng.randint(need, groups),
                         renorm=rng.random() < 0.6)
            else:
                c.update(sequences=rng.choice([0, 0, 1, rng.randint(2, 64)]))
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return c


def work(c):
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        eb = {"bf16": 2, "fp16": 2, "mxfp4": 0.5}
        a, b = M * K * eb.get(c["kind"], 1), N * K * eb.get(c["kind"], 0.5 if c["kind"] == "int4" else 1)
        scales = {"bf16": 0, "fp16": 0, "mxfp4": (M + N) * K // 32, "fp8_block": 4 * (M * K // 128 + -(-N // 128) * K // 128)}
        byt = a + b + scales.get(c["kind"], 4 * (M + N)) + 2 * M * N * (2 if c["residual"] else 1) + (2 * N if c["bias"] else 0)
        return {"bytes": byt, "flops": 2 * M * N * K}
    T, E, k, es = c["T"], c["E"], c["k"], 4 if c["dtype"] == "fp32" else 2
    logits = T * E * es * (2 if c["grad"] else 1)          # read, and the gradient written
    mask = T if c["masked"] else 0
    if c["op"] == "topk":
        return {"bytes": logits + T * k * (12 if c["grad"] else 8) + mask + (4 * E if c["bias"] else 0), "flops": 5 * T * E}
    return {"bytes": logits + 4 * T * k + 4 * E + mask, "flops": 5 * T * E * (2 if c["grad"] else 1)}


# ---- inputs --------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _row_quant(x, dtype, qmax):
    """Symmetric per-row quantization: codes and fp32 scales [rows]."""
    s = x.abs().amax(dim=1, keepdim=True) / qmax
    s = torch.where(s == 0, torch.ones_like(s), s)
    y = x / s
    if dtype == torch.int8:
        y = y.round_().clamp_(-qmax, qmax)
    return y.to(dtype), s.reshape(-1)


def _block_quant(x, br, bc=128):
    """fp8 codes and fp32 scales [ceil(R/br), C/bc] of br x bc blocks."""
    R, C = x.shape
    rp = -(-R // br) * br
    if rp != R:
        x = torch.cat([x, x.new_zeros(rp - R, C)])
    t = x.view(rp // br, br, C // bc, bc)
    s = t.abs().amax(dim=(1, 3), keepdim=True) / 448.0
    s = torch.where(s == 0, torch.ones_like(s), s)
    return (t / s).view(rp, C)[:R].to(FP8), s.view(rp // br, C // bc)


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E2M1_MID = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _mx_quant(x):
    """MXFP4: e2m1 codes [R, C] (uint8) and E8M0 scale bytes [R, C/32]."""
    R, C = x.shape
    b = x.view(R, C // 32, 32)
    e = torch.ceil(torch.log2(b.abs().amax(dim=2).clamp_min(1e-30) / 6.0)).clamp(-126, 126)
    y = b / torch.exp2(e)[:, :, None]
    code = torch.bucketize(y.abs(), torch.tensor(_E2M1_MID, device=x.device)).to(torch.uint8)
    code |= (y < 0).to(torch.uint8) << 3
    return code.view(R, C), (e + 127).to(torch.uint8)


def _linear_inputs(c, seed):
    """Activations of a normalized layer, weights that keep their scale, and what the epilogue adds."""
    g = _gen(seed)
    M, N, K, kind, ot = c["M"], c["N"], c["K"], c["kind"], T16[c["out"]]
    a = torch.randn(M, K, generator=g, device="cuda")
    b = torch.randn(N, K, generator=g, device="cuda").div_(math.sqrt(K))
    sa = sb = None
    if kind in T16:
        a, b = a.to(T16[kind]), b.to(T16[kind])
    elif kind == "fp8_block":
        (a, sa), (b, sb) = _block_quant(a, 1), _block_quant(b, 128)
    elif kind == "mxfp4":
        a, sa = _mx_quant(torch.cat([a, a.new_zeros(-M % 32, K)]))
        b, sb = _mx_quant(b)
    else:
        qt, qa, qb = {"fp8": (FP8, 448.0, 448.0), "int8": (torch.int8, 127.0, 127.0), "int4": (torch.int8, 127.0, 7.0)}[kind]
        (a, sa), (b, sb) = _row_quant(a, qt, qa), _row_quant(b, qt, qb)
    bias = torch.randn(N, generator=g, device="cuda").mul_(0.5).to(ot) if c["bias"] else None
    res = torch.randn(M, N, generator=g, device="cuda").to(ot) if c["residual"] else None
    return dict(a=a, b=b, sa=sa, sb=sb, bias=bias, res=res)


def _router_inputs(c, seed):
    """Logits whose experts differ in popularity; padded rows hold whatever was there (NaN among it)."""
    g = _gen(seed)
    T, E, k = c["T"], c["E"], c["k"]
    x = torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")
    s = dict(x=x.to(T16[c["dtype"]]), mask=None)
    if c["masked"]:
        s["mask"] = torch.rand(T, generator=g, device="cuda") < 0.9
        s["x"][~s["mask"]] = float("nan")
    if c["op"] == "topk":
        s["bias"] = torch.randn(E, generator=g, device="cuda").mul_(0.1) if c["bias"] else None
        s["dw"] = torch.randn(T, k, generator=g, device="cuda")
        return s
    s["ids"] = torch.sort(x.nan_to_num(), dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
    if c["masked"]:
        s["ids"][~s["mask"]] = -1
    s["cu"] = None
    if c["sequences"]:
        # ragged lengths, an empty sequence among them where there are several, and rows behind the last
        cut = torch.sort(torch.randint(0, T + 1, (c["sequences"],), generator=g, device="cuda")).values
        if c["sequences"] > 2:
            cut[1] = cut[0]
        s["cu"] = torch.cat([cut.new_zeros(1), cut]).to(torch.int32)
    return s


def prepare(case, seed):
    c = case
    if c["op"] != "linear":
        s = dict(case=c, **_router_inputs(c, seed))
        if own:
            from flydsl_amd import moe

            s["moe"] = moe
            s["x"].requires_grad_(c["grad"])
        return s
    s = dict(case=c, **_linear_inputs(c, seed))
    if own:
        _linear_plan(s)
    return s


def _linear_plan(s):
    """Weights laid out once, and the pre-bound launcher that a serving loop keeps."""
    import flydsl_amd as fly
    from flydsl_amd import fp4
    from flydsl_amd.kernels.blockscale_preshuffle_gemm import compile_blockscale_preshuffle_gemm_epilogue
    from flydsl_amd.kernels.preshuffle_gemm import compile_preshuffle_gemm_epilogue

    c = s["case"]
    M, N, K, kind, dev = c["M"], c["N"], c["K"], c["kind"], s["a"].device
    sb = s["sb"]
    if kind == "mxfp4":
        s["fp4"] = fp4
        b, sb = fp4.shuffle_weight_w4(fp4.pack_fp4(s["b"])), fp4.shuffle_scale_w4(sb)
    else:
        b = fly.shuffle_weight(s["b"])
        if kind == "int4":
            b = fly.pack_int4(b)
    if s["sa"] is None:
        s["sa"] = sb = torch.empty(0, dtype=torch.float32, device=dev)
    kw = dict(M=M, N=N, K=K, tile_m=64, tile_n=64, out_dtype=c["out"], activation=c["act"])
    if kind == "fp8_block":
        launch = compile_blockscale_preshuffle_gemm_epilogue(tile_k=128, **kw)
    else:
        tile_k = {"mxfp4": 256, "fp8": 128, "bf16": 32, "fp16": 32}.get(kind, 64)
        launch = compile_preshuffle_gemm_epilogue(tile_k=tile_k, in_dtype="fp4" if kind == "mxfp4" else kind, **kw)
    out = torch.empty(M, N, dtype=T16[c["out"]], device=dev)
    s.update(out=out, args=(out, s["a"], b, s["sa"], sb, s["bias"], s["res"], M, N))
    s["launch"] = fly.compile(launch, *_linear_args(s), torch.cuda.current_stream())


def _linear_args(s):
    """The launcher's arguments, the activations laid out as it takes them: MXFP4 codes two to a byte and their scales in
    tiles, block scales K-block major."""
    kind = s["case"]["kind"]
    if kind not in ("mxfp4", "fp8_block"):
        return s["args"]
    out, a, b, sa, *rest = s["args"]
    if kind == "mxfp4":
        return out, s["fp4"].pack_fp4(a)[:rest[-2]], b, s["fp4"].shuffle_scale_w4(sa), *rest
    return out, a, b, sa.t().contiguous(), *rest


# ---- one pass ------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    c = s["case"]
    if c["op"] == "linear":
        s["launch"](*_linear_args(s), torch.cuda.current_stream())
        return s["out"]
    moe = s["moe"]
    if c["op"] == "topk":
        ids, w = moe.moe_topk(s["x"], c["k"], scoring=c["scoring"], correction_bias=s["bias"], num_groups=c["groups"],
                              topk_groups=c["topk_groups"], renormalize=c["renorm"], token_mask=s["mask"])
        if not c["grad"]:
            return ids, w
        return ids, w.detach(), *torch.autograd.grad(w, s["x"], s["dw"])
    loss, counts = moe.moe_balance_loss(s["x"], s["ids"], scoring=c["scoring"], token_mask=s["mask"], cu_seqlens=s["cu"])
    if not c["grad"]:
        return loss, counts
    return loss.detach(), counts, *torch.autograd.grad(loss, s["x"])


def _run_plain(s):
    c = s["case"]
    return {"linear": _plain_linear, "topk": _plain_topk, "balance": _plain_balance}[c["op"]](s, c)


def _mx_value(code, scale, dt):
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=dt, device=code.device)
    R, C = code.shape
    return (table[code.int()].view(R, C // 32, 32) * torch.exp2(scale.to(dt) - 127.0)[:, :, None]).view(R, C)


def _product(s, c, dt):
    """The scaled product, in dt."""
    M, N, K, kind = c["M"], c["N"], c["K"], c["kind"]
    if kind == "mxfp4":
        return _mx_value(s["a"], s["sa"], dt)[:M] @ _mx_value(s["b"], s["sb"], dt).t()
    a, b = s["a"].to(dt), s["b"].to(dt)
    if kind == "fp8_block":
        a = a * s["sa"].to(dt).repeat_interleave(128, dim=1)
        b = b * s["sb"].to(dt).repeat_interleave(128, dim=0)[:N].repeat_interleave(128, dim=1)
        return a @ b.t()
    v = a @ b.t()
    if s["sa"] is not None:
        v = v * s["sa"].to(dt)[:, None] * s["sb"].to(dt)
    return v


def _plain_linear(s, c):
    v = _product(s, c, torch.float32)
    if s["bias"] is not None:
        v = v + s["bias"].float()
    if c["act"] == "relu":
        v = torch.where(v < 0, torch.zeros_like(v), v)
    elif c["act"] == "gelu":
        v = 0.5 * v * torch.erfc(v * -math.sqrt(0.5))
    elif c["act"] == "gelu_tanh":
        v = v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    elif c["act"] == "silu":
        v = v / (1.0 + torch.exp(-v))
    if s["res"] is not None:
        v = v + s["res"].float()
    return v.to(T16[c["out"]])


def _scores(x, scoring):
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _choose(x, s, c):
    """ids [T, k] (-1 where no expert is left) from logits of padding-free rows."""
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    key = x.double()
    if s["bias"] is not None:
        key = _scores(key, c["scoring"]) + s["bias"].double()
    low = torch.full_like(key, -math.inf)
    key = torch.where(x > -math.inf, key, low)
    if G > 1:
        two = torch.sort(key.view(T, G, E // G), dim=2, descending=True).values[:, :, :2]
        score = two[:, :, 0] if s["bias"] is None else two[:, :, 0] + torch.where(
            two[:, :, 1] > -math.inf, two[:, :, 1], torch.zeros_like(two[:, :, 1]))
        order = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :c["topk_groups"]]
        kept = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, order, True)
        key = torch.where(kept[:, :, None].expand(T, G, E // G).reshape(T, E), key, low)
    key, idx = torch.sort(key, dim=1, descending=True, stable=True)
    return torch.where(key[:, :k] > -math.inf, idx[:, :k], torch.full_like(idx[:, :k], -1))


def _plain_topk(s, c):
    x = s["x"].float()
    if s["mask"] is not None:
        x = torch.where(s["mask"][:, None], x, torch.zeros_like(x))
    ids = _choose(x, s, c)
    score = _scores(x, c["scoring"])
    if s["mask"] is not None:
        ids = torch.where(s["mask"][:, None], ids, torch.full_like(ids, -1))
    have = ids >= 0
    at = ids.clamp_min(0)
    q = torch.where(have, score.gather(1, at), torch.zeros_like(score[:, :1]))
    total = q.sum(dim=1, keepdim=True) if c["renorm"] else torch.ones_like(q[:, :1])
    total = torch.where(total > 0, total, torch.ones_like(total))
    w = q / total
    out = (ids.to(torch.int32), w)
    if not c["grad"]:
        return out
    dq = torch.where(have, s["dw"], torch.zeros_like(w))
    if c["renorm"]:
        dq = (dq - (w * dq).sum(dim=1, keepdim=True)) / total
    ds = torch.zeros_like(score).scatter_add_(1, at, torch.where(have, dq, torch.zeros_like(dq)))
    if c["scoring"] == "sigmoid":
        dx = ds * score * (1.0 - score)
    else:
        dx = score * (ds - (score * ds).sum(dim=1, keepdim=True))
    return *out, dx.to(s["x"].dtype)


def _sequence(s, c, dev):
    """The sequence of each row (or one for all), -1 for rows of none, and their number."""
    if s["cu"] is None:
        seq, B = torch.zeros(c["T"], dtype=torch.int64, device=dev), 1
    else:
        B = c["sequences"]
        seq = torch.bucketize(torch.arange(c["T"], device=dev), s["cu"].long(), right=True) - 1
        seq = torch.where(seq < B, seq, torch.full_like(seq, -1))
    if s["mask"] is not None:
        seq = torch.where(s["mask"], seq, torch.full_like(seq, -1))
    return seq, B


def _plain_balance(s, c):
    T, E, k, dev = c["T"], c["E"], c["k"], s["x"].device
    seq, B = _sequence(s, c, dev)
    valid = seq >= 0
    x = torch.where(valid[:, None], s["x"].float(), torch.zeros_like(s["x"], dtype=torch.float32))
    score = _scores(x, c["scoring"])
    p = score / score.sum(dim=1, keepdim=True) if c["scoring"] == "sigmoid" else score
    member = seq[None, :] == torch.arange(B, device=dev)[:, None]
    n = member.sum(dim=1).double()
    if B == 1:
        psum = torch.where(member.view(T, 1), p, torch.zeros_like(p)).sum(dim=0, dtype=torch.float64).view(1, E)
    else:
        psum = member.double() @ p.double()
    row = torch.where(valid[:, None] & (s["ids"] >= 0), seq[:, None] * E + s["ids"], torch.full_like(s["ids"], B * E).long())
    count = torch.zeros(B * E + 1, dtype=torch.int64, device=dev).scatter_add_(0, row.view(-1), torch.ones_like(row).view(-1))
    count = count[:-1].view(B, E)
    some = (n > 0).sum().clamp_min(1)
    n1 = n.clamp_min(1)
    f = count.double() * E / (k * n1)[:, None]
    loss = ((f * psum).sum(dim=1) / n1).sum() / some
    out = (loss.float(), count.sum(dim=0).to(torch.int32))
    if not c["grad"]:
        return out
    h = (f / (n1 * some)[:, None]).float()[seq.clamp_min(0)]
    dx = p * (h - (p * h).sum(dim=1, keepdim=True))
    if c["scoring"] == "sigmoid":
        dx = dx * (1.0 - score)
    return *out, torch.where(valid[:, None], dx, torch.zeros_like(dx)).to(s["x"].dtype)


# ---- the definitions in 64 bits ------------------------------------------------------------
def exact(case, seed):
    c = case
    if c["op"] == "linear":
        return _exact_linear(c, _linear_inputs(c, seed))
    s = _router_inputs(c, seed)
    return (_exact_topk if c["op"] == "topk" else _exact_balance)(c, s)


def _exact_linear(c, s):
    v = _product(s, c, torch.float64)
    if c["bias"]:
        v += s["bias"].double()
    act = c["act"]
    if act == "relu":
        v = v.clamp_min(0.0)
    elif act == "gelu":
        v = v * torch.special.ndtr(v)
    elif act == "gelu_tanh":
        v = v * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * v * (1.0 + 0.044715 * v.square()))
    elif act == "silu":
        v = v * torch.special.expit(v)
    if c["residual"]:
        v += s["res"].double()
    return v


def _exact_topk(c, s):
    E, k, G = c["E"], c["k"], c["groups"]
    x = s["x"].double()
    on = s["mask"][:, None] if s["mask"] is not None else torch.ones_like(x[:, :1], dtype=torch.bool)
    x = x.masked_fill(~on, 0.0)
    score = torch.special.expit(x) if c["scoring"] == "sigmoid" else torch.softmax(x, dim=1)
    key = x if s["bias"] is None else score + s["bias"].double()
    if G > 1:
        per = key.unflatten(1, (G, E // G))
        gs = per.amax(dim=2) if s["bias"] is None else per.topk(2, dim=2).values.sum(dim=2)
        rank = gs.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        key = key.masked_fill((rank >= c["topk_groups"]).repeat_interleave(E // G, dim=1), -math.inf)
    ids = key.argsort(dim=1, descending=True, stable=True)[:, :k]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    out = (ids.masked_fill(~on, -1).to(torch.int32), w.masked_fill(~on, 0.0))
    if not c["grad"]:
        return out
    # the Jacobian's transpose applied to dw
    dw, q = s["dw"].double(), score.gather(1, ids)
    if c["renorm"]:
        dlog = w * (dw - (w * dw).sum(dim=1, keepdim=True))     # with respect to log q
    else:
        dlog = q * dw
    hot = torch.zeros_like(x).scatter_(1, ids, dlog)
    if c["scoring"] == "sigmoid":
        dx = hot * torch.special.expit(-x)                     # d log s / dx
    else:
        dx = hot - score * hot.sum(dim=1, keepdim=True)
    return *out, dx.masked_fill(~on, 0.0)


def _exact_balance(c, s):
    T, E, k = c["T"], c["E"], c["k"]
    x = s["x"].double()
    bounds = [0, T] if s["cu"] is None else s["cu"].tolist()
    on = s["mask"] if s["mask"] is not None else torch.ones(T, dtype=torch.bool, device=x.device)
    total, grad = x.new_zeros(()), torch.zeros_like(x)
    counts = torch.zeros(E, dtype=torch.int64, device=x.device)
    groups = []
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        rows = torch.nonzero(on[lo:hi]).view(-1) + lo
        if len(rows):
            groups.append(rows)
    for rows in groups:
        n, xs, chosen = len(rows), x[rows], s["ids"][rows].long().view(-1)
        cnt = torch.bincount(chosen[chosen >= 0], minlength=E)
        counts += cnt
        score = torch.special.expit(xs)
        p = score / score.sum(dim=1, keepdim=True) if c["scoring"] == "sigmoid" else torch.softmax(xs, dim=1)
        f = cnt.double() * E / (k * n)
        total += (f * p.mean(dim=0)).sum() / len(groups)
        dp = f / (n * len(groups))
        dx = p * (dp - (p @ dp)[:, None])
        grad[rows] = dx * torch.special.expit(-xs) if c["scoring"] == "sigmoid" else dx
    return (total, counts.to(torch.int32)) + ((grad,) if c["grad"] else ())
