"""The router's kernels where fp32 cannot tell groups apart, on special values with several rows to a wave, and at sizes
near their limits, against the oracle in 64 bits (oracle/router.py): ids are equal, and weights within the bounds of
test_gpu_router.py."""
import pytest
import torch

from flydsl_amd import moe
from test_gpu_router import DT, U, check_topk, logits, np64, within
from oracle import router as orr

pytestmark = pytest.mark.gpu


# (experts, groups): groups of whole lanes, a power of two of them, are ranked in registers, others through LDS; 8192
# tokens up, or more than 256 experts, several rows to a wave
@pytest.mark.parametrize("T,E,groups", [(300, 256, 8), (300, 60, 4), (8200, 256, 8), (8200, 60, 4), (8200, 6, 3), (300, 512, 16),
                                        (300, 510, 10)])
@pytest.mark.parametrize("size", [1e3, 2.0 ** 17])
def test_groups_whose_two_largest_keys_cancel(gpu, T, E, groups, size):
    """The two largest keys of every other group are +-size and leave errors of an fp32 step of that (6e-5, 2^-7) in its
    score; the other groups' scores are exact to 1e-6.  Any of them may rank first."""
    per = E // groups
    x = logits(T, E, "fp32", gpu, E)
    bias = torch.full((groups, per), -4.0 * size)
    for g in range(groups):
        bias[g, :2] = torch.tensor([size, -size]) if g % 2 == 0 else 0.0
    if per > 2:                                     # not always the first two
        bias = bias.gather(1, torch.rand(groups, per, generator=torch.Generator().manual_seed(E)).argsort(dim=1))
    bias = bias.view(E).to(gpu)
    for topk_groups in (1, 2, groups - 1):
        k = 2 * topk_groups
        for scoring in ("sigmoid", "softmax"):
            check_topk(x, min(k, 16), scoring=scoring, bias=bias, groups=groups, topk_groups=topk_groups, grad=False)


@pytest.mark.parametrize("T", [1, 8200])
def test_a_group_behind_two_that_fp32_orders(gpu, T):
    """Scores .7, .9 and .8: in fp32 the first group's keys 2^24 + .1 and .6 - 2^24 add up to 1, so that it ranks first
    and the second, whose score is sure, last."""
    s = torch.tensor([0.1, 0.6, 0.5, 0.4, 0.45, 0.35], dtype=torch.float64)
    x = torch.log(s / (1 - s)).float().expand(T, 6).contiguous().to(gpu)
    bias = torch.tensor([2.0 ** 24, -2.0 ** 24, 0, 0, 0, 0], device=gpu)
    check_topk(x, 4, scoring="sigmoid", bias=bias, groups=3, topk_groups=2, grad=False)


@pytest.mark.parametrize("T,E", [(40, 16), (8200, 16), (40, 12), (8200, 12), (40, 512)])
def test_group_scores_past_the_largest_float(gpu, T, E):
    """Sums of two keys that are infinite in fp32 and not in 64 bits, on both sides; and biases of +inf."""
    x = logits(T, E, "fp32", gpu, 2)
    per = E // 4
    top = torch.tensor([2.0e38, 2.5e38, 3.0e38, 1.5e38])
    for sign in (1.0, -1.0):
        bias = torch.full((4, per), -3.4e38)
        bias[:, 0], bias[:, 1] = sign * top, sign * top / 1.2
        for topk_groups in (1, 2, 3):
            check_topk(x, 2 * topk_groups, scoring="sigmoid", bias=bias.view(E).to(gpu), groups=4, topk_groups=topk_groups, grad=False)
    bias = torch.zeros(4, per)
    bias[1, 1] = bias[3, 0] = bias[3, 2] = float("inf")
    for topk_groups in (1, 2, 3):
        check_topk(x, 3, scoring="sigmoid", bias=bias.view(E).to(gpu), groups=4, topk_groups=topk_groups, grad=False)


def test_sizes_that_do_not_fit_32_bits_are_refused(gpu):
    """Numbers of ids and of sequences that would reach the kernels without their upper bits (expanded tensors: nothing
    of that size is allocated)."""
    x = torch.zeros(1, 4, device=gpu)
    ids = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="do not fit 32 bits"):
        moe.moe_balance_loss(x, ids.expand(1, 2**32 + 1))
    with pytest.raises(ValueError, match="do not fit 32 bits"):
        moe.moe_balance_loss(x, ids, cu_seqlens=ids[0].expand(2**32 + 2))


def same_rows(t):
    """Whether all rows are equal, without a copy of the whole."""
    return all(bool((part == t[:1]).all()) for part in t.split(1 << 24))


@pytest.mark.parametrize("T,E,k", [(2**26 + 5, 17, 17), (2**28 + 7, 2, 1)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_topk_of_more_workgroups_than_one_dimension_takes(gpu, T, E, k, with_bias):
    """2^32 threads and more, one row to a wave and four: every row of a broadcast one gives what that row gives."""
    x = torch.randn(1, E, generator=torch.Generator().manual_seed(E)).to(gpu)
    bias = torch.zeros(E, device=gpu) if with_bias else None
    leaf = x.expand(T, E).requires_grad_()
    ids, w = moe.moe_topk(leaf, k, scoring="softmax", correction_bias=bias, renormalize=False)
    rid, rw = orr.topk(np64(x), k, "softmax", None, 1, 1, False)
    assert ids[0].tolist() == rid[0].tolist() and same_rows(ids)
    # 2 R + 32 steps of 2^-23, as in test_gpu_router.py, with R < 8
    within(w[:1], rw, 48 * U * rw, "weights")
    assert same_rows(w.detach())
    dw = torch.randn(1, k, generator=torch.Generator().manual_seed(1)).to(gpu)
    (dx,) = torch.autograd.grad(w, leaf, dw.expand(T, k))
    ref = orr.topk_grad(np64(x), rid, np64(dw), "softmax", False)
    within(dx[:1], ref, 64 * U * orr.scores(np64(x)[0], "softmax") * (abs(np64(dw[0, :]))[None].max() * 2) + 1e-37, "gradient")
    assert same_rows(dx)


def test_balance_gradient_of_more_workgroups_than_one_dimension_takes(gpu):
    """2^28 tokens of one row of logits, all of them with expert 0: f = (2, 0), P = p, and every row's gradient
    p (f - f.p) / T."""
    T = 2**28 + 7
    x = torch.tensor([[0.3, -0.4]], device=gpu)
    leaf = x.expand(T, 2).requires_grad_()
    loss, counts = moe.moe_balance_loss(leaf, torch.zeros(1, 1, dtype=torch.int32, device=gpu).expand(T, 1))
    p = torch.softmax(x.double(), dim=1)[0].cpu()
    assert counts.tolist() == [T, 0]
    assert abs(loss.item() - 2 * p[0].item()) <= (2 + 32 + 4096) * U * 2 * p[0].item()
    (dx,) = torch.autograd.grad(loss, leaf)
    h = torch.tensor([2.0, 0.0], dtype=torch.float64) / T
    want = p * (h - (p * h).sum())
    assert ((dx[0].cpu() - want).abs() <= 50 * U * p * 2 * h.max()).all()
    assert same_rows(dx)


def test_balance_of_more_sequences_than_one_dimension_takes(gpu):
    """2^22 sequences, most of them empty, of one token each otherwise: L_b = E p[id] and f = E at the token's expert."""
    T, E, B = 1000, 3, 2**22 + 11
    x = logits(T, E, "fp32", gpu, 1)
    ids = torch.arange(T, device=gpu).remainder(E).to(torch.int32)[:, None]
    cu = (torch.arange(B + 1, device=gpu) * T // B).to(torch.int32)
    leaf = x.clone().requires_grad_()
    loss, counts = moe.moe_balance_loss(leaf, ids, cu_seqlens=cu)
    p = torch.softmax(x.double(), dim=1)
    want = E * p.gather(1, ids.long()).mean()
    assert counts.tolist() == [334, 333, 333]
    assert abs(loss.item() - want.item()) <= (2 * 12 + 33) * U * want.item()
    (dx,) = torch.autograd.grad(loss, leaf)
    h = torch.zeros_like(p).scatter_(1, ids.long(), E / T)
    want = p * (h - (p * h).sum(dim=1, keepdim=True))
    assert ((dx - want).abs() <= (2 * 12 + 48) * U * p * 2 * E / T + 1e-37).all()


def special_rows(T, E, dev):
    """Rows of infinities, NaN and the type's lowest value, ordinary ones between and behind them; a mask."""
    inf, nan = float("inf"), float("nan")
    x = logits(T, E, "fp32", dev, 3)
    low = torch.finfo(torch.float32).min
    x[0] = -inf
    x[1, 3:] = -inf
    x[2, 0] = -inf
    x[3] = low
    x[5, 5:] = low
    x[6, 7] = nan
    x[7] = nan
    x[9, 9] = inf
    x[10] = inf
    x[11, ::2], x[11, 1::2] = inf, -inf
    x[12, 0], x[12, 1], x[12, 2] = nan, inf, -inf
    x[13] *= 1e4
    x[14] -= 500.0                     # sigmoid underflows in fp32
    x[15] += 500.0
    x[17, 3] = -low
    x[18] = -low
    x[19:22] = nan                     # masked
    x[22] = inf
    x[-1, E - 1] = nan                 # of the last wave, which may have rows to spare
    mask = torch.ones(T, dtype=torch.bool, device=dev)
    mask[19:23] = False
    return x, mask


@pytest.mark.parametrize("T,E,k", [(8201, 40, 6), (8201, 40, 16), (8203, 60, 4), (101, 512, 8), (102, 300, 16)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_special_values_with_several_rows_to_a_wave(gpu, T, E, k, scoring):
    x, mask = special_rows(T, E, gpu)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(2)).mul_(0.1).to(gpu)
    special = bias.clone()
    special[4], special[9], special[11] = float("-inf"), float("nan"), float("inf")
    tied = torch.zeros_like(bias)
    for b in (None, bias, special, tied):
        for g, tg in ((1, 1), (5 if E % 5 == 0 else 4, 3)):
            if k <= E // g * tg:
                check_topk(x, k, scoring=scoring, bias=b, groups=g, topk_groups=tg, renorm=b is not bias, mask=mask, grad=b is bias)


@pytest.mark.parametrize("T", [40, 8200])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_subnormal_logits_are_ordered(gpu, T, dtype):
    """Logits that are all below the type's smallest normal number, of both signs, and zeros of both signs among them."""
    fin = torch.finfo(DT[dtype])
    step = fin.smallest_normal * fin.eps
    n = torch.randint(-40, 41, (T, 60), generator=torch.Generator().manual_seed(0)).double()
    x = (n * step).to(DT[dtype]).to(gpu)
    assert x.double().abs().max().item() == 40 * step and x[0].unique().numel() > 20
    x[:, 7] = -0.0
    check_topk(x, 8, grad=False)
    check_topk(x, 8, groups=4, topk_groups=2, scoring="sigmoid", grad=False)
