"""Refusals of the router that need no GPU: the C entry points' on made-up addresses (every one of them returns before
a launch), and the Python functions' own."""
import pytest
import torch

from flydsl_amd import _lib, moe

X, IDS, W, OUT, AUX, SCRATCH = (0x10000000 * i for i in range(1, 7))
F32, SOFTMAX = _lib.QUANT_IN["fp32"], _lib.SCORING["softmax"]


def topk(tokens, experts=8, k=2):
    return _lib.load().flygemm_moe_topk(IDS, W, X, 0, None, None, tokens, experts, k, 1, 1, F32, SOFTMAX, 1, 1.0, None)


def topk_grad(tokens, experts=8, k=2):
    return _lib.load().flygemm_moe_topk_grad(OUT, W, IDS, X, 0, tokens, experts, k, F32, SOFTMAX, 1, 1.0, None)


def balance(tokens, experts=8, k=2, sequences=1, cu=None):
    return _lib.load().flygemm_moe_balance(W, OUT, AUX, SCRATCH, X, 0, IDS, None, cu, tokens, experts, k, sequences, F32, SOFTMAX,
                                           0, None)


def balance_grad(tokens, experts=8):
    return _lib.load().flygemm_moe_balance_grad(OUT, W, AUX, X, 0, None, None, tokens, experts, 1, F32, SOFTMAX, None)


@pytest.mark.parametrize("entry", [topk, topk_grad, balance, balance_grad])
@pytest.mark.parametrize("tokens", [2**31 - 1, 2**31 - 129, 2**31 - 256, _lib.MOE_ROUTER_MAX_TOKENS + 1])
def test_tokens_whose_rows_do_not_fit_32_bits(entry, tokens):
    assert entry(tokens) != 0
    assert f"tokens={tokens} must be at most" in _lib.load().flygemm_last_error().decode()


def test_balance_scratch_at_the_largest_sizes():
    scratch = _lib.load().flygemm_moe_balance_scratch
    most = _lib.MOE_ROUTER_MAX_TOKENS
    assert scratch(most + 1, 8, 1) == scratch(2**31 - 1, 8, 1) == -1
    slots = -(-most // 4096) + 1                    # chunks of 4096 rows: float and int parts of 64 experts, a count
    assert scratch(most, 8, 1) == 2 * slots * 64 * 4 + -(-slots * 4 // 16) * 16


@pytest.mark.parametrize("call", [lambda x: moe.moe_topk(x, 2), lambda x: moe.moe_balance_loss(x, x[:, :2])])
def test_functions_refuse_too_many_tokens(call):
    x = torch.zeros(1, 8).expand(_lib.MOE_ROUTER_MAX_TOKENS + 1, 8)
    with pytest.raises(ValueError, match="tokens: the router's kernels take at most"):
        call(x)


@pytest.mark.parametrize("tokens,k", [(1, 2**27 - 1), (1, 2**27 - 64), (25600, 21474836)])
def test_balance_ids_of_a_chunk_do_not_fit_32_bits(tokens, k):
    """Chunks of 16 and of 100 rows, whose ids' last place is below 2^31 and a workgroup's next one above it."""
    assert balance(tokens, k=k) != 0
    assert f"topk={k} too large" in _lib.load().flygemm_last_error().decode()
