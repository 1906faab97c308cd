"""Token log probabilities of rows with NaN before a masked span, and of logits near
their type's largest value (GPU).  Bounds as derived at the head of test_logprobs.py."""

import numpy as np
import pytest
import torch

from test_logprobs import _check, _logits

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(300, 40000), (3, 300004), (17, 140000)])
@pytest.mark.parametrize("offset", [0, 1])
def test_nan_before_a_masked_span(cuda, dtype, rows, V, offset):
    """A NaN (a whole vector's, or one before the first 16-byte boundary), then steps of nothing but -inf, then ordinary logits."""
    x, tok = _logits(cuda, 5, V, dtype, V + offset)
    nan, none = float("nan"), -float("inf")
    x[0, 77], x[0, 8192:40000 - 8192] = nan, none
    x[1, 0], x[1, 1:30000] = nan, none
    x[2, 8], x[2, 9:] = nan, none
    x[3, V - 1], x[3, 100:V - 1] = nan, none           # behind the masked span
    buf = torch.zeros(rows * V + offset, dtype=dtype, device=cuda)
    view = buf[offset:].view(rows, V)
    at = torch.linspace(0, rows - 1, 5).long() if rows >= 5 else torch.arange(rows)
    view[at.to(cuda)] = x[:len(at)]
    all_tok = torch.zeros(rows, dtype=torch.int32, device=cuda)
    all_tok[at.to(cuda)] = tok[:len(at)]
    from tinyvllm_b200 import layers
    for k in (0, 1, 20):
        got = layers.token_logprobs(view, all_tok, k)
        _check(x[:len(at)], tok[:len(at)], k, layers.TokenLogprobs(*(t[at.to(cuda)] for t in got)))
        assert torch.isnan(got.logprobs[at[:3].to(cuda)]).all() and torch.isnan(got.entropy[at[:3].to(cuda)]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(4, 5000), (300, 20000), (4, 9)])
def test_logits_near_the_largest_value(cuda, dtype, rows, V):
    """One logit (or two) at the type's largest value, or at half of it, the others 0 or the lowest value."""
    from tinyvllm_b200 import layers
    big, low = torch.finfo(dtype).max, torch.finfo(dtype).min
    x = torch.zeros(4, V, device=cuda, dtype=dtype)
    x[0, V // 2] = big
    x[1], x[1, V - 1] = low, big
    x[2, 3], x[2, V - 3] = big, big
    x[3, V // 2] = big / 2
    tok = torch.tensor([V // 2, V - 1, 3, 0], dtype=torch.int32, device=cuda)
    view, all_tok = torch.zeros(rows, V, device=cuda, dtype=dtype), torch.zeros(rows, dtype=torch.int32, device=cuda)
    at = torch.linspace(0, rows - 1, 4).long().to(cuda)
    view[at], all_tok[at] = x, tok
    for k in (0, 1):
        got = layers.token_logprobs(view, all_tok, k)
        _check(x, tok, k, layers.TokenLogprobs(*(t[at] for t in got)))
