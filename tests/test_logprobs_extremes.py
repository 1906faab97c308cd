"""Token log probabilities of rows with NaN before a masked span, of logits near their
type's largest value, and of rows of ties (GPU).  Bounds as derived at the head of test_logprobs.py."""

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


def _time(fn, n=5):
    fn()
    best = float("inf")
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("kind", ["constant", "descending", "masked"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_ties_are_not_pushed_again_step_after_step(cuda, dtype, kind):
    """Once the K best are known exactly, nothing further of such rows is a candidate: the slow way through a full buffer is
    taken once, not for the whole row.  A row is 31 (bf16) or 62 (fp32) full steps long."""
    from tinyvllm_b200 import layers
    rows, V, k = 296, 256000, 20
    ordinary = torch.randn(rows, V, device=cuda).to(dtype)
    tok = torch.zeros(rows, dtype=torch.int32, device=cuda)
    base = _time(lambda: layers.token_logprobs(ordinary, tok, k))
    if kind == "constant":
        x = torch.full((rows, V), 1.5, device=cuda, dtype=dtype)
    elif kind == "descending":
        x = (-torch.arange(V, device=cuda) * 2.0 ** -8).to(dtype).expand(rows, V).contiguous()
    else:
        x = torch.full((rows, V), -float("inf"), device=cuda, dtype=dtype)
        x[:, 1000::20000] = 1.0
    took = _time(lambda: layers.token_logprobs(x, tok, k))
    print(f"{dtype} {kind}: {took * 1e3:.0f} us, ordinary {base * 1e3:.0f} us")
    assert took <= 4 * base, f"{kind} rows take {took / base:.1f} times ordinary ones"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(300, 40000), (3, 200000)])
def test_thresholds_of_full_buffers(cuda, dtype, rows, V):
    """Rows that overflow the candidate buffer and then hold better, equal and fewer tokens; NaN at the row's first places."""
    from tinyvllm_b200 import layers
    nan, none = float("nan"), -float("inf")
    x = torch.zeros(8, V, device=cuda)
    x[0, V - 50:] = torch.arange(50, device=cuda) * 0.25          # the K best come last
    x[1, ::3] = 0.5
    x[2] = none
    x[2, ::V // 7] = 1.0                                           # fewer tokens than alternatives
    x[3, :] = nan
    x[4, :2] = nan
    x[5] = torch.arange(V, device=cuda) // 2000 * 0.125            # steps up: every threshold falls behind
    x[6] = -(torch.arange(V, device=cuda) // 2000) * 0.125
    x[7, 0], x[7, 9000:9020] = nan, 3.0
    x = x.to(dtype)
    tok = torch.arange(8, dtype=torch.int32, device=cuda) * 5
    if rows == 3:
        parts = [torch.arange(0, 3), torch.arange(3, 6), torch.arange(5, 8)]
    else:
        parts = [torch.arange(8)]
    for k in (1, 2, 20, 32):
        for part in parts:
            view = torch.zeros(rows, V, device=cuda, dtype=dtype)
            at = torch.linspace(0, rows - 1, len(part)).long().to(cuda)
            p = part.to(cuda)
            all_tok = torch.zeros(rows, dtype=torch.int32, device=cuda)
            view[at], all_tok[at] = x[p], tok[p]
            got = layers.token_logprobs(view, all_tok, k)
            _check(x[p], tok[p], k, layers.TokenLogprobs(*(t[at] for t in got)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [300, 3])
def test_ties_between_the_last_elements_and_later_ones(cuda, dtype, rows):
    """The elements behind the last whole vector are looked at first: of equal ones in between, which come later, the smaller
    index counts."""
    from tinyvllm_b200 import layers
    V = 160007
    x = torch.zeros(4, V, device=cuda)
    x[:, 5], x[:, V - 1] = 2.0, 1.0
    x[1, 50000] = 1.0
    x[2, V - 40], x[2, V - 2] = 1.0, 1.0
    x[3, 100000:100300] = 1.0
    x = x[:rows].to(dtype)
    view = torch.zeros(rows, V, device=cuda, dtype=dtype)
    at = torch.linspace(0, rows - 1, len(x)).long().to(cuda)
    view[at] = x
    tok = torch.zeros(rows, dtype=torch.int32, device=cuda)
    for k in (2, 3, 5):
        got = layers.token_logprobs(view, tok, k)
        _check(x, tok[:len(x)], k, layers.TokenLogprobs(*(t[at] for t in got)))
