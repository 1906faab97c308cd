"""Token log probabilities on the GPU against the 64-bit restatement.

Bounds (natural units; d = x - max, E over the row's distribution): every exponential is off by
|d| 2^-23 (its argument is rounded twice) + 2^-21 (the unit), the sum of V of them by another
(V / 512 + 32) 2^-24, so log S is off by
  a = E|d| 2^-23 + 2^-21 + (V / 512 + 32) 2^-24
a log probability by a + (|logp| + |log S| + 1) 2^-23, and the entropy log S - T / S by
  a (2 + 2 E|d|) + E d^2 2^-22 + (H + E|d| + 1) 2^-22.
Top tokens are whole numbers and equal.
"""

import numpy as np
import pytest
import torch

from oracle import q8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(logits, tokens, k, got=None):
    from tinyvllm_b200 import layers
    got = got or layers.token_logprobs(logits, tokens, k)
    lp, ent, top, ids, e1, e2 = q8.token_logprobs(logits.double().cpu().numpy(), tokens.cpu().numpy(), k)
    np.testing.assert_array_equal(got.top_tokens.cpu().numpy(), ids)
    V = logits.shape[1]
    with np.errstate(all="ignore"):
        a = e1 * 2.0 ** -23 + 2.0 ** -21 + (V / 512 + 32) * 2.0 ** -24

    def near(x, want, bound):
        x = x.cpu().double().numpy()
        fine = np.isfinite(want)
        np.testing.assert_array_equal(np.where(fine, 0.0, x), np.where(fine, 0.0, want))
        over = np.where(fine, np.abs(x - np.where(fine, want, 0.0)) - np.where(np.isfinite(bound), bound, 0.0), 0.0)
        assert not over.size or over.max() <= 0, f"{over.max()} over the bound at {over.argmax()}"

    with np.errstate(all="ignore"):
        room = lambda v: (np.abs(v) + np.log(V) + 1) * 2.0 ** -23
        near(got.logprobs, lp, a + room(lp))
        near(got.top_logprobs, top, a[:, None] + room(top))
        near(got.entropy, ent, a * (2 + 2 * e1) + e2 * 2.0 ** -22 + (np.abs(ent) + e1 + 1) * 2.0 ** -22)


def _logits(dev, rows, V, dtype, seed, spread=3.0):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(rows, V)) * spread
    return torch.from_numpy(x).to(dtype).to(dev), torch.from_numpy(rng.integers(0, V, rows).astype(np.int32)).to(dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 31, 33, 500, 4096, 16385, 32000, 50001, 128256])
def test_vocabularies(cuda, dtype, V):
    for k in (0, 1, min(V, 5), min(V, 32)):
        _check(*_logits(cuda, 3, V, dtype, V + k), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 5, 17, 64, 149, 300, 700])
def test_row_counts(cuda, dtype, rows):
    _check(*_logits(cuda, rows, 4001, dtype, rows), 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,stride", [(0, 5003), (1, 5001), (3, 5010), (7, 5008)])
def test_strided_and_misaligned_rows(cuda, dtype, offset, stride):
    x, tok = _logits(cuda, 6, 5000, dtype, 3)
    buf = torch.full((offset + 6 * stride,), float("nan"), dtype=dtype, device=cuda)
    view = buf[offset:].as_strided((6, 5000), (stride, 1))
    view.copy_(x)
    _check(view, tok, 9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [100, 5000, 70000])
def test_ties_and_sorted_rows(cuda, dtype, V):
    """Constant rows, sorted rows, few distinct values: more candidates than the buffer holds."""
    ramp = torch.linspace(-20, 20, V)
    rows = torch.stack([torch.zeros(V), ramp, ramp.flip(0), torch.arange(V) % 3 * 1.0, torch.full((V,), -5.0), (torch.arange(V) // 1000) * 0.25,
                        torch.where(torch.arange(V) % 2 == 0, torch.zeros(V), -torch.zeros(V))])
    for k in (1, 20, 32):
        _check(rows.to(dtype).to(cuda), torch.arange(len(rows), dtype=torch.int32, device=cuda), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 3001, 40000])
def test_masks(cuda, dtype, V):
    """-inf and the type's lowest value in masked places; rows with one token, with none; tokens outside the vocabulary."""
    x, tok = _logits(cuda, 10, V, dtype, V)
    low = torch.finfo(dtype).min
    x[0, ::2] = -float("inf")
    x[1, 1:] = -float("inf")
    x[2] = -float("inf")
    x[3] = low
    x[4, 3:] = low
    x[5, :-1] = low
    x[6, : V // 2] = low
    x[6, V // 2:] = -float("inf")
    tok[1], tok[2], tok[3] = 0, 5, V - 1
    tok[7], tok[8], tok[9] = -1, V, 2 ** 31 - 1
    for k in (0, 2, 32):
        _check(x, tok, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinite_logits(cuda, dtype):
    x, tok = _logits(cuda, 6, 9000, dtype, 8)
    x[0, 77] = float("nan")
    x[1, 8999] = float("inf")
    x[2, 5:600] = float("nan")
    x[3] = float("nan")
    x[4, 10], x[4, 11] = float("inf"), float("inf")
    for k in (0, 3, 32):
        _check(x, tok, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_and_flat_rows(cuda, dtype):
    for spread in (0.0, 0.01, 1.0, 30.0, 1000.0):
        _check(*_logits(cuda, 4, 32000, dtype, 9, spread), 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [20000, 150001, 300004])
def test_long_rows_of_many(cuda, dtype, V):
    """More rows than share a GPU by clusters, each a CTA's with many steps: six kinds of rows among 260."""
    from tinyvllm_b200 import layers
    rng = np.random.default_rng(V)
    x = rng.normal(size=(6, V)) * 4
    x[1] = np.sort(x[1])                          # every step beats the ones before: the buffer runs over
    x[2] = np.sort(x[2])[::-1]
    x[3] = 1.5
    x[4, rng.random(V) < 0.9] = -np.inf
    x[5, :V - 40] = -np.inf
    at = np.asarray([0, 51, 103, 148, 200, 259])
    few = torch.from_numpy(x).to(dtype).to(cuda)
    logits = torch.randn(260, V, device=cuda, dtype=torch.float32).to(dtype)
    logits[torch.from_numpy(at).to(cuda)] = few
    tok = torch.from_numpy(rng.integers(0, V, 260).astype(np.int32)).to(cuda)
    for k in (0, 1, 5, 32):
        got = layers.token_logprobs(logits, tok, k)
        idx = torch.from_numpy(at).to(cuda)
        _check(few, tok[idx], k, layers.TokenLogprobs(*(t[idx] for t in got)))


def test_agrees_with_greedy_argmax(cuda):
    from tinyvllm_b200 import layers
    x, tok = _logits(cuda, 64, 32000, torch.float16, 4)
    best = layers.greedy_argmax(x)
    r = layers.token_logprobs(x, best, 1)
    assert torch.equal(r.top_tokens[:, 0], best) and torch.equal(r.top_logprobs[:, 0], r.logprobs)


def test_refusals(cuda):
    from tinyvllm_b200 import layers
    x, tok = _logits(cuda, 4, 100, torch.float16, 1)
    for bad, err in (((x.double(), tok, 1), TypeError), ((x, tok.long(), 1), TypeError), ((x, tok[:3], 1), TypeError), ((x[:, ::2], tok, 1), ValueError),
                     ((x[0], tok, 1), ValueError), ((x, tok, 33), ValueError), ((x, tok, -1), ValueError), ((x[:, :3], tok, 4), ValueError),
                     ((x[:1].expand(4, 100), tok, 1), ValueError)):
        with pytest.raises(err):
            layers.token_logprobs(*bad)
    r = layers.token_logprobs(x[:0], tok[:0], 2)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 2)


def test_graph_and_streams(cuda):
    from tinyvllm_b200 import layers
    x, tok = _logits(cuda, 5, 32000, torch.bfloat16, 2)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        layers.token_logprobs(x, tok, 5)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        r = layers.token_logprobs(x, tok, 5)
    y, tok2 = _logits(cuda, 5, 32000, torch.bfloat16, 3)
    for data in (x.clone(), y):
        x.copy_(data)
        g.replay()
        torch.cuda.synchronize()
        _check(x, tok, 5, r)
