"""The engine's bookkeeping of log probabilities when a step's kernel wait runs out (CPU: the model and the device calls are
stand-ins; the scheduler, the blocks and the engine's own steps are real)."""

from types import SimpleNamespace

import pytest
import torch

from tinyvllm_b200 import engine as engine_module
from tinyvllm_b200 import layers
from tinyvllm_b200._lib import TvkError
from tinyvllm_b200.engine import LLMEngine, SamplingParams

VOCAB = 53


class _Model:
    """Logits that follow from the last token and the position alone, so a step done again gives the same token."""

    def __init__(self):
        self.config = SimpleNamespace(n_layers=1, n_heads=2, n_kv_heads=1, head_dim=32, vocab_size=VOCAB, max_seq_len=64, torch_dtype=torch.float32)
        self.device = torch.device("cpu")
        self.output = torch.zeros(1)

    def _logits(self, tok, pos):
        rows = [torch.randn(VOCAB, generator=torch.Generator().manual_seed(1000 * int(t) + int(p))) for t, p in zip(tok, pos)]
        return torch.stack(rows)

    def prefill(self, tok, pos, cu, longest, slots, cache):
        last = cu[1:].long() - 1
        return self._logits(tok[last], pos[last])

    def decode(self, tok, pos, bt, ctx, slots, cache, order):
        return self._logits(tok, pos)


def _token_logprobs(logits, tokens, k):
    logp = torch.log_softmax(logits.float(), -1)
    top = torch.topk(logp, k, dim=-1)
    return layers.TokenLogprobs(logp.gather(1, tokens.long()[:, None])[:, 0], -(logp.exp() * logp).sum(-1), top.values, top.indices.int())


class _Checks:
    """The checks of the workspace's status, one per eager prefill or decode step: those numbered in ``bad`` report a time-out."""

    def __init__(self):
        self.bad, self.n = (), 0

    def __call__(self, device, kind, what):
        self.n += 1
        if self.n in self.bad:
            raise TvkError(f"{what}: a bounded wait inside the kernel timed out")


@pytest.fixture
def checks(monkeypatch):
    c = _Checks()
    monkeypatch.setattr(engine_module, "check_workspace", c)
    monkeypatch.setattr(layers, "greedy_argmax", lambda x: x.argmax(-1).int())
    monkeypatch.setattr(layers, "token_logprobs", _token_logprobs)
    return c


def _run(eng):
    outs = {}
    while eng.has_unfinished():
        try:
            for o in eng.step():
                outs[o.request_id] = o
        except TvkError:
            pass
    return outs


def _engine(**kw):
    kw = {"max_batch_size": 3, "num_blocks": 32, "block_size": 4, "kv_order": "append_first", **kw}
    return LLMEngine(_Model(), **kw)


def _both(checks, bad, make):
    """Outputs of ``make()``'s engine without a time-out, and with those of the numbered checks."""
    want = _run(make())
    checks.bad, checks.n = bad, 0
    got = _run(make())
    assert checks.n >= max(bad) and got.keys() == want.keys()
    return want, got


@pytest.mark.parametrize("bad", [(1,), (2,), (3, 4), (1, 2, 5)])
def test_log_probabilities_stay_with_their_tokens_after_a_time_out(checks, bad):
    """A caller that catches the error and steps on gets one entry per token, of that token."""
    ask = [2, None, 0]

    def make():
        eng = _engine()
        for i, prompt in enumerate([[3, 4, 5], [7], [9, 1, 2, 2, 8]]):
            eng.add_request(prompt, SamplingParams(max_tokens=5 + i, logprobs=ask[i]))
        return eng

    want, got = _both(checks, bad, make)
    for i, n in enumerate(ask):
        assert got[i].tokens == want[i].tokens and got[i].logprobs == want[i].logprobs
        assert n is None or [x.token for x in got[i].logprobs] == got[i].tokens


@pytest.mark.parametrize("bad", [(1,), (1, 2)])
def test_a_given_first_token_has_one_empty_entry_after_a_time_out(checks, bad):
    """A request whose K/V are there already, admitted with one whose prefill runs out of time."""
    def make():
        eng = _engine()
        eng.add_prefilled_request([5, 6, 7], SamplingParams(max_tokens=4, logprobs=1), first_token=11)
        eng.add_request([3, 4], SamplingParams(max_tokens=4, logprobs=1))
        return eng

    want, got = _both(checks, bad, make)
    for i in (0, 1):
        entries = got[i].logprobs
        assert len(entries) == len(got[i].tokens) == 4
        assert [x and x.token for x in entries] == ([None] if i == 0 else got[1].tokens[:1]) + got[i].tokens[1:]
    assert got[1].logprobs == want[1].logprobs


@pytest.mark.parametrize("bad", [(1,), (1, 2)])
def test_a_prefill_done_again_advances_given_sequences_once(checks, bad):
    """The step that admits a request with resident K/V beside one to prefill runs out of time, and is done again."""
    def make():
        eng = _engine()
        eng.add_prefilled_request([5, 6, 7], SamplingParams(max_tokens=4), first_token=11)
        eng.add_request([3, 4], SamplingParams(max_tokens=4))
        return eng

    want, got = _both(checks, bad, make)
    assert [got[i].tokens for i in (0, 1)] == [want[i].tokens for i in (0, 1)]
    checks.bad, checks.n = bad, 0
    eng = make()
    for _ in bad:
        with pytest.raises(TvkError):
            eng.step()
    eng.step()
    bm = eng.block_manager
    assert [bm.get_context_length(s) for s in sorted(eng.scheduler.running)] == [3, 2]


@pytest.mark.parametrize("steps", [1, 3])
@pytest.mark.parametrize("bad", [(3,), (4,), (3, 4), (6,)])
def test_sequences_that_finished_before_a_time_out_end_there(checks, bad, steps):
    """A sequence that reaches its length in a step whose later part raises gets no further token, and is reported."""
    def make():
        eng = _engine(num_scheduler_steps=steps, max_batch_size=2)
        for i, n in enumerate([6, 1, 1, 2, 3]):
            eng.add_request([3 + i, 4], SamplingParams(max_tokens=n, logprobs=0))
        return eng

    want, got = _both(checks, bad, make)
    assert {i: o.tokens for i, o in got.items()} == {i: o.tokens for i, o in want.items()}
    assert [len(got[i].logprobs) for i in range(5)] == [6, 1, 1, 2, 3]


def test_a_finished_sequence_that_is_aborted_before_its_step_is_done_again_is_not_reported(checks):
    eng = _engine(max_batch_size=2)
    a = eng.add_request([3, 4], SamplingParams(max_tokens=6))
    eng.step()
    b = eng.add_request([5, 4], SamplingParams(max_tokens=1))
    checks.bad = (checks.n + 2,)                 # b's prefill is fine and ends it; the decode step behind it is not
    with pytest.raises(TvkError):
        eng.step()
    assert eng.abort_request(b)
    got = _run(eng)
    assert list(got) == [a] and len(got[a].tokens) == 6
