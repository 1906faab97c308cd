"""The 8-bit cache and the log probabilities as the engine uses them: write, attend, logits, log
probabilities, step after step (GPU)."""

import numpy as np
import pytest
import torch

from oracle import q8

pytestmark = pytest.mark.gpu


def _model(dtype, heads=8, kv_heads=4, dim=256, **kw):
    from tinyvllm_b200.model import Llama, LlamaConfig
    return Llama(LlamaConfig(dim=dim, n_layers=2, n_heads=heads, n_kv_heads=kv_heads, vocab_size=97, hidden_dim=2 * dim, max_seq_len=256,
                             dtype=dtype, **kw), device="cuda", seed=3, init_std=0.25)


def _serve(model, logprobs=None, n=9, **kw):
    from tinyvllm_b200.engine import LLMEngine, SamplingParams
    rng = np.random.default_rng(5)
    eng = LLMEngine(model, max_batch_size=4, num_blocks=64, **kw)
    outs, i = {}, 0
    while i < n or eng.has_unfinished():
        for _ in range(2):
            if i < n:
                eng.add_request(rng.integers(0, 97, int(rng.integers(1, 60))).tolist(),
                                SamplingParams(max_tokens=int(rng.integers(2, 40)), logprobs=None if logprobs is None else logprobs(i)))
                i += 1
        for o in eng.step():
            outs[o.request_id] = o
    return outs, eng


class _Spy:
    """Feeds one layer's K/V rows, as the model computes them, to the 64-bit restatement of the cache."""

    def __init__(self, cache):
        self.k = [np.zeros(tuple(t.shape)) for t in cache.k_cache]
        self.ks = [np.zeros(tuple(t.shape)) for t in cache.k_scale]

    def write(self, layer, k, slots):
        self.k[layer], self.ks[layer] = q8.write_kv_slots(k.double().cpu().numpy(), slots.cpu().numpy(), self.k[layer], self.ks[layer])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("order", ["reference", "append_first"])
def test_engine_cache_holds_what_the_restatement_holds(cuda, dtype, order, monkeypatch):
    """Prompts, steps, finished sequences and blocks used again: codes and scales stay equal bit for bit."""
    from tinyvllm_b200.model import KVCache
    spies = {}
    real = KVCache.write_slots

    def write(self, layer, k, v, slots):
        spies.setdefault(id(self), _Spy(self)).write(layer, k, slots)
        real(self, layer, k, v, slots)

    monkeypatch.setattr(KVCache, "write_slots", write)
    _, eng = _serve(_model(dtype), kv_order=order, kv_cache_dtype="float8_e4m3fn")
    spy = spies[id(eng.kv_cache)]
    for i in range(2):
        np.testing.assert_array_equal(eng.kv_cache.k_scale[i].cpu().double().numpy(), spy.ks[i])
        np.testing.assert_array_equal(eng.kv_cache.k_cache[i].cpu().view(torch.uint8).view(torch.float8_e4m3fn).double().numpy(), spy.k[i])
    k, _ = eng.kv_cache.read_kv_blocks(1, [5, 3], 20)
    np.testing.assert_array_equal(k.cpu().double().numpy(), (spy.k[1][[5, 3]] * spy.ks[1][[5, 3]][:, None, :, None]).reshape(32, 4, 32)[:20])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 256), (8, 1, 512), (8, 8, 512)])
def test_graphs_and_eager_steps_give_the_same_tokens(cuda, dtype, heads, kv_heads, dim):
    model = _model(dtype, heads, kv_heads, dim)
    runs = [_serve(model, kv_cache_dtype="float8_e4m3fn", use_cuda_graphs=g, kv_order="append_first")[0] for g in (False, True)]
    # the projections run at other (padded) row counts in the graphs, so a near tie may fall differently
    same = [runs[0][r].tokens == runs[1][r].tokens for r in runs[0]]
    assert sum(same) >= len(same) - 2


def test_run_of_write_attend_and_logprobs(cuda):
    """Decode steps by hand over an 8-bit cache, each compared with 64 bits on the cache as it stands: attention
    within its rounding, log probabilities of the picks within theirs."""
    from tinyvllm_b200 import layers
    from tinyvllm_b200.model import KVCache
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    hq, hkv, d, vocab, B = 32, 8, 128, 5003, 5
    cache = KVCache(1, 40, 16, hkv, d, torch.float8_e4m3fn, "cuda")
    assert cache.get_memory_bytes() == 2 * 40 * (16 * hkv * d + 4 * hkv)
    head = rnd(hq * d, vocab) * 0.2
    lens = [0, 15, 16, 31, 100]
    tables = torch.arange(B * 8, device="cuda").view(B, 8).flip(0).int().contiguous()
    for b, n in enumerate(lens):
        if n:
            t = torch.arange(n, device="cuda")
            cache.write_slots(0, rnd(n, hkv, d), rnd(n, hkv, d), tables[b].long()[t // 16] * 16 + t % 16)
    for step in range(6):
        pos = torch.tensor([n + step for n in lens], device="cuda")
        slots = tables.gather(1, (pos // 16)[:, None])[:, 0].long() * 16 + pos % 16
        cache.write_slots(0, rnd(B, hkv, d), rnd(B, hkv, d), slots)
        q = rnd(B, 1, hq, d)
        out = cache.attend(0, q, tables, (pos + 1).int(), hq)
        codes = lambda c: c.cpu().view(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
        n64 = lambda t: t.cpu().double().numpy()
        ref, mass, span, wide, vmax = q8.paged_decode(n64(q), codes(cache.k_cache[0]), codes(cache.v_cache[0]), n64(cache.k_scale[0]),
                                                      n64(cache.v_scale[0]), tables.cpu().numpy(), (pos + 1).cpu().numpy())
        ds = (d + 16) * 2.0 ** -23 * span[:, None, :, None] + 2.0 ** -25 * wide[:, None, :, None]
        bound = 2.0 ** -11 * np.abs(ref) * 1.02 + (2.0 ** -10 + 2 * ds + 128 * 2.0 ** -23) * mass + 128 * 2.0 ** -23 * vmax[:, None, :, None]
        assert (np.abs(n64(out) - ref) <= bound).all()
        logits = torch.matmul(out.view(B, -1), head)
        pick = layers.greedy_argmax(logits)
        r = layers.token_logprobs(logits, pick, 4)
        lp, ent, top, ids, e1, _ = q8.token_logprobs(n64(logits), pick.cpu().numpy(), 4)
        np.testing.assert_array_equal(r.top_tokens.cpu().numpy(), ids)
        assert torch.equal(r.top_tokens[:, 0], pick)
        room = e1 * 2.0 ** -23 + 2.0 ** -21 + (vocab / 512 + 32) * 2.0 ** -24 + (np.abs(lp) + np.log(vocab) + 1) * 2.0 ** -23
        assert (np.abs(n64(r.logprobs) - lp) <= room).all()


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("kv", [None, "float8_e4m3fn"])
def test_engine_reports_log_probabilities(cuda, graphs, kv):
    model = _model("float16")
    ask = lambda i: [None, 0, 3, 5][i % 4]
    outs, _ = _serve(model, logprobs=ask, use_cuda_graphs=graphs, kv_cache_dtype=kv)
    plain, _ = _serve(model, use_cuda_graphs=graphs, kv_cache_dtype=kv)
    for rid, o in outs.items():
        assert o.tokens == plain[rid].tokens and plain[rid].logprobs is None      # asking changes no token
        if ask(rid) is None:
            assert o.logprobs is None
            continue
        assert [x.token for x in o.logprobs] == o.tokens
        for x in o.logprobs:
            assert len(x.top) == ask(rid) and 0 <= x.entropy <= np.log(97) + 1e-5 and x.logprob <= 0
            if x.top:
                assert x.top[0] == (x.token, x.logprob)        # greedy: the pick is the most likely token
                assert [p for _, p in x.top] == sorted((p for _, p in x.top), reverse=True)


def test_prefilled_requests_have_no_log_probability_for_their_given_token(cuda):
    from tinyvllm_b200.engine import LLMEngine, SamplingParams
    eng = LLMEngine(_model("float16"), max_batch_size=2, num_blocks=16, kv_cache_dtype="float8_e4m3fn")
    eng.add_prefilled_request([1, 2, 3], SamplingParams(max_tokens=4, logprobs=2), first_token=7)
    (o,) = list(eng.run())
    assert o.logprobs[0] is None and [x.token for x in o.logprobs[1:]] == o.tokens[1:]


def test_engine_refusals(cuda):
    from tinyvllm_b200.engine import LLMEngine, SamplingParams
    model = _model("float16")
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLMEngine(model, kv_cache_dtype="int8")
    eng = LLMEngine(model, num_blocks=8)
    for n in (-1, 33):
        with pytest.raises(ValueError, match="logprobs"):
            eng.add_request([1, 2], SamplingParams(logprobs=n))
