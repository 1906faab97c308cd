"""The 8-bit decode in recorded graphs: time-outs of calls of different sizes, graph and eager engine runs that agree to the
bit, and block sizes of several tiles (GPU)."""

import numpy as np
import pytest
import torch

from test_q8_cache import TYPES, _case, _check, _run
from test_q8_engine import _model

pytestmark = pytest.mark.gpu

LIMIT_NS = 5_000_000


def _arm():
    from tinyvllm_b200 import _lib
    assert _lib.lib().tvk_debug_arm_wait_timeout(LIMIT_NS) == 0


def test_time_out_of_a_call_before_a_larger_one_is_told(cuda):
    """The larger call takes a larger workspace; the smaller one's time-out (test hook) is still in the status word."""
    from tinyvllm_b200.attention import status_word, workspace_status
    small = _case(cuda, 2, 8, 2, 64, 16, [70, 300], torch.float16, 1)
    large = _case(cuda, 64, 8, 2, 64, 16, [40] * 64, torch.float16, 2)
    want = [_run(c).clone() for c in (small, large)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    told = torch.zeros(2, dtype=torch.int32, device=cuda)
    graphs = []
    for armed in (False, True):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            if armed:
                _arm()
            _run(small)
            out = _run(large)
            told[int(armed)].copy_(status_word(cuda, "decode_q8")[0])
        graphs.append((g, out))
    for _ in range(2):
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[1])
        assert told.tolist() == [0, 1]
    with torch.cuda.stream(torch.cuda.Stream()):      # the same without a recording
        _arm()
        _run(small)
        _run(large)
        assert workspace_status(cuda, "decode_q8") == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bs", [256, 384, 1024])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_blocks_of_several_tiles(cuda, dtype, bs, d):
    ctx = [1, 127, 128, 129, bs - 1, bs, bs + 1, 2 * bs + 130, 9 * bs + 5]
    c = _case(cuda, len(ctx), 8, 4, d, bs, ctx, dtype, bs + d)
    _check(c, _run(c, check=True))


def _padded(model, eng):
    """Makes the eager engine run the model at the row counts, table widths and padding that its graphs would run at."""
    from tinyvllm_b200.engine import _GRAPH_BATCHES, _PREFILL_TOKEN_QUANTUM
    from tinyvllm_b200.model import prefill_staging_layout, stage_prefill_inputs
    real_decode, real_prefill, dev = model.decode, model.prefill, model.device

    def pad(t, n, value):
        return torch.cat([t, torch.full((n - t.shape[0], *t.shape[1:]), value, dtype=t.dtype, device=dev)])

    def decode(tok, pos, bt, ctx, slots, cache, order):
        B = tok.shape[0]
        cap = next((b for b in _GRAPH_BATCHES if b >= B), -(-B // 64) * 64)
        wide = torch.zeros(cap, eng._graph_width, dtype=torch.int32, device=dev)
        wide[:B, :bt.shape[1]] = bt
        return real_decode(pad(tok, cap, 0), pad(pos, cap, 0), wide, pad(ctx, cap, 1), pad(slots, cap, -1), cache, order)[:B]

    def prefill(tok, pos, cu, longest, slots, cache):
        n, t = cu.shape[0] - 1, tok.shape[0]
        T = -(-(t + 1) // _PREFILL_TOKEN_QUANTUM) * _PREFILL_TOKEN_QUANTUM
        off_cu, off_slots, words = prefill_staging_layout(n, T)
        h = np.zeros(words, dtype=np.int32)
        lens = (cu[1:] - cu[:-1]).tolist()
        stage_prefill_inputs(h, n, T, tok.cpu().numpy(), pos.cpu().numpy(), lens, slots.cpu().numpy())
        d = torch.from_numpy(h).to(dev)
        return real_prefill(d[:T], d[T:2 * T], d[off_cu:off_cu + n + 2], T, d[off_slots:].view(torch.int64), cache, n_out=n)

    return decode, prefill


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 256), (8, 1, 512), (8, 8, 512)])
@pytest.mark.parametrize("order", ["reference", "append_first"])
def test_graphs_and_eager_steps_agree_to_the_bit(cuda, dtype, heads, kv_heads, dim, order, monkeypatch):
    """The same prompts through an engine of graphs and one of eager steps padded alike: every token, every log probability and
    every byte of the cache."""
    from tinyvllm_b200.engine import LLMEngine, SamplingParams
    model = _model(dtype, heads, kv_heads, dim)
    runs = []
    for graphs in (True, False):
        eng = LLMEngine(model, max_batch_size=4, num_blocks=64, kv_order=order, kv_cache_dtype="float8_e4m3fn", use_cuda_graphs=graphs)
        if not graphs:
            decode, prefill = _padded(model, eng)
            monkeypatch.setattr(model, "decode", decode)
            monkeypatch.setattr(model, "prefill", prefill)
        rng = np.random.default_rng(6)
        for _ in range(9):
            eng.add_request(rng.integers(0, 97, int(rng.integers(1, 60))).tolist(),
                            SamplingParams(max_tokens=int(rng.integers(2, 40)), logprobs=2))
        outs = {o.request_id: o for o in eng.run()}
        runs.append((outs, eng.kv_cache))
    (a, ca), (b, cb) = runs
    assert a.keys() == b.keys() and len(a) == 9
    for r in a:
        assert a[r].tokens == b[r].tokens and a[r].logprobs == b[r].logprobs
    for x, y in zip(ca.k_cache + ca.v_cache + ca.k_scale + ca.v_scale, cb.k_cache + cb.v_cache + cb.k_scale + cb.v_scale):
        # blocks 0 on: padding rows write nothing, and both engines hand out blocks alike
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
