"""Log probabilities of a sharded engine's requests stay with the rank that owns them (CPU, gloo)."""

import multiprocessing as mp
import os
import traceback

import pytest

from test_distributed import _free_port

PROMPTS = [[3, 4, 5], [7], [9, 1, 2, 2, 8], [6, 6], [1, 2, 3, 4], [10]]
ASK = [2, None, 0, 3, 1, 2]


def _worker(rank, world, port, q):
    import datetime
    import torch
    import torch.distributed as dist
    import test_engine_logprobs as t
    from tinyvllm_b200.distributed import ShardedEngine
    from tinyvllm_b200.engine import SamplingParams
    try:
        t.engine_module.check_workspace = t._Checks()
        t.layers.greedy_argmax = lambda x: x.argmax(-1).int()
        t.layers.token_logprobs = t._token_logprobs
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=20))
        local = t._engine(max_batch_size=2, num_scheduler_steps=2)
        eng = ShardedEngine(local, rank, world, torch.device("cpu"))
        for i, (p, n) in enumerate(zip(PROMPTS, ASK)):
            eng.add_request(p, SamplingParams(max_tokens=3 + i, logprobs=n))
        partial = []
        while eng.has_unfinished():
            eng.step()
            partial.append([None if r.logprobs is None else len(r.logprobs) - len(r.tokens) for r in eng.requests.values()])
        rows = [(eng.owner(i), r.tokens, r.logprobs and [(x.token, len(x.top)) for x in r.logprobs]) for i, r in eng.requests.items()]
        q.put((rank, rows, partial))
        dist.destroy_process_group()
    except Exception:
        q.put((rank, traceback.format_exc(), None))


@pytest.mark.slow
def test_owner_has_the_log_probabilities_of_its_requests():
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = dict((r[0], r[1:]) for r in (q.get(timeout=90) for _ in procs))
    for p in procs:
        p.join(timeout=60)
    assert all(isinstance(r[0], list) for r in res.values()), res
    owners = {row[0] for row in res[0][0]}
    assert owners == {0, 1}
    for rank in (0, 1):
        rows, partial = res[rank]
        for (owner, tokens, got), n in zip(rows, ASK):
            if owner != rank or n is None:
                assert got is None
            else:                            # one entry a token, of that token, with as many alternatives as asked for
                assert got == [(t, n) for t in tokens]
        assert all(x in (None, 0) for step in partial for x in step)      # and after every step as many as tokens
