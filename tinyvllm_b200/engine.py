"""Continuous-batching engine over the sm_100a kernels.

Mirrors ``tinyvllm/core/engine.py``, ``core/scheduler.py`` and ``core/sequence.py``
for the hot path: FCFS admission up to ``max_batch_size`` (scheduler.py:32-54),
prefill of newly admitted sequences then ``num_scheduler_steps`` batched decode
iterations (engine.py:114-196), blocks freed when a sequence finishes
(scheduler.py:56-64).  Differences, all on the device side:

* newly admitted prompts are prefilled in one ragged kernel call per layer
  (the reference runs one prompt at a time, engine.py:125-132); block
  allocation still happens prompt by prompt in admission order, so the slots
  are the reference's;
* each decode step builds its block tables and context lengths in one numpy
  pass (engine.py:235-255) and writes all sequences' new K/V with one launch
  per layer (the reference issues batch x layers writes, llama.py:381-386);
* sampling is greedy only (temperature < 1e-5): an on-device argmax; the
  reference's random sampling paths (sampling.py) are not part of this build;
* with ``use_cuda_graphs`` a decode step replays a CUDA graph per padded batch
  size and a prefill step one per (prompt count, token count rounded up to
  128), the latter over a token buffer whose tail is a padding prompt that
  stores nothing; up to 64 prefill graphs are kept, further shapes run eagerly.

``kv_cache_dtype="float8_e4m3fn"`` keeps the K/V cache in 8 bits with one scale per block
and KV head (half the bytes of a 16-bit cache, values off by up to 2^-4 of themselves; steps of long contexts
get faster, of short ones slower; no counterpart in the reference).
``SamplingParams.logprobs = n`` returns for each sampled token its log probability, the
entropy of its distribution and the n most likely tokens, from the step's logits.

``kv_order="reference"`` (default) reproduces the reference decode exactly:
tables padded / truncated to 64 blocks (engine.py:81, llama.py:368-374),
attention over ``position + 1`` slots before the step's own K/V is written.
``kv_order="append_first"`` writes first and uses full-width tables.
"""

from __future__ import annotations

import time
from dataclasses import dataclass, field
from enum import Enum, auto
from typing import Any, Callable, Dict, Iterator, List, Optional, Tuple

import numpy as np
import torch

from . import layers
from .attention import check_workspace
from .block_manager import BlockManager
from .model import KVCache, Llama

_SAMPLING_EPS = 1e-5
_GRAPH_BATCHES = (1, 2, 4, 8, 16, 24, 32, 48, 64, 96, 128, 192, 256, 384, 512)
# prefill graphs hold a whole number of these tokens (the live prompts plus at least one padding token)
_PREFILL_TOKEN_QUANTUM = 128
# prefill graphs an engine keeps; a step of another (prompt count, token count) shape runs eagerly
_MAX_PREFILL_GRAPHS = 64


@dataclass
class SamplingParams:
    """core/sampling.py:12-18.  Only greedy decoding (temperature < 1e-5) is run here.
    ``logprobs``: None, or how many most likely tokens (0 to 32) to report with each
    token's log probability."""
    temperature: float = 0.0
    top_k: int = 40
    top_p: float = 0.95
    repetition_penalty: float = 1.0
    max_tokens: int = 1024
    logprobs: Optional[int] = None


@dataclass
class SampledLogprobs:
    """What ``SamplingParams.logprobs`` asks for, of one sampled token (natural logarithms)."""
    token: int
    logprob: float
    entropy: float
    top: List[Tuple[int, float]]      # (token, log probability), most likely first


class SequenceStatus(Enum):
    WAITING = auto()
    RUNNING = auto()
    FINISHED = auto()


@dataclass
class Sequence:
    seq_id: int
    request_id: int
    prompt_tokens: List[int]
    output_tokens: List[int] = field(default_factory=list)
    status: SequenceStatus = SequenceStatus.WAITING
    # one entry per output token where asked for (None: a first token that was given, not sampled)
    logprobs: Optional[List[Optional[SampledLogprobs]]] = None

    def get_all_tokens(self) -> List[int]:
        return self.prompt_tokens + self.output_tokens

    def get_len(self) -> int:
        return len(self.prompt_tokens) + len(self.output_tokens)

    def get_prompt_len(self) -> int:
        return len(self.prompt_tokens)

    def get_output_len(self) -> int:
        return len(self.output_tokens)

    def append_token(self, token_id: int) -> None:
        self.output_tokens.append(token_id)

    def is_finished(self) -> bool:
        return self.status == SequenceStatus.FINISHED


@dataclass
class Request:
    request_id: int
    prompt: Any
    prompt_tokens: List[int]
    sampling_params: SamplingParams
    arrival_time: float = field(default_factory=time.time)
    sequence: Optional[Sequence] = None
    prefilled_first_token: Optional[int] = None


@dataclass
class SchedulerOutput:
    scheduled_seqs: List[Sequence] = field(default_factory=list)


@dataclass
class GenerationOutput:
    request_id: int
    text: str
    tokens: List[int]
    finish_reason: str  # 'eos', 'length' or 'abort'
    logprobs: Optional[List[Optional[SampledLogprobs]]] = None   # as SamplingParams.logprobs asks for


class Scheduler:
    """FCFS continuous batching (core/scheduler.py:10-88)."""

    def __init__(self, max_batch_size: int, block_manager: BlockManager, gpu_id: int = 0):
        self.max_batch_size = max_batch_size
        self.block_manager = block_manager
        self.gpu_id = gpu_id
        self.waiting: List[Request] = []
        self.running: Dict[int, Sequence] = {}
        self.next_seq_id = 0

    def add_request(self, request: Request) -> None:
        self.waiting.append(request)

    def has_unfinished(self) -> bool:
        return bool(self.waiting) or bool(self.running)

    def schedule(self) -> SchedulerOutput:
        batch = SchedulerOutput(scheduled_seqs=list(self.running.values()))
        while len(batch.scheduled_seqs) < self.max_batch_size and self.waiting:
            request = self.waiting.pop(0)
            self.block_manager.register_sequence(self.next_seq_id, self.gpu_id)
            seq = Sequence(self.next_seq_id, request.request_id, request.prompt_tokens,
                           status=SequenceStatus.RUNNING,
                           logprobs=None if request.sampling_params.logprobs is None else [])
            request.sequence = seq
            self.next_seq_id += 1
            self.running[seq.seq_id] = seq
            batch.scheduled_seqs.append(seq)
        return batch

    def update(self, finished_seqs: List[int]) -> None:
        for seq_id in finished_seqs:
            seq = self.running.pop(seq_id, None)
            if seq is not None:
                seq.status = SequenceStatus.FINISHED
                self.block_manager.free_sequence(seq_id)

    def get_num_waiting(self) -> int:
        return len(self.waiting)

    def get_num_running(self) -> int:
        return len(self.running)

    def abort_request(self, request_id: int) -> bool:
        for i, req in enumerate(self.waiting):
            if req.request_id == request_id:
                self.waiting.pop(i)
                return True
        for seq_id, seq in list(self.running.items()):
            if seq.request_id == request_id:
                del self.running[seq_id]
                self.block_manager.free_sequence(seq_id)
                return True
        return False


class TokenIdTokenizer:
    """Pass-through tokenizer: prompts are lists of token ids; ``eos_id`` defaults to
    an id outside any vocabulary so generation runs to ``max_tokens``."""

    def __init__(self, eos_id: int = -1):
        self.eos_id = eos_id

    def encode(self, prompt) -> List[int]:
        return list(prompt)

    def decode(self, tokens: List[int]) -> str:
        return " ".join(map(str, tokens))


class LLMEngine:
    def __init__(self, model: Llama, tokenizer: Any = None, max_batch_size: int = 8, num_blocks: int = 1024,
                 block_size: int = 16, num_scheduler_steps: int = 1, kv_order: str = "reference",
                 max_table_blocks: Optional[int] = None, gpu_id: int = 0,
                 output_callback: Optional[Callable[[GenerationOutput], None]] = None,
                 use_cuda_graphs: bool = False, kv_cache_dtype: Optional[str] = None):
        if kv_order not in ("reference", "append_first"):
            raise ValueError("kv_order must be 'reference' or 'append_first'")
        if kv_cache_dtype not in (None, "float8_e4m3fn"):
            raise ValueError("kv_cache_dtype must be None (the model's dtype) or 'float8_e4m3fn'")
        self.model = model
        self.tokenizer = tokenizer or TokenIdTokenizer()
        self.max_batch_size = max_batch_size
        self.block_size = block_size
        self.num_scheduler_steps = num_scheduler_steps
        self.kv_order = kv_order
        # the reference pads / truncates decode tables to 64 blocks (engine.py:81)
        self.table_width = max_table_blocks or (64 if kv_order == "reference" else None)
        cfg = model.config
        self.device = model.device
        self.block_manager = BlockManager(num_gpus=gpu_id + 1, blocks_per_gpu=num_blocks, block_size=block_size)
        self.gpu_id = gpu_id
        self.kv_cache = KVCache(cfg.n_layers, num_blocks, block_size, cfg.n_kv_heads, cfg.head_dim,
                                cfg.torch_dtype if kv_cache_dtype is None else torch.float8_e4m3fn, self.device)
        self.scheduler = Scheduler(max_batch_size, self.block_manager, gpu_id)
        self.next_request_id = 0
        self.requests: Dict[int, Request] = {}
        self.output_callback = output_callback
        self._outputs: List[GenerationOutput] = []
        self.stats = {"prefill_tokens": 0, "decode_tokens": 0, "decode_steps": 0}
        # decode graphs, one per padded batch size (the reference keeps one TinyJit per batch size)
        self.use_cuda_graphs = use_cuda_graphs
        self._graphs = {}
        # prefill graphs, one per (prompt count, padded token count); they replay one at
        # a time on one stream, so they share one memory pool
        self._prefill_graphs = {}
        self._prefill_pool = None
        self._prefill_stream = None
        self._graph_width = self.table_width or -(-2 * cfg.max_seq_len // block_size)
        self._finished: List[int] = []     # sequences whose last token is there, until their step reports them
        self._step_logprobs: Dict[int, SampledLogprobs] = {}   # of the tokens being sampled, by sequence

    # ------------------------------------------------------------------ API
    def add_request(self, prompt, sampling_params: Optional[SamplingParams] = None,
                    request_id: Optional[int] = None) -> int:
        sp = sampling_params or SamplingParams()
        if sp.temperature >= _SAMPLING_EPS:
            raise ValueError("only greedy decoding (temperature < 1e-5) is supported by this engine")
        if sp.logprobs is not None and not 0 <= sp.logprobs <= min(32, self.model.config.vocab_size):
            raise ValueError("logprobs must be None or from 0 to 32 (and no more than the vocabulary)")
        tokens = self.tokenizer.encode(prompt)
        if not tokens:
            raise ValueError("empty prompt")
        if request_id is None:
            request_id = self.next_request_id
            self.next_request_id += 1
        elif request_id in self.requests:
            raise ValueError(f"Request ID {request_id} already exists")
        elif request_id >= self.next_request_id:
            self.next_request_id = request_id + 1
        req = Request(request_id, prompt, tokens, sp)
        self.requests[request_id] = req
        self.scheduler.add_request(req)
        return request_id

    def add_prefilled_request(self, context_tokens, sampling_params: Optional[SamplingParams] = None,
                              first_token: int = 0, request_id: Optional[int] = None) -> int:
        """Admit a sequence whose K/V for ``context_tokens`` is already resident in the
        pool contents (e.g. synthetic K/V for a decode benchmark): on admission its
        blocks are allocated and its position advanced as a prefill would, no
        prefill is run, and ``first_token`` is taken as the prompt's sampled token."""
        rid = self.add_request(context_tokens, sampling_params, request_id)
        self.requests[rid].prefilled_first_token = int(first_token)
        return rid

    def has_unfinished(self) -> bool:
        return self.scheduler.has_unfinished()

    def abort_request(self, request_id: int) -> bool:
        return self.scheduler.abort_request(request_id)

    def run(self) -> Iterator[GenerationOutput]:
        while self.scheduler.has_unfinished():
            yield from self.step()

    # ----------------------------------------------------------------- step
    def step(self) -> List[GenerationOutput]:
        batch = self.scheduler.schedule()
        if not batch.scheduled_seqs:
            return []
        # not empty only where the step before raised after they finished (some may have been aborted since)
        finished = self._finished = [i for i in self._finished if i in self.scheduler.running]
        prefill = [s for s in batch.scheduled_seqs if s.get_output_len() == 0]
        decode = [s for s in batch.scheduled_seqs if s.get_output_len() > 0 and s.seq_id not in finished]
        if prefill:
            first = self._prefill(prefill)
            for seq, tok in zip(prefill, first):
                self._append(seq, tok)
                if self._check_finished(seq):
                    finished.append(seq.seq_id)
        for _ in range(self.num_scheduler_steps):
            if not decode:
                break
            next_tokens = self._decode(decode)
            still = []
            for seq, tok in zip(decode, next_tokens):
                self._append(seq, tok)
                if self._check_finished(seq):
                    finished.append(seq.seq_id)
                else:
                    still.append(seq)
            decode = still
        self.scheduler.update(finished)
        self._finished = []
        outs = []
        for sid in finished:
            for rid, req in list(self.requests.items()):
                if req.sequence is not None and req.sequence.seq_id == sid:
                    out = GenerationOutput(rid, self.tokenizer.decode(req.sequence.output_tokens),
                                           list(req.sequence.output_tokens), self._reason(req.sequence),
                                           req.sequence.logprobs)
                    outs.append(out)
                    if self.output_callback:
                        self.output_callback(out)
                    del self.requests[rid]
                    break
        return outs

    def _append(self, seq: Sequence, token: int) -> None:
        """Takes a sampled token with its log probabilities: together, once the step's checks have passed, so
        that a step that raised leaves neither."""
        seq.append_token(token)
        entry = self._step_logprobs.pop(seq.seq_id, None)
        if seq.logprobs is not None:
            seq.logprobs.append(entry)

    def _reason(self, seq: Sequence) -> str:
        return "eos" if seq.output_tokens[-1] == self.tokenizer.eos_id else "length"

    def _check_finished(self, seq: Sequence) -> bool:
        req = self.requests[seq.request_id]
        return seq.output_tokens[-1] == self.tokenizer.eos_id or seq.get_output_len() >= req.sampling_params.max_tokens

    # --------------------------------------------------------------- device
    def _prefill(self, seqs: List[Sequence]) -> List[int]:
        bm = self.block_manager
        first = {}
        live = []
        for s in seqs:
            tok = self.requests[s.request_id].prefilled_first_token
            if tok is None:
                live.append(s)
            else:                      # K/V already resident: allocate, and advance below
                bm.slot_mapping(s.seq_id, 0, s.get_prompt_len())
                first[s.seq_id] = tok
        if live:
            for s, t in zip(live, self._prefill_live(live)):
                first[s.seq_id] = t
        for s in seqs:                 # after the prefill, which may raise: a step done again advances once
            if self.requests[s.request_id].prefilled_first_token is not None:
                bm.advance_position(s.seq_id, s.get_prompt_len())
        return [first[s.seq_id] for s in seqs]

    def _prefill_live(self, seqs: List[Sequence]) -> List[int]:
        bm = self.block_manager
        lens = [s.get_prompt_len() for s in seqs]
        slots = np.concatenate([bm.slot_mapping(s.seq_id, 0, L) for s, L in zip(seqs, lens)])
        toks = np.concatenate([np.asarray(s.prompt_tokens, dtype=np.int32) for s in seqs])
        pos = np.concatenate([np.arange(L, dtype=np.int32) for L in lens])
        cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        dev = self.device
        n, t_pad = len(seqs), -(-(int(cu[-1]) + 1) // _PREFILL_TOKEN_QUANTUM) * _PREFILL_TOKEN_QUANTUM
        graph = self._prefill_graphs.get((n, t_pad)) if self.use_cuda_graphs else None
        if self.use_cuda_graphs and (graph is not None or len(self._prefill_graphs) < _MAX_PREFILL_GRAPHS):
            if graph is None:
                if self._prefill_pool is None:
                    self._prefill_pool = torch.cuda.graph_pool_handle()
                    self._prefill_stream = torch.cuda.Stream(dev)
                    # one for all prefill graphs: it is read before the next of them runs
                    self._prefill_logits = torch.empty(self.max_batch_size, self.model.config.vocab_size,
                                                       dtype=self.model.output.dtype, device=dev)
                graph = self.model.capture_prefill(n, t_pad, self.kv_cache, self._prefill_pool, self._prefill_stream,
                                                   self._prefill_logits)
                self._prefill_graphs[(n, t_pad)] = graph
            sampled = graph.run(toks, pos, lens, slots).tolist()   # raises if a kernel wait timed out
            self._add_logprobs(graph.logits, graph.out[:n], seqs)
        else:
            logits = self.model.prefill(torch.from_numpy(toks).to(dev), torch.from_numpy(pos).to(dev),
                                        torch.from_numpy(cu).to(dev), max(lens), torch.from_numpy(slots).to(dev),
                                        self.kv_cache)
            sampled = self._sample(logits, seqs)
            check_workspace(dev, "prefill", "prefill step")     # a kernel wait that timed out raises here
        for s, L in zip(seqs, lens):
            bm.advance_position(s.seq_id, L)
        self.stats["prefill_tokens"] += int(sum(lens))
        return sampled

    def _decode(self, seqs: List[Sequence]) -> List[int]:
        bm = self.block_manager
        ids = [s.seq_id for s in seqs]
        pos = np.asarray([s.get_len() - 1 for s in seqs], dtype=np.int32)
        ctx = pos + 1

        def new_slots():
            out = np.empty(len(ids), dtype=np.int64)
            for j, i in enumerate(ids):
                _, blk, off = bm.get_slot(i)           # allocates a block when the position needs one
                out[j] = blk * self.block_size + off
            return out

        if self.kv_order == "reference":
            # tables are built before the new slot is allocated (engine.py:247, llama.py:383)
            bt = bm.block_table_array(ids, self.table_width)
            slots = new_slots()
        else:
            slots = new_slots()
            bt = bm.block_table_array(ids, self.table_width)
        if self.use_cuda_graphs:
            B = len(seqs)
            cap = next((b for b in _GRAPH_BATCHES if b >= B), -(-B // 64) * 64)
            graph = self._graphs.get(cap)
            if graph is None:
                graph = self.model.capture_decode(cap, self._graph_width, self.kv_cache, self.kv_order)
                self._graphs[cap] = graph
            toks = np.asarray([s.output_tokens[-1] for s in seqs], dtype=np.int32)
            sampled = graph.run(toks, pos, bt, ctx, slots).tolist()
            self._add_logprobs(graph.logits[:B], graph.out[:B], seqs)
        else:
            dev = self.device
            tok = torch.tensor([s.output_tokens[-1] for s in seqs], dtype=torch.int32, device=dev)
            logits = self.model.decode(tok, torch.from_numpy(pos).to(dev), torch.from_numpy(bt).to(dev),
                                       torch.from_numpy(ctx).to(dev), torch.from_numpy(slots).to(dev),
                                       self.kv_cache, self.kv_order)
            sampled = None
        if sampled is None:
            sampled = self._sample(logits, seqs)
            check_workspace(self.device, self.kv_cache.decode_kind, "decode step")
        for i in ids:
            bm.advance_position(i)
        self.stats["decode_tokens"] += len(seqs)
        self.stats["decode_steps"] += 1
        return sampled

    def _sample(self, logits: torch.Tensor, seqs: List[Sequence]) -> List[int]:
        """Greedy pick for each row of ``logits`` [len(seqs), vocab] (sampling.py:133-134)."""
        tokens = layers.greedy_argmax(logits)
        self._add_logprobs(logits, tokens, seqs)
        return tokens.cpu().tolist()

    def _add_logprobs(self, logits: torch.Tensor, tokens: torch.Tensor, seqs: List[Sequence]) -> None:
        """Log probabilities of this step's ``tokens`` (int32, one per row of ``logits``) for
        the sequences that asked for them, kept for ``_append``: one call over all rows, read back once."""
        self._step_logprobs = {}
        want = [self.requests[s.request_id].sampling_params.logprobs for s in seqs]
        n = max((w for w in want if w is not None), default=None)
        if n is None:
            return
        r = layers.token_logprobs(logits, tokens, n)
        host = torch.cat([tokens[:, None].double(), r.logprobs[:, None].double(), r.entropy[:, None].double(),
                          r.top_tokens.double(), r.top_logprobs.double()], dim=1).tolist()
        for s, w, row in zip(seqs, want, host):
            if w is not None:
                top = [(int(t), lp) for t, lp in zip(row[3:3 + w], row[3 + n:3 + n + w])]
                self._step_logprobs[s.seq_id] = SampledLogprobs(int(row[0]), row[1], row[2], top)


def generate_batch(engine: LLMEngine, prompts: List, sampling_params: Optional[SamplingParams] = None) -> List[str]:
    """core/engine.py:258-266: completions in input order."""
    ids = [engine.add_request(p, sampling_params) for p in prompts]
    results = {o.request_id: o.text for o in engine.run()}
    return [results[i] for i in ids]
