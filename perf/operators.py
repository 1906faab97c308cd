"""The measured cases of three serving operators: paged decode attention over an 8-bit K/V
cache, the write that fills that cache, and the log probabilities of picked tokens.

The 8-bit cache holds ``torch.float8_e4m3fn`` codes [num_blocks, block_size, n_kv_heads,
head_dim] and one fp32 scale per (block, KV head), for K and for V: a value is code * scale.
Scales that the write makes are powers of two, the smallest 2^k with amax <= 448 * 2^k.

``own`` selects who computes: False, plain torch operations in 32 bits; True, the package.
"""

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
E4M3_MAX = 448.0
MIN_SCALE_EXP = -100

# Padded K/V elements (batch x longest context x KV heads x head_dim), written rows and logits that no drawn case passes.
_MAX_DECODE = 256 * 4096 * 8 * 128
_MAX_WRITE = 8192 * 8 * 128
_MAX_LOGITS = 2048 * 128256


def listed():
    return [
        # one user's chat at the end of a 64-block table: nothing but latency
        dict(name="decode_one", op="decode", batch=1, n_heads=32, n_kv_heads=4, head_dim=64, block_size=16,
             ctx_lo=1023, ctx_hi=1023, empty=False, dtype="float16"),
        # a decode step of the engine: 64 requests of 40 to 640 tokens, and one padding row without context
        dict(name="decode_step", op="decode", batch=64, n_heads=32, n_kv_heads=4, head_dim=64, block_size=16,
             ctx_lo=40, ctx_hi=640, empty=True, dtype="float16"),
        # a large serving batch of ragged contexts
        dict(name="decode_batch", op="decode", batch=256, n_heads=32, n_kv_heads=8, head_dim=128, block_size=16,
             ctx_lo=128, ctx_hi=4096, empty=False, dtype="bfloat16"),
        # few users with long documents, larger blocks
        dict(name="decode_long", op="decode", batch=3, n_heads=32, n_kv_heads=8, head_dim=128, block_size=64,
             ctx_lo=20001, ctx_hi=65536, empty=False, dtype="bfloat16"),
        # a model run in fp32 to check another one: the smallest benchmark batch
        dict(name="decode_fp32", op="decode", batch=4, n_heads=32, n_kv_heads=4, head_dim=64, block_size=16,
             ctx_lo=17, ctx_hi=255, empty=False, dtype="float32"),
        # the K/V of one decode step of 64 requests
        dict(name="write_step", op="write", kind="step", rows=64, n_kv_heads=4, head_dim=64, block_size=16,
             num_blocks=1024, dtype="float16"),
        # the same for the large batch
        dict(name="write_batch", op="write", kind="step", rows=256, n_kv_heads=8, head_dim=128, block_size=16,
             num_blocks=1024, dtype="bfloat16"),
        # the K/V of a prefill of ragged prompts, 8,192 tokens in all
        dict(name="write_prompts", op="write", kind="prompts", rows=8192, n_kv_heads=8, head_dim=128, block_size=16,
             num_blocks=1024, dtype="bfloat16"),
        # the answer of one user's step, with five alternatives
        dict(name="logprobs_one", op="logprobs", rows=1, vocab=128256, top_k=5, dtype="bfloat16"),
        # a decode step of 64 requests with 20 alternatives
        dict(name="logprobs_step", op="logprobs", rows=64, vocab=32000, top_k=20, dtype="float16"),
        # scoring the tokens of a long prompt, no alternatives asked for but the best
        dict(name="logprobs_prompt", op="logprobs", rows=2048, vocab=128256, top_k=1, dtype="bfloat16"),
        # fp32 logits of an odd vocabulary
        dict(name="logprobs_fp32", op="logprobs", rows=37, vocab=50001, top_k=8, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "write", "logprobs"])
    if op == "decode":
        hq, hkv, d = rng.choice([(32, 4, 64), (32, 8, 128), (8, 8, 32), (12, 4, 64), (16, 1, 128), (20, 5, 64), (16, 8, 128),
                                 (16, 16, 64)])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        most = _MAX_DECODE // (8 if dtype == "float32" else 1)
        batch = _log_int(rng, 1, 256)
        hi = _log_int(rng, 1, min(65536, most // (batch * hkv * d)))
        return dict(op="decode", batch=batch, n_heads=hq, n_kv_heads=hkv, head_dim=d, block_size=rng.choice([8, 16, 16, 32, 64]),
                    ctx_lo=_log_int(rng, 1, hi), ctx_hi=hi, empty=rng.random() < 0.3, dtype=dtype)
    dtype = rng.choice(["float16", "bfloat16", "float32"])
    if op == "write":
        kind = rng.choice(["step", "prompts"])
        hkv, d = rng.choice([(4, 64), (8, 128), (8, 32), (1, 128), (5, 64)])
        bs = rng.choice([8, 16, 32, 64])
        rows = _log_int(rng, 1, 256) if kind == "step" else _log_int(rng, 1, 8192)
        need = rows if kind == "step" else 2 * rows // bs + 64
        return dict(op="write", kind=kind, rows=rows, n_kv_heads=hkv, head_dim=d, block_size=bs, num_blocks=need + rng.randint(0, 256),
                    dtype=dtype)
    vocab = _log_int(rng, 1000, 131072)
    return dict(op="logprobs", rows=_log_int(rng, 1, _MAX_LOGITS // (131072 * (2 if dtype == "float32" else 1))), vocab=vocab,
                top_k=rng.choice([0, 1, 5, 8, 20, 32]), dtype=dtype)


# ------------------------------------------------------------------ the cache format
def _scale_for(amax):
    """The smallest power of two s >= 2^-100 with amax <= 448 s, of fp32 maxima."""
    m, e = torch.frexp(amax)                       # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    k = (e - 9 + (m > 0.875).int()).clamp(min=MIN_SCALE_EXP)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, k, torch.full_like(k, MIN_SCALE_EXP)))


def _to_e4m3(x):
    """fp32 values in [-448, 448] to e4m3, nearest, ties to even."""
    return x.to(torch.float8_e4m3fn)


def _pool(gen, num_blocks, bs, hkv, d, spread):
    """A cache that earlier writes filled: normal values, a few loud channels, per-block scales."""
    dev = gen.device
    codes = torch.empty(num_blocks, bs, hkv, d, dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty(num_blocks, hkv, dtype=torch.float32, device=dev)
    loud = 1.0 + spread * (torch.rand(hkv, d, generator=gen, device=dev) < 0.05).float()
    step = max(1, (1 << 26) // (bs * hkv * d))
    for i in range(0, num_blocks, step):
        x = torch.randn(min(step, num_blocks - i), bs, hkv, d, generator=gen, device=dev) * loud
        s = _scale_for(x.abs().amax(dim=(1, 3)))
        codes[i:i + step] = _to_e4m3(x / s[:, None, :, None])
        scale[i:i + step] = s
    return codes, scale


# ------------------------------------------------------------------ prepare
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    rng = torch.Generator().manual_seed(1000003 * seed + 29)
    if case["op"] == "decode":
        return _prepare_decode(case, gen, rng)
    if case["op"] == "write":
        return _prepare_write(case, gen, rng)
    dt = _DTYPES[case["dtype"]]
    rows, vocab = case["rows"], case["vocab"]
    # next-token logits: a normal bulk and a few hundred likely tokens
    logits = torch.randn(rows, vocab, generator=gen, device="cuda")
    logits.mul_(2.5)
    likely = torch.randint(0, vocab, (rows, 64), generator=gen, device="cuda")
    logits.scatter_add_(1, likely, 6.0 * torch.rand(rows, 64, generator=gen, device="cuda"))
    picked = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.7, likely[:, 0],
                         torch.randint(0, vocab, (rows,), generator=gen, device="cuda"))
    return dict(op="logprobs", logits=logits.to(dt), tokens=picked.int(), top_k=case["top_k"])


def _prepare_decode(case, gen, rng):
    B, bs, hq, hkv, d = (case[k] for k in ("batch", "block_size", "n_heads", "n_kv_heads", "head_dim"))
    ctx = _contexts(case, rng)
    need = (ctx + bs - 1) // bs
    n_blocks = int(math.ceil(1.1 * int(need.sum()))) + 1
    width = max(1, int(need.max()))
    perm = torch.randperm(n_blocks, generator=rng)
    at = torch.arange(width)[None, :]
    first = need.cumsum(0) - need
    tables = torch.where(at < need[:, None], perm[(first[:, None] + at).clamp(max=n_blocks - 1)], torch.zeros((), dtype=torch.int64))
    k, ks = _pool(gen, n_blocks, bs, hkv, d, 7.0)
    v, vs = _pool(gen, n_blocks, bs, hkv, d, 0.0)
    q = torch.randn(B, 1, hq, d, generator=gen, device="cuda").to(_DTYPES[case["dtype"]])
    return dict(op="decode", q=q, k=k, v=v, ks=ks, vs=vs, tables=tables.int().cuda(), ctx=ctx.int().cuda(), n_heads=hq, n_kv_heads=hkv,
                head_dim=d, block_size=bs)


def _contexts(case, rng):
    ctx = torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (case["batch"],), generator=rng)
    if case["empty"]:
        ctx[case["batch"] // 2] = 0
    return ctx


def _prepare_write(case, gen, rng):
    T, bs, hkv, d, nb = (case[k] for k in ("rows", "block_size", "n_kv_heads", "head_dim", "num_blocks"))
    perm = torch.randperm(nb, generator=rng)
    if case["kind"] == "step":           # one token each of T sequences, somewhere in its last block
        slots = perm[:T] * bs + torch.randint(0, bs, (T,), generator=rng)
    else:                                # prompts one after the other, each in whole blocks of its own
        lens, left = [], T
        while left > 0:
            n = min(left, int(torch.randint(1, max(2, T // 3), (1,), generator=rng)) if len(lens) < 32 else left)
            lens.append(n)
            left -= n
        starts, used = [], 0
        for n in lens:
            starts.append(perm[used + torch.arange(n) // bs] * bs + torch.arange(n) % bs)
            used += -(-n // bs)
        slots = torch.cat(starts)
    if T > 8:
        slots[T - 2] = -1                # a padding row
    dt = _DTYPES[case["dtype"]]
    k, ks = _pool(gen, nb, bs, hkv, d, 7.0)
    v, vs = _pool(gen, nb, bs, hkv, d, 0.0)
    loud = 1.0 + 7.0 * (torch.rand(hkv, d, generator=gen, device="cuda") < 0.05).float()
    new_k = (torch.randn(T, hkv, d, generator=gen, device="cuda") * loud).to(dt)
    new_v = torch.randn(T, hkv, d, generator=gen, device="cuda").to(dt)
    return dict(op="write", new_k=new_k, new_v=new_v, slots=slots.cuda(), k=k, v=v, ks=ks, vs=vs)


# ------------------------------------------------------------------ run
def run(s):
    if s["op"] == "decode":
        return _decode(s)
    if s["op"] == "write":
        return _write(s)
    return _logprobs(s)


def _decode(s):
    if own:
        from tinyvllm_b200.attention import paged_decode_attention_q8
        return paged_decode_attention_q8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["ctx"], s["n_heads"], s["n_kv_heads"],
                                         s["head_dim"], s["block_size"])
    B, W = s["tables"].shape
    hkv, d, bs = s["n_kv_heads"], s["head_dim"], s["block_size"]
    at = s["tables"].long()
    q = s["q"].float().view(B, hkv, s["n_heads"] // hkv, d)
    k = s["k"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float().mul_(s["ks"][at][:, :, None, :, None]).view(B, W * bs, hkv, d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)
    del k
    live = torch.arange(W * bs, device=q.device)[None, :] < s["ctx"][:, None]
    some = (s["ctx"] > 0)[:, None, None, None]
    score = score.masked_fill(~live[:, None, None, :], -math.inf)
    e = torch.exp(score - torch.where(some, score.amax(-1, keepdim=True), 0.0))
    p = e / torch.where(some, e.sum(-1, keepdim=True), 1.0)
    v = s["v"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float().mul_(s["vs"][at][:, :, None, :, None]).view(B, W * bs, hkv, d)
    out = torch.matmul(p, v.permute(0, 2, 1, 3))
    return out.view(B, 1, s["n_heads"], d).to(s["q"].dtype)


def _write(s):
    if own:
        from tinyvllm_b200 import layers
        layers.write_kv_slots_q8(s["new_k"], s["new_v"], s["slots"], s["k"], s["v"], s["ks"], s["vs"])
        return s["k"], s["v"], s["ks"], s["vs"]
    nb, bs = s["k"].shape[:2]
    slots, T = s["slots"], s["slots"].shape[0]
    ok = (slots >= 0) & (slots < nb * bs)
    row = torch.full((nb * bs + 1,), -1, dtype=torch.int64, device=slots.device)   # the last row given for each slot
    row = row.scatter_reduce(0, torch.where(ok, slots, nb * bs), torch.arange(T, device=slots.device), "amax")
    row = row[:-1].view(nb, bs)
    new = row >= 0
    touched, started = new.any(1)[:, None], new[:, 0][:, None]
    _write_one(s["new_k"], row, new, touched, started, s["k"], s["ks"])
    _write_one(s["new_v"], row, new, touched, started, s["v"], s["vs"])
    return s["k"], s["v"], s["ks"], s["vs"]


def _write_one(x, row, new, touched, started, codes, scale):
    y = x.float()[row.clamp(min=0)]
    fine = torch.isfinite(y) & new[:, :, None, None]
    need = _scale_for(torch.where(fine, y.abs(), 0.0).amax(dim=(1, 3)))
    old = torch.where(started | ~(scale > 0), 0.0, scale)
    now = torch.maximum(old, need)
    kept = torch.where(started[:, :, None, None], 0.0, codes.float() * (old / now)[:, None, :, None])
    y = torch.where(torch.isfinite(y), y / now[:, None, :, None], math.nan)
    y = torch.where(new[:, :, None, None], y, kept)
    codes.copy_(torch.where(touched[:, :, None, None], _to_e4m3(y).float(), codes.float()))
    scale.copy_(torch.where(touched, now, scale))


def _logprobs(s):
    x, tok, n = s["logits"], s["tokens"], s["top_k"]
    if own:
        from tinyvllm_b200 import layers
        r = layers.token_logprobs(x, tok, n)
        return r.logprobs, r.entropy, r.top_logprobs, r.top_tokens
    y = x.float()
    vocab = y.shape[-1]
    low = y - y.amax(-1, keepdim=True)
    e = torch.exp(low)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    t = tok.long()
    inside = (t >= 0) & (t < vocab)
    chosen = torch.gather(low, 1, t.clamp(0, vocab - 1)[:, None])[:, 0] - log_total[:, 0]
    chosen = torch.where(inside, chosen, -math.inf)
    entropy = log_total[:, 0] - torch.where(e > 0, e * low, 0.0).sum(-1) / total[:, 0]
    # larger values first, equal ones by index: one whole number per logit that orders both
    bits = (y + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 20) + (vocab - 1 - torch.arange(vocab, device=y.device))
    top = vocab - 1 - (torch.topk(order, n, dim=-1).values & ((1 << 20) - 1))
    return chosen, entropy, torch.gather(low, 1, top) - log_total, top.int()


# ------------------------------------------------------------------ work
def work(case):
    if case["op"] == "decode":
        # the mean context: what a call has to read of the pool depends on the seed's lengths
        tokens = case["batch"] * (case["ctx_lo"] + case["ctx_hi"]) / 2
        es = _DTYPES[case["dtype"]].itemsize
        kv = 2 * case["n_kv_heads"] * case["head_dim"]
        blocks = tokens / case["block_size"]
        return {"bytes": tokens * kv + blocks * (8 * case["n_kv_heads"] + 4) + 2 * case["batch"] * case["n_heads"] * case["head_dim"] * es
                + 4 * case["batch"], "flops": 4 * case["n_heads"] * case["head_dim"] * tokens}
    if case["op"] == "write":
        row = 2 * case["n_kv_heads"] * case["head_dim"]
        blocks = case["rows"] if case["kind"] == "step" else case["rows"] / case["block_size"]
        return {"bytes": case["rows"] * (row * (_DTYPES[case["dtype"]].itemsize + 1) + 8) + 16 * blocks * case["n_kv_heads"],
                "flops": 3 * case["rows"] * row}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * _DTYPES[case["dtype"]].itemsize + case["rows"] * (12 + 8 * case["top_k"]), "flops": 5 * n}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "decode":
        return _exact_decode(s)
    if s["op"] == "write":
        return _exact_write(s)
    x = s["logits"].double()
    lse = torch.logsumexp(x, -1)
    logp = x - lse[:, None]
    entropy = -(logp.exp() * logp).sum(-1)
    best = torch.sort(logp, dim=-1, descending=True).values[:, :s["top_k"]] if x.numel() < 1 << 24 else \
        torch.topk(logp, s["top_k"], dim=-1).values
    return logp[torch.arange(len(x), device=x.device), s["tokens"].long()], entropy, best, None


def _exact_decode(s):
    """One sequence at a time, each on its own live tokens only."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    bs, group = s["block_size"], s["n_heads"] // s["n_kv_heads"]
    for b, n in enumerate(s["ctx"].tolist()):
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        block, row = s["tables"][b].long()[at // bs], at % bs
        k = s["k"].view(torch.uint8)[block, row].view(torch.float8_e4m3fn).double() * s["ks"][block].double()[..., None]
        v = s["v"].view(torch.uint8)[block, row].view(torch.float8_e4m3fn).double() * s["vs"][block].double()[..., None]
        q = s["q"][b, 0].double().unflatten(0, (s["n_kv_heads"], group))
        w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) * s["head_dim"] ** -0.5, -1)
        out[b, 0] = torch.einsum("hgt,thd->hgd", w, v).flatten(0, 1)
    return out


def _round_e4m3(y):
    """Nearest value with three fraction bits and exponents from -6 up, ties to even, of doubles within +-448."""
    exponent = torch.frexp(y).exponent.clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(y), exponent - 3)
    return torch.round(y / step) * step


def _exact_write(s):
    nb, bs = s["k"].shape[:2]
    last = {}
    for t, slot in enumerate(s["slots"].tolist()):
        if 0 <= slot < nb * bs:
            last.setdefault(slot // bs, {})[slot % bs] = t
    blocks = torch.tensor(sorted(last), device="cuda", dtype=torch.int64)
    rows = torch.tensor([[last[b].get(o, -1) for o in range(bs)] for b in sorted(last)], device="cuda")
    outs = []
    for x, codes, scale in ((s["new_k"], s["k"], s["ks"]), (s["new_v"], s["v"], s["vs"])):
        value, size = codes.double(), scale.double()
        if len(blocks):
            x = x.double()[rows.clamp(min=0)] * (rows >= 0)[..., None, None]
            need = x.abs().amax(dim=(1, 3))
            need = torch.exp2(torch.ceil(torch.log2(need.clamp(min=2.0 ** MIN_SCALE_EXP * E4M3_MAX) / E4M3_MAX)))
            fresh = (rows[:, 0] >= 0)[:, None]
            old = torch.where(fresh, 0.0, size[blocks])
            now = torch.maximum(old, need)
            kept = torch.where(fresh[:, :, None, None], 0.0, value[blocks] * (old / now)[:, None, :, None])
            value[blocks] = _round_e4m3(torch.where((rows >= 0)[..., None, None], x / now[:, None, :, None], kept))
            size[blocks] = now
        outs += [value, size]
    return outs[0], outs[2], outs[1], outs[3]
