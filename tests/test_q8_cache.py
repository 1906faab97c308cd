"""The 8-bit K/V cache on the GPU: the write and the decode attention against 64-bit restatements.

The write is exact: codes and scales equal the restatement's bit for bit.  Attention errors are
bounded per element by what the kernel rounds (u = half a step of the output type):
  u |out|                          the output's rounding
  2^-10 sum p|v|                   weights as halves before P.V (16-bit queries): 2^-11 on the weight, and
                                   the sum that normalises them is not rounded, so twice that at most
  2 ds sum p|v|                    fp32 scores off by ds = (D + 16) 2^-23 max_t sum_d |q k| / sqrt(D), and with 16-bit
                                   queries by 2^-25 max|q| max_t sum_d |k| / sqrt(D): a query row, its maximum scaled to
                                   2^7 or more, is a sum of e4m3 parts, the last scaled by 2^8, down to half of 2^-17
  (n + 16) 2^-23 sum p|v|          n fp32 additions in the output and in the normaliser
  n 2^-23 max|v|                   weights below half the last step of their parts (2^-18, where the largest counts as
                                   2^4 or more: 2^-23 of the largest)
"""

import math

import numpy as np
import pytest
import torch

from oracle import q8

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _vals(codes):
    return codes.cpu().view(torch.uint8).view(torch.float8_e4m3fn).double().numpy()


def _codes(rng, shape, lo=-1.0, hi=1.0):
    return torch.from_numpy(np.clip(rng.normal(size=shape) * 60, -448, 448)).float().to(torch.float8_e4m3fn)


def _case(dev, B, hq, hkv, d, bs, ctx, dtype, seed, width=None, extra=3, scale=None, kscale=0.02):
    rng = np.random.default_rng(seed)
    need = [-(-c // bs) for c in ctx]
    n = sum(need) + extra
    width = width or max(1, max(need))
    bt = np.zeros((B, width), dtype=np.int32)
    perm, at = rng.permutation(n), 0
    for b, m in enumerate(need):
        bt[b, :m] = perm[at:at + m]
        at += m
    k, v = _codes(rng, (n, bs, hkv, d)), _codes(rng, (n, bs, hkv, d))
    ks = torch.from_numpy(kscale * 2.0 ** rng.integers(-2, 3, (n, hkv)) * rng.uniform(0.5, 1, (n, hkv))).float()
    vs = torch.from_numpy(0.02 * 2.0 ** rng.integers(-3, 4, (n, hkv))).float() if scale is None else scale(rng, n, hkv)
    q = torch.from_numpy(rng.normal(size=(B, 1, hq, d))).to(dtype)
    c = dict(q=q, k=k, v=v, ks=ks, vs=vs, bt=torch.from_numpy(bt), ctx=torch.tensor(ctx, dtype=torch.int32))
    c = {a: t.to(dev) for a, t in c.items()}
    c.update(hq=hq, hkv=hkv, d=d, bs=bs)
    return c


def _run(c, **kw):
    from tinyvllm_b200.attention import paged_decode_attention_q8
    return paged_decode_attention_q8(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["bt"], c["ctx"], c["hq"], c["hkv"], c["d"], c["bs"], **kw)


def _expect(c, mcl=None):
    n = lambda t: t.cpu().double().numpy()
    return q8.paged_decode(n(c["q"]), _vals(c["k"]), _vals(c["v"]), n(c["ks"]), n(c["vs"]), c["bt"].cpu().numpy(), c["ctx"].cpu().numpy(), mcl)


def _bound(c, ref):
    out, mass, span, wide, vmax = ref
    n = int(c["ctx"].max())
    ds = (c["d"] + 16) * 2.0 ** -23 * span[:, None, :, None]
    if c["q"].dtype != torch.float32:
        ds = ds + 2.0 ** -25 * wide[:, None, :, None]
    p = 2.0 ** -10 if c["q"].dtype != torch.float32 else 0.0
    return U[c["q"].dtype] * np.abs(out) * (1 + 2.0 ** -6) + (p + 2 * ds + (n + 16) * 2.0 ** -23) * mass + n * 2.0 ** -23 * vmax[:, None, :, None]


def _check(c, got, mcl=None, ref=None):
    ref = ref or _expect(c, mcl)
    g = got.cpu().double().numpy()
    assert np.isfinite(g).all()
    over = np.abs(g - ref[0]) - _bound(c, ref)
    assert over.max() <= 0, f"{over.max()} over the bound at {np.unravel_index(over.argmax(), over.shape)}"


TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 8), (12, 3), (32, 4), (32, 2), (5, 1), (9, 1), (20, 5)])
def test_head_layouts(cuda, dtype, d, hq, hkv):
    ctx = [1, 15, 16, 17, 63, 64, 65, 129, 300, 700]
    c = _case(cuda, len(ctx), hq, hkv, d, 16, ctx, dtype, hq * 7 + d)
    _check(c, _run(c, check=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bs", [1, 5, 8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_block_sizes(cuda, dtype, bs, d):
    ctx = [1, bs, bs + 1, 3 * bs + 2, 200]
    c = _case(cuda, len(ctx), 16, 4, d, bs, ctx, dtype, bs)
    _check(c, _run(c, check=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_truncated_and_padded_rows(cuda, dtype):
    c = _case(cuda, 6, 8, 2, 64, 16, [0, 40, 0, 64, 33, 0], dtype, 3, width=64)
    c["ctx"][5] = -4
    ref = _expect(c)
    out = _run(c)
    assert not out[0].any() and not out[2].any() and not out[5].any()
    _check(c, out, ref=ref)
    c["ctx"][3] = 5000                      # beyond the table: cut at its end
    c["bt"] = c["bt"][:, :4].contiguous()
    _check(c, _run(c))
    for mcl in (0, 1, 16, 17, 1000):
        _check(c, _run(c, max_context_len=mcl), mcl=mcl)
    c["ctx"].zero_()
    assert not _run(c).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,ctx", [(1, [5000]), (1, [33000]), (3, [9000, 1, 4097]), (2, [12000, 12000])])
def test_long_contexts_shared_by_ctas(cuda, dtype, B, ctx):
    c = _case(cuda, B, 8, 2, 128, 16, ctx, dtype, B + sum(ctx))
    _check(c, _run(c, check=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,d", [(1, 128), (4, 64), (7, 32), (16, 128)])
def test_one_head_shared_by_all_ctas(cuda, dtype, hq, d):
    """One KV head: every CTA has a part of its one unit (or of each few query heads), more parts than are joined at a time."""
    c = _case(cuda, 1, hq, 1, d, 16, [70001], dtype, hq)
    _check(c, _run(c, check=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences(cuda, dtype):
    rng = np.random.default_rng(4)
    ctx = [int(x) for x in rng.integers(0, 90, 700)]
    c = _case(cuda, len(ctx), 4, 2, 64, 16, ctx, dtype, 5)
    _check(c, _run(c, check=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_lies_behind_a_context_is_not_used(cuda, dtype):
    """NaN codes and scales in the rows and blocks behind the last token, and in table padding."""
    for d, bs in ((32, 16), (64, 8), (128, 16), (128, 64)):
        c = _case(cuda, 4, 8, 4, d, bs, [1, 17, 70, 130], dtype, 9, width=40)
        want = _run(c).clone()
        live = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
        for b, n in enumerate(c["ctx"].tolist()):
            for t in range(n):
                live[int(c["bt"][b, t // bs]), t % bs] = True
        dead = (~live).to(cuda)
        for x in (c["k"], c["v"]):
            x.view(torch.uint8)[dead] = 0x7F
        none = dead.all(1)
        c["ks"][none] = float("nan")
        c["vs"][none] = float("inf")
        pad = int(none.nonzero()[0])
        for b, n in enumerate(c["ctx"].tolist()):
            c["bt"][b, -(-n // bs):] = pad if b % 2 else 10 ** 6
        assert torch.equal(_run(c), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_block_ids_outside_the_pool_read_as_zeros(cuda, dtype):
    c = _case(cuda, 3, 8, 4, 64, 16, [40, 100, 64], dtype, 10)
    c["bt"][0, 1], c["bt"][1, 0], c["bt"][2, 3] = -1, c["k"].shape[0], 2 ** 31 - 1
    _check(c, _run(c))


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_in_a_live_row_reaches_its_heads_only(cuda, dtype):
    c = _case(cuda, 2, 8, 4, 64, 16, [40, 100], dtype, 11)
    c["k"].view(torch.uint8)[c["bt"][0, 1].long(), 3, 2, 5] = 0x7F
    out = _run(c)
    assert torch.isnan(out[0, 0, 4:6]).all()
    assert torch.isfinite(out[0, 0, :4]).all() and torch.isfinite(out[0, 0, 6:]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_far_apart(cuda, dtype):
    """Block scales of 2^-40 to 2^12 in one sequence: each block counts as it is."""
    c = _case(cuda, 3, 8, 2, 128, 16, [300, 64, 1000], dtype, 12,
              scale=lambda rng, n, h: torch.from_numpy(2.0 ** rng.integers(-40, 7, (n, h))).float())
    _check(c, _run(c))


def test_loud_and_quiet_queries(cuda):
    """bf16 queries beyond the range of a half, and rows of zeros."""
    for mul, ks in ((2.0 ** 30, 2.0 ** -36), (2.0 ** -40, 2.0 ** 34)):
        c = _case(cuda, 3, 8, 2, 64, 16, [100, 64, 30], torch.bfloat16, 13, kscale=ks)
        c["q"] = c["q"] * mul
        c["q"][1, 0, 3] = 0
        c["q"][2, 0, 0, 1:] = 0
        _check(c, _run(c))


def test_repeated_and_relabelled_calls_agree_to_the_bit(cuda):
    c = _case(cuda, 5, 32, 8, 128, 16, [3000, 1, 700, 64, 9000], torch.bfloat16, 14)
    a = _run(c)
    for _ in range(5):
        assert torch.equal(_run(c), a)
    n = c["k"].shape[0]
    perm = torch.randperm(n, device=cuda)
    inv = torch.empty_like(perm)
    inv[perm] = torch.arange(n, device=cuda)
    for x in ("ks", "vs"):
        c[x] = c[x][perm].contiguous()
    for x in ("k", "v"):
        c[x] = c[x].view(torch.uint8)[perm].view(torch.float8_e4m3fn).contiguous()
    c["bt"] = inv[c["bt"].long()].int()
    assert torch.equal(_run(c), a)


def test_offsets_beyond_32_bits(cuda):
    """A pool of more than 2^32 codes a side; the sequence lies at its end."""
    n, bs, hkv, d = 131100 * 2, 16, 8, 128
    k = torch.zeros(n, bs, hkv, d, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    v = torch.zeros(n, bs, hkv, d, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    ks, vs = torch.zeros(n, hkv, device=cuda), torch.zeros(n, hkv, device=cuda)
    from tinyvllm_b200 import layers
    rng = np.random.default_rng(1)
    ctx = 50
    blocks = [n - 1, 3, n - 7, 131073]
    x = [torch.from_numpy(rng.normal(size=(ctx, hkv, d))).half().to(cuda) for _ in range(2)]
    slots = torch.tensor([blocks[t // bs] * bs + t % bs for t in range(ctx)], device=cuda)
    layers.write_kv_slots_q8(x[0], x[1], slots, k, v, ks, vs)
    small = [t[torch.tensor(blocks, device=cuda)] for t in (k.view(torch.uint8), v.view(torch.uint8), ks, vs)]
    for dtype in (torch.float16, torch.float32):
        c = dict(q=torch.from_numpy(rng.normal(size=(1, 1, 32, d))).to(dtype).to(cuda), k=k, v=v, ks=ks, vs=vs,
                 bt=torch.tensor([blocks], dtype=torch.int32, device=cuda), ctx=torch.tensor([ctx], dtype=torch.int32, device=cuda), hq=32, hkv=hkv, d=d,
                 bs=bs)
        got = _run(c)
        c.update(k=small[0].view(torch.float8_e4m3fn), v=small[1].view(torch.float8_e4m3fn), ks=small[2], vs=small[3],
                 bt=torch.arange(4, dtype=torch.int32, device=cuda)[None])
        assert small[2].count_nonzero() == 4 * hkv
        _check(c, got)


# ------------------------------------------------------------------ the write
def _write_case(dev, T, hkv, d, bs, n, dtype, seed, slots):
    rng = np.random.default_rng(seed)
    x = [torch.from_numpy(rng.normal(size=(T, hkv, d)) * 2.0 ** rng.integers(-9, 9, (T, hkv, 1))).to(dtype).to(dev) for _ in range(2)]
    codes = [_codes(rng, (n, bs, hkv, d)).to(dev) for _ in range(2)]
    scale = [torch.from_numpy(2.0 ** rng.integers(-9, 4, (n, hkv))).float().to(dev) for _ in range(2)]
    return x, codes, scale, torch.tensor(slots(rng), dtype=torch.int64, device=dev)


def _check_write(x, codes, scale, slots):
    from tinyvllm_b200 import layers
    want = [q8.write_kv_slots(x[i].double().cpu().numpy(), slots.cpu().numpy(), _vals(codes[i]), scale[i].cpu().numpy()) for i in range(2)]
    layers.write_kv_slots_q8(x[0], x[1], slots, codes[0], codes[1], scale[0], scale[1])
    for i in range(2):
        np.testing.assert_array_equal(scale[i].cpu().double().numpy(), want[i][1])
        np.testing.assert_array_equal(_vals(codes[i]), want[i][0])


SLOTS = {
    "one": lambda n, bs, T: lambda rng: [int(rng.integers(0, n * bs))] * 1 + [-1] * (T - 1),
    "one_each": lambda n, bs, T: lambda rng: (rng.permutation(n)[:T] * bs + rng.integers(0, bs, T)).tolist() if T <= n else rng.permutation(n * bs)[:T].tolist(),
    "run": lambda n, bs, T: lambda rng: (bs // 2 + np.arange(T)).tolist(),
    "reversed": lambda n, bs, T: lambda rng: (bs // 2 + np.arange(T))[::-1].tolist(),
    "any": lambda n, bs, T: lambda rng: rng.integers(-5, n * bs + 5, T).tolist(),       # with repeats, skips and rows of one block far apart
    "same": lambda n, bs, T: lambda rng: [bs + 1] * T,
    "nothing": lambda n, bs, T: lambda rng: [-1, n * bs, 2 ** 62, -2 ** 62][:T] + [-7] * max(0, T - 4),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("kind", sorted(SLOTS))
@pytest.mark.parametrize("hkv,d,bs", [(4, 64, 16), (1, 128, 8), (5, 32, 64), (8, 128, 16), (3, 48, 7), (2, 256, 1)])
def test_write_matches_bit_for_bit(cuda, dtype, T, kind, hkv, d, bs):
    n = 60
    _check_write(*_write_case(cuda, T, hkv, d, bs, n, dtype, T + bs, SLOTS[kind](n, bs, T)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,n", [(3000, 300), (2500, 40), (700, 700)])
def test_write_many_rows(cuda, dtype, T, n):
    bs = 16
    kind = "run" if T > n * bs // 4 and n == 300 else "any"
    _check_write(*_write_case(cuda, T, 2, 64, bs, n, dtype, T, SLOTS[kind](n, bs, T)))


@pytest.mark.parametrize("dtype", TYPES)
def test_write_of_special_values(cuda, dtype):
    """Infinities and NaN become NaN and leave the scale alone; zeros, the smallest and the largest values; bad old scales."""
    bs, n, hkv, d = 16, 6, 2, 32
    x, codes, scale, slots = _write_case(cuda, 8, hkv, d, bs, n, dtype, 5, lambda rng: [0, 1, 17, 33, 50, 64, 65, 81])
    big = torch.finfo(dtype).max
    for y in x:
        y[0, 0, 3], y[1, 1, 0], y[2, 0, 1] = float("inf"), float("nan"), -float("inf")
        y[3] = 0
        y[4, 0] = float("nan")
        y[5], y[6] = big, torch.finfo(dtype).smallest_normal
    for s in scale:
        s[1, 0], s[1, 1], s[2, 0], s[2, 1] = float("nan"), -1.0, 0.0, float("inf")
    _check_write(x, codes, scale, slots)


def test_write_twice_changes_nothing(cuda):
    x, codes, scale, slots = _write_case(cuda, 40, 4, 64, 16, 60, torch.float16, 6, SLOTS["any"](60, 16, 40))
    _check_write(x, codes, scale, slots)
    before = [t.clone() for t in (*[c.view(torch.uint8) for c in codes], *scale)]
    from tinyvllm_b200 import layers
    layers.write_kv_slots_q8(x[0], x[1], slots, codes[0], codes[1], scale[0], scale[1])
    for a, b in zip(before, (*[c.view(torch.uint8) for c in codes], *scale)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [8192, 8193, 30011])
@pytest.mark.parametrize("kind", ["run", "reversed", "any", "same", "nothing", "prompts"])
def test_write_of_many_rows(cuda, T, kind):
    """Calls that look for a block's rows by classes of blocks, and the last that does not."""
    n, bs = T // 16 + 40, 16

    def prompts(rng):                       # runs over blocks in any order, each from a block's start, with skipped rows
        blocks, out = list(rng.permutation(n)), []
        while len(out) < T:
            m = int(rng.integers(1, 400))
            own = [blocks.pop() for _ in range(-(-m // bs))] if len(blocks) * bs > 400 else []
            out += [int(b) * bs + o for b in own for o in range(bs)][:m] if own else [-1] * m
        return out[:T]

    make = prompts if kind == "prompts" else SLOTS[kind](n, bs, T)
    _check_write(*_write_case(cuda, T, 1, 32, bs, n, torch.bfloat16, T, make))


def test_long_writes_at_once_and_recorded(cuda):
    """Long calls on two streams and from two graphs at the same time, each with a workspace of its own."""
    from tinyvllm_b200 import layers
    T, n = 20000, 1300
    cs = [_write_case(cuda, T, 2, 64, 16, n, torch.float16, s, lambda rng: (rng.permutation(n - 1)[:, None] * 16 + np.arange(16)).reshape(-1)[:T].tolist()) for s in (1, 2)]
    want = []
    for x, codes, scale, slots in cs:
        c, s = [t.clone() for t in codes], [t.clone() for t in scale]
        layers.write_kv_slots_q8(x[0], x[1], slots, *c, *s)
        want.append([t.view(torch.uint8).clone() for t in c])
    streams, graphs, rec = [torch.cuda.Stream(), torch.cuda.Stream()], [], torch.cuda.Stream()
    call = lambda c: layers.write_kv_slots_q8(c[0][0], c[0][1], c[3], *c[1], *c[2])
    torch.cuda.synchronize()
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=rec):
            call(c)
        graphs.append(g)
    for use in (lambda i: call(cs[i]), lambda i: graphs[i].replay()):
        for c in cs:
            for t in c[1]:
                t.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        for _ in range(8):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    use(i)
        torch.cuda.synchronize()
        for c, w in zip(cs, want):
            started = torch.zeros(n, dtype=torch.bool, device=cuda)
            started[c[3][c[3] % 16 == 0] // 16] = True
            assert all(torch.equal(t.view(torch.uint8)[started], v[started]) for t, v in zip(c[1], w))


# ------------------------------------------------------------------ how they are called
def test_python_refusals(cuda):
    from tinyvllm_b200 import layers
    from tinyvllm_b200._lib import TvkError
    c = _case(cuda, 2, 8, 4, 64, 16, [40, 100], torch.float16, 1)
    for name, bad, err in (("k", c["k"].float(), TypeError), ("ks", c["ks"].half(), TypeError), ("vs", c["vs"][:, :2], ValueError),
                           ("bt", c["bt"].long(), TypeError), ("ctx", c["ctx"][:1], ValueError), ("q", c["q"].double(), TypeError),
                           ("q", c["q"][:, :, ::2], ValueError), ("v", c["v"].view(torch.uint8)[:-1].view(torch.float8_e4m3fn), ValueError),
                           ("q", torch.zeros(2 * 8 * 64 + 1, dtype=torch.float16, device=cuda)[1:].view(2, 1, 8, 64), TvkError)):
        with pytest.raises(err):
            _run({**c, name: bad})
    with pytest.raises(ValueError):
        _run(c, out=torch.empty(2, 1, 8, 64, device=cuda))
    room = torch.zeros(2 * c["q"].numel(), dtype=c["q"].dtype, device=cuda)
    q = room[:c["q"].numel()].view(c["q"].shape)
    for off in (0, 8, c["q"].numel() - 8):
        with pytest.raises(TvkError, match="overlap"):
            _run({**c, "q": q}, out=room[off:off + q.numel()].view(q.shape))
    x, codes, scale, slots = _write_case(cuda, 4, 2, 64, 16, 8, torch.float16, 6, lambda rng: [0, 1, 2, 3])
    good = [*x, slots, *codes, *scale]
    for i, bad, err in ((0, x[0].double(), TypeError), (2, slots.int(), TypeError), (2, slots[:3], TypeError), (3, codes[0].float(), TypeError),
                        (5, scale[0][:4], ValueError), (6, scale[1].double(), TypeError), (1, x[1][:, :1], ValueError), (0, x[0][:, :, ::2], ValueError)):
        with pytest.raises(err):
            layers.write_kv_slots_q8(*[bad if j == i else t for j, t in enumerate(good)])


def test_two_streams_and_captured_graphs(cuda):
    """Calls on two streams at once, each with its own workspace, and a graph replayed between eager calls."""
    cs = [_case(cuda, 3, 32, 8, 128, 16, [5000, 700, 9000], torch.bfloat16, s) for s in (1, 2)]
    want = [_run(c).clone() for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_run(cs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    out = torch.empty_like(want[0])
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        _run(cs[0], out=out)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        _run(cs[0], out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        other = _run(cs[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(other, want[1])


def test_two_graphs_recorded_on_one_stream_replay_at_once(cuda):
    """Each recorded graph has a workspace of its own: both split their sequences over CTAs, and run on two streams."""
    cs = [_case(cuda, B, 32, 8, 128, 16, ctx, torch.bfloat16, s) for s, B, ctx in ((1, 3, [5000, 700, 9000]), (2, 40, [3000] * 40))]
    want = [_run(c).clone() for c in cs]
    outs, graphs = [torch.empty_like(w) for w in want], []
    rec = torch.cuda.Stream()
    for c, o in zip(cs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=rec):
            for _ in range(3):
                _run(c, out=o)
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_branches_of_one_graph_and_many_recordings(cuda):
    """Two branches of a graph that may run at once each have a workspace, and recordings of graphs that are dropped leave no memory behind."""
    cs = [_case(cuda, 3, 32, 8, 128, 16, ctx, torch.float16, s) for s, ctx in ((1, [5000, 700, 9000]), (2, [8000, 0, 3000]))]
    want = [_run(c).clone() for c in cs]
    outs = [torch.empty_like(w) for w in want]
    main, side = torch.cuda.Stream(), torch.cuda.Stream()

    def record():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=main):
            side.wait_stream(main)
            with torch.cuda.stream(side):
                for _ in range(4):
                    _run(cs[1], out=outs[1])
            for _ in range(4):
                _run(cs[0], out=outs[0])
            main.wait_stream(side)
        return g

    g = record()
    for _ in range(10):
        for o in outs:
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    held = []
    for _ in range(6):
        del g
        g = record()
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated())
    assert held[-1] == held[1]


def test_wait_that_runs_out_is_told_and_the_next_call_is_right(cuda):
    """The producers issue nothing (test hook): the kernel's waits run out, it says so and returns."""
    from tinyvllm_b200 import _lib
    from tinyvllm_b200.attention import workspace_status
    c = _case(cuda, 6, 32, 8, 128, 16, [5, 70, 300, 900, 1500, 21000], torch.float16, 41)
    want = _run(c, check=True).clone()
    assert _lib.lib().tvk_debug_arm_wait_timeout(5_000_000) == 0
    with pytest.raises(_lib.TvkError, match="timed out"):
        _run(c, check=True)
    assert workspace_status(cuda, "decode_q8") == 0
    assert torch.equal(_run(c, check=True), want)
