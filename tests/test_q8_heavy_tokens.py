"""8-bit decode where one token has nearly all of the weight and a long tail shares the rest (GPU).

A first token that every later one attends to is ordinary, and its value is often small, so the tail's
weights, each 2^-20 to 2^-30 of the largest, make a good part of the output.  Bound per output element (u: half a
step of the output type; n tokens; p, v the exact weights and values):
  u |out|                     the output's rounding
  2^-14 sum p|v|              a weight of 16-bit queries is the sum of four e5m2 parts: what is left of w < 2^(e + 1) is at
                              most 2^(e - 3) after the first, and that as a half 2^(e - 15), which the other three hold
                              exactly; 2^-15 of w, and the sum that normalises them is not rounded, so twice that at most
  2 ds sum p|v|               fp32 scores off by ds = (D + 16) 2^-23 max_t sum_d |q k| / sqrt(D), with 16-bit queries and
                              2^-25 max|q| max_t sum_d |k| / sqrt(D)
  (n + 16) 2^-23 sum p|v|     n fp32 additions in the output and in the normaliser
  n 2^-36 max|v|              a half is off by 2^-25 at least, where the largest weight counts as 2^11 or more
"""

import math

import numpy as np
import pytest
import torch

from oracle import q8

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BS = 16


def _round_codes(x):
    return torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn)


def _sequence(hq, hkv, d, n, heavy, dtype, seed):
    """One sequence of n tokens whose first has about ``heavy`` of every head's weight and values of some 0.02; the others' values
    scatter about a mean of their own in every dim."""
    rng = np.random.default_rng(seed)
    g, blocks = hq // hkv, -(-n // BS)
    u = rng.normal(size=(hkv, 1, d))
    q = torch.from_numpy((u + 0.3 * rng.normal(size=(hkv, g, d))).reshape(1, 1, hq, d)).to(dtype)
    k = rng.normal(size=(blocks * BS, hkv, d)) * 60
    ks = 2.0 ** -6
    want = math.log(heavy / (1 - heavy) * n) + 0.5         # of scores N(0, 1) each exp() is worth e^0.5
    k[0] = u[:, 0] * (want * math.sqrt(d) / (ks * (u * u).sum(-1)))
    v = (rng.normal(size=(1, hkv, d)) + 0.5 * rng.normal(size=(blocks * BS, hkv, d))) * 64
    v[0] = rng.normal(size=(hkv, d)) * 0.02 * 64
    shape = (blocks, BS, hkv, d)
    scale = torch.full((blocks, hkv), 2.0 ** -6)
    return q, _round_codes(k.reshape(shape)), _round_codes(v.reshape(shape)), scale


def _vals(codes):
    return codes.view(torch.uint8).view(torch.float8_e4m3fn).double().numpy()


def _bound(ref, d, n, dtype):
    out, mass, span, wide, vmax = ref
    few = dtype != torch.float32
    ds = (d + 16) * 2.0 ** -23 * span[:, None, :, None] + (2.0 ** -25 * wide[:, None, :, None] if few else 0.0)
    return U[dtype] * np.abs(out) * (1 + 2.0 ** -6) + ((2.0 ** -14 if few else 0.0) + 2 * ds + (n + 16) * 2.0 ** -23) * mass \
        + n * 2.0 ** -36 * vmax[:, None, :, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 128), (32, 2, 128), (8, 2, 64), (16, 2, 64), (8, 4, 32)])
@pytest.mark.parametrize("n,heavy,batch", [(8192, 0.999, 160), (16384, 0.99, 160), (28000, 0.99, 160), (50000, 0.9999, 48), (20000, 0.999, 1)])
def test_tail_behind_a_heavy_first_token(cuda, dtype, hq, hkv, d, n, heavy, batch):
    """A large batch, so that one CTA holds most of a sequence (all rows are the same sequence), and one by itself."""
    from tinyvllm_b200.attention import paged_decode_attention_q8
    q, k, v, scale = _sequence(hq, hkv, d, n, heavy, dtype, n + hq + d)
    tables = torch.randperm(k.shape[0], generator=torch.Generator().manual_seed(n)).int()[None]
    at = torch.empty_like(k.view(torch.uint8)), torch.empty_like(v.view(torch.uint8))
    for dst, src in zip(at, (k, v)):
        dst[tables[0].long()] = src.view(torch.uint8)
    k, v = (x.view(torch.float8_e4m3fn) for x in at)
    ctx = torch.tensor([n], dtype=torch.int32)
    n64 = lambda t: t.double().numpy()
    ref = q8.paged_decode(n64(q), _vals(k), _vals(v), n64(scale), n64(scale), tables.numpy(), ctx.numpy())
    many = lambda t: t.to(cuda).expand(batch, *t.shape[1:]).contiguous()
    got = paged_decode_attention_q8(many(q), k.to(cuda), v.to(cuda), scale.to(cuda), scale.to(cuda), many(tables), ctx.to(cuda).expand(batch).contiguous(),
                                    hq, hkv, d, BS, check=True).cpu().double().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - ref[0]) - _bound(ref, d, n, dtype)
    off = (np.abs(got - ref[0]) / ref[1]).max()
    assert over.max() <= 0, f"{over.max()} over the bound; off by {off} of sum p|v|"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,d", [(4, 128), (16, 128), (8, 64), (4, 32)])
@pytest.mark.parametrize("at", [0, 700, 1999])
def test_heavy_token_anywhere(cuda, dtype, hq, d, at):
    """The reference moves when the heavy token comes: weights before it shrink, those behind it start small."""
    from tinyvllm_b200.attention import paged_decode_attention_q8
    n = 2000
    q, k, v, scale = _sequence(hq, 1, d, n, 0.9999, dtype, hq + d)
    for x in (k, v):
        rows = x.view(torch.uint8).view(-1, 1, d)
        first = rows[0].clone()
        rows[0] = rows[at]
        rows[at] = first
    tables, ctx = torch.arange(n // BS).int()[None], torch.tensor([n], dtype=torch.int32)
    n64 = lambda t: t.double().numpy()
    ref = q8.paged_decode(n64(q), _vals(k), _vals(v), n64(scale), n64(scale), tables.numpy(), ctx.numpy())
    batch = 300
    many = lambda t: t.to(cuda).expand(batch, *t.shape[1:]).contiguous()
    got = paged_decode_attention_q8(many(q), k.to(cuda), v.to(cuda), scale.to(cuda), scale.to(cuda), many(tables), ctx.to(cuda).expand(batch).contiguous(),
                                    hq, 1, d, BS, check=True).cpu().double().numpy()
    over = np.abs(got - ref[0]) - _bound(ref, d, n, dtype)
    assert over.max() <= 0, f"{over.max()} over the bound"
