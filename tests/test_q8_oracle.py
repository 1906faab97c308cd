"""The 64-bit restatements behind the 8-bit cache and log-probability tests, and every refusal that
needs no GPU (CPU)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import q8


def test_e4m3_values_and_rounding_match_torch():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    np.testing.assert_array_equal(q8.e4m3_values(), codes.double().numpy())
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.normal(size=5000) * s for s in (1e-3, 0.1, 1, 30, 150)] + [q8._POS, -q8._POS, (q8._POS[1:] + q8._POS[:-1]) / 2])
    x = np.clip(x, -448, 448).astype(np.float32)
    np.testing.assert_array_equal(q8.e4m3_round(x), torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("amax,k", [(0.0, -100), (448.0, 0), (448.0001, 1), (1.75, -8), (1.7500001, -7), (3.0e38, 120), (1e-40, -100)])
def test_scale_is_the_smallest_power_of_two(amax, k):
    assert q8.scale_for(amax) == 2.0 ** k


def test_growing_scale_keeps_the_rows_already_there():
    """Powers of two: a block's rows survive a louder row exactly unless they become subnormal."""
    x = np.array([[[1.0, -0.4375, 0.0625, 0.0]]])
    codes, scale = q8.write_kv_slots(x, [0], np.zeros((1, 4, 1, 4)), np.zeros((1, 1)))
    before = codes[0, 0, 0] * scale[0, 0]
    codes, scale = q8.write_kv_slots(x * 16, [1], codes, scale)
    np.testing.assert_array_equal(codes[0, 0, 0] * scale[0, 0], before)
    np.testing.assert_array_equal(before, x[0, 0])


def test_starting_a_block_drops_what_it_held_and_the_last_row_wins():
    codes, scale = np.full((1, 4, 1, 2), 300.0), np.full((1, 1), 8.0)
    codes, scale = q8.write_kv_slots(np.array([[[9.0, 9.0]], [[1.0, 0.5]], [[2.0, 3.0]]]), [0, 2, 0], codes, scale)
    np.testing.assert_array_equal(codes[0, :, 0] * scale[0, 0], [[2, 3], [0, 0], [1, 0.5], [0, 0]])
    assert scale[0, 0] == 2.0 ** -7          # 3 / 448: the row of nines does not count


def test_logprobs_rank_ties_by_index_and_nan_first():
    x = np.array([[1.0, 3.0, 3.0, -0.0, 0.0], [np.nan, 1.0, np.nan, 2.0, 0.0]])
    _, _, _, top, _, _ = q8.token_logprobs(x, [0, 0], 5)
    assert top.tolist() == [[1, 2, 0, 3, 4], [0, 2, 3, 1, 4]]


# ------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def lib():
    from tinyvllm_b200 import build
    build.build()
    from tinyvllm_b200 import _lib
    return _lib.lib()


P = 1 << 20      # an aligned address that nothing reads: every call below is refused first


def _decode(lib, **kw):
    a = dict(q=P, k=P, v=P, ks=P, vs=P, bt=P, ctx=P, out=P << 1, batch=2, hq=8, hkv=2, d=64, bs=16, nb=8, mb=4, mcl=-1, dt=1, ws=P, n=1 << 30)
    a.update(kw)
    rc = lib.tvk_paged_decode_attention_q8(*[a[k] for k in ("q", "k", "v", "ks", "vs", "bt", "ctx", "out", "batch", "hq", "hkv", "d", "bs",
                                                            "nb", "mb", "mcl", "dt", "ws", "n")], None)
    return rc, lib.tvk_last_error().decode()


@pytest.mark.parametrize("kw,rc,say", [
    (dict(q=None), -1, "null"), (dict(ks=None), -1, "null"), (dict(vs=None), -1, "null"), (dict(q=P + 4), -1, "aligned"),
    (dict(k=P + 8), -1, "aligned"), (dict(batch=-1), -1, "batch"), (dict(hq=7), -1, "multiple"), (dict(hq=64), -1, "exceeds"),
    (dict(d=96), -2, "head_dim"), (dict(d=256), -2, "head_dim"), (dict(bs=0), -1, "positive"), (dict(dt=3), -1, "dtype"),
    (dict(ws=None), -4, "workspace"), (dict(n=4096), -4, "workspace"), (dict(ws=P + 4), -1, "aligned"),
    (dict(out=P), -1, "overlap"), (dict(out=P + 2032), -1, "overlap"), (dict(out=P - 16), -1, "overlap"), (dict(mb=1 << 28), -1, "2^31"), (dict(batch=1 << 20, mb=1 << 20), -1, "32-bit"),
])
def test_decode_refuses(lib, kw, rc, say):
    got, msg = _decode(lib, **kw)
    assert got == rc and say in msg


def test_empty_calls_are_fine(lib):
    assert _decode(lib, batch=0, q=None, ws=None)[0] == 0
    assert lib.tvk_write_kv_slots_q8(None, None, None, None, None, None, None, 0, 2, 64, 8, 16, 1, None, 0, None) == 0
    assert lib.tvk_token_logprobs(None, None, None, None, None, None, 0, 10, 10, 0, 1, None) == 0


@pytest.mark.parametrize("args,rc,say", [
    ((None, P, P, P, P, P, P, 4, 2, 64, 8, 16, 1), -1, "null"), ((P, P, P, P, P, None, P, 4, 2, 64, 8, 16, 1), -1, "null"),
    ((P + 2, P, P, P, P, P, P, 4, 2, 64, 8, 16, 1), -1, "aligned"), ((P, P, P, P, P, P, P, -1, 2, 64, 8, 16, 1), -1, "n_tokens"),
    ((P, P, P, P, P, P, P, 4, 2, 24, 8, 16, 1), -1, "head_dim"), ((P, P, P, P, P, P, P, 4, 2, 64, 8, 2048, 1), -2, "block_size"),
    ((P, P, P, P, P, P, P, 4, 0, 64, 8, 16, 1), -1, "positive"), ((P, P, P, P, P, P, P, 4, 2, 64, 8, 16, 7), -1, "dtype"),
    ((P, P, P, P, P, P, P, 8193, 2, 64, 8, 16, 1), -4, "workspace"),
])
def test_write_refuses(lib, args, rc, say):
    assert lib.tvk_write_kv_slots_q8(*args, None, 0, None) == rc
    assert say in lib.tvk_last_error().decode()


@pytest.mark.parametrize("args,rc,say", [
    ((None, P, P, P, P, P, 4, 100, 100, 2, 1), -1, "null"), ((P, P, P, P, None, P, 4, 100, 100, 2, 1), -1, "null"),
    ((P, P, P, P, P, P, 4, 100, 99, 2, 1), -1, "shape"), ((P, P, P, P, P, P, 4, 100, 100, 33, 1), -1, "top_k"),
    ((P, P, P, P, P, P, 4, 5, 5, 6, 1), -1, "top_k"), ((P, P, P, P, P, P, 4, 100, 100, -1, 1), -1, "top_k"),
    ((P + 1, P, P, P, P, P, 4, 100, 100, 2, 1), -1, "aligned"), ((P, P, P, P, P, P, 4, 100, 100, 2, 9), -1, "dtype"),
])
def test_logprobs_refuses(lib, args, rc, say):
    assert lib.tvk_token_logprobs(*args, None) == rc
    assert say in lib.tvk_last_error().decode()


def test_workspace_size(lib):
    a, b = lib.tvk_paged_decode_q8_workspace_size(1, 1), lib.tvk_paged_decode_q8_workspace_size(256, 8)
    assert b - a == 4 * 4 * (256 * 8 - 1)      # up to four counters per (sequence, KV head)


def test_python_entry_points_refuse_cpu_tensors():
    from tinyvllm_b200 import attention, layers
    z = torch.zeros(1)
    with pytest.raises(RuntimeError, match="CUDA"):
        attention.paged_decode_attention_q8(z, z, z, z, z, z, z, 1, 1, 64, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        layers.write_kv_slots_q8(z, z, z, z, z, z, z)
    with pytest.raises(RuntimeError, match="CUDA"):
        layers.token_logprobs(z, z)
