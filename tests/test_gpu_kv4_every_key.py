"""Attention over the 4-bit cache takes every key once: cases in which a key left out, counted twice or
taken with another's value shows, at the edges of tiles, waves, rounds and pieces as anywhere."""
import numpy as np
import pytest

from nimbleml_amd import kernels as K
from oracle import kv4_ref as R
from test_gpu_kv4 import cache_of, normal

pytestmark = pytest.mark.gpu

DTYPES = [np.float16, np.float32]


def check_every_key(dtype, dk, kv, group, seq, lens, counts=None):
    """Equal scores (keys of zero): an output is Σ v / (keys seen). Key j has one value, a power of two
    at dim j % dk; a call's keys of one dim have different powers, so the sum names its keys. As many
    calls as it takes for every key to have had a value."""
    b, p = len(lens), max(1, max(lens))
    r = np.random.RandomState(dk + seq)
    q = r.randn(b, kv * group, seq, dk).astype(dtype)
    # powers that a sum holds exactly beside the division's rounding and, in float16, the output's
    bits = 8 if dtype == np.float16 else 20
    j = np.arange(p)
    n = [seq] * b if counts is None else list(counts)
    k = np.zeros((b, kv, p, dk), dtype)
    for first in range(0, p, dk * bits):
        here = (j >= first) & (j < first + dk * bits)
        row = np.zeros((p, dk))
        row[j[here], j[here] % dk] = 2.0 ** ((j[here] - first) // dk)
        v = np.broadcast_to(row, (b, kv, p, dk)).astype(dtype)
        got = K.kv4_attention(q, cache_of(k, v), np.array(lens), 1.0, counts).numpy()
        got = got.reshape(b, seq, kv * group, dk).astype(np.float64)
        upto = np.concatenate([np.zeros((1, dk)), np.cumsum(row, 0)])
        for i in range(b):
            for t in range(n[i]):
                seen = min(p, lens[i] - n[i] + t + 1)
                want = upto[seen] / seen if seen > 0 else np.zeros(dk)
                # p = 1 and the sums exact: the division rounds, then the output
                assert (np.abs(got[i, t] - want) <= want * (2.0**-22 + np.finfo(dtype).eps / 2)).all(), (i, t, first)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(64, 1, 1), (128, 2, 1), (32, 1, 5), (80, 3, 2), (256, 1, 1)])
def test_long_rows(gpu, dtype, dk, group, seq):
    check_every_key(dtype, dk, 1, group, seq, [3001, 128, 129, 1, 1280])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(64, 1, 40), (128, 3, 7), (32, 2, 17)])
def test_prompt_pieces_over_long_rows(gpu, dtype, dk, group, seq):
    check_every_key(dtype, dk, 1, group, seq, [2600, 3, 2049, 40], [seq, min(seq, 9), 1, 0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(32, 1, 1), (64, 3, 2)])
def test_one_long_row_among_short_ones(gpu, dtype, dk, group, seq):
    lens = np.random.RandomState(dk).randint(0, 4, 40).tolist()
    lens[17] = 9001
    check_every_key(dtype, dk, 1, group, seq, lens)


@pytest.mark.parametrize("dk", [32, 64, 96, 128, 192])
def test_every_length_to_two_rounds(gpu, dk):
    """Rows of 1 … 530 keys in one call (eight waves of 32 keys twice, and over), one after another in
    two calls' worth of tiles."""
    check_every_key(np.float32, dk, 1, 1, 1, list(range(1, 531)))


@pytest.mark.parametrize("dk", [32, 64, 128])
def test_many_rows_and_two_long_ones(gpu, dk):
    lens = np.random.RandomState(dk).randint(0, 4, 130).tolist()
    lens[0], lens[64], lens[-1] = 2500, 257, 2499
    check_every_key(np.float32, dk, 1, 1, 2, lens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_workgroups_of_four_waves(gpu, dtype):
    """Tiles enough for them: 97 rows × 33 heads."""
    lens = np.random.RandomState(3).randint(0, 200, 97).tolist()
    lens[5], lens[96] = 300, 259
    check_every_key(dtype, 64, 33, 1, 1, lens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk", [32, 64, 80, 128, 256])
@pytest.mark.parametrize("n", [33, 300, 2049, 5000])
def test_one_key_takes_it_all(gpu, dtype, dk, n):
    """Sixteen query heads, each with a key of its own at an edge that scores far above the others: the
    output is that key's value, whichever way K and V could come apart."""
    r = np.random.RandomState(n + dk)
    edges = np.unique(np.clip(np.r_[0, 1, 15, 16, 31, 32, 255, 256, 511, 512, 1023, 1024, 2047, 2048,
                                    n - 33, n - 32, n - 2, n - 1, r.randint(0, n, 6)], 0, n - 1))
    v = r.randn(2, 1, n, dk).astype(dtype)
    hv = R.held(v)
    for some in np.array_split(edges, -(-len(edges) // 16)):
        marks = r.choice([-1.0, 1.0], (len(some), dk))
        k = np.zeros((2, 1, n, dk), dtype)
        k[:, 0, some] = 6 * marks
        q = np.broadcast_to(marks[None, :, None], (2, len(some), 1, dk)).astype(dtype)
        got = K.kv4_attention(q, cache_of(k, v), [n, n], 0.25).numpy().reshape(2, len(some), dk)
        # own score 24·dk ≥ 768, the others' at most 24·(marks·marks') < 24·(dk − 4): e^-96 of it
        cross = np.abs(marks @ marks.T - dk * np.eye(len(some))).max() if len(some) > 1 else 0
        assert cross <= dk - 4
        want = hv[:, 0, some]
        assert np.abs(got.astype(np.float64) - want).max() <= np.abs(want).max() * (2.0**-20 + np.finfo(dtype).eps / 2)


def errors_of(q, k, v, scale, dtype):
    """(output, largest error) of one query over its keys, per dim. A score is off by δ = (dk + 4)·2^-24·
    Σ|q·k| / scale, its exponential by that, by the rounding of its argument (2^-24 of each of its two
    terms) and by 2^-22; a probability enters with 17 bits (float16) or 24; sums are of 32 products,
    then of tiles one after another: 64 + keys / 32 roundings; the output rounds by half a step."""
    s = k @ q / scale
    w = np.exp(s - s.max())
    w /= w.sum()
    out = w @ v
    eps = (k.shape[1] + 4) * 2.0**-24 * (np.abs(k) @ np.abs(q)) / scale + \
        2.0**-24 * 1.5 * (np.abs(s) + np.abs(s.max())) + 2.0**-22
    rel = 2.0 ** (-17 if dtype == np.float16 else -24) + 2 * (64 + len(k) / 32) * 2.0**-24
    size = w @ np.abs(v) + np.abs(out)
    return out, (w * eps) @ (np.abs(v) + np.abs(out)) + rel * size + np.abs(out) * np.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(32, 2, 1), (64, 1, 1), (64, 3, 2), (80, 1, 1), (128, 4, 1), (256, 1, 1)])
def test_random_rows_within_their_own_errors(gpu, dtype, dk, group, seq):
    """Random keys and values, each output against an error of its own keys' weights."""
    r = np.random.RandomState(dk + group)
    lens = [3001, 700, 257, 33]
    k, v = normal(r, (4, 1, 3001, dk), dtype), normal(r, (4, 1, 3001, dk), dtype)
    q, scale = normal(r, (4, group, seq, dk), dtype), 2.0 * np.sqrt(dk)
    got = K.kv4_attention(q, cache_of(k, v), lens, scale).numpy().reshape(4, seq, group, dk)
    hk, hv = R.held(k), R.held(v)
    scale = float(np.float32(scale))
    told = 0
    for i, n in enumerate(lens):
        for t in range(seq):
            for h in range(group):
                keys = n - seq + t + 1
                want, err = errors_of(q[i, h, t].astype(np.float64), hk[i, 0, :keys], hv[i, 0, :keys], scale, dtype)
                assert (np.abs(got[i, t, h].astype(np.float64) - want) <= err).all(), (i, t, h)
                # how many of the keys would be missed
                s = hk[i, 0, :keys] @ q[i, h, t].astype(np.float64) / scale
                w = np.exp(s - s.max())
                w /= w.sum()
                told += ((w / (1 - w))[:, None] * np.abs(hv[i, 0, :keys] - want) > 2 * err).any(1).mean()
    assert told > 0.5 * 4 * seq * group, told / (4 * seq * group)
