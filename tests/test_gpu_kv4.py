"""The 4-bit KV cache against the 64-bit statements of oracle/kv4_ref.py: bytes written (exactly),
values read back (exactly), and attention over the held values, at the sizes and in the places
where each can go wrong."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [np.float16, np.float32]


def filled(batch, heads, max_seq, dk, byte=0xAB):
    """A cache whose every byte is `byte` (a scale of that byte is an ordinary one)."""
    c = K.KV4Cache(batch, heads, max_seq, dk)
    for a in (c.k_codes, c.k_scales, c.v_codes, c.v_scales):
        N.check(N.lib.nml_memset(a.ptr, byte, a.nbytes))
    return c


def cache_of(k, v, max_seq=None):
    """A cache holding k and v (batch, heads, n, dk) from position 0 on."""
    b, h, n, dk = k.shape
    c = filled(b, h, max_seq or n, dk)
    K.kv4_write(c, k, v)
    return c


def normal(r, shape, dtype):
    x = r.randn(*shape)
    x[..., 3::16] *= 4
    return x.astype(dtype)


# ------------------------------------------------------------------ write and read

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk", [1, 8, 31, 32, 33, 64, 80, 128, 200, 256])
def test_bytes_written_and_values_read(gpu, dtype, dk):
    r = np.random.RandomState(dk)
    b, h, s, p = 4, 3, 5, 23
    k, v = normal(r, (b, h, s, dk), dtype), normal(r, (b, h, s, dk), dtype)
    k[0, 0, 0], v[1, 1, 1] = 0, -0.0
    pos, counts = np.array([0, 18, 7, 3]), np.array([5, 5, 0, 2])
    c = filled(b, h, p, dk)
    before = [a.numpy() for a in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]
    K.kv4_write(c, k, v, pos, counts)
    for i, x in ((0, k), (2, v)):
        codes, scales = R.quantise(x)
        for row in range(b):  # the rest of the cache is as it was
            at = slice(pos[row], pos[row] + counts[row])
            before[i][row, :, at] = codes[row, :, :counts[row]]
            before[i + 1][row, :, at] = scales[row, :, :counts[row]]
    for got, want in zip((c.k_codes, c.k_scales, c.v_codes, c.v_scales), before):
        assert np.array_equal(got.numpy(), want)
    for got, x in zip(K.kv4_read(c, s, pos, counts, dtype), (k, v)):
        want = R.held(x)
        for row in range(b):
            want[row, :, counts[row]:] = 0
        assert np.array_equal(got.numpy().astype(np.float64), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, pad", [(64, 0), (64, 8), (40, 0), (40, 3), (33, 0)])
def test_projection_layout_and_odd_strides(gpu, dtype, dk, pad):
    """(batch, seq, 3, heads, dk) as one projection leaves it, with and without padding."""
    r = np.random.RandomState(5)
    b, s, h = 2, 6, 5
    qkv = normal(r, (b, s, 3, h, dk + pad), dtype)
    dev = N.DeviceArray.from_host(qkv)
    es, row = qkv.itemsize, h * (dk + pad)
    c = filled(b, h, 9, dk)
    pos = N.DeviceArray.from_host(np.array([3, 0], np.int32))
    N.check(N.lib.nml_kv4_write_device(
        dev.ptr + es * row, dev.ptr + es * 2 * row, s * 3 * row, dk + pad, 3 * row, *c.pointers,
        pos.ptr, None, b, h, s, 9, dk, None, N.np_dtype_code(dtype)))
    got = K.kv4_read(c, s, pos, None, dtype)
    for i in (1, 2):
        want = R.held(np.ascontiguousarray(qkv[:, :, i, :, :dk].transpose(0, 2, 1, 3)))
        assert np.array_equal(got[i - 1].numpy().astype(np.float64), want)


def test_every_float16_value_and_block_of_every_size(gpu):
    bits = np.arange(65536, dtype=np.uint16).view(np.float16)
    x = bits[np.isfinite(bits)]
    r = np.random.RandomState(1)
    near = np.sort(x)[: len(x) // 32 * 32].reshape(1, 1, -1, 32)  # blocks of like magnitude
    mixed = r.permutation(x)[: len(x) // 32 * 32].reshape(1, 1, -1, 32)
    c = cache_of(np.ascontiguousarray(near), mixed)
    for got, want in zip(K.kv4_read(c, near.shape[2], dtype=np.float16), (near, mixed)):
        got = got.numpy()
        assert np.isfinite(got).all()  # no code stands for more than float16 holds
        assert np.array_equal(got.astype(np.float64), R.held(np.ascontiguousarray(want)))


def test_float32_magnitudes_and_ties(gpu):
    r = np.random.RandomState(2)
    e = np.linspace(-149, 127.9, 2000)
    x = ((2.0 ** e)[:, None] * r.uniform(-1, 1, (2000, 32))).astype(np.float32)
    # every midpoint between codes, under every scale that a block can have, and just beside it
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    t = np.zeros((246, 32), np.float32)
    t[:, 0], t[:, 1:8] = 6.0, mids
    t[:, 8:15], t[:, 15:22] = -mids, np.nextafter(mids.astype(np.float32), np.float32(9))
    t[:, 22:29] = np.nextafter(mids.astype(np.float32), np.float32(0))
    t = (t * 2.0 ** np.arange(-120, 126)[:, None]).astype(np.float32)
    c = K.KV4Cache(1, 1, 2246, 32)
    both = np.concatenate([x, t])[None, None]
    K.kv4_write(c, both, -both)
    codes, scales = R.quantise(both)
    assert np.array_equal(c.k_codes.numpy(), codes) and np.array_equal(c.k_scales.numpy(), scales)
    assert np.array_equal(c.v_codes.numpy(), R.quantise(-both)[0])
    got = K.kv4_read(c, 2246, dtype=np.float32)[0].numpy()
    assert np.array_equal(got.astype(np.float64), R.held(both))
    with np.errstate(over="ignore"):  # past float16's range: infinite there
        want = R.held(both).astype(np.float32).astype(np.float16)
    assert np.array_equal(K.kv4_read(c, 2246, dtype=np.float16)[0].numpy(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_that_are_not_finite_read_as_nan(gpu, dtype):
    r = np.random.RandomState(3)
    k = normal(r, (1, 1, 4, 80), dtype)
    k[0, 0, 0, 5], k[0, 0, 1, 40], k[0, 0, 2, 79] = np.nan, np.inf, -np.inf
    got = K.kv4_read(cache_of(k, k), 4, dtype=dtype)[1].numpy()
    want = R.held(k)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got).sum() == 32 + 32 + 16
    assert np.array_equal(got[~np.isnan(got)].astype(np.float64), want[~np.isnan(want)])


def test_positions_and_counts_outside_the_cache(gpu):
    r = np.random.RandomState(4)
    x = normal(r, (3, 2, 4, 32), np.float32)
    for pos, counts in (([-2, 0, 6], [4, 4, 4]), ([0, 0, 0], [4, 5, -1])):
        c = filled(3, 2, 8, 32)
        with pytest.raises(ValueError, match="outside"):
            K.kv4_write(c, x, x, pos, counts)
        want = filled(3, 2, 8, 32).v_codes.numpy()
        codes = R.quantise(x)[0]
        for b in range(3):
            for s in range(min(4, max(0, counts[b]))):
                if 0 <= pos[b] + s < 8:
                    want[b, :, pos[b] + s] = codes[b, :, s]
        assert np.array_equal(c.v_codes.numpy(), want)
        with pytest.raises(ValueError, match="outside"):
            K.kv4_read(c, 4, pos, counts, np.float32)
    out = [N.DeviceArray.from_host(np.full((3, 2, 4, 32), 7, np.float32)) for _ in range(2)]
    pd = N.DeviceArray.from_host(np.array([-2, 8, 6], np.int32))
    cd = N.DeviceArray.from_host(np.array([4, 2, 3], np.int32))
    N.check(N.lib.nml_kv4_read_device(*c.pointers, pd.ptr, cd.ptr, out[0].ptr, out[1].ptr, 3, 2, 4,
                                      8, 32, None, N.F32))
    got = out[0].numpy()
    assert (got[0, :, :2] == 0).all() and (got[1, :, :2] == 0).all() and (got[2, :, 2] == 0).all()
    assert (got[1, :, 2:] == 7).all() and (got[2, :, 3] == 7).all()  # left as they were


# ---------------------------------------------------------------------- attention

def bound(q, k, v, scale, dtype):
    """Largest error of an output, per (row, head): scores are float32 sums of dk exact products
    (of values split without loss), so each is off by at most (dk + 4)·2^-24·Σ|q·k| / scale and
    its exponential by twice that, relative; exponent and sums in float32 add (keys + 16)·2^-24;
    probabilities enter the product with at least 17 bits (float16) or 24 (float32); the output
    rounds by half a step. An output is at most the largest value it averages."""
    b, h = q.shape[:2]
    g = h // k.shape[1]
    kk, vv = np.abs(np.nan_to_num(k)), np.abs(np.nan_to_num(v))
    dots = max((np.abs(q[i, j].astype(np.float64)) @ kk[i, j // g].T).max()
               for i in range(b) for j in range(h)) / scale
    keys, dk = k.shape[2], k.shape[3]
    rel = 2 * ((dk + 4) * dots + keys + 16) * 2.0**-24 + 2.0 ** (-17 if dtype == np.float16 else -24)
    return vv.max() * (rel + np.finfo(dtype).eps / 2)


def check_attention(r, dtype, dk, kv, group, seq, lens, counts=None, max_seq=None):
    b, lens = len(lens), np.asarray(lens)
    p = max_seq or max(1, int(lens.max()))
    k, v = normal(r, (b, kv, p, dk), dtype), normal(r, (b, kv, p, dk), dtype)
    q = normal(r, (b, kv * group, seq, dk), dtype)
    c = cache_of(k, v)
    scale = float(np.sqrt(dk))
    got = K.kv4_attention(q, c, lens, scale, counts).numpy().astype(np.float64)
    hk, hv = R.held(k), R.held(v)
    want = R.attention(q, hk, hv, lens, counts, scale)
    assert got.shape == want.shape
    err = np.abs(got - want).max()
    assert err <= bound(q, hk, hv, scale, dtype), (err, bound(q, hk, hv, scale, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk", [1, 8, 16, 32, 33, 64, 80, 96, 128, 130, 192, 256])
def test_one_token_every_head_dim_at_edge_lengths(gpu, dtype, dk):
    check_attention(np.random.RandomState(dk), dtype, dk, 2, 1, 1,
                    [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 257, 300])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv, group", [(1, 1), (1, 2), (2, 3), (2, 4), (1, 7), (1, 8), (1, 16), (1, 33)])
@pytest.mark.parametrize("dk", [32, 64, 128])
def test_shared_kv_heads(gpu, dtype, kv, group, dk):
    check_attention(np.random.RandomState(group), dtype, dk, kv, group, 1, [1, 40, 200])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seq", [2, 3, 5, 8, 16, 17, 40])
@pytest.mark.parametrize("dk, group", [(32, 1), (64, 2), (80, 1), (128, 4), (256, 1)])
def test_several_tokens_are_causal(gpu, dtype, seq, dk, group):
    check_attention(np.random.RandomState(seq), dtype, dk, 2, group, seq,
                    [seq, seq + 1, 64, 65 + seq, 190])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seq", [1, 4, 19])
def test_rows_that_see_nothing_give_zeros(gpu, dtype, seq):
    """Lengths of zero, and lengths below the count: the first tokens see no key."""
    check_attention(np.random.RandomState(7), dtype, 64, 2, 2, seq, [0, 1, 2, 50], max_seq=70)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged_counts_leave_the_padding(gpu, dtype):
    r = np.random.RandomState(8)
    b, h, seq, dk, p = 5, 3, 6, 64, 90
    lens, counts = np.array([90, 40, 3, 6, 0]), np.array([6, 1, 3, 0, 2])
    check_attention(r, dtype, dk, h, 1, seq, lens, counts, p)
    k, q = normal(r, (b, h, p, dk), dtype), normal(r, (b, h, seq, dk), dtype)
    c = cache_of(k, k)
    dev = [N.DeviceArray.from_host(x) for x in (q, lens.astype(np.int32), counts.astype(np.int32),
                                                np.full((b, seq, h * dk), 7, dtype))]
    need = N.C.c_size_t()
    N.check(N.lib.nml_kv4_attention_workspace(b, h, h, seq, p, dk, N.C.byref(need)))
    ws = N.DeviceArray.from_host(np.zeros(need.value, np.uint8))
    N.check(N.lib.nml_kv4_attention_device(dev[0].ptr, *c.pointers, dev[1].ptr, dev[2].ptr,
                                           dev[3].ptr, b, h, h, seq, p, dk, 8.0, ws.ptr, need.value,
                                           None, N.np_dtype_code(dtype)))
    got = dev[3].numpy()
    for i in range(b):
        assert (got[i, counts[i]:] == 7).all()
    assert (got[4, :2] == 0).all()


def test_lengths_and_counts_out_of_range_are_clamped_and_reported(gpu):
    r = np.random.RandomState(9)
    k, q = normal(r, (2, 2, 50, 32), np.float32), normal(r, (2, 2, 2, 32), np.float32)
    c = cache_of(k, k)
    for lens, counts in (([51, 5], None), ([-1, 5], None), ([5, 5], [3, 1]), ([5, 5], [2, -1])):
        with pytest.raises(ValueError, match="outside"):
            K.kv4_attention(q, c, lens, 5.0, counts)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seq, dk", [(1, 64), (5, 64), (5, 128), (3, 40)])
def test_what_lies_past_a_row_never_matters(gpu, dtype, seq, dk):
    """Cache positions from lens on hold NaN blocks: the outputs are bit for bit those of a cache
    that ends there or holds other values."""
    r = np.random.RandomState(10)
    k, v = normal(r, (3, 2, 150, dk), dtype), normal(r, (3, 2, 150, dk), dtype)
    q, lens = normal(r, (3, 2, seq, dk), dtype), np.array([7, 64, 101])
    clean = K.kv4_attention(q, cache_of(k, v), lens, 8.0).numpy()
    for i, n in enumerate(lens):
        k[i, :, n:], v[i, :, n:] = np.nan, np.nan
    dirty = K.kv4_attention(q, cache_of(k, v), lens, 8.0).numpy()
    assert np.isfinite(clean).all() and np.array_equal(clean, dirty)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group", [(64, 1), (128, 2), (96, 1)])
def test_nan_blocks_reach_the_tokens_that_see_them(gpu, dtype, dk, group):
    """A NaN block of V makes its 32 output values NaN, one of K the whole output, for the
    tokens at or after its key; the others are as without it."""
    r = np.random.RandomState(11)
    seq, lens = 6, np.array([40, 75])
    k, v = normal(r, (2, 2, 80, dk), dtype), normal(r, (2, 2, 80, dk), dtype)
    q = normal(r, (2, 2 * group, seq, dk), dtype)
    clean = K.kv4_attention(q, cache_of(k, v), lens, 8.0).numpy()
    k[0, 0, 37, 5] = np.nan     # seen by tokens 3, 4, 5 of row 0 (positions 37 …)
    v[1, 1, 72, 40] = np.inf    # by tokens 3, 4, 5 of row 1
    got = K.kv4_attention(q, cache_of(k, v), lens, 8.0).numpy()
    want_nan = np.zeros((2, seq, 2 * group, dk), bool)
    want_nan[0, 3:, :group] = True
    want_nan[1, 3:, group:, 32:64] = True
    want_nan = want_nan.reshape(got.shape)
    assert np.array_equal(np.isnan(got), want_nan)
    assert np.array_equal(got[~want_nan], clean[~want_nan])


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_queries_and_extreme_values(gpu, dtype):
    """An infinite or NaN query makes its own output NaN and no other; large scores stay exact
    (the largest wins alone); tiny probabilities of far keys keep their share."""
    r = np.random.RandomState(12)
    k, v = normal(r, (1, 2, 70, 64), dtype), normal(r, (1, 2, 70, 64), dtype)
    q = normal(r, (1, 2, 3, 64), dtype)
    c = cache_of(k, v)
    clean = K.kv4_attention(q, c, [70], 8.0).numpy().reshape(3, 2, 64)
    q[0, 0, 1, 3], q[0, 1, 2, 0] = np.inf, np.nan
    got = K.kv4_attention(q, c, [70], 8.0).numpy().reshape(3, 2, 64)
    assert np.isnan(got[1, 0]).all() and np.isnan(got[2, 1]).all()
    for t, h in ((0, 0), (0, 1), (1, 1), (2, 0)):
        assert np.array_equal(got[t, h], clean[t, h])
    # one key scores 600 above the others: its value alone
    k[:] = 0.0
    k[0, :, 33] = 6.0
    q[:] = 6.0
    got = K.kv4_attention(q, cache_of(k, v), [70], 3.0).numpy().reshape(3, 2, 64)
    assert np.array_equal(got[2].astype(np.float64), R.held(v)[0, :, 33])


def test_small_probabilities_are_not_lost(gpu):
    """4000 keys of probability e^-12 of the best one's each: their values' sum shows."""
    dk, n = 32, 4001
    k = np.zeros((1, 1, n, dk), np.float16)
    v = np.zeros((1, 1, n, dk), np.float16)
    k[0, 0, 0, 0], v[0, 0, 1:] = 6.0, 4.0
    q = np.zeros((1, 1, 1, dk), np.float16)
    q[..., 0] = 2.0
    got = K.kv4_attention(q, cache_of(k, v), [n], 1.0).numpy().astype(np.float64)
    w = 4000 * np.exp(-12.0)
    # float16 output, probabilities with 17 bits
    assert np.abs(got - 4 * w / (1 + w)).max() <= 4 * w / (1 + w) * (2.0**-11 + 2.0**-16)


def test_offsets_past_32_bits(gpu):
    """64 rows × 16 heads × 65,600 positions of dk 128: 4.3 GB of codes, read in the last row."""
    r = np.random.RandomState(13)
    b, h, p, dk = 64, 16, 65600, 128
    c = K.KV4Cache(b, h, p, dk)
    assert c.k_codes.nbytes > 2**32
    n = 90
    k, v = normal(r, (b, h, n, dk), np.float16), normal(r, (b, h, n, dk), np.float16)
    pos = np.full(b, p - n)
    K.kv4_write(c, k, v, pos)
    got = K.kv4_read(c, n, pos, dtype=np.float16)[0].numpy()[-1]
    assert np.array_equal(got.astype(np.float64), R.held(k[-1:])[0])
    # the zeroed positions before hold zeros: every score there is 0, every value 0
    lens = np.full(b, 1)
    lens[-1] = p
    q = normal(r, (b, h, 1, dk), np.float16)
    out = K.kv4_attention(q, c, lens, 11.0).numpy()[-1].astype(np.float64).reshape(h, dk)
    hk, hv = R.held(k[-1:])[0], R.held(v[-1:])[0]
    for j in range(h):
        x = hk[j] @ q[-1, j, 0].astype(np.float64) / 11.0
        w = np.exp(x)
        want = w @ hv[j] / (w.sum() + p - n)
        tol = np.abs(hv[j]).max() * w.sum() / p * 1e-3 + 2.0**-11 * np.abs(want).max() + 2.0**-25
        assert np.abs(out[j] - want).max() <= tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(64, 1, 1), (128, 2, 1), (32, 1, 5), (80, 3, 2), (256, 1, 1)])
def test_long_rows_in_pieces(gpu, dtype, dk, group, seq):
    """Few rows and long ones: a row's keys in many pieces, beside rows of one piece and of a
    piece and a key."""
    check_attention(np.random.RandomState(dk), dtype, dk, 1, group, seq, [3001, 128, 129, 1, 1280])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(64, 1, 40), (128, 3, 7), (32, 2, 17)])
def test_prompt_pieces_over_long_rows(gpu, dtype, dk, group, seq):
    """More queries than a tile holds over rows in pieces; rows with fewer tokens than the call, and
    a row whose first tokens see no key."""
    check_attention(np.random.RandomState(seq), dtype, dk, 1, group, seq, [2600, 3, 2049, 40],
                    [seq, min(seq, 9), 1, 0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_of_very_different_scores(gpu, dtype):
    """One piece holds scores hundreds above the others', one holds a NaN block that the last
    token alone sees."""
    r = np.random.RandomState(14)
    dk, n = 64, 2050
    k, v = normal(r, (1, 1, n, dk), dtype), normal(r, (1, 1, n, dk), dtype)
    q = normal(r, (1, 1, 2, dk), dtype)
    k[0, 0, 700:720] *= 40
    scale = 8.0
    got = K.kv4_attention(q, cache_of(k, v), [n], scale).numpy().astype(np.float64)
    hk, hv = R.held(k), R.held(v)
    err = np.abs(got - R.attention(q, hk, hv, [n], None, scale)).max()
    assert err <= bound(q, hk, hv, scale, dtype)
    clean = got
    v[0, 0, n - 1, 10] = np.inf
    got = K.kv4_attention(q, cache_of(k, v), [n], scale).numpy().astype(np.float64)[0]
    assert np.array_equal(got[0], clean[0, 0])
    assert np.isnan(got[1, :32]).all() and np.array_equal(got[1, 32:], clean[0, 1, 32:])
    k[0, 0, n - 1, 40] = np.nan
    got = K.kv4_attention(q, cache_of(k, v), [n], scale).numpy().astype(np.float64)[0]
    assert np.array_equal(got[0], clean[0, 0]) and np.isnan(got[1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(32, 1, 1), (64, 3, 2)])
def test_one_long_row_among_short_ones(gpu, dtype, dk, group, seq):
    """One row's keys in more pieces than are merged at a time, beside forty rows of a few."""
    r = np.random.RandomState(dk)
    lens = r.randint(0, 4, 40)
    lens[17] = 9001
    check_attention(r, dtype, dk, 1, group, seq, lens)


def test_many_rows(gpu):
    """More rows than a wave's lanes, with and without keys, tokens or both."""
    r = np.random.RandomState(15)
    lens, counts = r.randint(0, 150, 200), r.randint(0, 4, 200)
    lens[::7] = 0
    check_attention(r, np.float16, 32, 2, 1, 3, lens, counts, 150)


@pytest.mark.parametrize("rows", [65, 128, 513, 1030])
@pytest.mark.parametrize("dk, long", [(32, 7000), (64, 5000), (128, 3)])
def test_many_rows_and_two_long_ones(gpu, rows, dk, long):
    """More rows than one wave, or one load of all eight, looks through: two long ones in pieces,
    the rest of a few keys or none; first and last rows among them."""
    r = np.random.RandomState(rows)
    kv, seq, p = 1, 2, max(long, 4)
    lens = r.randint(0, 4, rows).astype(np.int32)
    lens[0], lens[-1] = long, long - 1
    picked = np.unique(np.r_[0, 1, 62:65, rows // 2, rows - 2:rows])
    c = K.KV4Cache(rows, kv, p, dk)
    k, v = (np.zeros((rows, kv, 4, dk), np.float16) for _ in range(2))
    k[:], v[:] = normal(r, k.shape, np.float16), normal(r, v.shape, np.float16)
    K.kv4_write(c, k, v)  # the first four keys of every row
    tail = [normal(r, (1, kv, p, dk), np.float16) for _ in range(2)]
    blocks = -(-dk // 32)
    for row in (0, rows - 1):  # all of the two long ones
        ptrs = [a.ptr + row * kv * p * blocks * size for a, size in
                ((c.k_codes, 16), (c.k_scales, 1), (c.v_codes, 16), (c.v_scales, 1))]
        dev = [N.DeviceArray.from_host(x) for x in tail]
        N.check(N.lib.nml_kv4_write_device(dev[0].ptr, dev[1].ptr, 0, p * dk, dk, *ptrs, None, None, 1, kv,
                                           p, p, dk, None, N.np_dtype_code(np.float16)))
    q = normal(r, (rows, kv, seq, dk), np.float16)
    got = K.kv4_attention(q, c, lens, 8.0).numpy().astype(np.float64)
    for i in picked:
        hk, hv = (R.held(t if i in (0, rows - 1) else x[i:i + 1]) for t, x in zip(tail, (k, v)))
        want = R.attention(q[i:i + 1], hk, hv, lens[i:i + 1], None, 8.0)
        assert np.abs(got[i] - want[0]).max() <= bound(q[i:i + 1], hk, hv, 8.0, np.float16), i
    none = lens == 0
    assert (got[none] == 0).all()
    with pytest.raises(ValueError, match="outside"):
        lens[rows - 5] = p + 1
        K.kv4_attention(q, c, lens, 8.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk, group, seq", [(32, 1, 1), (64, 2, 3), (128, 1, 1), (256, 1, 1)])
def test_many_tiles_of_every_length(gpu, dtype, dk, group, seq):
    """Tiles far more than the card holds at once, one row in pieces; rows picked by length."""
    r = np.random.RandomState(dk + seq)
    rows, kv, p = 100, 33, 700
    lens = r.randint(0, 40, rows)
    lens[[3, 50, 99]] = 0, p, 300
    k, v = normal(r, (1, kv, p, dk), dtype), normal(r, (1, kv, p, dk), dtype)
    q = normal(r, (rows, kv * group, seq, dk), dtype)
    one, c = cache_of(k, v), K.KV4Cache(rows, kv, p, dk)
    for i in range(rows):  # every row holds the same keys
        for a, b in ((one.k_codes, c.k_codes), (one.k_scales, c.k_scales), (one.v_codes, c.v_codes),
                     (one.v_scales, c.v_scales)):
            N.check(N.lib.nml_memcpy_d2d(b.ptr + i * a.nbytes, a.ptr, a.nbytes))
    got = K.kv4_attention(q, c, lens, 8.0).numpy().astype(np.float64)
    hk, hv = R.held(k), R.held(v)
    for i in (0, 3, 49, 50, 51, 98, 99):
        want = R.attention(q[i:i + 1], hk, hv, lens[i:i + 1], None, 8.0)
        assert np.abs(got[i] - want[0]).max() <= bound(q[i:i + 1], hk, hv, 8.0, dtype), i


def test_one_workspace_serves_calls_of_any_size(gpu):
    """Calls of different shapes follow each other on one workspace, zeroed once."""
    r = np.random.RandomState(16)
    shapes = [(3, 2, 1, 1, 64, 900), (1, 1, 4, 5, 32, 3000), (40, 4, 1, 1, 128, 260),
              (2, 2, 2, 3, 256, 700), (1, 1, 1, 1, 16, 5000)]
    need = N.C.c_size_t()
    most = 0
    for b, kv, g, s, dk, n in shapes:
        N.check(N.lib.nml_kv4_attention_workspace(b, kv * g, kv, s, n, dk, N.C.byref(need)))
        most = max(most, need.value)
    ws = N.DeviceArray.from_host(np.zeros(most, np.uint8))
    made = []
    for b, kv, g, s, dk, n in shapes:
        k, v, q = normal(r, (b, kv, n, dk), np.float32), normal(r, (b, kv, n, dk), np.float32), \
            normal(r, (b, kv * g, s, dk), np.float32)
        lens = r.randint(s, n + 1, b)
        c = cache_of(k, v)
        made.append((c, N.DeviceArray.from_host(q), N.DeviceArray.from_host(lens.astype(np.int32)),
                     K.kv4_attention(q, c, lens, 8.0).numpy()))
    for _ in range(3):
        for (b, kv, g, s, dk, n), (c, q, lens, want) in zip(shapes, made):
            out = N.DeviceArray((b, s, kv * g * dk), np.float32)
            N.check(N.lib.nml_kv4_attention_device(
                q.ptr, *c.pointers, lens.ptr, None, out.ptr, b, kv * g, kv, s, n, dk, 8.0, ws.ptr,
                most, None, N.F32))
            assert np.array_equal(out.numpy(), want)
