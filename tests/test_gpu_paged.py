"""The paged KV cache on the GPU: written exactly, attended to within float32's roundings."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import draft_ref as R

pytestmark = pytest.mark.gpu

HALF = {np.float32: 2.0 ** -24, np.float16: 2.0 ** -11}  # half a step, relative


def upload(a):
    return N.DeviceArray.from_host(np.ascontiguousarray(a))


class Cache:
    """A cache with random (or given) contents, a table of scattered pages, and both on the host."""

    def __init__(self, batch, kv, dk, page, max_pages, dtype, seed=0, spare=3, table=None):
        r = np.random.RandomState(seed)
        total = batch * max_pages + spare
        self.c = K.PagedKVCache(total, page, kv, dk, dtype)
        self.k = r.randn(total, kv, page, dk).astype(dtype)
        self.v = r.randn(total, kv, page, dk).astype(dtype)
        self.table = r.permutation(total)[:batch * max_pages].reshape(batch, max_pages).astype(np.int32) \
            if table is None else table
        self.push()

    def push(self):
        for pool, x in ((self.c.k_pages, self.k), (self.c.v_pages, self.v)):
            x = np.ascontiguousarray(x)
            N.check(N.lib.nml_memcpy_h2d(pool.ptr, x.ctypes.data, x.nbytes))

    def attend(self, q, lens, counts=None, scale=None):
        scale = np.sqrt(q.shape[3]) if scale is None else scale
        return K.paged_attention(q, self.c, self.table, lens, scale, counts).numpy()


def check(cache, q, lens, counts, scale=None):
    dtype, (batch, heads, seq, dk) = q.dtype.type, q.shape
    scale = np.sqrt(dk) if scale is None else scale
    got = cache.attend(q, lens, counts, scale).reshape(batch, seq, heads, dk).astype(np.float64)
    full = np.full(batch, seq) if counts is None else counts
    want, size, spread = R.paged_attention(q, cache.k, cache.v, cache.table, lens, full, scale)
    # a score is a float32 sum of dk products and is rounded three times more, the exponential of that
    # error is a relative one of p, twice (the sum of them); the sums over the keys round once a
    # key at most; a float16 probability is held in two parts of 11 bits, or, for more than 32 queries
    # of a KV head, in one: half a step of 2^-10 of it, and of the sum of them
    n = max(int(np.max(lens)), 1)
    ds = 2.0 ** -24 * (dk + 4) * spread
    one = dtype == np.float16 and seq > 1 and heads // cache.k.shape[1] * seq > 32 and dk % 8 == 0
    part = 2.0 ** -10 if one else 2.0 ** -21
    tol = size * (2 * ds + 2.0 ** -24 * (n + 32) + part) + HALF[dtype] * np.abs(want) + 2.0 ** -25 * (dtype == np.float16)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    if one:
        # as a whole: two roundings that know nothing of each other, of 2^-11/√3 of what they round in
        # the mean at most (Σ(p·v)² is the output's square in the mean, for values of either sign)
        off, norm = (np.sqrt((x ** 2).sum()) for x in (got - want, want))
        assert off <= 2.0 ** -11 * np.sqrt(2 / 3) * norm * 1.02
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def queries(batch, heads, seq, dk, dtype, seed):
    return np.random.RandomState(seed + 1000).randn(batch, heads, seq, dk).astype(dtype)


# batch, kv heads, queries a KV head, head dim, page, pages a row, new tokens
SHAPES = [
    (1, 1, 1, 64, 8, 1, 1), (1, 2, 1, 32, 16, 5, 1), (3, 2, 4, 128, 16, 9, 1), (2, 1, 7, 80, 32, 4, 1),
    (2, 2, 1, 1, 8, 6, 3), (2, 1, 2, 7, 8, 6, 5), (1, 2, 3, 33, 16, 7, 4), (2, 1, 1, 250, 8, 8, 2),
    (1, 1, 2, 256, 64, 3, 1), (2, 2, 2, 192, 32, 3, 6), (1, 3, 1, 40, 256, 1, 17), (1, 2, 2, 64, 16, 20, 100),
    (1, 1, 1, 128, 64, 8, 300), (2, 1, 4, 128, 8, 40, 70), (1, 1, 3, 96, 16, 17, 129), (1, 2, 1, 16, 1024, 1, 65),
    (70, 1, 1, 64, 8, 7, 2), (130, 1, 2, 32, 16, 3, 1), (1, 2, 1, 64, 16, 400, 1), (1, 1, 8, 128, 64, 80, 5),
    (3, 1, 1, 256, 32, 70, 2), (2, 1, 1, 72, 32, 60, 40),
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, kv, group, dk, page, pages, seq", SHAPES)
def test_attention(gpu, batch, kv, group, dk, page, pages, seq, dtype):
    seed = batch + kv * 3 + dk + seq
    cache = Cache(batch, kv, dk, page, pages, dtype, seed)
    r, room = np.random.RandomState(seed), page * pages
    q = queries(batch, kv * group, seq, dk, dtype, seed)
    check(cache, q, np.full(batch, room, np.int32), None)
    # ragged: rows with no key, fewer keys than tokens, tokens that are padding
    lens, counts = r.randint(0, room + 1, batch).astype(np.int32), r.randint(0, seq + 1, batch).astype(np.int32)
    lens[0], counts[-1] = room, seq
    check(cache, q, lens, counts)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("group, dk", [(1, 64), (3, 72), (5, 96), (2, 128), (1, 136), (2, 192), (3, 200), (2, 256), (1, 252)])
def test_many_new_tokens_behind_a_long_cache(gpu, group, dk, dtype):
    """Several tiles of queries of a row, whose keys are cut into pieces of a size that differs with the row."""
    cache = Cache(3, 2, dk, 16, 130, dtype, dk)
    q = queries(3, 2 * group, 257, dk, dtype, dk)
    check(cache, q, np.array([2080, 700, 257], np.int32), None)
    check(cache, q, np.array([1999, 100, 0], np.int32), np.array([129, 256, 3], np.int32))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, kv, group, dk, seq", [
    (1, 1, 16, 128, 1), (1, 3, 4, 64, 6), (2, 1, 1, 256, 3), (1, 2, 5, 200, 9), (5, 3, 9, 32, 2), (1, 11, 1, 16, 1), (3, 5, 1, 96, 30)])
def test_many_pieces(gpu, batch, kv, group, dk, seq, dtype):
    """Few rows of many keys: pieces of every tile merged, KV heads in eights and not, one tile and several."""
    cache = Cache(batch, kv, dk, 64, 130, dtype, dk + seq)
    q, r = queries(batch, kv * group, seq, dk, dtype, dk), np.random.RandomState(seq)
    check(cache, q, np.full(batch, 8320, np.int32), None)
    lens = r.randint(0, 8321, batch).astype(np.int32)
    lens[0] = 8001
    check(cache, q, lens, r.randint(0, seq + 1, batch).astype(np.int32))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seq", [1, 5, 150])
def test_what_is_not_seen_does_not_matter(gpu, dtype, seq):
    """NaN and infinities past a row's length, in other pages, and in the tokens after a token."""
    cache = Cache(2, 2, 64, 16, 20, dtype, 5)
    lens = np.array([203, 161], np.int32)
    q = queries(2, 4, seq, 64, dtype, 5)
    used = np.zeros(cache.k.shape[:1] + (cache.k.shape[2],), bool)
    for b in range(2):
        for p in range(lens[b]):
            used[cache.table[b, p // 16], p % 16] = True
    for x, fill in ((cache.k, np.nan), (cache.v, np.inf)):
        x.transpose(0, 2, 1, 3)[~used] = fill
    cache.push()
    check(cache, q, lens, None)
    if seq > 1:
        clean = cache.attend(q, lens).reshape(2, seq, 4, 64)
        for x, fill in ((cache.k, np.nan), (cache.v, -np.inf)):  # the rows' last token
            for b in range(2):
                x[cache.table[b, (lens[b] - 1) // 16], :, (lens[b] - 1) % 16] = fill
        cache.push()
        got = cache.attend(q, lens).reshape(2, seq, 4, 64)
        # (a tile that is formed again, key by key, sums in another order)
        assert np.abs(got[:, :-1].astype(np.float64) - clean[:, :-1]).max() <= (2 ** -18 if dtype == np.float32 else 2 ** -9)
        assert np.isnan(got[:, -1]).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seq", [1, 5, 150])
def test_an_infinite_value_that_is_seen(gpu, dtype, seq):
    cache = Cache(1, 1, 32, 8, 40, dtype, 6)
    q = queries(1, 2, seq, 32, dtype, 6)
    length = 300
    cache.v[cache.table[0, 100 // 8], 0, 100 % 8, 3] = np.inf
    cache.push()
    got = cache.attend(q, np.array([length], np.int32)).reshape(seq, 2, 32)
    assert (got[..., 3] == np.inf).all()
    assert np.isfinite(np.delete(got, 3, -1)).all()


@pytest.mark.parametrize("seq", [1, 150])
def test_large_values_stay_finite(gpu, seq):
    """Averages of float32 values near its largest, over pieces of a long row too."""
    cache = Cache(1, 1, 64, 64, 80, np.float32, 7)
    cache.v[:] = np.where(np.arange(64) % 2, 3.0e38, -1.5e38)
    cache.push()
    got = cache.attend(queries(1, 1, seq, 64, np.float32, 7), np.array([5000], np.int32)).reshape(seq, 64)
    want = np.where(np.arange(64) % 2, 3.0e38, -1.5e38)
    assert (np.abs(got / want - 1) <= 2.0 ** -24 * 5100).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("seq", [1, 200])
def test_sharp_and_flat_scores(gpu, dtype, seq):
    """Scores far apart (one key has all the weight, maxima that keep rising) and all equal."""
    cache = Cache(1, 1, 64, 16, 60, dtype, 8)
    for p in range(960):
        cache.k[cache.table[0, p // 16], 0, p % 16] = p / 960 * 3
    cache.push()
    q = np.abs(queries(1, 2, seq, 64, dtype, 8))
    check(cache, q, np.array([960], np.int32), None)
    check(cache, (q * 0).astype(dtype), np.array([959], np.int32), None)
    check(cache, (-4 * q).astype(dtype), np.array([955], np.int32), None, scale=1.0)


def test_rows_may_share_pages(gpu):
    table = np.array([[5, 2, 0], [5, 2, 1], [5, 3, 4]], np.int32)
    cache = Cache(3, 2, 64, 16, 2, np.float16, 9, table=table)
    check(cache, queries(3, 4, 2, 64, np.float16, 9), np.array([48, 40, 33], np.int32), None)


def test_rows_behind_a_count_are_left_as_they_were(gpu):
    cache = Cache(3, 1, 64, 16, 4, np.float32, 10)
    q, lens, counts = queries(3, 2, 6, 64, np.float32, 10), np.array([20, 64, 0], np.int32), np.array([2, 0, 6], np.int32)
    out = upload(np.full((3, 6, 128), 7.0, np.float32))
    need = N.sz()
    N.check(N.lib.nml_paged_attention_workspace(3, 2, 1, 6, 4, 16, 64, 0, N.C.byref(need)))
    ws = upload(np.zeros(max(1, need.value), np.uint8))
    args = [upload(x) for x in (q, cache.table, lens, counts)]
    N.check(N.lib.nml_paged_attention_device(
        args[0].ptr, cache.c.k_pages.ptr, cache.c.v_pages.ptr, args[1].ptr, args[2].ptr, args[3].ptr, out.ptr, 3, 2, 1,
        6, 4, 16, cache.c.num_pages, 64, 8.0, ws.ptr, need.value, None, 0))
    got = out.numpy()
    assert (got[0, 2:] == 7.0).all() and (got[1] == 7.0).all() and (got[2] == 0.0).all()
    assert (got[0, :2] != 7.0).all()


# ------------------------------------------------------------------------- write

@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, kv, dk, page, pages, seq", [
    (1, 1, 64, 8, 1, 1), (3, 2, 128, 16, 5, 20), (2, 3, 80, 32, 3, 50), (4, 1, 1, 8, 9, 60), (2, 2, 33, 64, 2, 31),
    (1, 5, 256, 16, 4, 64), (70, 1, 40, 8, 2, 3), (2, 1, 7, 1024, 1, 900)])
def test_write(gpu, batch, kv, dk, page, pages, seq, dtype):
    cache = Cache(batch, kv, dk, page, pages, dtype, 11)
    r = np.random.RandomState(11)
    k, v = (r.randn(batch, kv, seq, dk).astype(dtype) for _ in range(2))
    pos = r.randint(0, page * pages - seq + 1, batch).astype(np.int32)
    counts = r.randint(0, seq + 1, batch).astype(np.int32)
    counts[0] = seq
    K.paged_write(cache.c, k, v, cache.table, pos, counts)
    for x, pool, new in ((cache.k, cache.c.k_pages, k), (cache.v, cache.c.v_pages, v)):
        for b in range(batch):
            for s in range(counts[b]):
                p = pos[b] + s
                x[cache.table[b, p // page], :, p % page] = new[b, :, s]
        assert np.array_equal(pool.numpy(), x)


@pytest.mark.parametrize("dk, skip", [(64, 0), (64, 1), (40, 8), (33, 0)])
def test_write_from_a_projection(gpu, dk, skip):
    """K and V as they lie in a (batch, seq, 3, heads, dk) projection, `skip` values from its start."""
    cache = Cache(2, 3, dk, 16, 4, np.float16, 12)
    r = np.random.RandomState(12)
    qkv = r.randn(2, 30, 3, 3, dk).astype(np.float16)
    flat = np.concatenate([np.zeros(skip, np.float16), qkv.reshape(-1)])
    src, table = upload(flat), upload(cache.table)
    base, es = src.ptr + 2 * skip, 2
    N.check(N.lib.nml_paged_write_device(
        base + es * 3 * dk, base + es * 6 * dk, 30 * 9 * dk, dk, 9 * dk, cache.c.k_pages.ptr, cache.c.v_pages.ptr,
        table.ptr, None, None, 2, 3, 30, 4, 16, cache.c.num_pages, dk, None, 1))
    for x, pool, i in ((cache.k, cache.c.k_pages, 1), (cache.v, cache.c.v_pages, 2)):
        for b in range(2):
            for p in range(30):
                x[cache.table[b, p // 16], :, p % 16] = qkv[b, p, i]
        assert np.array_equal(pool.numpy(), x)


def test_out_of_range_is_told_and_not_written(gpu):
    cache = Cache(2, 1, 32, 8, 3, np.float32, 13)
    k = np.ones((2, 1, 10, 32), np.float32)
    before = cache.c.k_pages.numpy()
    with pytest.raises(ValueError, match="position"):
        K.paged_write(cache.c, k, k, cache.table, np.array([20, -3], np.int32))
    after = cache.c.k_pages.numpy()
    changed = (before != after).any((1, 3))
    want = np.zeros_like(changed)
    for p in range(20, 24):
        want[cache.table[0, p // 8], p % 8] = True
    for p in range(0, 7):
        want[cache.table[1, p // 8], p % 8] = True
    assert np.array_equal(changed, want)
    for page in (-1, cache.c.num_pages, 1 << 30):
        bad = cache.table.copy()
        bad[1, 1] = page
        before = cache.c.k_pages.numpy()
        with pytest.raises(ValueError, match="page"):
            K.paged_write(cache.c, 2 * k, k, bad, np.array([0, 10], np.int32), np.array([0, 4], np.int32))
        assert np.array_equal(before, cache.c.k_pages.numpy())
        # a table on the device is checked there (and read in bounds), one on the host before the call
        q = queries(2, 2, 1, 32, np.float32, 13)
        for table in (upload(bad), bad):
            with pytest.raises(ValueError, match="page"):
                K.paged_attention(q, cache.c, table, np.array([24, 12], np.int32), 4.0)
        K.paged_attention(q, cache.c, upload(bad), np.array([24, 8], np.int32), 4.0)
    with pytest.raises(ValueError, match="length"):
        K.paged_attention(q, cache.c, upload(cache.table), np.array([25, 1], np.int32), 4.0)
    with pytest.raises(ValueError, match="count"):
        K.paged_attention(q, cache.c, cache.table, np.array([24, 1], np.int32), 4.0, np.array([2, 1], np.int32))


def test_pages_past_32_bits(gpu):
    """Pools of 4.6 GB each: the pages used lie past the first 4 GiB."""
    page, dk, total = 256, 128, 70000
    c = K.PagedKVCache(total, page, 1, dk, np.float16)
    r = np.random.RandomState(14)
    table = np.array([[total - 1, total - 7, 66000, 3]], np.int32)
    k, v = (r.randn(1, 1, 1000, dk).astype(np.float16) for _ in range(2))
    K.paged_write(c, k, v, table)
    q = queries(1, 4, 3, dk, np.float16, 14)
    got = K.paged_attention(q, c, table, np.array([1000], np.int32), np.sqrt(dk)).numpy().reshape(3, 4, dk)
    fill = [np.zeros((4, 1, page, dk), np.float16) for _ in range(2)]
    for x, new in zip(fill, (k, v)):
        x.reshape(1024, dk)[:1000] = new[0, 0]
    want, _, _ = R.paged_attention(q, *fill, np.arange(4)[None], [1000], [3], np.sqrt(dk))
    assert np.abs(got - want[0]).max() <= 2.0 ** -11 * np.abs(want).max() * 2


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_out_of_range_is_told_with_many_new_tokens(gpu, dtype):
    cache = Cache(2, 1, 32, 8, 40, dtype, 15)
    q, lens = queries(2, 1, 150, 32, dtype, 15), np.array([320, 200], np.int32)
    good = K.paged_attention(q, cache.c, cache.table, lens, 4.0).numpy().reshape(2, 150, 32)
    for page in (-1, cache.c.num_pages, 1 << 30):
        bad = cache.table.copy()
        bad[1, 24] = page  # (its keys 192 … 199, the last that it has)
        with pytest.raises(ValueError, match="page"):
            K.paged_attention(q, cache.c, upload(bad), lens, 4.0)
        short = np.array([320, 192], np.int32)  # (the page is not read then)
        got = K.paged_attention(q, cache.c, upload(bad), short, 4.0).numpy().reshape(2, 150, 32)
        assert np.array_equal(got[0], good[0])
    for lens, counts, match in (([321, 200], [150, 3], "length"), ([320, -1], [150, 3], "length"),
                                ([320, 200], [151, 3], "count"), ([320, 200], [150, -1], "count")):
        with pytest.raises(ValueError, match=match):
            K.paged_attention(q, cache.c, upload(cache.table), upload(np.array(lens, np.int32)), 4.0,
                              np.array(counts, np.int32))
