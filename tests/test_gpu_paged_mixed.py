"""Attention over pages of batches whose rows differ: a piece of a prompt beside rows of one token, long rows
beside short ones, more rows than the card has workgroups."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from test_gpu_kv4_graphs import Graph, hip  # noqa: F401  (the fixture)
from test_gpu_paged import Cache, check, queries, upload

pytestmark = pytest.mark.gpu

# batch, kv heads, queries a KV head, head dim, page, pages a row, tokens a row
MIXED = [(9, 2, 1, 64, 16, 130, 300), (64, 2, 1, 64, 16, 70, 600), (5, 1, 4, 128, 64, 40, 90), (3, 3, 2, 96, 32, 60, 150),
         (4, 2, 1, 192, 64, 30, 260), (7, 1, 2, 256, 64, 20, 260), (2, 5, 1, 32, 8, 300, 280), (70, 1, 1, 40, 16, 40, 140),
         (520, 1, 1, 64, 64, 9, 130)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, kv, group, dk, page, pages, seq", MIXED)
def test_a_piece_of_a_prompt_beside_rows_of_few_tokens(gpu, batch, kv, group, dk, page, pages, seq, dtype):
    cache, room = Cache(batch, kv, dk, page, pages, dtype, batch + dk), page * pages
    r = np.random.RandomState(batch)
    q = queries(batch, kv * group, seq, dk, dtype, dk)
    for many in (0, batch - 1, batch // 2):  # the row of many tokens
        lens = r.randint(room // 2, room + 1, batch).astype(np.int32)
        counts = r.randint(0, 3, batch).astype(np.int32)
        counts[many], lens[many] = seq, r.randint(seq, room + 1)
        check(cache, q, lens, counts)
        if batch > 100:
            break


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("batch, kv, group, dk, page, pages, seq", [
    (4, 1, 1, 64, 16, 250, 129), (66, 4, 1, 64, 16, 100, 33), (3, 2, 2, 128, 64, 50, 130), (2, 1, 8, 80, 8, 200, 40)])
def test_long_rows_beside_short_ones(gpu, batch, kv, group, dk, page, pages, seq, dtype):
    """As many new tokens everywhere, keys from none to all of the room."""
    cache, room = Cache(batch, kv, dk, page, pages, dtype, batch), page * pages
    lens = np.full(batch, 5, np.int32)
    lens[batch // 2], lens[-1], lens[0] = room, room // 3, 0
    check(cache, queries(batch, kv * group, seq, dk, dtype, 3), lens, None)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_one_workspace_serves_calls_of_any_mixture(gpu, dtype):
    """Mixed batches, batches of one token and again: what one call leaves in the workspace does not matter."""
    batch, kv, dk, page, pages, seq = 6, 2, 64, 16, 120, 200
    cache, room, code = Cache(batch, kv, dk, page, pages, dtype, 1), page * pages, N.np_dtype_code(dtype)
    table, r = upload(cache.table), np.random.RandomState(4)
    sizes = [(s, N.sz()) for s in (seq, 1)]
    for s, need in sizes:
        N.check(N.lib.nml_paged_attention_workspace(batch, kv, kv, s, pages, page, dk, code, N.C.byref(need)))
    most = max(n.value for _, n in sizes)
    ws = upload(np.zeros(most, np.uint8))
    for i in range(6):
        s = sizes[i % 2][0]
        q = queries(batch, kv, s, dk, dtype, i)
        lens = r.randint(0, room + 1, batch).astype(np.int32)
        counts = r.randint(0, s + 1, batch).astype(np.int32)
        lens[i], counts[i] = room, s
        d = [upload(x) for x in (q, lens, counts)]
        out = upload(np.zeros((batch, s, kv * dk), dtype))
        N.check(N.lib.nml_paged_attention_device(
            d[0].ptr, cache.c.k_pages.ptr, cache.c.v_pages.ptr, table.ptr, d[1].ptr, d[2].ptr, out.ptr, batch, kv, kv, s,
            pages, page, cache.c.num_pages, dk, 8.0, ws.ptr, most, None, code))
        assert np.array_equal(out.numpy(), K.paged_attention(q, cache.c, cache.table, lens, 8.0, counts).numpy())


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_a_captured_call_follows_lengths_and_counts(gpu, hip, dtype):  # noqa: F811
    """One graph, replayed over batches that are cut into pieces in other ways each time."""
    batch, kv, group, dk, page, pages, seq = 8, 4, 1, 64, 16, 160, 130
    cache, room, code, heads = Cache(batch, kv, dk, page, pages, dtype, 2), page * pages, N.np_dtype_code(dtype), kv * group
    r, need = np.random.RandomState(6), N.sz()
    q = queries(batch, heads, seq, dk, dtype, 9)
    d = [upload(x) for x in (q, cache.table, np.zeros(batch, np.int32), np.zeros(batch, np.int32))]
    N.check(N.lib.nml_paged_attention_workspace(batch, heads, kv, seq, pages, page, dk, code, N.C.byref(need)))
    ws, out = upload(np.zeros(need.value, np.uint8)), upload(np.zeros((batch, seq, heads * dk), dtype))

    def work():
        N.check(N.lib.nml_paged_attention_device(
            d[0].ptr, cache.c.k_pages.ptr, cache.c.v_pages.ptr, d[1].ptr, d[2].ptr, d[3].ptr, out.ptr, batch, heads, kv,
            seq, pages, page, cache.c.num_pages, dk, 8.0, ws.ptr, need.value, None, code))

    graph = Graph(hip, work)
    try:
        for i in range(6):
            lens = r.randint(0, room + 1, batch).astype(np.int32)
            counts = r.randint(0, (seq if i % 2 else 3) + 1, batch).astype(np.int32)
            lens[i], counts[i] = room, seq
            if i == 2:
                lens[:], counts[:] = room, seq
            if i == 3:
                counts[:] = 0
            for x, new in zip((d[2], d[3], out), (lens, counts, np.zeros(out.shape, dtype))):
                N.check(N.lib.nml_memcpy_h2d(x.ptr, new.ctypes.data, new.nbytes))
            N.synchronize()
            graph.run()
            graph.wait()
            got = out.numpy()
            assert np.array_equal(got, K.paged_attention(q, cache.c, cache.table, lens, 8.0, counts).numpy()), i
            assert counts.any() or not got.any()
    finally:
        graph.close()
