"""A drafting model trained from a large one, and both serving: distillation, drafted tokens checked
in one cached forward, verification, caches taken back; and the operators over a paged cache in
turn, captured into graphs and replayed, on streams of the caller's."""
import ctypes as C

import numpy as np
import pytest

import nimbleml_amd as nm
from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import draft_ref as R
from test_gpu_kv4_graphs import Graph, hip  # noqa: F401  (the fixture)
from test_gpu_paged import Cache, queries, upload

pytestmark = pytest.mark.gpu


@pytest.fixture
def models(gpu):
    nm.set_dtype("float32")
    np.random.seed(3)
    target, drafter = nm.GPT(96, 64, 4, 2, 96), nm.GPT(96, 32, 2, 1, 96)
    for _, p in [*nm.named_parameters(target), *nm.named_parameters(drafter)]:
        if p.data.size > 96:
            p.data[...] = p.data * 4  # (distributions that are not flat)
    return target, drafter


def step(target, drafter, tc, dc, last, n, t, rng):
    """One round for rows whose caches hold everything but their last token: what each row gains."""
    batch = last.shape[0]
    drafts, seen, ids = np.zeros((batch, n), np.int64), [], last
    for i in range(n + 1):  # (the last draft is fed as well: the cache then has it, if it stands)
        logits, _ = drafter.forward_with_cache(ids[:, None], dc)
        if i == n:
            break
        x = np.asarray(logits.data).reshape(batch, 96)
        ids = K.sample_tokens(x, temperature=t, uniforms=rng.rand(batch) if t > 0 else None)
        drafts[:, i] = ids
        seen.append(x)
    logits, _ = target.forward_with_cache(np.concatenate([last[:, None], drafts], 1), tc)
    x = np.asarray(logits.data).reshape(batch, n + 1, 96)
    u, q = rng.rand(batch, n + 1), np.stack(seen, 1)
    a, tokens = (y.numpy() for y in K.verify_drafts(logits.data.reshape(batch, n + 1, 96), drafts, u, draft_logits=q,
                                                    temperature=t))
    wa, wt = R.verify(x, drafts, u, q, np.full(batch, n), t)
    assert np.array_equal(a, wa) and np.array_equal(tokens, wt)
    return a, tokens


@pytest.mark.parametrize("kv_bits", [None, 4])
@pytest.mark.parametrize("t", [0.0, 1.0])
def test_drafted_generation(models, t, kv_bits):
    """Greedy: exactly the target's own tokens. Sampled: every round as the 64-bit statement has it."""
    target, drafter = models
    rng = np.random.RandomState(0)
    prompts = [np.arange(5), np.arange(20) * 3 % 96, np.arange(11) * 7 % 96]
    new, n = 30, 4
    _, tc = target.prefill_ragged([p[:-1] for p in prompts], kv_bits=kv_bits)
    _, dc = drafter.prefill_ragged([p[:-1] for p in prompts])
    rows = [list(p) for p in prompts]
    while min(len(r) - len(p) for r, p in zip(rows, prompts)) < new:
        a, tokens = step(target, drafter, tc, dc, np.array([r[-1] for r in rows]), n, t, rng)
        for b, row in enumerate(rows):
            row += tokens[b, :a[b] + 1].tolist()
            if len(row) > len(prompts[b]) + new:  # done: held where it is
                del row[len(prompts[b]) + new:]
        for c in (tc, dc):
            c.truncate([len(r) - 1 for r in rows])
    if t == 0:
        want = nm.generate(target, prompts, max_new_tokens=new, temperature=0.0, kv_bits=kv_bits)
        for row, w in zip(rows, want):
            assert row == w.tolist()


def test_truncate(models):
    target, _ = models
    ids = np.arange(24).reshape(2, 12) * 5 % 96
    whole, cache = target.forward_with_cache(ids)
    whole = whole.numpy()
    cache.truncate([7, 12])
    assert cache.length == 7
    with pytest.raises(ValueError, match="out of range"):
        cache.truncate([8, 12])
    with pytest.raises(ValueError, match="out of range"):
        cache.truncate(-1)
    cache.truncate(4)
    again, _ = target.forward_with_cache(ids[:, 4:], cache)
    assert np.allclose(again.numpy(), whole[:, 4:], atol=1e-4)
    cache.truncate(0)
    empty, _ = target.forward_with_cache(ids[:, :3], cache)
    assert np.allclose(empty.numpy(), whole[:, :3], atol=1e-4)


def test_distillation_step(models):
    """The gradient that a drafter's training step takes is the loss's: against differences along the
    gradient, of the float32 forward."""
    target, drafter = models
    ids = np.random.RandomState(1).randint(0, 96, (2, 48))
    top = target.log_probs(ids, np.zeros_like(ids), top_k=16)

    def loss():
        return nm.distill_loss(drafter.forward(ids), top["top_ids"], top["top_logp"], temperature=1.5)

    out = loss()
    out.backward(np.full(out.shape, 1 / 96, np.float32))
    params = [p for _, p in nm.named_parameters(drafter)]
    grads = [p.grad.copy().astype(np.float64) for p in params]
    norm = np.sqrt(sum((g ** 2).sum() for g in grads))
    h, start = 2e-3, [p.data.copy() for p in params]
    at = []
    for sign in (1, -1):
        for p, s, g in zip(params, start, grads):
            p.data[...] = s + (sign * h * g / norm).reshape(s.shape)
        drafter.to_device()
        with nm.no_grad():
            at.append(np.asarray(loss().data, dtype=np.float64).mean())
    # the difference is off by h² times a third derivative (of the norm's order) and by the two
    # losses' roundings, 2^-20 each at the most, over 2h
    assert abs((at[0] - at[1]) / (2 * h) - norm) <= 0.01 * norm + 2 * 2.0 ** -20 / (2 * h)


def test_pieces_drafts_and_steps_over_pages(gpu):
    """A prompt in pieces, drafted tokens of which some are refused and written over, steps: each as
    attention over everything at once has it."""
    r = np.random.RandomState(2)
    batch, kv, group, dk, page, pages = 3, 2, 2, 64, 16, 12
    cache = Cache(batch, kv, dk, page, pages, np.float32, 21)
    cache.k[:] = np.nan
    cache.v[:] = np.nan
    cache.push()
    total = page * pages
    k, v = (r.randn(batch, kv, total, dk).astype(np.float32) for _ in range(2))
    q = r.randn(batch, kv * group, total, dk).astype(np.float32)
    mask = np.triu(np.full((total, total), -np.inf, np.float32), 1)
    flat = [x.reshape(batch * kv * group, total, dk) for x in (q, np.repeat(k, group, 1), np.repeat(v, group, 1))]
    whole, _ = K.fused_sdpa_forward(*flat, np.sqrt(dk), mask)
    whole = whole.numpy().reshape(batch, kv * group, total, dk).transpose(0, 2, 1, 3)
    done = np.zeros(batch, np.int64)
    for s in [40, 33, 1, 5, 5, 5, 1, 1, 64]:
        counts = np.minimum(r.randint(1, s + 1, batch), total - done).astype(np.int32)
        counts[0] = min(s, total - done[0])
        take = [np.stack([np.concatenate([x[b, :, done[b]:done[b] + counts[b]],
                                          np.zeros((x.shape[1], s - counts[b], dk), np.float32)], 1)
                          for b in range(batch)]) for x in (q, k, v)]
        if s == 5:  # drafts: written, attended to, two of them given up
            wrong = [x + 1 for x in take]
            K.paged_write(cache.c, wrong[1], wrong[2], cache.table, done.astype(np.int32), counts)
            K.paged_attention(wrong[0], cache.c, cache.table, (done + counts).astype(np.int32), 8.0, counts)
            counts = np.maximum(counts - 2, 0).astype(np.int32)
        K.paged_write(cache.c, take[1], take[2], cache.table, done.astype(np.int32), counts)
        got = K.paged_attention(take[0], cache.c, cache.table, (done + counts).astype(np.int32), np.sqrt(dk),
                                counts).numpy().reshape(batch, s, kv * group, dk)
        for b in range(batch):
            assert np.allclose(got[b, :counts[b]], whole[b, done[b]:done[b] + counts[b]], atol=2e-5)
        done += counts


def test_captured_and_replayed(gpu, hip):  # noqa: F811
    """A round of the serving operators and a training step's loss in one graph; inputs change between
    replays, with eager work on another stream among them."""
    r = np.random.RandomState(4)
    cache = Cache(2, 2, 64, 16, 200, np.float16, 22)
    q, lens, counts = queries(2, 4, 3, 64, np.float16, 1), np.array([3200, 77], np.int32), np.array([3, 2], np.int32)
    new = r.randn(2, 2, 3, 64).astype(np.float16)
    logits, draft = r.randn(4, 6, 3000).astype(np.float32), r.randn(4, 5, 3000).astype(np.float32)
    drafts, u = r.randint(0, 3000, (4, 5)), r.rand(4, 6)
    x, ids, y, dl = r.randn(30, 999).astype(np.float16), r.randint(0, 999, (30, 8)), r.randn(30, 8).astype(np.float32), \
        r.randn(30).astype(np.float32)
    d = {n: upload(a) for n, a in dict(q=q, lens=lens, counts=counts, new=new, table=cache.table, logits=logits,
                                       draft=draft, drafts=drafts, u=u, x=x, ids=ids, y=y, dl=dl,
                                       pos=(lens - counts).astype(np.int32)).items()}
    need = N.sz()
    N.check(N.lib.nml_paged_attention_workspace(2, 4, 2, 3, 200, 16, 64, 1, C.byref(need)))
    ws = upload(np.zeros(need.value, np.uint8))
    assert need.value  # (a row in pieces: counters that have to be left zero)
    N.check(N.lib.nml_verify_drafts_workspace(4, 5, 3000, C.byref(need)))
    vws, out = upload(np.zeros(need.value, np.uint8)), N.DeviceArray((2, 3, 256), np.float16)
    acc, tok = N.DeviceArray((4,), np.int32), N.DeviceArray((4, 6), np.int64)
    stats, dx = [N.DeviceArray((30,), np.float32) for _ in range(3)], N.DeviceArray((30, 999), np.float16)

    def work():
        N.check(N.lib.nml_paged_write_device(
            d["new"].ptr, d["new"].ptr, 2 * 3 * 64, 3 * 64, 64, cache.c.k_pages.ptr, cache.c.v_pages.ptr, d["table"].ptr,
            d["pos"].ptr, d["counts"].ptr, 2, 2, 3, 200, 16, cache.c.num_pages, 64, None, 1))
        N.check(N.lib.nml_paged_attention_device(
            d["q"].ptr, cache.c.k_pages.ptr, cache.c.v_pages.ptr, d["table"].ptr, d["lens"].ptr, d["counts"].ptr, out.ptr,
            2, 4, 2, 3, 200, 16, cache.c.num_pages, 64, 8.0, ws.ptr, ws.nbytes, None, 1))
        N.check(N.lib.nml_verify_drafts_device(
            d["logits"].ptr, 3000, d["draft"].ptr, 3000, d["drafts"].ptr, None, d["u"].ptr, 4, 5, 3000, 1.0, acc.ptr,
            tok.ptr, vws.ptr, vws.nbytes, None, 0))
        N.check(N.lib.nml_distill_device(d["x"].ptr, 999, d["ids"].ptr, d["y"].ptr, 30, 999, 8, 1.0,
                                         *(s.ptr for s in stats), None, 1))
        N.check(N.lib.nml_distill_backward_device(
            d["x"].ptr, 999, d["ids"].ptr, d["y"].ptr, stats[1].ptr, stats[2].ptr, d["dl"].ptr, 30, 999, 8, 1.0, dx.ptr,
            999, None, 1))

    def results():
        return [o.numpy() for o in (out, acc, tok, *stats, dx, cache.c.k_pages)]

    N.check(N.lib.nml_memset(out.ptr, 0, out.nbytes))
    graph = Graph(hip, work)
    try:
        for i in range(4):
            for name in ("q", "new", "logits", "u", "x", "y"):
                a = r.rand(*d[name].shape) if name == "u" else r.randn(*d[name].shape)
                a = np.ascontiguousarray(a, dtype=d[name].dtype)
                N.check(N.lib.nml_memcpy_h2d(d[name].ptr, a.ctypes.data, a.nbytes))
            N.synchronize()
            graph.run()
            K.token_logprobs(np.zeros((3, 50), np.float32), np.zeros(3, np.int64))  # eager, on the library's stream
            graph.wait()
            replayed = results()
            work()
            for a, b in zip(replayed, results()):
                assert np.array_equal(a, b, equal_nan=True), i
    finally:
        graph.close()


def test_two_streams_at_once(gpu, hip):  # noqa: F811
    """Calls on two streams, each with its own workspaces, over one cache: as one after another."""
    r = np.random.RandomState(5)
    cache = Cache(2, 2, 128, 16, 130, np.float16, 23)
    lens = upload(np.array([2080, 900], np.int32))
    table = upload(cache.table)
    V, batch, n = 20001, 5, 4
    need = N.sz()
    sides = []
    for seq in (4, 300):
        q = upload(queries(2, 4, seq, 128, np.float16, seq))
        N.check(N.lib.nml_paged_attention_workspace(2, 4, 2, seq, 130, 16, 128, 1, C.byref(need)))
        ws = upload(np.zeros(need.value, np.uint8))
        N.check(N.lib.nml_verify_drafts_workspace(batch, n, V, C.byref(need)))
        vws = upload(r.randint(0, 256, need.value).astype(np.uint8))
        logits, drafts, u = upload(r.randn(batch, n + 1, V).astype(np.float32)), upload(r.randint(0, V, (batch, n))), \
            upload(r.rand(batch, n + 1))
        out, acc, tok = N.DeviceArray((2, seq, 512), np.float16), N.DeviceArray((batch,), np.int32), \
            N.DeviceArray((batch, n + 1), np.int64)

        def work(seq=seq, q=q, ws=ws, vws=vws, logits=logits, drafts=drafts, u=u, out=out, acc=acc, tok=tok):
            N.check(N.lib.nml_paged_attention_device(
                q.ptr, cache.c.k_pages.ptr, cache.c.v_pages.ptr, table.ptr, lens.ptr, None, out.ptr, 2, 4, 2, seq, 130, 16,
                cache.c.num_pages, 128, 11.0, ws.ptr, ws.nbytes, None, 1))
            N.check(N.lib.nml_verify_drafts_device(
                logits.ptr, V, None, 0, drafts.ptr, None, u.ptr, batch, n, V, 1.0, acc.ptr, tok.ptr, vws.ptr, vws.nbytes,
                None, 0))

        work()
        N.synchronize()
        sides.append((work, (out, acc, tok), [o.numpy() for o in (out, acc, tok)]))
        for o in (out, acc, tok):
            N.check(N.lib.nml_memset(o.ptr, 0xff, o.nbytes))
    N.synchronize()
    graphs = [Graph(hip, side[0]) for side in sides]  # (each on a stream of its own)
    try:
        for _ in range(3):
            for _ in range(5):
                for g in graphs:
                    g.run()
            for g in graphs:
                g.wait()
            for _, outs, want in sides:
                for o, w in zip(outs, want):
                    assert np.array_equal(o.numpy(), w)
    finally:
        for g in graphs:
            g.close()


def test_empty_batches(gpu):
    loss, m, lsum = K.distill(np.zeros((0, 7), np.float32), np.zeros((0, 2)), np.zeros((0, 2)))
    assert loss.shape == m.shape == lsum.shape == (0,)
    accepted, tokens = K.verify_drafts(np.zeros((0, 3, 7), np.float32), np.zeros((0, 2)), np.zeros((0, 3)))
    assert accepted.shape == (0,) and tokens.shape == (0, 3)
    cache = K.PagedKVCache(2, 8, 1, 16, np.float16)
    none = np.zeros((0, 1, 2, 16), np.float16)
    K.paged_write(cache, none, none, np.zeros((0, 1)))
    assert K.paged_attention(none, cache, np.zeros((0, 1)), np.zeros(0), 4.0).shape == (0, 2, 16)
    no_tokens = np.zeros((2, 1, 0, 16), np.float16)
    K.paged_write(cache, no_tokens, no_tokens, np.zeros((2, 1)))
    assert K.paged_attention(no_tokens, cache, np.zeros((2, 1)), np.zeros(2), 4.0).shape == (2, 0, 16)
