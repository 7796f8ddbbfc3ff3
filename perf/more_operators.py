"""The operators that train a small drafting model from a large one and serve with both, as cases
to be measured.

Each case is one pass through an operator, in its plain form (elementary torch operations) or,
where ``own`` is true, through the framework's C entry points on device buffers:

  distill  the divergence of a model's distributions from a teacher's top logits, row by row
  dgrad    its gradient with respect to the model's logits
  verify   drafted tokens accepted or replaced by the target's distribution, from given uniforms
  store    K and V of new tokens written to the pages of a cache
  attend   attention of a row's newest tokens (one, a few drafted ones, a piece of a prompt) over
           the pages of its cache

A paged cache is two pools (pages, kv_heads, page_size, dk) and, for each row of the batch, the ids
of its pages in the order of its positions.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32}
CODES = {"float32": 0, "float16": 1}


def listed():
    return [
        # A training batch of the Small configuration (8 x 256 tokens) at the default dtype.
        {"name": "distill_small_f32", "op": "distill", "rows": 2048, "vocab": 4096, "top_k": 20,
         "temperature": 2.0, "absent": True, "dtype": "float32"},
        # 4096 tokens at a vocabulary of 32000 with as many teacher logits as log_probs gives.
        {"name": "distill_f16", "op": "distill", "rows": 4096, "vocab": 32000, "top_k": 64,
         "temperature": 1.0, "absent": False, "dtype": "float16"},
        # The gradients of the two.
        {"name": "dgrad_small_f32", "op": "dgrad", "rows": 2048, "vocab": 4096, "top_k": 20,
         "temperature": 2.0, "absent": True, "dtype": "float32"},
        {"name": "dgrad_f16", "op": "dgrad", "rows": 4096, "vocab": 32000, "top_k": 64,
         "temperature": 1.0, "absent": False, "dtype": "float16"},
        # One sequence's four drafted tokens: latency.
        {"name": "verify_b1_f32", "op": "verify", "batch": 1, "drafted": 4, "vocab": 32000,
         "temperature": 0.8, "sampled": True, "ragged": False, "dtype": "float32"},
        # A batch of 32, up to five drafted tokens a row.
        {"name": "verify_b32_f16", "op": "verify", "batch": 32, "drafted": 5, "vocab": 50304,
         "temperature": 1.0, "sampled": True, "ragged": True, "dtype": "float16"},
        # One layer's new K and V of a batched decode step: 32 rows at their own positions.
        {"name": "store_step_f16", "op": "store", "batch": 32, "heads": 16, "dk": 64, "seq": 1,
         "max_seq": 2048, "lo": 128, "hi": 1280, "page": 16, "ragged": False, "dtype": "float16"},
        # One layer's K and V of the first 4096 tokens of four prompts.
        {"name": "store_prompt_f16", "op": "store", "batch": 4, "heads": 16, "dk": 128,
         "seq": 4096, "max_seq": 4096, "lo": 0, "hi": 0, "page": 64, "ragged": False,
         "dtype": "float16"},
        # One layer's attention of a single sequence's decode step: latency.
        {"name": "attend_b1_f16", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 16,
         "dk": 64, "seq": 1, "max_seq": 2048, "lo": 1023, "hi": 1023, "page": 16, "ragged": False,
         "dtype": "float16"},
        # Decode of long sequences of ragged length with four query heads to a KV head.
        {"name": "attend_long_f16", "op": "attend", "batch": 16, "heads": 32, "kv_heads": 8,
         "dk": 128, "seq": 1, "max_seq": 8192, "lo": 1024, "hi": 8192, "page": 64, "ragged": False,
         "dtype": "float16"},
        # Up to five drafted tokens a row, default dtype, head dim 32, a page that ends anywhere.
        {"name": "attend_verify_f32", "op": "attend", "batch": 16, "heads": 8, "kv_heads": 8,
         "dk": 32, "seq": 5, "max_seq": 2048, "lo": 1, "hi": 2048, "page": 32, "ragged": True,
         "dtype": "float32"},
        # The last 2048 tokens of a prompt of 8192, prefilled in pieces.
        {"name": "attend_chunk_f16", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8,
         "dk": 128, "seq": 2048, "max_seq": 8192, "lo": 8192, "hi": 8192, "page": 64,
         "ragged": False, "dtype": "float16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: vocabularies, head dims and lengths of any size, ragged and
    empty rows, shared KV heads, pages of 8 to 256 tokens, both dtypes."""
    while True:
        c = _draw(rng)
        w = work(c)
        flops = w["flops"] * (8 if c["dtype"] == "float32" else 1)  # (products of 32 bits)
        if w["bytes"] <= 5.2e8 and flops <= 2.4e11 and _held(c) <= 2.5e9:
            return c


def _draw(rng):
    op = rng.choice(["distill", "dgrad", "verify", "verify", "store", "attend", "attend", "attend"])
    c = {"op": op, "dtype": rng.choice(["float16", "float32"])}
    if op in ("distill", "dgrad"):
        c.update(rows=_log_int(rng, 1, 4096), vocab=_log_int(rng, 100, 130000),
                 temperature=rng.choice([1.0, 1.0, 2.0, 0.7, 4.0]), absent=rng.random() < 0.4)
        c["top_k"] = min(c["vocab"], rng.choice([1, 5, 20, 50, 64, 100, rng.randint(1, 256)]))
        return c
    if op == "verify":
        c.update(batch=_log_int(rng, 1, 64), drafted=rng.choice([1, 2, 3, 4, 5, 8, 16]),
                 vocab=_log_int(rng, 100, 130000), temperature=rng.choice([1.0, 0.8, 0.6, 1.3, 0.0]),
                 sampled=rng.random() < 0.7, ragged=rng.random() < 0.5)
        return c
    dk = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 192, 256, rng.randint(1, 256)])
    max_seq = _log_int(rng, 16, 16384)
    c.update(batch=_log_int(rng, 1, 32), dk=dk, max_seq=max_seq, ragged=rng.random() < 0.5,
             page=rng.choice([8, 16, 16, 32, 64, 128, 256]))
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8, 12, 16])
        c.update(kv_heads=kv, heads=kv * rng.choice([1, 1, 1, 2, 4, 7, 8]),
                 seq=min(max_seq, rng.choice([1, 1, 1, 2, 5, 17, _log_int(rng, 2, 2048),
                                              _log_int(rng, 64, 2048)])))
        hi = rng.randint(c["seq"], max_seq) if c["seq"] > 1 else _log_int(rng, 1, max_seq)
        c.update(lo=rng.choice([0, hi // 8, hi]), hi=hi)
        return c
    seq = _log_int(rng, 1, max_seq)
    lo = rng.randint(0, max_seq - seq)
    c.update(heads=rng.choice([1, 4, 8, 12, 16]), seq=seq, lo=lo, hi=rng.randint(lo, max_seq - seq))
    return c


def _held(c):
    """About what the plain form holds of its largest tensor, in bytes."""
    if c["op"] in ("distill", "dgrad"):
        return 4 * c["rows"] * c["vocab"]
    if c["op"] == "verify":
        return 8 * c["batch"] * (c["drafted"] + 1) * c["vocab"]
    pages = 4 * c["batch"] * c.get("kv_heads", c["heads"]) * c["max_seq"] * c["dk"]
    if c["op"] == "store":
        return pages
    return max(pages, 4 * c["batch"] * c["heads"] * c["seq"] * c["max_seq"])


# ------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6151 + 17)
    return g


def _normal(g, shape, dtype, std=1.0):
    t = torch.empty(shape, device="cuda", dtype=torch.float32)
    t.normal_(0.0, std, generator=g)
    return t.to(dtype)


def _kv(g, shape, dtype):
    """Keys or values (..., dk): unit normal, one channel in 16 four times as large, as the keys
    of trained models have them."""
    t = _normal(g, shape, torch.float32)
    t[..., 5::16] *= 4.0
    return t.to(dtype)


def _ints(case, seed, lo, hi, salt):
    r = np.random.RandomState((int(seed) * 31 + salt) % (1 << 31))
    return torch.from_numpy(r.randint(lo, hi + 1, size=case["batch"]).astype(np.int32)).cuda()


def _logit_inputs(case, g, dt):
    n, v, k = case["rows"], case["vocab"], case["top_k"]
    s = {"logits": _normal(g, (n, v), dt, 2.5)}
    # a teacher that the model has come near to
    teacher = s["logits"].float() + _normal(g, (n, v), torch.float32, 0.7)
    top = torch.topk(teacher, k, dim=-1)
    s["top_logits"], s["top_ids"] = top.values.contiguous(), top.indices.contiguous()
    if case["absent"]:
        s["top_ids"][::7] = -1  # rows without a teacher (padding)
        s["top_ids"][1::5, k // 2:] = -1
    if case["op"] == "dgrad":
        # the forward's statistics, which a training step keeps, and the gradient of its losses
        x = s["logits"].double()
        m = x.amax(-1)
        s["m"] = m.float()
        s["l"] = ((x - m[:, None]) / case["temperature"]).exp().sum(-1).float()
        s["dloss"] = _normal(g, (n,), torch.float32)
    return s


def _verify_inputs(case, seed, g, dt):
    b, n, v, t = case["batch"], case["drafted"], case["vocab"], case["temperature"]
    s = {"logits": _normal(g, (b, n + 1, v), dt, 2.5)}
    draft = (s["logits"][:, :n].float() + _normal(g, (b, n, v), torch.float32, 0.7)).to(dt)
    if t > 0 and case["sampled"]:
        p = torch.softmax(draft.float() / t, -1).flatten(0, 1)
        s["drafts"] = torch.multinomial(p, 1, generator=g).view(b, n)
        s["draft_logits"] = draft
    else:
        s["drafts"] = draft.argmax(-1)
        s["draft_logits"] = None
    s["u"] = torch.rand((b, n + 1), device="cuda", dtype=torch.float64, generator=g)
    s["counts"] = _ints(case, seed, 0, n, 3) if case["ragged"] else \
        torch.full((b,), n, device="cuda", dtype=torch.int32)
    return s


def _pages(case):
    per_row = -(-case["max_seq"] // case["page"])
    return per_row, case["batch"] * per_row + 3


def _cache_inputs(case, seed, g, dt):
    b, dk, seq = case["batch"], case["dk"], case["seq"]
    kv = case.get("kv_heads", case["heads"])
    per_row, pages = _pages(case)
    s = {"counts": _ints(case, seed, 0, seq, 11) if case["ragged"] else
         torch.full((b,), seq, device="cuda", dtype=torch.int32)}
    s["counts"][0] = seq
    order = torch.randperm(pages, device="cuda", generator=g)[:b * per_row]
    s["table"] = order.to(torch.int32).view(b, per_row).contiguous()
    pool = (pages, kv, case["page"], dk)
    s["k_pages"], s["v_pages"] = _kv(g, pool, dt), _kv(g, pool, dt)
    if case["op"] == "store":
        # K and V as the QKV projection leaves them: (batch, seq, 3, heads, dk)
        s["qkv"] = _kv(g, (b, seq, 3, kv, dk), dt)
        s["pos"] = _ints(case, seed, case["lo"], case["hi"], 5)
    else:
        s["q"] = _normal(g, (b, case["heads"], seq, dk), dt)
        s["lens"] = _ints(case, seed, case["lo"], case["hi"], 5)
    return s


def _inputs(case, seed):
    """The tensors of one call, from the seed alone (prepare and exact both start here)."""
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    if case["op"] in ("distill", "dgrad"):
        return _logit_inputs(case, g, dt)
    if case["op"] == "verify":
        return _verify_inputs(case, seed, g, dt)
    return _cache_inputs(case, seed, g, dt)


def prepare(case, seed):
    s, op, dt = _inputs(case, seed), case["op"], DTYPES[case["dtype"]]
    if op == "distill":
        s["out"] = {k: torch.zeros((case["rows"],), device="cuda") for k in ("loss", "m", "l")}
    elif op == "dgrad":
        s["out"] = torch.zeros_like(s["logits"])
    elif op == "verify":
        b, n = case["batch"], case["drafted"]
        s["out"] = {"accepted": torch.zeros((b,), device="cuda", dtype=torch.int32),
                    "tokens": torch.zeros((b, n + 1), device="cuda", dtype=torch.int64)}
    elif op == "attend":
        s["out"] = torch.zeros((case["batch"], case["seq"], case["heads"] * case["dk"]),
                               device="cuda", dtype=dt)
    s["err"] = torch.zeros((1,), device="cuda", dtype=torch.int32)
    s["case"] = dict(case)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------- the plain forms

def _teacher(s, t, f):
    """(which entries are present, their ids, the teacher's probabilities, their logarithms)."""
    there = s["top_ids"] >= 0
    y = torch.where(there, s["top_logits"].to(f) / t, torch.full_like(s["top_logits"], -math.inf).to(f))
    top = y.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(y - top)
    z = e.sum(-1, keepdim=True)
    safe = torch.where(z == 0, torch.ones_like(z), z)
    logq = torch.where(there, y - top - torch.log(safe), torch.zeros_like(y))
    return there, s["top_ids"].clamp_min(0), e / safe, logq


def _distill_plain(s, c):
    t = c["temperature"]
    x = s["logits"].float()
    m = x.amax(-1)
    l = torch.exp((x - m[:, None]) / t).sum(-1)
    there, ids, q, logq = _teacher(s, t, torch.float32)
    logp = (x.gather(1, ids) - m[:, None]) / t - torch.log(l)[:, None]
    loss = (q * torch.where(there, logq - logp, torch.zeros_like(q))).sum(-1)
    taught = there.any(-1)
    zero = torch.zeros((), device="cuda")
    return {"loss": loss, "m": torch.where(taught, m, zero), "l": torch.where(taught, l, zero)}


def _dgrad_plain(s, c):
    t = c["temperature"]
    there, ids, q, _ = _teacher(s, t, torch.float32)
    d = torch.exp((s["logits"].float() - s["m"][:, None]) / t) / s["l"][:, None]
    d.scatter_add_(1, ids, torch.where(there, -q, torch.zeros_like(q)))
    d *= (s["dloss"] / t)[:, None]
    d = torch.where(there.any(-1)[:, None], d, torch.zeros_like(d))
    return d.to(DTYPES[c["dtype"]])


def _soft64(x, t):
    x = x.double()
    e = torch.exp((x - x.amax(-1, keepdim=True)) / t)
    return e / e.sum(-1, keepdim=True)


def _verify_plain(s, c):
    # in 64 bits: a draw falls to the next token where a running sum passes a uniform number
    b, n = c["batch"], c["drafted"]
    drafts, counts, u = s["drafts"], s["counts"].long(), s["u"]
    live = torch.arange(n, device="cuda") < counts[:, None]
    rows = torch.arange(b, device="cuda")
    if c["temperature"] <= 0:
        best = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True).indices[..., 0]
        ok = live & (drafts == best[:, :n])
        accepted = ok.long().cumprod(-1).sum(-1)
        token = best[rows, accepted]
    else:
        p = _soft64(s["logits"], c["temperature"])
        pd = p[:, :n].gather(-1, drafts[..., None])[..., 0]
        if s["draft_logits"] is not None:
            q = _soft64(s["draft_logits"], c["temperature"])
        else:
            q = torch.zeros_like(p[:, :n]).scatter_(-1, drafts[..., None], 1.0)
        qd = q.gather(-1, drafts[..., None])[..., 0]
        ok = live & (u[:, :n] * qd < pd)
        accepted = ok.long().cumprod(-1).sum(-1)
        last = p[rows, accepted]
        left = (last - q[rows, accepted.clamp_max(n - 1)]).clamp_min(0.0)
        use = (accepted < counts) & (left.sum(-1) > 0)
        w = torch.where(use[:, None], left, last)
        run = w.cumsum(-1)
        token = (run <= (u[:, n] * run[:, -1])[:, None]).sum(-1)
        at = torch.arange(c["vocab"], device="cuda")
        token = torch.minimum(token, torch.where(w > 0, at, torch.zeros_like(at)).amax(-1))
    i = torch.arange(n + 1, device="cuda")
    tokens = torch.cat([drafts, drafts[:, :1]], 1)
    tokens = torch.where(i < accepted[:, None], tokens, torch.full_like(tokens, -1))
    tokens[rows, accepted] = token
    return {"accepted": accepted.to(torch.int32), "tokens": tokens}


def _store_plain(s, c):
    t = torch.arange(c["seq"], device="cuda")
    row, tok = (t < s["counts"][:, None]).nonzero(as_tuple=True)
    at = s["pos"].long()[row] + tok
    page = s["table"].long()[row, at // c["page"]]
    for i, name in ((1, "k_pages"), (2, "v_pages")):
        s[name][page, :, at % c["page"]] = s["qkv"][row, tok, i]
    return [s["k_pages"], s["v_pages"]]


def _in_order(pages, table, kv, dk):
    """(batch, kv_heads, positions, dk) of the rows' pages, in 32 bits."""
    x = pages[table.long()].float()  # (batch, pages of a row, kv, page, dk)
    return x.transpose(1, 2).reshape(table.shape[0], kv, -1, dk)


def _attend_plain(s, c):
    b, h, kv, seq, dk = c["batch"], c["heads"], c["kv_heads"], c["seq"], c["dk"]
    k, v = (_in_order(s[n], s["table"], kv, dk) for n in ("k_pages", "v_pages"))
    at = torch.arange(k.shape[2], device="cuda")
    # (of positions past a row's length nothing is known)
    there = (at < s["lens"][:, None])[:, None, :, None]
    k, v = (torch.where(there, x, torch.zeros_like(x)) for x in (k, v))
    q = s["q"].float().reshape(b, kv, h // kv * seq, dk)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dk)
    x = x.reshape(b, kv, h // kv, seq, -1)
    t = torch.arange(seq, device="cuda")
    last = s["lens"][:, None] - s["counts"][:, None] + t  # (batch, seq): the last key attended
    seen = (at <= last[..., None])[:, None, None]
    x.masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(x - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.reshape(b, kv, h // kv * seq, -1), v).reshape(b, h, seq, dk)
    o = torch.where((t < s["counts"][:, None])[:, None, :, None], o, torch.zeros_like(o))
    return o.transpose(1, 2).reshape(b, seq, h * dk).to(DTYPES[c["dtype"]])


_PLAIN = {"distill": _distill_plain, "dgrad": _dgrad_plain, "verify": _verify_plain,
          "store": _store_plain, "attend": _attend_plain}


# --------------------------------------------------------------- the framework's calls

def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(N, s, size, *args):
    """The workspace of the call's sizes, which a program makes once and keeps."""
    if "ws" not in s:
        n = N.sz()
        N.check(size(*args, N.C.byref(n)))
        s["ws"] = torch.zeros((max(1, n.value),), device="cuda", dtype=torch.uint8)
        torch.cuda.synchronize()
    return s["ws"].data_ptr(), s["ws"].numel()


def _distill_own(N, s, c):
    o = s["out"]
    N.check(N.lib.nml_distill_device(
        s["logits"].data_ptr(), c["vocab"], s["top_ids"].data_ptr(), s["top_logits"].data_ptr(),
        c["rows"], c["vocab"], c["top_k"], c["temperature"], o["loss"].data_ptr(), o["m"].data_ptr(),
        o["l"].data_ptr(), s["err"].data_ptr(), CODES[c["dtype"]]))
    return o


def _dgrad_own(N, s, c):
    N.check(N.lib.nml_distill_backward_device(
        s["logits"].data_ptr(), c["vocab"], s["top_ids"].data_ptr(), s["top_logits"].data_ptr(),
        s["m"].data_ptr(), s["l"].data_ptr(), s["dloss"].data_ptr(), c["rows"], c["vocab"],
        c["top_k"], c["temperature"], s["out"].data_ptr(), c["vocab"], s["err"].data_ptr(),
        CODES[c["dtype"]]))
    return s["out"]


def _verify_own(N, s, c):
    ws = _workspace(N, s, N.lib.nml_verify_drafts_workspace, c["batch"], c["drafted"], c["vocab"])
    N.check(N.lib.nml_verify_drafts_device(
        s["logits"].data_ptr(), c["vocab"], _ptr(s["draft_logits"]), c["vocab"],
        s["drafts"].data_ptr(), s["counts"].data_ptr(), s["u"].data_ptr(), c["batch"], c["drafted"],
        c["vocab"], c["temperature"], s["out"]["accepted"].data_ptr(), s["out"]["tokens"].data_ptr(),
        *ws, s["err"].data_ptr(), CODES[c["dtype"]]))
    return s["out"]


def _store_own(N, s, c):
    k, v = s["qkv"][:, :, 1], s["qkv"][:, :, 2]
    per_row, pages = _pages(c)
    N.check(N.lib.nml_paged_write_device(
        k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(2), k.stride(1), s["k_pages"].data_ptr(),
        s["v_pages"].data_ptr(), s["table"].data_ptr(), s["pos"].data_ptr(), s["counts"].data_ptr(),
        c["batch"], c["heads"], c["seq"], per_row, c["page"], pages, c["dk"], s["err"].data_ptr(),
        CODES[c["dtype"]]))
    return [s["k_pages"], s["v_pages"]]


def _attend_own(N, s, c):
    per_row, pages = _pages(c)
    code = CODES[c["dtype"]]
    ws = _workspace(N, s, N.lib.nml_paged_attention_workspace, c["batch"], c["heads"],
                    c["kv_heads"], c["seq"], per_row, c["page"], c["dk"], code)
    N.check(N.lib.nml_paged_attention_device(
        s["q"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["table"].data_ptr(),
        s["lens"].data_ptr(), s["counts"].data_ptr(), s["out"].data_ptr(), c["batch"], c["heads"],
        c["kv_heads"], c["seq"], per_row, c["page"], pages, c["dk"], math.sqrt(c["dk"]), *ws,
        s["err"].data_ptr(), code))
    return s["out"]


_OWN = {"distill": _distill_own, "dgrad": _dgrad_own, "verify": _verify_own, "store": _store_own,
        "attend": _attend_own}


def run(state):
    c = state["case"]
    if own:
        from nimbleml_amd import _native as N

        N.ensure_init()
        return _OWN[c["op"]](N, state, c)
    return _PLAIN[c["op"]](state, c)


# --------------------------------------------------------------------------- work

def work(case):
    es, op = 2 if case["dtype"] == "float16" else 4, case["op"]
    if op in ("distill", "dgrad"):
        n = case["rows"] * case["vocab"]
        # rows without a teacher: one in seven
        live = n * (6 / 7 if case["absent"] and case["rows"] > 6 else 1)
        small = (12 * case["top_k"] + 12) * case["rows"]
        return {"bytes": es * live + (es * n if op == "dgrad" else 0) + small, "flops": 5 * live}
    some = 0.5 if case["ragged"] and case["batch"] > 1 else 1
    if op == "verify":
        drafted = case["batch"] * case["drafted"] * some
        rows = drafted * (2 if case["sampled"] and case["temperature"] > 0 else 1) + case["batch"]
        return {"bytes": es * rows * case["vocab"] + 24 * drafted, "flops": 4 * rows * case["vocab"]}
    tokens = case["batch"] * case["seq"] * some
    if op == "store":
        moved = 4 * es * tokens * case["heads"] * case["dk"]
        return {"bytes": moved, "flops": moved / es / 4}
    keys = case["batch"] * max(1.0, (case["lo"] + case["hi"]) / 2)
    pairs = tokens / case["batch"] * (keys - 0.5 * min(keys, tokens))  # a token sees what is before it
    return {"bytes": 2 * es * case["dk"] * (case["kv_heads"] * keys + tokens * case["heads"]),
            "flops": 4 * max(pairs, 1.0) * case["heads"] * case["dk"]}


# --------------------------------------------------------------------------- exact

def _exact_distill(case, s):
    t, n = case["temperature"], case["rows"]
    logp = torch.log_softmax(s["logits"].double() / t, -1)
    here = s["top_ids"] != -1
    y = (s["top_logits"].double() / t).masked_fill(~here, -math.inf)
    taught = here.any(-1)
    logq = y - torch.logsumexp(torch.where(taught[:, None], y, torch.zeros_like(y)), -1, keepdim=True)
    q = torch.where(here, logq.exp(), torch.zeros_like(y))
    at = torch.where(here, s["top_ids"], torch.zeros_like(s["top_ids"]))
    if case["op"] == "dgrad":
        # from the statistics that the call is given
        p = ((s["logits"].double() - s["m"].double()[:, None]) / t - s["l"].double().log()[:, None]).exp()
        full = torch.zeros_like(p).scatter_add_(1, at, q)
        return (p - full) * (s["dloss"].double() / t * taught)[:, None]
    terms = torch.where(here, q * (logq - logp.gather(1, at)), torch.zeros_like(q))
    top = s["logits"].double().amax(-1)
    return {"loss": terms.sum(-1), "m": top * taught,
            "l": (torch.logsumexp(s["logits"].double() / t, -1) - top / t).exp() * taught}


def _exact_verify(case, s):
    """Row by row and draft by draft, as the rule is told."""
    t, v = case["temperature"], case["vocab"]
    u, counts, drafts = s["u"].tolist(), s["counts"].tolist(), s["drafts"].tolist()
    accepted = torch.zeros((case["batch"],), device="cuda", dtype=torch.int32)
    tokens = torch.full((case["batch"], case["drafted"] + 1), -1, device="cuda", dtype=torch.int64)

    def dist(x):
        x = x.double()
        if t <= 0:
            hot = torch.zeros_like(x)
            hot[int((x == x.max()).nonzero()[0])] = 1.0
            return hot
        return torch.softmax(x / t, -1)

    for b in range(case["batch"]):
        i, w = 0, None
        while i < counts[b]:
            p, d = dist(s["logits"][b, i]), drafts[b][i]
            if t > 0 and s["draft_logits"] is not None:
                q = dist(s["draft_logits"][b, i])
            else:
                q = torch.zeros((v,), device="cuda", dtype=torch.float64)
                q[d] = 1.0
            pd, qd = float(p[d]), float(q[d])
            if (pd == 1.0) if t <= 0 else (u[b][i] * qd < pd):
                tokens[b, i] = d
                i += 1
                continue
            w = torch.relu(p - q) if t > 0 else p
            if float(w.sum()) == 0.0:
                w = p
            break
        if w is None:
            w = dist(s["logits"][b, i])
        accepted[b] = i
        run = torch.cumsum(w, 0)
        past = (run > u[b][-1] * run[-1]).nonzero()
        tokens[b, i] = int(past[0]) if len(past) and t > 0 else int(w.nonzero()[-1])
    return {"accepted": accepted, "tokens": tokens}


def _exact_store(case, s):
    out = [s["k_pages"].double(), s["v_pages"].double()]
    table, pos, counts = s["table"].tolist(), s["pos"].tolist(), s["counts"].tolist()
    size = case["page"]
    for b in range(case["batch"]):
        done = 0
        while done < counts[b]:
            at = pos[b] + done
            n = min(size - at % size, counts[b] - done)
            for i in (0, 1):
                new = s["qkv"][b, done:done + n, i + 1].double()
                out[i][table[b][at // size], :, at % size:at % size + n] = new.transpose(0, 1)
            done += n
    return out


def _exact_attend(case, s):
    group, dk, size = case["heads"] // case["kv_heads"], case["dk"], case["page"]
    out = torch.zeros((case["batch"], case["seq"], case["heads"], dk), device="cuda",
                      dtype=torch.float64)
    counts = s["counts"].tolist()
    for b, length in enumerate(s["lens"].tolist()):
        n, used = counts[b], -(-length // size)
        if n == 0 or length == 0:
            continue
        ids = s["table"][b, :used].long()
        k, v = (torch.cat(list(s[name][ids].double()), 1)[:, :length] for name in ("k_pages", "v_pages"))
        last = torch.arange(length - n, length, device="cuda")
        seen = torch.arange(length, device="cuda")[None] <= last[:, None]
        for h in range(case["heads"]):
            w = s["q"][b, h, :n].double() @ k[h // group].T.contiguous() / math.sqrt(dk)
            w = torch.softmax(w.masked_fill(~seen, -math.inf), -1)
            w = torch.where(seen.any(-1, keepdim=True), w, torch.zeros_like(w))
            out[b, :n, h] = w @ v[h // group]
    return out.flatten(-2)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("distill", "dgrad"):
        return _exact_distill(case, s)
    return {"verify": _exact_verify, "store": _exact_store, "attend": _exact_attend}[case["op"]](case, s)
