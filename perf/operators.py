"""The operators that serve from a 4-bit KV cache and score tokens, as cases to be measured.

Each case is one pass through an operator, in its plain form (elementary torch operations in
32 bits) or, where ``own`` is true, through the framework's C entry points on device buffers:

  store   K and V of new tokens quantised into the cache, then read back from it
  read    a cached prefix as values in the compute dtype
  attend  attention of new tokens over the cache (decode, several tokens, shared KV heads)
  score   log probabilities of given tokens with entropy and the best alternatives
  grad    the gradient of log probabilities and entropies with respect to the logits

The cache holds blocks of 32 values along a head's vector: 32 E2M1 codes (two a byte, the first
in the low four bits) and one scale byte e standing for 2^(e - 127), 255 for NaN.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32}
CODES = {"float32": 0, "float16": 1}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MIDS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between neighbours of GRID
IGNORE = -100


def listed():
    return [
        # One layer's new K and V of a batched decode step: 32 rows at their own positions.
        {"name": "store_step_f16", "op": "store", "batch": 32, "heads": 16, "dk": 64, "seq": 1,
         "max_seq": 2048, "lo": 128, "hi": 1280, "ragged": False, "dtype": "float16"},
        # One layer's K and V of a 4 x 4096 prompt, written to an empty cache.
        {"name": "store_prompt_f16", "op": "store", "batch": 4, "heads": 16, "dk": 128,
         "seq": 4096, "max_seq": 4096, "lo": 0, "hi": 0, "ragged": False, "dtype": "float16"},
        # A ragged prefix read back for the next piece of a prompt, at a head dim that fills no
        # whole number of blocks.
        {"name": "read_ragged_f32", "op": "read", "batch": 8, "heads": 12, "dk": 80, "seq": 1000,
         "max_seq": 1000, "lo": 0, "hi": 0, "ragged": True, "dtype": "float32"},
        # The whole 4 x 4096 prefix of one layer.
        {"name": "read_prefix_f16", "op": "read", "batch": 4, "heads": 16, "dk": 128, "seq": 4096,
         "max_seq": 4096, "lo": 0, "hi": 0, "ragged": False, "dtype": "float16"},
        # One layer's attention of a single sequence's decode step: latency.
        {"name": "attend_b1_f16", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 16,
         "dk": 64, "seq": 1, "max_seq": 2048, "lo": 1023, "hi": 1023, "ragged": False,
         "dtype": "float16"},
        # The same of a batch of 32 rows of ragged length.
        {"name": "attend_b32_f16", "op": "attend", "batch": 32, "heads": 16, "kv_heads": 16,
         "dk": 64, "seq": 1, "max_seq": 2048, "lo": 128, "hi": 1280, "ragged": False,
         "dtype": "float16"},
        # Long sequences with four query heads to a KV head: what the 4-bit cache is for.
        {"name": "attend_long_f16", "op": "attend", "batch": 8, "heads": 32, "kv_heads": 8,
         "dk": 128, "seq": 1, "max_seq": 32768, "lo": 8192, "hi": 32768, "ragged": False,
         "dtype": "float16"},
        # Up to five guessed tokens a row checked at once, default dtype, head dim 32.
        {"name": "attend_verify_f32", "op": "attend", "batch": 16, "heads": 8, "kv_heads": 8,
         "dk": 32, "seq": 5, "max_seq": 2048, "lo": 1, "hi": 2048, "ragged": True,
         "dtype": "float32"},
        # Scoring 4096 given tokens over a vocabulary of 50304.
        {"name": "score_f16", "op": "score", "rows": 4096, "vocab": 50304, "top_k": 0,
         "ignored": False, "dtype": "float16"},
        # A decode step's chosen tokens with their 20 best alternatives.
        {"name": "score_top_f32", "op": "score", "rows": 32, "vocab": 32000, "top_k": 20,
         "ignored": False, "dtype": "float32"},
        # The gradient over a training batch's logits.
        {"name": "grad_f16", "op": "grad", "rows": 4096, "vocab": 32000, "ignored": True,
         "dtype": "float16"},
        # The same of the Small configuration (8 x 256 tokens) at the default dtype.
        {"name": "grad_small_f32", "op": "grad", "rows": 2048, "vocab": 4096, "ignored": True,
         "dtype": "float32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: any head dim, ragged and empty rows, several new tokens,
    shared KV heads, vocabularies of any size, both dtypes."""
    while True:
        c = _draw(rng)
        limit = 1.1e9 if c["op"] == "grad" else 4.2e8
        if work(c)["bytes"] <= limit and _plain_bytes(c) <= 2.5e9:
            return c


def _draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "attend", "score", "score", "grad"])
    c = {"op": op, "dtype": rng.choice(["float16", "float32"])}
    if op in ("score", "grad"):
        c.update(rows=_log_int(rng, 1, 4096), vocab=_log_int(rng, 100, 100000),
                 ignored=rng.random() < 0.3)
        if op == "score":
            c["top_k"] = rng.choice([0, 0, 1, 5, 20, 50])
        return c
    dk = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 192, 256, rng.randint(1, 256)])
    max_seq = _log_int(rng, 16, 32768)
    c.update(batch=_log_int(rng, 1, 48), dk=dk, max_seq=max_seq, ragged=rng.random() < 0.5)
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8, 12, 16])
        c.update(kv_heads=kv, heads=kv * rng.choice([1, 1, 1, 2, 4, 7, 8]),
                 seq=min(max_seq, rng.choice([1, 1, 1, 2, 3, 5, 8, 17])))
        hi = _log_int(rng, 1, max_seq)
        c.update(lo=rng.choice([0, hi // 8, hi]), hi=hi)
        return c
    seq = _log_int(rng, 1, max_seq)
    lo = rng.randint(0, max_seq - seq)
    c.update(heads=rng.choice([1, 4, 8, 12, 16]), seq=seq, lo=lo,
             hi=rng.randint(lo, max_seq - seq))
    return c


def _plain_bytes(c):
    """What the plain form holds of the largest tensor, in bytes."""
    if c["op"] in ("score", "grad"):
        return 4 * c["rows"] * c["vocab"]
    return 4 * c["batch"] * c.get("kv_heads", c["heads"]) * c["max_seq"] * 32 * _blocks(c)


# ------------------------------------------------------------------------- inputs

def _blocks(case):
    return -(-case["dk"] // 32)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
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
    return r.randint(lo, hi + 1, size=case["batch"]).astype(np.int32)


def _inputs(case, seed):
    """The tensors of one call, from the seed alone (prepare and exact both start here)."""
    g, dt, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    if op in ("score", "grad"):
        n, v = case["rows"], case["vocab"]
        s = {"logits": _normal(g, (n, v), dt, 2.5),
             "targets": torch.randint(0, v, (n,), device="cuda", dtype=torch.int64, generator=g)}
        if case["ignored"]:
            s["targets"][::7] = IGNORE
        if op == "grad":
            # the forward's statistics, which a training step keeps, and the two gradients
            x = s["logits"].double()
            m = x.amax(-1)
            e = (x - m[:, None]).exp()
            z = e.sum(-1)
            s["m"], s["l"] = m.float(), z.float()
            s["entropy"] = (z.log() - (e * (x - m[:, None])).sum(-1) / z).float()
            s["dlogp"], s["dentropy"] = _normal(g, (n,), torch.float32), _normal(g, (n,), torch.float32, 0.1)
        return s
    b, dk, seq = case["batch"], case["dk"], case["seq"]
    counts = np.full(b, seq, np.int32)
    if case["ragged"]:
        counts = _ints(case, seed, 0, seq, 11)
        counts[0] = seq
    s = {"counts": torch.from_numpy(counts).cuda()}
    if op == "store":
        # K and V as the QKV projection leaves them: (batch, seq, 3, heads, dk)
        s["qkv"] = _kv(g, (b, seq, 3, case["heads"], dk), dt)
        s["pos"] = torch.from_numpy(_ints(case, seed, case["lo"], case["hi"], 5)).cuda()
        return s
    kv = case.get("kv_heads", case["heads"])
    cached = (b, kv, case["max_seq"], dk)
    s["k"], s["v"] = _kv(g, cached, dt), _kv(g, cached, dt)
    if op == "read":
        s["pos"] = torch.from_numpy(_ints(case, seed, case["lo"], case["hi"], 5)).cuda()
        return s
    s["q"] = _normal(g, (b, case["heads"], seq, dk), dt)
    s["lens"] = torch.from_numpy(_ints(case, seed, case["lo"], case["hi"], 5)).cuda()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "store":
        shape = (case["batch"], case["heads"], case["max_seq"], _blocks(case))
        s["cache"] = [torch.zeros(shape + (16,) * (i % 2 == 0), device="cuda", dtype=torch.uint8)
                      for i in range(4)]
    elif op in ("read", "attend"):
        s["cache"] = [t for x in (s.pop("k"), s.pop("v")) for t in _quantise(x)]
    if op in ("store", "read"):
        shape = (case["batch"], case["heads"], case["seq"], case["dk"])
        s["out"] = [torch.zeros(shape, device="cuda", dtype=dt) for _ in range(2)]
    elif op == "attend":
        s["out"] = torch.zeros((case["batch"], case["seq"], case["heads"] * case["dk"]),
                               device="cuda", dtype=dt)
    elif op == "score":
        n, k = case["rows"], case["top_k"]
        s["out"] = {name: torch.zeros((n,), device="cuda") for name in ("logp", "entropy", "m", "l")}
        if k:
            s["out"]["top_ids"] = torch.zeros((n, k), device="cuda", dtype=torch.int64)
            s["out"]["top_logp"] = torch.zeros((n, k), device="cuda")
    else:
        s["out"] = torch.zeros_like(s["logits"])
    s["err"] = torch.zeros((1,), device="cuda", dtype=torch.int32)
    s["case"] = dict(case)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------- the plain forms

def _quantise(x):
    """(codes (..., blocks, 16), scales (..., blocks)) of values (..., dk)."""
    dk, top = x.shape[-1], 13 if x.dtype == torch.float16 else 125
    x = torch.nn.functional.pad(x.float(), (0, -dk % 32))
    x = x.reshape(x.shape[:-1] + (-1, 32))
    amax = x.abs().amax(-1)
    m, k = torch.frexp(amax)  # amax = m * 2^k, 1/2 <= m < 1
    e = (k.int() - 3 + (m >= 0.875).int()).clamp(-120, top)
    e = torch.where(amax == 0, torch.full_like(e, -120), e)
    finite = torch.isfinite(amax)
    # 2^-e takes two factors: one alone overflows at the smallest scales
    half = -e // 2
    a = x.abs() * torch.exp2(half.float())[..., None] * torch.exp2((-e - half).float())[..., None]
    mids = torch.tensor(MIDS, device=x.device)
    # a tie goes to the even code: of the midpoints with even index below, of the others above
    c = torch.bucketize(a, mids) + ((a == 0.75) | (a == 1.75) | (a == 3.5)).long()
    c = c + 8 * torch.signbit(x).long()
    c = torch.where(finite[..., None], c, torch.zeros_like(c)).to(torch.uint8)
    scale = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), scale


def _values(codes, scales, dk):
    """The float32 values (..., dk) that a cache's codes and scales stand for."""
    table = torch.tensor(GRID + tuple(-x for x in GRID), device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    e = torch.exp2(scales.float() - 127)
    e = torch.where(scales == 255, torch.full_like(e, math.nan), e)
    return (v * e[..., None]).flatten(-2)[..., :dk]


def _rows(case, s):
    """(index of the cache's positions (batch, seq), which of them are written or read)."""
    t = torch.arange(case["seq"], device="cuda")
    at = s["pos"].long()[:, None] + t
    live = t < s["counts"][:, None]
    return at.clamp(0, case["max_seq"] - 1), live


def _read_one(s, c, codes, scales):
    at, live = _rows(c, s)
    b = torch.arange(c["batch"], device="cuda")[:, None]
    x = _values(codes[b, :, at], scales[b, :, at], c["dk"])  # (batch, seq, heads, dk)
    x = torch.where(live[:, :, None, None], x, torch.zeros_like(x))
    return x.permute(0, 2, 1, 3).to(DTYPES[c["dtype"]]).contiguous()


def _read_plain(s, c):
    return [_read_one(s, c, *s["cache"][:2]), _read_one(s, c, *s["cache"][2:])]


def _store_one(s, c, x, codes, scales):
    at, live = _rows(c, s)
    b = torch.arange(c["batch"], device="cuda")[:, None]
    new_codes, new_scales = _quantise(x)  # (batch, seq, heads, ...)
    live = live[:, :, None, None]
    codes[b, :, at] = torch.where(live[..., None], new_codes, codes[b, :, at])
    scales[b, :, at] = torch.where(live, new_scales, scales[b, :, at])


def _store_plain(s, c):
    _store_one(s, c, s["qkv"][:, :, 1], *s["cache"][:2])
    _store_one(s, c, s["qkv"][:, :, 2], *s["cache"][2:])
    return _read_plain(s, c)


def _attend_plain(s, c):
    b, h, kv, seq, dk = c["batch"], c["heads"], c["kv_heads"], c["seq"], c["dk"]
    k, v = (_values(*s["cache"][i:i + 2], dk) for i in (0, 2))
    q = s["q"].float().reshape(b, kv, h // kv * seq, dk)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dk)
    x = x.reshape(b, kv, h // kv, seq, -1)
    t = torch.arange(seq, device="cuda")
    last = s["lens"][:, None] - s["counts"][:, None] + t  # (batch, seq): the last key attended
    seen = torch.arange(c["max_seq"], device="cuda") <= last[..., None]
    seen = seen[:, None, None]
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - top), torch.zeros_like(x))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.reshape(b, kv, h // kv * seq, -1), v).reshape(b, h, seq, dk)
    o = torch.where((t < s["counts"][:, None])[:, None, :, None], o, torch.zeros_like(o))
    return o.transpose(1, 2).reshape(b, seq, h * dk).to(DTYPES[c["dtype"]])


def _score_plain(s, c):
    x, target = s["logits"].float(), s["targets"]
    kept = target != IGNORE
    zero = torch.zeros((), device="cuda")
    top = x.amax(-1, keepdim=True)
    t = x - top
    e = torch.exp(t)
    z = e.sum(-1)
    entropy = torch.log(z) - (e * torch.where(e == 0, zero, t)).sum(-1) / z
    logp = t.gather(1, target.clamp_min(0)[:, None])[:, 0] - torch.log(z)
    out = {"logp": torch.where(kept, logp, zero), "entropy": torch.where(kept, entropy, zero),
           "m": torch.where(kept, top[:, 0], zero), "l": torch.where(kept, z, zero)}
    if c["top_k"]:
        best, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        ids, best = ids[:, :c["top_k"]], best[:, :c["top_k"]] - top - torch.log(z)[:, None]
        out["top_ids"] = torch.where(kept[:, None], ids, torch.full_like(ids, -1))
        out["top_logp"] = torch.where(kept[:, None], best, zero)
    return out


def _grad_plain(s, c):
    logp = s["logits"].float() - s["m"][:, None] - torch.log(s["l"])[:, None]
    p = torch.exp(logp)
    d = -s["dlogp"][:, None] * p
    d -= s["dentropy"][:, None] * p * torch.where(p == 0, torch.zeros_like(p),
                                                  logp + s["entropy"][:, None])
    d.scatter_add_(1, s["targets"].clamp_min(0)[:, None], s["dlogp"][:, None])
    d = torch.where((s["targets"] != IGNORE)[:, None], d, torch.zeros_like(d))
    return d.to(DTYPES[c["dtype"]])


_PLAIN = {"store": _store_plain, "read": _read_plain, "attend": _attend_plain,
          "score": _score_plain, "grad": _grad_plain}


# --------------------------------------------------------------- the framework's calls

def _read_own(N, s, c):
    N.check(N.lib.nml_kv4_read_device(
        *(t.data_ptr() for t in s["cache"]), s["pos"].data_ptr(), s["counts"].data_ptr(),
        *(t.data_ptr() for t in s["out"]), c["batch"], c["heads"], c["seq"], c["max_seq"], c["dk"],
        s["err"].data_ptr(), CODES[c["dtype"]]))
    return s["out"]


def _store_own(N, s, c):
    k, v = s["qkv"][:, :, 1], s["qkv"][:, :, 2]
    N.check(N.lib.nml_kv4_write_device(
        k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(2), k.stride(1),
        *(t.data_ptr() for t in s["cache"]), s["pos"].data_ptr(), s["counts"].data_ptr(),
        c["batch"], c["heads"], c["seq"], c["max_seq"], c["dk"], s["err"].data_ptr(),
        CODES[c["dtype"]]))
    return _read_own(N, s, c)


def _attend_own(N, s, c):
    sizes = (c["batch"], c["heads"], c["kv_heads"], c["seq"], c["max_seq"], c["dk"])
    if "ws" not in s:  # a program keeps one workspace for its sizes
        n = N.sz()
        N.check(N.lib.nml_kv4_attention_workspace(*sizes, N.C.byref(n)))
        s["ws"] = torch.zeros((max(1, n.value),), device="cuda", dtype=torch.uint8)
        torch.cuda.synchronize()
    N.check(N.lib.nml_kv4_attention_device(
        s["q"].data_ptr(), *(t.data_ptr() for t in s["cache"]), s["lens"].data_ptr(),
        s["counts"].data_ptr(), s["out"].data_ptr(), *sizes, math.sqrt(c["dk"]),
        s["ws"].data_ptr(), s["ws"].numel(), s["err"].data_ptr(), CODES[c["dtype"]]))
    return s["out"]


def _score_own(N, s, c):
    o, k = s["out"], c["top_k"]
    N.check(N.lib.nml_token_logprobs_device(
        s["logits"].data_ptr(), c["vocab"], s["targets"].data_ptr(), c["rows"], c["vocab"], IGNORE,
        1, k, o["logp"].data_ptr(), o["entropy"].data_ptr(), o["m"].data_ptr(), o["l"].data_ptr(),
        o["top_ids"].data_ptr() if k else None, o["top_logp"].data_ptr() if k else None,
        s["err"].data_ptr(), CODES[c["dtype"]]))
    return o


def _grad_own(N, s, c):
    N.check(N.lib.nml_token_logprobs_backward_device(
        s["logits"].data_ptr(), c["vocab"], s["targets"].data_ptr(), s["m"].data_ptr(),
        s["l"].data_ptr(), s["entropy"].data_ptr(), s["dlogp"].data_ptr(), s["dentropy"].data_ptr(), c["rows"],
        c["vocab"], IGNORE, 1, s["out"].data_ptr(), c["vocab"], s["err"].data_ptr(),
        CODES[c["dtype"]]))
    return s["out"]


_OWN = {"store": _store_own, "read": _read_own, "attend": _attend_own, "score": _score_own,
        "grad": _grad_own}


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
    if op in ("score", "grad"):
        n = case["rows"] * case["vocab"]
        if op == "grad":
            return {"bytes": 2 * es * n + 28 * case["rows"], "flops": 8 * n}
        return {"bytes": es * n + (24 + 12 * case["top_k"]) * case["rows"], "flops": 6 * n}
    tokens = case["batch"] * case["seq"] * (0.5 if case["ragged"] and case["batch"] > 1 else 1)
    if op != "attend":
        vectors = 2 * tokens * case["heads"]  # K's and V's
        cache, values = 17 * _blocks(case), es * case["dk"]
        moved = cache + values * (2 if op == "store" else 1)
        return {"bytes": vectors * moved, "flops": (2 if op == "read" else 6) * vectors * case["dk"]}
    keys = case["batch"] * max(1.0, (case["lo"] + case["hi"]) / 2)
    return {"bytes": 34 * _blocks(case) * case["kv_heads"] * keys +
            2 * es * tokens * case["heads"] * case["dk"],
            "flops": 4 * keys * tokens / case["batch"] * case["heads"] * case["dk"]}


# --------------------------------------------------------------------------- exact

def _held64(x):
    """The values that the cache holds of x (..., dk), in 64 bits: per block of 32 the power of
    two, then the nearest of the 15 values, the one of even code where two are as near."""
    shape, dk = x.shape, x.shape[-1]
    limit = 13 if x.dtype == torch.float16 else 125
    x = x.double()
    wide = torch.zeros(shape[:-1] + (-(-dk // 32) * 32,), device=x.device, dtype=torch.float64)
    wide[..., :dk] = x
    wide = wide.view(shape[:-1] + (-(-dk // 32), 32))
    big = wide.abs().amax(-1, keepdim=True)
    k = torch.floor(torch.log2(big.clamp_min(1e-300)))
    k = k + (2.0 ** (k + 1) <= big).double() - (2.0 ** k > big).double()
    e = k - 2 + (big >= 1.75 * 2.0 ** k).double()
    step = 2.0 ** e.clamp(-120, limit)
    a = wide.abs() / step
    # below 2 the values are half a unit apart, below 4 a unit, above two units; the rounding of
    # each stretch is to the even multiple, which is the even code
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    held = r.clamp_max(6) * step * torch.sign(wide)
    return held.flatten(-2)[..., :dk]


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op in ("score", "grad"):
        x, t = s["logits"].double(), s["targets"]
        keep = (t != IGNORE).double()
        at = t.clamp_min(0)[:, None]
        if op == "grad":
            lp = x - s["m"].double()[:, None] - s["l"].double().log()[:, None]
            p = lp.exp()
            hot = torch.zeros_like(x).scatter_(1, at, 1.0)
            d = s["dlogp"].double()[:, None] * (hot - p)
            d = d - s["dentropy"].double()[:, None] * p * (lp + s["entropy"].double()[:, None])
            return d * keep[:, None]
        lse = torch.logsumexp(x, -1)
        lp = x - lse[:, None]
        out = {"logp": lp.gather(1, at)[:, 0] * keep, "entropy": -(lp.exp() * lp).sum(-1) * keep,
               "m": x.amax(-1) * keep, "l": (x - x.amax(-1, keepdim=True)).exp().sum(-1) * keep}
        if case["top_k"]:
            out["top_ids"] = None
            out["top_logp"] = torch.topk(lp, case["top_k"], -1).values * keep[:, None]
        return out
    n = s["counts"].tolist()
    if op in ("store", "read"):
        out = []
        for i, name in enumerate(("k", "v")):
            y = torch.zeros((case["batch"], case["heads"], case["seq"], case["dk"]), device="cuda",
                            dtype=torch.float64)
            for b, p in enumerate(s["pos"].tolist()):
                src = s["qkv"][b, :n[b], i + 1].transpose(0, 1) if op == "store" else \
                    s[name][b, :, p:p + n[b]]
                y[b, :, :n[b]] = _held64(src)
            out.append(y)
        return out
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros((case["batch"], case["seq"], case["heads"], case["dk"]), device="cuda",
                      dtype=torch.float64)
    for b, length in enumerate(s["lens"].tolist()):
        k, v = _held64(s["k"][b, :, :length]), _held64(s["v"][b, :, :length])
        for t in range(n[b]):
            last = length - n[b] + t + 1
            if last <= 0:
                continue
            q = s["q"][b, :, t].double().view(case["kv_heads"], group, -1)
            w = torch.softmax(q @ k[:, :last].transpose(1, 2).contiguous() / math.sqrt(case["dk"]), -1)
            out[b, t] = (w @ v[:, :last]).reshape(case["heads"], -1)
    return out.flatten(-2)
