"""Array-level device ops under the reference kernel names (NimbleML/kernels/).

Each takes host arrays or ``DeviceArray``s in the compute dtype and returns
``DeviceArray`` results computed by the HIP kernels:
  fused_rmsnorm_forward       kernels/fused_rmsnorm.py:130-162
  fused_gelu_forward          kernels/fused_gelu.py:57-83
  fused_sdpa_forward          kernels/fused_sdpa.py:256-289 (any additive mask, or none)
  decode_attention            one cached decode step of that attention (the KV-cache seam of
                              models/generate.py:93-100; no reference kernel)
  KV4Cache, kv4_write, kv4_read, kv4_attention
                              a KV cache in 4 bits: quantised as it is written, read back,
                              attended to by one or several new tokens (no reference kernel)
  PagedKVCache, paged_write, paged_attention, paged_attention_workspace
                              a KV cache in pages: written, attended to by one or several new
                              tokens (no reference kernel)
  token_logprobs, token_logprobs_backward
                              log probabilities of given tokens, entropies and the best
                              alternatives, and their gradient (no reference kernel)
  distill, distill_backward   divergence from a teacher's top logits and its gradient (no
                              reference kernel)
  verify_drafts               drafted tokens accepted or replaced by the target's distribution
                              (no reference kernel)
  embedding_lookup            kernels/embedding_scatter.py:25-36
  fused_tied_crossentropy_forward  kernels/fused_tied_crossentropy.py:8-24 (loss only)
  linear                      the `x @ W + b` of neural_network/_fused_arrays.py:25-30
  sample_tokens               models/generate.py:23-59 on a (batch, vocab) logits block
  adamw_step                  native adamw_step (native/src/adamw.cpp:6-20), in place
  clip_grad_norm              native clip_grad_norm (native/src/adamw.cpp:22-37), in place
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from nimbleml_amd import _native as N
from nimbleml_amd import np_backend
from nimbleml_amd.tensor import Tensor

EPI_NONE, EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESID = 0, 1, 2, 3


def _dev(x, dtype=None):
    if isinstance(x, N.DeviceArray):
        if dtype is not None and x.dtype != np.dtype(dtype):
            raise TypeError(f"expected {np.dtype(dtype)}, got {x.dtype}")
        return x
    return N.DeviceArray.from_host(np.asarray(x, dtype=dtype if dtype is not None else None))


def _float_dtype(x):
    dt = np.dtype(x.dtype) if hasattr(x, "dtype") else np.dtype(np_backend.dtype)
    N.np_dtype_code(dt)
    return dt


def fused_rmsnorm_forward(x, gamma, epsilon=1e-5):
    """Returns (out, x, ms, rms) with ms/rms shaped (rows, 1) like the reference."""
    dt = _float_dtype(x)
    xd, gd = _dev(x, dt), _dev(gamma, dt)
    d = xd.shape[-1]
    rows = xd.size // d
    out = N.DeviceArray(xd.shape, dt)
    ms = N.DeviceArray((rows, 1), np.float32)
    rms = N.DeviceArray((rows, 1), np.float32)
    N.check(N.lib.nml_rmsnorm_forward_device(xd.ptr, gd.ptr, out.ptr, ms.ptr, rms.ptr, rows, d,
                                             float(epsilon), N.np_dtype_code(dt)))
    return out, xd, ms, rms


def fused_gelu_forward(x):
    """Returns (out, tanh_u) — tanh_u in float32 as in the reference."""
    dt = _float_dtype(x)
    xd = _dev(x, dt)
    out = N.DeviceArray(xd.shape, dt)
    tu = N.DeviceArray(xd.shape, np.float32)
    N.check(N.lib.nml_gelu_forward_device(xd.ptr, out.ptr, tu.ptr, xd.size, N.np_dtype_code(dt)))
    return out, tu


def fused_sdpa_forward(q, k, v, scale, mask_arr=None, *, batch=None, num_heads=None):
    """Attention over (bh, seq, dk) (kernels/fused_sdpa.py:256-289); ``scale`` is the
    sqrt(dk) divisor. ``mask_arr``: None attends to every key (the reference's
    ``_matmul_sdpa_forward`` without a mask); the causal mask (−inf above the diagonal)
    runs the causal kernels; any other additive (seq, seq) mask is added to the scaled
    scores. Returns ``(out, None)``: no probability matrix is formed."""
    dt = _float_dtype(q)
    qd, kd, vd = _dev(q, dt), _dev(k, dt), _dev(v, dt)
    bh, seq, dk = qd.shape
    causal, md = 0, None
    if mask_arr is not None:
        m = np.ascontiguousarray(np.asarray(mask_arr).astype(dt, copy=False))
        if m.shape != (seq, seq):
            raise ValueError(f"mask must be ({seq}, {seq}), got {m.shape}")
        if np.array_equal(m, np.triu(np.full((seq, seq), -np.inf, dtype=dt), k=1)):
            causal = 1
        else:
            md = N.DeviceArray.from_host(m)
    out = N.DeviceArray((bh, seq, dk), dt)
    N.check(N.lib.nml_sdpa_forward_device(qd.ptr, kd.ptr, vd.ptr, N.ptr(md), out.ptr, bh, seq, dk,
                                          float(scale), causal, N.np_dtype_code(dt)))
    return out, None


def flash_sdpa_forward(q, k, v, scale):
    """The reference's native flash path (kernels/fused_sdpa.py:91-115): float32 causal
    attention over (bh, seq, dk) with ``scale`` the sqrt(dk) divisor, returning
    ``(out, m, l)`` — m, l the per-row softmax max and sum from
    ``flash_sdpa_forward_device`` called with the multiplier ``1/scale``."""
    qd, kd, vd = _dev(q, np.float32), _dev(k, np.float32), _dev(v, np.float32)
    bh, seq, dk = qd.shape
    out = N.DeviceArray((bh, seq, dk), np.float32)
    m = N.DeviceArray((bh, seq), np.float32)
    lsum = N.DeviceArray((bh, seq), np.float32)
    N.check(N.lib.nml_flash_sdpa_forward_device(qd.ptr, kd.ptr, vd.ptr, out.ptr, m.ptr, lsum.ptr,
                                                bh, seq, dk, float(1.0 / scale)))
    return out, m, lsum


def decode_attention(q, kcache, vcache, lens, scale):
    """Attention of one new query per (row, head) over a KV cache: ``q`` (batch, heads, dk),
    ``kcache``/``vcache`` (batch, heads, max_seq, dk), ``lens`` (batch,) keys attended per
    row, ``scale`` the sqrt(dk) divisor (kernels/fused_sdpa.py:71-78 on the cached keys).
    Returns the merged-head output (batch, heads·dk). Raises ValueError for a length
    outside [1, max_seq]."""
    dt = _float_dtype(q)
    qd, kd, vd = _dev(q, dt), _dev(kcache, dt), _dev(vcache, dt)
    batch, heads, max_seq, dk = kd.shape
    if qd.shape != (batch, heads, dk) or vd.shape != kd.shape:
        raise ValueError(f"decode_attention: q {qd.shape}, kcache {kd.shape}, vcache {vd.shape}")
    ln = _dev(np.ascontiguousarray(lens, dtype=np.int32) if not isinstance(lens, N.DeviceArray)
              else lens, np.int32)
    if ln.shape != (batch,):
        raise ValueError(f"decode_attention: lens must be ({batch},), got {ln.shape}")
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    out = N.DeviceArray((batch, heads * dk), dt)
    N.check(N.lib.nml_decode_attention_device(qd.ptr, kd.ptr, vd.ptr, ln.ptr, out.ptr, batch,
                                              heads, max_seq, dk, float(scale), err.ptr,
                                              N.np_dtype_code(dt)))
    if int(err.numpy()[0]):
        raise ValueError(f"decode_attention: a length is outside [1, {max_seq}]")
    return out


def flash_sdpa_backward(grad_out, q, k, v, m, lsum, scale):
    """``flash_sdpa_backward_device`` (kernels/fused_sdpa.py:118-140): float32 gradients
    (grad_q, grad_k, grad_v) of the causal flash forward, ``scale`` the sqrt(dk) divisor."""
    arrs = [_dev(a, np.float32) for a in (grad_out, q, k, v, m, lsum)]
    bh, seq, dk = arrs[1].shape
    gq, gk, gv = (N.DeviceArray((bh, seq, dk), np.float32) for _ in range(3))
    N.check(N.lib.nml_flash_sdpa_backward_device(*[a.ptr for a in arrs], gq.ptr, gk.ptr, gv.ptr,
                                                 bh, seq, dk, float(1.0 / scale)))
    return gq, gk, gv


def fused_rmsnorm_backward(grad, x, gamma, epsilon=1e-5):
    """``rmsnorm_backward_device`` (kernels/fused_rmsnorm.py:104-128 device branch, float32):
    returns (grad_x, grad_gamma)."""
    gd, xd, gmd = _dev(grad, np.float32), _dev(x, np.float32), _dev(gamma, np.float32)
    d = xd.shape[-1]
    rows = xd.size // d
    gx = N.DeviceArray(xd.shape, np.float32)
    gg = N.DeviceArray((d,), np.float32)
    N.check(N.lib.nml_rmsnorm_backward_device(gd.ptr, xd.ptr, gmd.ptr, None, None, gx.ptr, gg.ptr,
                                              rows, d, float(epsilon)))
    return gx, gg


def embedding_lookup(weights, ids, pos_weights=None):
    """``weights[ids]`` (plus ``pos_weights[s]`` when given) on the device."""
    dt = _float_dtype(weights)
    wd = _dev(weights, dt)
    ids_np = np.asarray(ids, dtype=np.int64)
    shape = ids_np.shape
    ids2 = ids_np.reshape(1, -1) if ids_np.ndim != 2 else ids_np
    vocab, dim = wd.shape
    if ids2.size and (int(ids2.min()) < 0 or int(ids2.max()) >= vocab):
        raise ValueError(f"Token ID out of range [0, {vocab})")
    b, s = ids2.shape
    if pos_weights is None:
        pd = N.DeviceArray((max(s, 1), dim), dt)
        N.check(N.lib.nml_memset(pd.ptr, 0, pd.nbytes))
    else:
        pd = _dev(pos_weights, dt)
    idd = N.DeviceArray.from_host(ids2)
    out = N.DeviceArray((b, s, dim), dt)
    N.check(N.lib.nml_embedding_gather_device(wd.ptr, pd.ptr, idd.ptr, out.ptr, b, s, dim, vocab,
                                              pd.shape[0], None, None, N.np_dtype_code(dt)))
    return out.reshape(*shape, dim)


def linear(x, weights, bias=None, *, epilogue=None, resid=None):
    """``epi(x @ weights + bias)`` with ``weights`` in the reference layout (in, out)."""
    dt = _float_dtype(x)
    xd = _dev(x, dt)
    w = np.ascontiguousarray(np.asarray(weights, dtype=dt).T)
    wd = N.DeviceArray.from_host(w)
    n_out, k = w.shape
    rows = xd.size // k
    if epilogue is None:
        epilogue = EPI_BIAS if bias is not None else EPI_NONE
    bd = _dev(bias, dt) if bias is not None else None
    rd = _dev(resid, dt) if resid is not None else None
    out = N.DeviceArray((rows, n_out), dt)
    N.check(N.lib.nml_linear_device(xd.ptr, k, wd.ptr, N.ptr(bd), N.ptr(rd), out.ptr, rows, k,
                                    n_out, int(epilogue), N.np_dtype_code(dt)))
    return out


def linear_t(x, w_t, bias=None, *, epilogue=None):
    """``epi(x @ w_tᵀ + bias)`` with ``w_t`` a DeviceArray already in the device layout
    (out, in) and ``bias`` a DeviceArray or None: no host copy of the weights."""
    dt = _float_dtype(x)
    xd = _dev(x, dt)
    n_out, k = w_t.shape
    rows = xd.size // k
    if epilogue is None:
        epilogue = EPI_BIAS if bias is not None else EPI_NONE
    out = N.DeviceArray((rows, n_out), dt)
    N.check(N.lib.nml_linear_device(xd.ptr, k, w_t.ptr, N.ptr(bias), None, out.ptr, rows, k,
                                    n_out, int(epilogue), N.np_dtype_code(dt)))
    return out


def fused_tied_crossentropy_forward(hidden, weights, label_indices, ignore_index=None):
    """Mean CE of ``hidden @ weights.T`` against labels (float)."""
    dt = _float_dtype(hidden)
    hd, wd = _dev(hidden, dt), _dev(weights, dt)
    rows, dim = hd.shape
    labels = np_backend.as_label_indices(label_indices, batch_size=rows)
    ld = N.DeviceArray.from_host(labels)
    loss = C.c_double()
    has = ignore_index is not None
    N.check(N.lib.nml_tied_ce_forward_device(hd.ptr, wd.ptr, ld.ptr, rows, dim, wd.shape[0],
                                             int(ignore_index) if has else 0, int(has),
                                             C.byref(loss), N.np_dtype_code(dt)))
    return float(loss.value)


def sample_tokens(logits, *, temperature, top_k=0, top_p=1.0, uniforms=None, history=None,
                  repetition_penalty=1.0):
    """One token per row of (batch, vocab) logits with ``_sample_logits`` semantics;
    ``uniforms[b]`` replaces row b's RandomState draw; ``history`` is a list of the
    token ids already in each row (repetition penalty)."""
    dt = _float_dtype(logits)
    ld = _dev(logits, dt)
    batch, vocab = ld.shape
    ud = None
    if temperature > 0:
        ud = N.DeviceArray.from_host(np.asarray(uniforms, dtype=np.float64).reshape(batch))
    hd = hl = None
    stride = 0
    if history is not None:
        stride = max(1, max(len(h) for h in history))
        hist = np.zeros((batch, stride), dtype=np.int64)
        for b, h in enumerate(history):
            hist[b, :len(h)] = h
        hd = N.DeviceArray.from_host(hist)
        hl = N.DeviceArray.from_host(np.asarray([len(h) for h in history], dtype=np.int32))
    out = N.DeviceArray((batch,), np.int64)
    N.check(N.lib.nml_sample_device(ld.ptr, batch, vocab, float(temperature), int(top_k or 0),
                                    float(top_p if top_p is not None else 1.0),
                                    float(repetition_penalty), N.ptr(ud), N.ptr(hd), stride,
                                    N.ptr(hl), out.ptr, N.np_dtype_code(dt)))
    return out.numpy()


def adamw_step(param, grad, m, v, lr, beta1, beta2, bias1, bias2, eps, weight_decay):
    """AdamW update of float32 ``DeviceArray``s in place, the reference native kernel's
    arithmetic (``native.adamw_step``, module.cpp:175-188): bias1/bias2 are the caller's
    ``1 − β^t`` bias corrections, as optimizers/adam.py:93-94 passes them."""
    arrs = [param, grad, m, v]
    for a in arrs:
        if not isinstance(a, N.DeviceArray) or a.dtype != np.float32:
            raise TypeError("adamw_step takes float32 DeviceArrays")
    n = param.size
    if any(a.size != n for a in arrs):
        raise ValueError("adamw_step: param, grad, m and v must have the same size")
    N.check(N.lib.nml_adamw_step_device(param.ptr, grad.ptr, m.ptr, v.ptr, n, float(lr),
                                        float(beta1), float(beta2), float(bias1), float(bias2),
                                        float(eps), float(weight_decay)))


def clip_grad_norm(grads, max_norm):
    """Global L2 norm of float32 gradient ``DeviceArray``s, scaled in place to max_norm
    when above it (``native.clip_grad_norm``, module.cpp:190-200). Returns the norm."""
    grads = list(grads)
    for g in grads:
        if not isinstance(g, N.DeviceArray) or g.dtype != np.float32:
            raise TypeError("clip_grad_norm takes float32 DeviceArrays")
    ptrs = (C.c_void_p * max(1, len(grads)))(*[g.ptr for g in grads])
    sizes = (C.c_size_t * max(1, len(grads)))(*[g.size for g in grads])
    norm = C.c_float()
    N.check(N.lib.nml_clip_grad_norm_device(ptrs, sizes, len(grads), float(max_norm),
                                            C.byref(norm)))
    return float(norm.value)


class KV4Cache:
    """K and V of ``max_seq`` positions a row in 4 bits (blocks of 32 E2M1 codes and a
    power-of-two scale): ``k_codes``/``v_codes`` uint8 (batch, kv_heads, max_seq, blocks, 16),
    ``k_scales``/``v_scales`` uint8 (batch, kv_heads, max_seq, blocks). Starts zeroed."""

    def __init__(self, batch, kv_heads, max_seq, dk):
        self.batch, self.kv_heads = int(batch), int(kv_heads)
        self.max_seq, self.dk = int(max_seq), int(dk)
        shape = (self.batch, self.kv_heads, self.max_seq, -(-self.dk // 32))
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = arrs = [
            N.DeviceArray(shape + (16,) * (i % 2 == 0), np.uint8) for i in range(4)]
        for a in arrs:
            N.check(N.lib.nml_memset(a.ptr, 0, a.nbytes))

    @property
    def pointers(self):
        return (self.k_codes.ptr, self.k_scales.ptr, self.v_codes.ptr, self.v_scales.ptr)


def _rows_i32(x, batch, what):
    """A device int32 (batch,) array, or None."""
    if x is None:
        return None
    d = _dev(x if isinstance(x, N.DeviceArray) else np.ascontiguousarray(x, dtype=np.int32),
             np.int32)
    if d.shape != (batch,):
        raise ValueError(f"{what} must be ({batch},), got {d.shape}")
    return d


def _check_flag(err, message):
    if int(err.numpy()[0]):
        raise ValueError(message)


def kv4_write(cache, k, v, pos=None, counts=None):
    """Quantise K and V (batch, kv_heads, seq, dk) of new tokens into ``cache``: token s of row
    b, s < ``counts[b]`` (None: all), goes to position ``pos[b] + s`` (None: s). Raises
    ValueError for a position outside the cache (the others are written) or a count outside
    [0, seq]."""
    dt = _float_dtype(k)
    kd, vd = _dev(k, dt), _dev(v, dt)
    want = (cache.batch, cache.kv_heads, kd.shape[2] if kd.ndim == 4 else -1, cache.dk)
    if kd.shape != want or vd.shape != want:
        raise ValueError(f"kv4_write: k {kd.shape}, v {vd.shape} for a cache of ({cache.batch}, "
                         f"{cache.kv_heads}, seq, {cache.dk})")
    seq = want[2]
    pd = _rows_i32(pos, cache.batch, "kv4_write: pos")
    cd = _rows_i32(counts, cache.batch, "kv4_write: counts")
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_kv4_write_device(
        kd.ptr, vd.ptr, cache.kv_heads * seq * cache.dk, seq * cache.dk, cache.dk,
        *cache.pointers, N.ptr(pd), N.ptr(cd), cache.batch, cache.kv_heads, seq, cache.max_seq,
        cache.dk, err.ptr, N.np_dtype_code(dt)))
    _check_flag(err, f"kv4_write: a position is outside [0, {cache.max_seq}) or a count outside "
                     f"[0, {seq}]")


def kv4_read(cache, seq, pos=None, counts=None, dtype=None):
    """The values (K, V), each (batch, kv_heads, seq, dk) in ``dtype`` (None: the compute
    dtype), that ``cache`` holds at positions ``pos[b] …`` (None: 0); zeros from ``counts[b]``
    on. Raises ValueError for a position outside the cache."""
    dt = np.dtype(np_backend.dtype if dtype is None else dtype)
    pd = _rows_i32(pos, cache.batch, "kv4_read: pos")
    cd = _rows_i32(counts, cache.batch, "kv4_read: counts")
    out = [N.DeviceArray((cache.batch, cache.kv_heads, int(seq), cache.dk), dt) for _ in range(2)]
    if cd is not None:
        for o in out:
            N.check(N.lib.nml_memset(o.ptr, 0, o.nbytes))
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_kv4_read_device(
        *cache.pointers, N.ptr(pd), N.ptr(cd), out[0].ptr, out[1].ptr, cache.batch,
        cache.kv_heads, int(seq), cache.max_seq, cache.dk, err.ptr, N.np_dtype_code(dt)))
    _check_flag(err, f"kv4_read: a position is outside [0, {cache.max_seq}) or a count outside "
                     f"[0, {seq}]")
    return out[0], out[1]


def kv4_attention(q, cache, lens, scale, counts=None):
    """Causal attention of each row's ``counts[b]`` (None: all ``seq``) last cached tokens over
    ``cache``: ``q`` (batch, heads, seq, dk), ``lens`` (batch,) tokens cached per row, these
    included, ``scale`` the sqrt(dk) divisor; query head h reads KV head
    h // (heads // kv_heads). Returns the merged-head output (batch, seq, heads·dk), zeros for
    tokens from ``counts[b]`` on and for tokens that see no key. Raises ValueError for a length
    outside [0, max_seq] or a count outside [0, seq]."""
    dt = _float_dtype(q)
    qd = _dev(q, dt)
    if qd.ndim != 4 or qd.shape[0] != cache.batch or qd.shape[3] != cache.dk:
        raise ValueError(f"kv4_attention: q {qd.shape} for a cache of {cache.batch} rows, head "
                         f"dim {cache.dk}")
    batch, heads, seq, dk = qd.shape
    ld = _rows_i32(lens, batch, "kv4_attention: lens")
    if ld is None:
        raise ValueError("kv4_attention: lens is required")
    cd = _rows_i32(counts, batch, "kv4_attention: counts")
    sizes = (batch, heads, cache.kv_heads, seq, cache.max_seq, dk)
    need = C.c_size_t()
    N.check(N.lib.nml_kv4_attention_workspace(*sizes, C.byref(need)))
    ws = N.DeviceArray((need.value,), np.uint8) if need.value else None
    if ws is not None:
        N.check(N.lib.nml_memset(ws.ptr, 0, ws.nbytes))
    out = N.DeviceArray((batch, seq, heads * dk), dt)
    if cd is not None:
        N.check(N.lib.nml_memset(out.ptr, 0, out.nbytes))
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_kv4_attention_device(
        qd.ptr, *cache.pointers, ld.ptr, N.ptr(cd), out.ptr, *sizes, float(scale), N.ptr(ws),
        need.value, err.ptr, N.np_dtype_code(dt)))
    _check_flag(err, f"kv4_attention: a length is outside [0, {cache.max_seq}] or a count outside "
                     f"[0, {seq}]")
    return out


def _logit_rows(logits, targets):
    dt = _float_dtype(logits)
    ld = _dev(logits, dt)
    rows = ld.size // ld.shape[-1]
    td = targets
    if not isinstance(td, N.DeviceArray):
        td = N.DeviceArray.from_host(np.ascontiguousarray(targets, dtype=np.int64).reshape(-1))
    if td.dtype != np.int64 or td.size != rows:
        raise ValueError(f"label count ({td.size}) must match batch size ({rows})")
    return ld, td, rows, ld.shape[-1], N.np_dtype_code(dt)


def token_logprobs(logits, targets, top_k=0, ignore_index=None):
    """Log probabilities of ``targets`` (rows,) under ``logits`` (..., vocab), row by row:
    ``(logp, entropy, m, l, top_ids, top_logp)`` as ``DeviceArray``s — float32 (rows,) each (m, l:
    the largest logit and Σ exp(x − m)), the ``top_k`` most probable ids (int64) and their log
    probabilities (rows, top_k), most probable first, or None without ``top_k``. Rows whose target
    is ``ignore_index`` give zeros and ids −1. Raises ValueError for a target outside [0, vocab)."""
    if not 0 <= top_k <= 64:
        raise ValueError(f"token_logprobs: top_k must be in [0, 64], got {top_k}")
    ld, td, rows, vocab, code = _logit_rows(logits, targets)
    logp, entropy, m, lsum = (N.DeviceArray((rows,), np.float32) for _ in range(4))
    ids = top = None
    if top_k:
        ids, top = N.DeviceArray((rows, top_k), np.int64), N.DeviceArray((rows, top_k), np.float32)
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    has = ignore_index is not None
    N.check(N.lib.nml_token_logprobs_device(
        ld.ptr, vocab, td.ptr, rows, vocab, int(ignore_index) if has else 0, int(has), int(top_k),
        logp.ptr, entropy.ptr, m.ptr, lsum.ptr, N.ptr(ids), N.ptr(top), err.ptr, code))
    _check_flag(err, f"label out of range [0, {vocab})")
    return logp, entropy, m, lsum, ids, top


def token_logprobs_backward(logits, targets, m, lsum, entropy, dlogp=None, dentropy=None,
                            ignore_index=None):
    """The gradient with respect to ``logits`` (its shape and dtype) of Σ dlogp·logp +
    dentropy·entropy, from ``token_logprobs``' ``m``, ``l`` and ``entropy``; ``dlogp``, ``dentropy``
    (rows,) float32 or None."""
    ld, td, rows, vocab, code = _logit_rows(logits, targets)
    stats = []
    for name, x in (("m", m), ("l", lsum), ("entropy", entropy), ("dlogp", dlogp),
                    ("dentropy", dentropy)):
        d = None if x is None else _dev(x, np.float32)
        if d is not None and d.size != rows:
            raise ValueError(f"token_logprobs_backward: {name} must have {rows} values, got {d.size}")
        stats.append(d)
    out = N.DeviceArray(ld.shape, ld.dtype)
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    has = ignore_index is not None
    N.check(N.lib.nml_token_logprobs_backward_device(
        ld.ptr, vocab, td.ptr, *(N.ptr(s) for s in stats), rows, vocab,
        int(ignore_index) if has else 0, int(has), out.ptr, vocab, err.ptr, code))
    _check_flag(err, f"label out of range [0, {vocab})")
    return out


def _page_count(lengths, page_size):
    return -(-np.maximum(np.asarray(lengths, dtype=np.int64), 0) // page_size)


def _check_pages(what, table, lengths, page_size, num_pages, counts=None):
    """Raises ValueError where a row of ``lengths`` positions needs more pages than ``table`` (host
    arrays) has or, unless its count is 0, one outside [0, num_pages)."""
    need = _page_count(lengths, page_size)
    if need.size and int(need.max()) > table.shape[1]:
        raise ValueError(f"{what}: a row of {int(np.max(lengths))} positions needs {int(need.max())} "
                         f"pages of {page_size}, the table has {table.shape[1]}")
    used = np.arange(table.shape[1]) < need[:, None]
    if counts is not None:
        used &= np.asarray(counts)[:, None] != 0
    bad = used & ((table < 0) | (table >= num_pages))
    if bad.any():
        raise ValueError(f"{what}: page {int(table[bad][0])} is outside [0, {num_pages})")


class PagedKVCache:
    """K and V in ``num_pages`` pages of ``page_size`` (a power of two in [8, 1024]) positions:
    ``k_pages``/``v_pages`` (num_pages, kv_heads, page_size, dk) in ``dtype`` (None: the compute
    dtype). Which pages a row has is the caller's table; rows may share pages that none of them
    writes. Starts zeroed."""

    def __init__(self, num_pages, page_size, kv_heads, dk, dtype=None):
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.kv_heads, self.dk = int(kv_heads), int(dk)
        if self.page_size < 8 or self.page_size > 1024 or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size must be a power of two in [8, 1024], got {page_size}")
        if self.num_pages < 1:
            raise ValueError(f"num_pages must be at least 1, got {num_pages}")
        self.dtype = np.dtype(np_backend.dtype if dtype is None else dtype)
        N.np_dtype_code(self.dtype)
        shape = (self.num_pages, self.kv_heads, self.page_size, self.dk)
        self.k_pages, self.v_pages = (N.DeviceArray(shape, self.dtype) for _ in range(2))
        for a in (self.k_pages, self.v_pages):
            N.check(N.lib.nml_memset(a.ptr, 0, a.nbytes))


def _page_table(cache, table, what):
    """(the table as a host array or None, its shape (batch, pages of a row))."""
    host = None if isinstance(table, N.DeviceArray) else np.ascontiguousarray(table, dtype=np.int32)
    shape = table.shape if host is None else host.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{what}: the table must be (batch, pages of a row), got {shape}")
    return host, shape


def paged_write(cache, k, v, table, pos=None, counts=None):
    """Write K and V (batch, kv_heads, seq, dk) of new tokens into ``cache``: token s of row b, s <
    ``counts[b]`` (None: all), goes to position ``pos[b] + s`` (None: s), position p of row b being
    position p % page_size of page ``table[b, p // page_size]``. No two tokens may go to one place.
    Raises ValueError for a position past the table, a page outside the cache (the other tokens are
    written) or a count outside [0, seq]."""
    host, (batch, max_pages) = _page_table(cache, table, "paged_write")
    shape = (batch, cache.kv_heads, k.shape[2] if np.ndim(k) == 4 else -1, cache.dk)
    if tuple(k.shape) != shape or tuple(v.shape) != shape:
        raise ValueError(f"paged_write: k {k.shape}, v {v.shape} for {batch} rows of a cache of "
                         f"{cache.kv_heads} heads, head dim {cache.dk}")
    seq = shape[2]
    kd, vd = _dev(k, cache.dtype), _dev(v, cache.dtype)
    td = _dev(host if host is not None else table, np.int32)
    pd = _rows_i32(pos, batch, "paged_write: pos")
    cd = _rows_i32(counts, batch, "paged_write: counts")
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_paged_write_device(
        kd.ptr, vd.ptr, cache.kv_heads * seq * cache.dk, seq * cache.dk, cache.dk,
        cache.k_pages.ptr, cache.v_pages.ptr, td.ptr, N.ptr(pd), N.ptr(cd), batch, cache.kv_heads,
        seq, max_pages, cache.page_size, cache.num_pages, cache.dk, err.ptr,
        N.np_dtype_code(cache.dtype)))
    _check_flag(err, f"paged_write: a position is outside [0, {max_pages * cache.page_size}), a page "
                     f"outside [0, {cache.num_pages}) or a count outside [0, {seq}]")


def _paged_attention_bytes(cache, *sizes):
    need = C.c_size_t()
    N.check(N.lib.nml_paged_attention_workspace(*sizes, cache.page_size, cache.dk,
                                                N.np_dtype_code(cache.dtype), C.byref(need)))
    return need.value


def paged_attention_workspace(cache, batch, heads, seq, max_pages):
    """A workspace for ``paged_attention`` over ``cache`` by ``heads`` query heads, ``seq`` new tokens
    and tables of (batch, max_pages): a uint8 ``DeviceArray``, zeroed, which calls that run one after
    another may share, also with other sizes that need no more. Calls of several threads that can
    run at the same time need one each."""
    ws = N.DeviceArray((_paged_attention_bytes(cache, batch, heads, cache.kv_heads, seq, max_pages),), np.uint8)
    N.check(N.lib.nml_memset(ws.ptr, 0, ws.nbytes))
    return ws


def paged_attention(q, cache, table, lens, scale, counts=None, *, workspace=None):
    """Causal attention of each row's ``counts[b]`` (None: all ``seq``) last cached tokens over its
    pages: ``q`` (batch, heads, seq, dk), ``table`` (batch, pages of a row), ``lens`` (batch,) tokens
    cached per row, these included, ``scale`` the sqrt(dk) divisor; query head h reads KV head
    h // (heads // kv_heads). Returns the merged-head output (batch, seq, heads·dk), zeros for
    tokens from ``counts[b]`` on and for tokens that see no key. ``workspace``: what
    ``paged_attention_workspace`` gave (None: made and freed here, for which a call takes 8 to 40 µs
    longer). Raises ValueError for a length outside the table, a count outside [0, seq], a page
    outside the cache or a workspace that is too small."""
    host, (batch, max_pages) = _page_table(cache, table, "paged_attention")
    if len(q.shape) != 4 or q.shape[0] != batch or q.shape[3] != cache.dk:
        raise ValueError(f"paged_attention: q {q.shape} for {batch} rows, head dim {cache.dk}")
    if lens is None:
        raise ValueError("paged_attention: lens is required")
    for name, x in (("lens", lens), ("counts", counts)):
        if x is not None and np.shape(x) != (batch,):
            raise ValueError(f"paged_attention: {name} must be ({batch},), got {np.shape(x)}")
    heads, seq, dk = q.shape[1:]
    # what is on the host is checked here, anything else by the kernel: pages of rows that attend
    if host is not None and seq and not any(isinstance(x, N.DeviceArray) for x in (lens, counts)):
        _check_pages("paged_attention", host, lens, cache.page_size, cache.num_pages, counts)
    qd = _dev(q, cache.dtype)
    td = _dev(host if host is not None else table, np.int32)
    ld = _rows_i32(lens, batch, "paged_attention: lens")
    cd = _rows_i32(counts, batch, "paged_attention: counts")
    code = N.np_dtype_code(cache.dtype)
    sizes = (batch, heads, cache.kv_heads, seq, max_pages, cache.page_size)
    if workspace is None:
        workspace = paged_attention_workspace(cache, batch, heads, seq, max_pages)
    elif workspace.nbytes < (need := _paged_attention_bytes(cache, *sizes[:-1])):
        raise ValueError(f"paged_attention: a workspace of {need} bytes is needed, got {workspace.nbytes}")
    out = N.DeviceArray((batch, seq, heads * dk), cache.dtype)
    if cd is not None:
        N.check(N.lib.nml_memset(out.ptr, 0, out.nbytes))
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_paged_attention_device(
        qd.ptr, cache.k_pages.ptr, cache.v_pages.ptr, td.ptr, ld.ptr, N.ptr(cd), out.ptr, *sizes,
        cache.num_pages, dk, float(scale), N.ptr(workspace), workspace.nbytes, err.ptr, code))
    _check_flag(err, f"paged_attention: a length is outside [0, {max_pages * cache.page_size}], a page "
                     f"outside [0, {cache.num_pages}) or a count outside [0, {seq}]")
    return out


def _teacher_rows(logits, top_ids, top_logits, what):
    """(logits, ids, values, rows, vocab, entries a row) of a distillation's arguments."""
    dt = _float_dtype(logits)
    shape = tuple(np.shape(logits))
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: logits must be (..., vocab), got {shape}")
    ld = _dev(logits, dt)
    vocab = ld.shape[-1]
    rows = ld.size // vocab
    idd = _dev(top_ids if isinstance(top_ids, N.DeviceArray) else
               np.ascontiguousarray(top_ids, dtype=np.int64), np.int64)
    top_k = idd.shape[-1] if idd.shape else 0
    yd = _dev(top_logits if isinstance(top_logits, N.DeviceArray) else
              np.ascontiguousarray(top_logits, dtype=np.float32), np.float32)
    if idd.size != rows * top_k or yd.shape != idd.shape:
        raise ValueError(f"{what}: top_ids {idd.shape} and top_logits {yd.shape} for {rows} rows")
    return ld, idd, yd, rows, vocab, top_k


def distill(logits, top_ids, top_logits, temperature=1.0):
    """KL(q || p) of each row of ``logits`` (..., vocab): p its softmax at ``temperature``, q that of
    the teacher's ``top_logits`` (..., k) of the tokens ``top_ids`` (..., k; log probabilities will
    do: ``token_logprobs``' alternatives are such entries); ids of −1 are absent, rows of nothing
    else give zeros. Returns ``(loss, m, l)``, float32 (rows,) ``DeviceArray``s; m, l: the largest
    logit and Σ exp((x − m) / temperature). Raises ValueError for an id outside [−1, vocab)."""
    ld, idd, yd, rows, vocab, top_k = _teacher_rows(logits, top_ids, top_logits, "distill")
    loss, m, lsum = (N.DeviceArray((rows,), np.float32) for _ in range(3))
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_distill_device(
        ld.ptr, vocab, idd.ptr, yd.ptr, rows, vocab, top_k, float(temperature), loss.ptr, m.ptr,
        lsum.ptr, err.ptr, N.np_dtype_code(ld.dtype)))
    _check_flag(err, f"distill: an id is outside [-1, {vocab})")
    return loss, m, lsum


def distill_backward(logits, top_ids, top_logits, m, lsum, dloss, temperature=1.0):
    """The gradient with respect to ``logits`` (its shape and dtype) of Σ dloss·loss, from
    ``distill``'s ``m`` and ``l``; ``dloss`` (rows,) float32."""
    ld, idd, yd, rows, vocab, top_k = _teacher_rows(logits, top_ids, top_logits, "distill_backward")
    stats = [_dev(x, np.float32) for x in (m, lsum, dloss)]
    for name, x in zip(("m", "l", "dloss"), stats):
        if x.size != rows:
            raise ValueError(f"distill_backward: {name} must have {rows} values, got {x.size}")
    out = N.DeviceArray(ld.shape, ld.dtype)
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_distill_backward_device(
        ld.ptr, vocab, idd.ptr, yd.ptr, *(x.ptr for x in stats), rows, vocab, top_k,
        float(temperature), out.ptr, vocab, err.ptr, N.np_dtype_code(ld.dtype)))
    _check_flag(err, f"distill_backward: an id is outside [-1, {vocab})")
    return out


def verify_drafts(logits, drafts, uniforms=None, *, draft_logits=None, counts=None, temperature=1.0):
    """Which drafted tokens stand, and the token after them, so that what a row gains is distributed
    as sampling from the target alone at ``temperature`` (≤ 0: as its largest logits).

    ``logits`` (batch, n + 1, vocab): the target's after the row's last token and after each draft,
    as ``GPT.forward_with_cache`` gives them for [last token, *drafts]; ``drafts`` (batch, n);
    ``draft_logits`` (batch, n, vocab): what the drafts were sampled from at the same temperature (None:
    they were chosen outright); ``uniforms`` (batch, n + 1) float64 in [0, 1), one a draft and the last
    for the final token; ``counts`` (batch,) drafts of each row (None: n).

    Returns ``(accepted, tokens)`` as ``DeviceArray``s: int32 (batch,) accepted drafts and int64
    (batch, n + 1), those drafts, one token more, then −1; ``KVCache.truncate`` takes a cache back to
    them. Raises ValueError for a draft outside [0, vocab), a count outside [0, n] or a row of
    logits that decides and has no distribution. Both logits may be Tensors."""
    logits, draft_logits = (x.data.reshape(x.shape) if isinstance(x, Tensor) else x
                            for x in (logits, draft_logits))
    dt = _float_dtype(logits)
    if len(logits.shape) != 3 or logits.shape[1] < 1:
        raise ValueError(f"verify_drafts: logits must be (batch, n + 1, vocab), got {logits.shape}")
    batch, n, vocab = logits.shape[0], logits.shape[1] - 1, logits.shape[2]
    greedy = temperature <= 0
    if uniforms is None and not greedy:
        raise ValueError("verify_drafts: uniforms are required at a temperature above 0")
    for name, x, shape in (("drafts", drafts, (batch, n)), ("uniforms", uniforms, (batch, n + 1)),
                           ("draft_logits", draft_logits, (batch, n, vocab))):
        if x is not None and tuple(np.shape(x)) != shape:
            raise ValueError(f"verify_drafts: {name} must be {shape}, got {tuple(np.shape(x))}")
    ld = _dev(logits, dt)
    dd = _dev(drafts if isinstance(drafts, N.DeviceArray) else
              np.ascontiguousarray(drafts, dtype=np.int64), np.int64)
    qd = None if draft_logits is None or greedy else _dev(draft_logits, dt)
    ud = None if greedy else _dev(uniforms if isinstance(uniforms, N.DeviceArray) else
                                  np.ascontiguousarray(uniforms, dtype=np.float64), np.float64)
    cd = _rows_i32(counts, batch, "verify_drafts: counts")
    need = C.c_size_t()
    N.check(N.lib.nml_verify_drafts_workspace(batch, n, vocab, C.byref(need)))
    ws = N.DeviceArray((need.value,), np.uint8)
    accepted, tokens = N.DeviceArray((batch,), np.int32), N.DeviceArray((batch, n + 1), np.int64)
    err = N.DeviceArray.from_host(np.zeros(1, np.int32))
    N.check(N.lib.nml_verify_drafts_device(
        ld.ptr, vocab, N.ptr(qd), vocab, dd.ptr, N.ptr(cd), N.ptr(ud), batch, n, vocab,
        float(temperature), accepted.ptr, tokens.ptr, ws.ptr, need.value, err.ptr,
        N.np_dtype_code(dt)))
    flag = int(err.numpy()[0])
    if flag & 1:
        raise ValueError(f"verify_drafts: a draft is outside [0, {vocab}) or a count outside [0, {n}]")
    if flag:
        raise ValueError("verify_drafts: a row of logits holds NaN or infinity, or nothing above -inf")
    return accepted, tokens
