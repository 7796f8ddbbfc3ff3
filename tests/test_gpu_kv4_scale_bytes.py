"""Every scale byte that the format has (a cache may have been written elsewhere): reading and attention
take the same values from it."""
import numpy as np
import pytest

from nimbleml_amd import _native as N
from nimbleml_amd import kernels as K
from oracle import kv4_ref as R

pytestmark = pytest.mark.gpu


def cache_with(codes_k, scales_k, codes_v, scales_v, dk):
    b, h, n = scales_k.shape[:3]
    c = K.KV4Cache(b, h, n, dk)
    c.k_codes, c.k_scales, c.v_codes, c.v_scales = (
        N.DeviceArray.from_host(np.ascontiguousarray(x)) for x in (codes_k, scales_k, codes_v, scales_v))
    return c


@pytest.mark.parametrize("dk", [32, 64, 128, 256])
def test_the_smallest_scales(gpu, dk):
    """Bytes 0, 1, 2, … of V (2^-127 and on), all codes; keys of equal score. Row b of the batch has
    one key with byte b."""
    r = np.random.RandomState(dk)
    nb, rows = dk // 32, 6
    codes = r.randint(0, 256, (rows, 1, 1, nb, 16)).astype(np.uint8)
    scales = np.broadcast_to(np.arange(rows, dtype=np.uint8)[:, None, None, None], (rows, 1, 1, nb))
    zero = np.zeros_like(codes)
    c = cache_with(zero, np.full_like(scales, 127), codes, scales, dk)
    want = R.values(codes, scales, dk)[:, 0, 0]
    assert np.array_equal(K.kv4_read(c, 1, dtype=np.float32)[1].numpy()[:, 0, 0].astype(np.float64), want)
    q = np.ones((rows, 1, 1, dk), np.float32)
    got = K.kv4_attention(q, c, np.ones(rows, np.int32), 1.0).numpy()[:, 0].astype(np.float64)
    # one key: its value, which float32 holds but for a denormal's step
    assert np.abs(got - want).max() <= 2.0**-149 + np.abs(want).max() * 2.0**-23, (got - want)


@pytest.mark.parametrize("dk", [32, 64, 128, 256])
@pytest.mark.parametrize("byte", [0, 1, 3])
def test_the_smallest_scales_of_keys(gpu, dk, byte):
    """Keys of such scales under queries large enough for scores of some size."""
    r = np.random.RandomState(dk + byte)
    nb, n = dk // 32, 70
    codes = r.randint(0, 256, (1, 1, n, nb, 16)).astype(np.uint8)
    v = r.randn(1, 1, n, dk).astype(np.float32)
    codes_v, scales_v = R.quantise(v)
    c = cache_with(codes, np.full((1, 1, n, nb), byte, np.uint8), codes_v, scales_v, dk)
    q = (2.0**118 * r.randint(-3, 4, (1, 1, 1, dk))).astype(np.float32)  # (one part of bf16: exact)
    scale = 2.0**-4
    got = K.kv4_attention(q, c, [n], scale).numpy()[0, 0].astype(np.float64)
    k = R.values(codes, np.full((1, 1, n, nb), byte, np.uint8), dk)
    hv = R.held(v)
    want = R.attention(q, k, hv, [n], None, scale)[0, 0]
    dots = (np.abs(q[0, 0].astype(np.float64)) @ np.abs(k[0, 0]).T).max() / scale
    rel = 2 * ((dk + 4) * dots + n + 16) * 2.0**-24 + 2.0**-23
    assert np.abs(got - want).max() <= np.abs(hv).max() * rel
