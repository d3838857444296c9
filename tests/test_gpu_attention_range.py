"""The paged attention where numbers are far from 1: queries whose elements differ by many powers of two, and cache scales near
the ends of fp32."""
import numpy as np
import pytest

import kv_ref as R
import q8mi
from gpu_common import NULL
from q8mi import hip, ok

pytestmark = pytest.mark.gpu


def attend(pools, q, n, scale):
    """fp32 rows q [rows, heads, dim], newest of one sequence of n tokens that lie in the pools' pages in order."""
    rows, heads, dim = q.shape
    pools.upload()
    L = q8mi.lib()
    dq, out = hip.to_device(np.ascontiguousarray(q, np.float32)), hip.DeviceBuffer(4 * q.size).fill(0xff)
    table, lens = hip.to_device(np.arange(pools.pages, dtype=np.int32)), hip.to_device(np.array([n], np.int32))
    scratch = hip.DeviceBuffer(L.q8mi_paged_attention_scratch_bytes(1, rows, heads, pools.kv_heads, dim, n))
    ok(L.q8mi_paged_attention(dq.ptr, 0, rows, heads * dim, pools.ref, table.ptr, pools.pages, lens.ptr, None, 1, rows, heads, n, scale,
                              out.ptr, 0, heads * dim, scratch.ptr, NULL), "paged_attention")
    hip.synchronize()
    return out.download(np.float32).reshape(rows, heads, dim)


@pytest.mark.parametrize("top", [1.0, 1.999, 2.0 ** 100, 2.0 ** -40, 2.0 ** -95])
@pytest.mark.parametrize("kind,k", [("f16", 2.0 ** 15), ("e4m3", 256.0)])
def test_small_elements_of_a_query(gpu, kind, k, top):
    """Two tokens, weighed by an element of the query far below the largest one, which meets a key of 0.  q is held to 2^-39 of its
    row's largest: the score, 0.45, is off by at most scale * k * top * 2^-39 = 0.25 (and a few roundings of fp32)."""
    pools = R.Pools(kind, 1, 16, 1, 64, fill=0)
    row = np.zeros((1, 64))
    row[0, 1] = k
    pools.put("k", 0, 1, R.encode(row, kind))
    pools.put("v", 0, 1, R.encode(np.ones((1, 64)), kind))
    q = np.zeros((1, 1, 64), np.float32)
    unit = 2.0 ** np.floor(np.log2(top))
    q[0, 0, 0], q[0, 0, 1] = top, 0.9 * unit * 2.0 ** -38
    scale = 2.0 ** 37 / k / unit                  # at most 2^124: beyond 2^127 the call is refused
    score = scale * k * float(q[0, 0, 1])
    p = attend(pools, q, 2, scale)[0, 0].astype(np.float64)
    assert abs(score - 0.45) < 0.01
    assert np.abs(np.log(p / (1 - p)) - score).max() <= scale * k * top * 2.0 ** -39 + 1e-5


@pytest.mark.parametrize("exponent", [-127, -130, -140, -149])
@pytest.mark.parametrize("kind,k", [("f16", 2.0 ** 15), ("e4m3", 256.0)])
def test_subnormal_queries(gpu, kind, k, exponent):
    """The largest element of a row is one of fp32's subnormals: a power of two, so that nothing but the sums' and the exponential's
    roundings is left (the bound of the score's own is 8 u of it, of p 16 u)."""
    pools = R.Pools(kind, 1, 16, 1, 64, fill=0)
    row = np.zeros((1, 64))
    row[0, 5] = k
    pools.put("k", 0, 1, R.encode(row, kind))
    pools.put("v", 0, 1, R.encode(np.ones((1, 64)), kind))
    q = np.zeros((1, 1, 64), np.float32)
    q[0, 0, 5] = 2.0 ** exponent
    scale = min(2.0 ** 126, 2.0 ** -1 / k / 2.0 ** exponent)
    score = scale * k * 2.0 ** exponent
    p = attend(pools, q, 2, scale)[0, 0].astype(np.float64)
    want = 1 / (1 + np.exp(-score))
    assert np.abs(p - want).max() <= (8 * score + 16) * R.U


@pytest.mark.parametrize("v_scale", [1.3 * 2.0 ** -124, 1.3 * 2.0 ** -100, 1.3 * 2.0 ** 120])
@pytest.mark.parametrize("n", [1, 50, 3000])
def test_value_scales_near_the_ends(gpu, n, v_scale):
    """Zero queries weigh all tokens alike; the mean is good to fp32's roundings of the sum, however small the scale (outputs that
    are subnormal: to half their step)."""
    rng = np.random.default_rng(n)
    v_scale = float(np.float32(v_scale))
    pages = (n + 15) // 16
    pools = R.Pools("e4m3", pages, 16, 2, 64, v_scale=v_scale, fill=0)
    v = np.zeros((n, 2, 64))
    for t in range(n):
        bits = R.e4m3_bits(4 * rng.standard_normal((2, 64)))
        pools.put("v", t // 16, t % 16, bits)
        v[t] = R.E4M3[bits] * v_scale
    got = attend(pools, np.zeros((1, 4, 64)), n, 1.0)[0].astype(np.float64)
    want, mag = v.mean(0).repeat(2, 0), np.abs(v).mean(0).repeat(2, 0)
    assert (np.abs(got - want) <= (6 * n ** 0.5 + 16) * R.U * mag + 2.0 ** -150).all()
