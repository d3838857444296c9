"""Inputs and outputs in one buffer, row by row side by side: no overlap, and the calls are served."""
import ctypes as C

import numpy as np
import pytest

import kv_ref as R
import q8mi
import test_gpu_paged_attention as attention
from gpu_common import NULL
from q8mi import hip, ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_first", [False, True])
@pytest.mark.parametrize("q_stride,out_stride,out_act", [(2, 2, "f32"), (3, 3, "f32"), (2, 2, "bf16"), (4, 2, "f32")])
def test_attention(gpu, q_stride, out_stride, out_act, out_first):
    """Strides in rows' widths; the last form (four rows of q and out each, of unlike strides) lets its outputs end behind q."""
    c = attention.Case([70, 33], [2, 2], 8, 4, 128, "f16", out_act=out_act, seed=1, spare_rows=0)
    w = c.width
    if q_stride != out_stride:      # rows of q at widths 0, 4, 8, 12; outputs at 1, 3, 5, 7 behind them: none meet
        out_first = False
    big = hip.DeviceBuffer(4 * w * 17).fill(0x5a)
    at_q, at_out = (4 * w, 0) if out_first else (0, 4 * w)
    for r in range(4):
        big.upload(c.q[r], at_q + 4 * w * q_stride * r)
    es = c.oes
    args = list(c.args())
    args[0], args[3], args[14], args[16] = big.at(at_q), w * q_stride, big.at(at_out), w * out_stride * 4 // es
    ok(q8mi.lib().q8mi_paged_attention(*args), "paged_attention")
    hip.synchronize()
    for r in range(4):
        c.dout.upload(big.download(np.uint8, w * es, at_out + 4 * w * out_stride * r), r * w * es)
        assert np.array_equal(big.download(np.float32, w, at_q + 4 * w * q_stride * r), c.q[r]), "q was written"
    c.check()


@pytest.mark.parametrize("tokens", [1, 7, 1400])
@pytest.mark.parametrize("place", ["in place", "behind v", "before q", "between heads"])
def test_append(gpu, tokens, place):
    """Rows [q k v] of one fused projection, the queries' results where they were, or beside them in the same rows."""
    heads, kv_heads, dim, rot = (1 if place == "between heads" else 6), 2, 128, 64
    rng = np.random.default_rng(tokens)
    lead = heads * dim if place == "before q" else 0
    q_at, k_at = lead, lead + heads * dim + (dim if place == "between heads" else 0)
    v_at = k_at + kv_heads * dim
    row = v_at + kv_heads * dim + heads * dim
    out_at = {"in place": q_at, "behind v": v_at + kv_heads * dim, "before q": 0, "between heads": q_at + dim}[place]
    x = rng.standard_normal((tokens, row)).astype(np.float32)
    buf = hip.to_device(x)
    freqs, positions = 1e4 ** (-np.arange(rot // 2) / (rot // 2)), np.arange(tokens, dtype=np.int32) + 100
    pages = (tokens + 15) // 16
    pools = R.Pools("bf16", pages, 16, kv_heads, dim)
    df, dp, ds = hip.to_device(freqs), hip.to_device(positions), hip.to_device(np.arange(tokens, dtype=np.int64))
    at = lambda i: C.c_void_p(buf.ptr + 4 * i)  # noqa: E731
    ok(q8mi.lib().q8mi_qk_norm_rope_append(at(q_at), at(k_at), at(v_at), at(out_at), 0, tokens, heads, row, dim, row, row, row, None, None, 1e-6,
                                           df.ptr, rot, 0, dp.ptr, ds.ptr, pools.ref, NULL), "append")
    hip.synchronize()
    got = buf.download(np.float32).reshape(tokens, row)
    want = R.norm_rope(x[:, q_at:q_at + heads * dim].reshape(tokens, heads, dim), None, 0, freqs, rot, False, positions)
    tol = 12 * R.U * R.partner_size(x[:, q_at:q_at + heads * dim].reshape(tokens, heads, dim), None, 0, rot, False)
    assert (np.abs(got[:, out_at:out_at + heads * dim].reshape(want.shape) - want) <= tol).all()
    left = x.copy()
    left[:, out_at:out_at + heads * dim] = got[:, out_at:out_at + heads * dim]
    assert np.array_equal(left, got), "something else was written"
    dev = pools.download()
    values = np.stack([R.decode(dev["v"][pools.at(t // 16, t % 16)], "bf16") for t in range(tokens)])
    v = x[:, v_at:v_at + kv_heads * dim].reshape(tokens, kv_heads, dim)
    assert (np.abs(values - v) <= R.HALF_STEP["bf16"] * np.abs(v)).all()
