"""Per-head norm + rotation + cache append against its 64-bit form.

Bounds: a head's sum of squares carries at most 6 sqrt(D) u relative error (probabilistic bound of D random roundings, half of
it after the root), root, quotient and the two products 4 u; the fraction of the angle is rounded once (2^-26 of a turn =
1.6 u in sine and cosine, which themselves are good to 2 u) and the rotation adds 3 u: below (3 sqrt(D) + 12) u of |a| + |b|.
A rounding to the cache's or the activations' type adds half a step of the value (e4m3: also half of its smallest step)."""
import ctypes as C

import numpy as np
import pytest

import kv_ref as R
import q8mi
from gpu_common import NULL
from q8mi import hip, ok

pytestmark = pytest.mark.gpu
EPS = 1e-6


def run(tokens, heads, kv_heads, dim, rot, kind="bf16", act="f32", interleaved=False, page=16, order="htd", gap=0, gated=False,
        pad=0, in_place=False, norms=True, slots=None, positions=None, seed=0, misalign=0, stream=NULL, scale=(1.0, 1.0), x=None):
    rng = np.random.default_rng(seed)
    wide = 2 if gated else 1
    sqh, sqr = wide * dim, heads * wide * dim + pad
    skr, svr, sor = kv_heads * dim + pad, kv_heads * dim + 2 * pad, heads * dim + (pad if not in_place else pad)
    q = (1.5 * rng.standard_normal((tokens, sqr))).astype(np.float32)
    k = (1.5 * rng.standard_normal((tokens, skr))).astype(np.float32)
    v = rng.standard_normal((tokens, svr)).astype(np.float32)
    if x is not None:
        x(q, k, v)
    q, k, v = (R.act_bits(a, act) for a in (q, k, v))
    qw = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) if norms else None
    kw = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) if norms else None
    freqs = 1e7 ** (-np.arange(rot // 2) / max(1, rot // 2))
    positions = np.asarray(positions if positions is not None else 70000 + np.arange(tokens), np.int32)
    pages = (tokens + page - 1) // page + 2
    if slots is None:
        slots = rng.permutation(pages * page)[:tokens]
    slots = np.asarray(slots, np.int64)
    pools = R.Pools(kind, pages, page, kv_heads, dim, order, gap, *scale)
    # a leading element or two of misalignment sends the call down the scalar path
    put = lambda a: hip.DeviceBuffer(a.nbytes + 64).upload(a, misalign * a.itemsize)  # noqa: E731
    dq, dk, dv = put(q), put(k), put(v)
    es = q.itemsize
    out = dq if in_place else hip.DeviceBuffer(tokens * sor * es + 64).fill(0xff)
    dqw, dkw = (hip.to_device(w) if norms else None for w in (qw, kw))
    df, dp, ds = hip.to_device(freqs) if rot else None, hip.to_device(positions), hip.to_device(slots)
    ptr = lambda b: b.ptr if b is not None else None  # noqa: E731
    at = lambda b: b.at(misalign * es)  # noqa: E731
    args = (at(dq), at(dk), at(dv), at(out), int(act == "bf16"), tokens, heads, sqr, sqh, skr, svr, sor, ptr(dqw), ptr(dkw), EPS,
            ptr(df), rot, int(interleaved), dp.ptr, ds.ptr, pools.ref, stream)
    keep = (dq, dk, dv, out, dqw, dkw, df, dp, ds)
    ok(q8mi.lib().q8mi_qk_norm_rope_append(*args), "append")
    hip.synchronize()

    qs = R.act_value(q[:, :heads * sqh], act).reshape(tokens, heads, wide, dim)[:, :, 0]
    ks = R.act_value(k[:, :kv_heads * dim], act).reshape(tokens, kv_heads, dim)
    vs = R.act_value(v[:, :kv_heads * dim], act).reshape(tokens, kv_heads, dim)
    want_q = R.norm_rope(qs, qw, EPS, freqs, rot, interleaved, positions)
    want_k = R.norm_rope(ks, kw, EPS, freqs, rot, interleaved, positions)
    rel = (3 * dim ** 0.5 + 12) * R.U
    tol_q = rel * R.partner_size(qs, qw, EPS, rot, interleaved)
    tol_k = rel * R.partner_size(ks, kw, EPS, rot, interleaved)

    got = out.download(q.dtype, tokens * sor, offset=misalign * es).reshape(tokens, sor)
    gq = R.act_value(got[:, :heads * dim], act).reshape(tokens, heads, dim)
    lim = tol_q + (R.HALF_STEP["bf16"] * (np.abs(want_q) + tol_q) if act == "bf16" else 0)
    bad = ~((np.abs(gq - want_q) <= lim) | (np.isnan(gq) & np.isnan(want_q)))
    assert not bad.any(), ("q", int(bad.sum()), np.argwhere(bad)[0], gq[bad][0], want_q[bad][0])
    if pad and not in_place:
        assert (got[:, heads * dim:].view(np.uint8) == 0xff).all(), "elements between the rows of q_out were written"

    dev = pools.download()
    for name, want, tol, sc in (("k", want_k, tol_k, scale[0]), ("v", vs, np.zeros_like(vs), scale[1])):
        left = pools.host[name].copy()
        for j, s in enumerate(slots):
            if not 0 <= s < pages * page:
                continue
            at_ = pools.at(s // page, s % page)
            left[at_] = dev[name][at_]
            g = R.decode(dev[name][at_], kind) * sc
            w = want[j]
            if kind == "e4m3":
                w = np.clip(w, -448 * sc, 448 * sc)
            step = R.HALF_STEP[kind] * (np.abs(w) + tol[j]) + {"e4m3": 2.0 ** -10 * sc, "f16": 2.0 ** -25, "bf16": 0}[kind]
            err = np.abs(g - w)
            # an e4m3 quotient is rounded to fp32 before the type: one more u
            bad = ~((err <= tol[j] + step * (1 + 2 * R.U)) | (np.isnan(g) & np.isnan(w)) | (g == w))
            assert not bad.any(), (name, j, np.argwhere(bad)[0], g[bad][0], w[bad][0])
        assert np.array_equal(left, dev[name]), f"{name}: rows outside the slots changed"
    return args, keep, out, pools


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim,heads,kv_heads,rot,interleaved", [(256, 24, 4, 64, False), (256, 3, 1, 256, False), (128, 5, 5, 128, True),
                                                               (128, 8, 2, 8, False), (64, 7, 1, 40, False), (64, 2, 2, 24, True),
                                                               (128, 4, 2, 0, False)])
def test_types_and_heads(gpu, dim, heads, kv_heads, rot, interleaved, kind, act):
    run(5, heads, kv_heads, dim, rot, kind, act, interleaved, seed=dim + rot, scale=(1 / 16, 1 / 32) if kind == "e4m3" else (1.0, 1.0))


@pytest.mark.parametrize("tokens", [1, 2, 63, 257, 1100])
def test_token_counts(gpu, tokens):
    run(tokens, 24, 4, 256, 64, seed=tokens, page=48)


@pytest.mark.parametrize("case", [dict(gated=True), dict(pad=8), dict(pad=3), dict(order="thd"), dict(gap=16), dict(in_place=True),
                                  dict(norms=False), dict(misalign=1), dict(misalign=2, act="bf16"), dict(page=1), dict(page=7, gated=True, pad=4)],
                         ids=str)
def test_strides_and_places(gpu, case):
    run(9, 6, 2, 128, 32, seed=3, **case)


def test_far_and_negative_positions(gpu):
    run(6, 4, 2, 256, 64, positions=[0, 1, -5, 1 << 20, 16777217, 2 ** 31 - 1], seed=4)


def test_padding_and_bad_slots(gpu):
    """Slots below zero and beyond the pools are skipped; the queries of those tokens are written all the same."""
    run(7, 4, 2, 128, 64, page=16, slots=[3, -1, 40, 1 << 40, 47, 48, -(1 << 62)], seed=5)


def test_values_out_of_range(gpu):
    """NaN and infinities of one head stay in it; e4m3 clamps what is beyond +-448."""
    def spoil(q, k, v):
        q[1, 5] = np.nan
        k[2, 130] = np.nan
        v[0, 0], v[0, 1], v[3, 200] = 1e6, -1e6, np.nan
    run(4, 4, 2, 128, 64, kind="e4m3", seed=6, x=spoil)


def test_stream_and_graph(gpu):
    """Captured on a stream of its own and replayed between other work: every replay gives the eager call's bits."""
    s = hip.Stream()
    args, keep, out, pools = run(33, 24, 4, 256, 64, "e4m3", seed=7, stream=s.handle)
    want, pool = out.download(np.uint32).copy(), pools.download()
    g = hip.Graph(s)
    with g:
        ok(q8mi.lib().q8mi_qk_norm_rope_append(*args), "append")
    for _ in range(3):
        out.fill(0)
        pools.upload()
        hip.synchronize()
        g.launch()
        s.synchronize()
        n = 33 * 24 * 256
        assert np.array_equal(out.download(np.uint32, n), want[:n])
        for name in "kv":
            assert np.array_equal(pools.download()[name], pool[name])


@pytest.mark.parametrize("case", [dict(gated=True), dict(pad=8), dict(pad=3), dict(order="thd"), dict(in_place=True), dict(norms=False),
                                  dict(misalign=1), dict(misalign=2, act="bf16"), dict(page=7, gated=True, pad=4), dict(rot=0),
                                  dict(rot=128, interleaved=True), dict(kind="e4m3", act="bf16", scale=(1 / 16, 1 / 32))], ids=str)
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 21, 3), (64, 40, 5), (256, 6, 1)])
def test_many_tokens(gpu, dim, heads, kv_heads, case):
    """A workgroup a token: the strides, forms and paddings once more, head counts that do not fill the waves."""
    case = {"rot": 32, **case}
    if case["rot"] > dim:
        case["rot"] = dim
    tokens = 1400
    slots = np.random.default_rng(9).permutation(tokens).astype(np.int64)
    slots[::13] = -1
    run(tokens, heads, kv_heads, dim, slots=slots, seed=dim, **case)


def test_two_calls_at_once(gpu):
    """Two streams on caches of their own: nothing is shared."""
    a, b = hip.Stream(), hip.Stream()
    first = run(40, 24, 4, 256, 64, seed=30, stream=a.handle)
    second = run(1500, 8, 2, 128, 128, "f16", "bf16", seed=31, stream=b.handle)
    want = [(o.download(np.uint8).copy(), p.download()) for _, _, o, p in (first, second)]
    for _, _, o, p in (first, second):
        o.fill(0)
        p.upload()
    hip.synchronize()
    ok(q8mi.lib().q8mi_qk_norm_rope_append(*first[0]), "append")
    ok(q8mi.lib().q8mi_qk_norm_rope_append(*second[0]), "append")
    a.synchronize()
    b.synchronize()
    for (_, _, o, p), (out, pool), n in zip((first, second), want, (40 * 24 * 256 * 4, 1500 * 8 * 128 * 2)):
        assert np.array_equal(o.download(np.uint8)[:n], out[:n])
        for name in "kv":
            assert np.array_equal(p.download()[name], pool[name])
