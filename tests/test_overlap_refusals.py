"""Outputs that overlap inputs are refused by the cache append and the paged attention, rows that lie side by side in one buffer
are not.  Every call here is refused on the host, for the one reason or another: the pointers are never followed, and no GPU is
needed."""
import ctypes as C
import random

import pytest

import q8mi

P = 1 << 20


def cache(stride_page, kv_heads=1, dim=64):
    return C.byref(q8mi.KvCache(k=64 * P, v=65 * P, dtype=q8mi.KV_BF16, pages=4, page_size=16, kv_heads=kv_heads, head_dim=dim,
                                stride_page=stride_page, stride_head=16 * dim, stride_token=dim, k_scale=1.0, v_scale=1.0))


def why_attention(q, q_is_bf16, sq, out, out_is_bf16, so, rows, heads=1):
    """The reason: the call's other fault, a pool beyond 64 GiB, is looked at later."""
    rc = q8mi.lib().q8mi_paged_attention(q, q_is_bf16, rows, sq, cache(1 << 36), 70 * P, 4, 71 * P, None, 1, 1, heads, 64, 1.0, out,
                                         out_is_bf16, so, 80 * P, None)
    assert rc == q8mi.REJECTED
    return q8mi.last_error()


def test_attention_against_all_bytes():
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(4000):
        rows, qb, ob = rng.randint(1, 7), rng.randint(0, 1), rng.randint(0, 1)
        wq, wo = 256 >> qb, 256 >> ob
        sq = wq + 16 * rng.choice([0, 1, rng.randint(0, 60)])
        so = rng.choice([sq, max(sq, wo), wo + 16 * rng.randint(0, 60)])
        if so < wo:
            so = wo
        q, out = P, P + 16 * rng.randint(-80, 80)
        if out == q:
            continue
        pieces = lambda at, s, w: {(at + i * s) // 16 + j for i in range(rows) for j in range(w // 16)}  # noqa: E731
        meet = bool(pieces(q, sq, wq) & pieces(out, so, wo))
        why = why_attention(q, qb, sq >> (1 if qb else 2), out, ob, so >> (1 if ob else 2), rows)
        assert ("out overlaps q" in why) == meet, (rows, qb, ob, sq, so, out - q, why)
        assert meet or "64 GiB" in why
        seen[meet] += 1
    assert min(seen) > 400


def append(q_out, k=2 * P, v=3 * P, q=P, tokens=3, q_heads=2, sqr=128, sqh=64, skr=64, svr=64, sor=128, is_bf16=0, kv_heads=1):
    rc = q8mi.lib().q8mi_qk_norm_rope_append(q, k, v, q_out, is_bf16, tokens, q_heads, sqr, sqh, skr, svr, sor, None, None, 1e-6, 4 * P, 64, 0,
                                             5 * P, 6 * P, cache(1 << 16, kv_heads), None)
    assert rc == q8mi.REJECTED
    return q8mi.last_error()


@pytest.mark.parametrize("case,why", [
    (dict(q_out=P + 4), "overlaps q"), (dict(q_out=P - 4), "overlaps q"), (dict(q_out=P + 512 * 3 - 4), "overlaps q"),
    (dict(q_out=P - 512 * 3 + 4), "overlaps q"), (dict(q_out=P + 512), "overlaps q"), (dict(q_out=P + 8, is_bf16=1), "overlaps q"),
    (dict(q_out=P + 4, tokens=1), "overlaps q"), (dict(q_out=P + 64 * 4, sqh=128, sqr=256), "overlaps q"),     # gates are no room for two heads
    (dict(q_out=P + 64 * 4, sqh=3 * 64, sqr=256, sor=160), "overlaps q"), (dict(q_out=2 * P), "k or v"), (dict(q_out=3 * P), "k or v"),
    (dict(q_out=2 * P + 3 * 256 - 4), "k or v"), (dict(q_out=3 * P - 3 * 512 + 4), "k or v"),
    (dict(q_out=P, k=P + 256, sqr=192, skr=192, sor=192), "k or v"),              # in place, k inside the queries' rows
    (dict(q_out=P, v=P + 512, sqr=190, svr=190, sor=190, skr=200, q_heads=3), "rows overlap")], ids=str)
def test_append(case, why):
    assert why in append(**case)


def test_reasons_of_the_bounds():
    """The refusals of the other arguments, on operands that lie apart: each names its own reason."""
    base = dict(q=P, qb=0, rows=4, sq=512, cache=cache(2 * 16 * 128, 2, 128), table=2 * P, stable=4, lens=3 * P, starts=None, n=2, new=2,
                heads=4, max_kv=64, scale=1.0, out=4 * P, ob=0, so=512, scratch=5 * P)
    for change, why in ((dict(q=0), "null"), (dict(out=0), "null"), (dict(table=0), "null"), (dict(lens=0), "null"), (dict(scratch=0), "null"),
                        (dict(heads=0), "query heads"), (dict(heads=5), "query heads"), (dict(heads=65538, sq=1 << 24, so=1 << 24), "query heads"),
                        (dict(new=0), "rows a sequence"), (dict(new=17), "rows a sequence"), (dict(max_kv=65), "page table"),
                        (dict(scale=float("nan")), "scale"), (dict(scale=3e38), "scale"), (dict(q=P + 4), "16-byte"), (dict(out=4 * P + 8), "16-byte"),
                        (dict(scratch=5 * P + 4), "16-byte"), (dict(sq=514), "16-byte"), (dict(so=510), "16-byte"), (dict(sq=256), "rows overlap"),
                        (dict(so=508), "rows overlap"), (dict(n=1 << 22), "too many"), (dict(out=P), "out is q")):
        a = {**base, **change}
        assert q8mi.lib().q8mi_paged_attention(*a.values(), None) == q8mi.REJECTED
        assert why in q8mi.last_error(), (change, q8mi.last_error())
    base = dict(q=P, k=2 * P, v=3 * P, q_out=4 * P, b=0, tokens=2, heads=4, sqr=512, sqh=128, skr=256, svr=256, sor=512, qw=None, kw=None, eps=1e-6,
                freqs=5 * P, rot=64, inter=0, positions=6 * P, slots=7 * P, cache=cache(2 * 16 * 128, 2, 128))
    for change, why in ((dict(q=0), "null"), (dict(k=0), "null"), (dict(v=0), "null"), (dict(q_out=0), "null"), (dict(slots=0), "null"),
                        (dict(freqs=0), "frequencies"), (dict(positions=0), "positions"), (dict(rot=60), "rotary_dim"), (dict(rot=136), "rotary_dim"),
                        (dict(heads=0), "query heads"), (dict(heads=65537, sqr=1 << 31), "query heads"), (dict(sqh=120), "rows overlap"),
                        (dict(sqr=508), "rows overlap"), (dict(skr=255), "rows overlap"), (dict(svr=100), "rows overlap"), (dict(sor=511), "rows overlap"),
                        (dict(q_out=P, sqh=256, sqr=1024), "in place"), (dict(q_out=P, sqr=1024), "in place"),
                        (dict(q=1 << 40, k=1 << 41, v=1 << 42, q_out=1 << 43, tokens=1 << 24), "too many")):
        a = {**base, **change}
        assert q8mi.lib().q8mi_qk_norm_rope_append(*a.values(), None) == q8mi.REJECTED
        assert why in q8mi.last_error(), (change, q8mi.last_error())
