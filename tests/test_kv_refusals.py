"""What the cache append, the paged attention and the sampler refuse: every refusal is taken on the host before anything is
enqueued, so these run without a GPU (the pointers are never followed)."""
import ctypes as C

import pytest

import q8mi

P = 4096           # an aligned address that is never followed
NAN, INF = float("nan"), float("inf")


def cache(**changed):
    d = dict(k=P, v=P, dtype=q8mi.KV_BF16, pages=4, page_size=16, kv_heads=2, head_dim=128, stride_page=2 * 16 * 128,
             stride_head=16 * 128, stride_token=128, k_scale=1.0, v_scale=1.0)
    d.update(changed)
    return C.byref(q8mi.KvCache(**d))


BAD_CACHES = [dict(k=0), dict(v=0), dict(dtype=3), dict(dtype=-1), dict(head_dim=96), dict(head_dim=0), dict(pages=0),
              dict(pages=1 << 31), dict(page_size=0), dict(page_size=65537), dict(kv_heads=0), dict(k=P + 8), dict(v=P + 2),
              dict(stride_token=120), dict(stride_token=132), dict(stride_head=4), dict(stride_page=4),
              dict(dtype=q8mi.KV_E4M3, stride_token=136), dict(dtype=q8mi.KV_E4M3, k_scale=0.0),
              dict(dtype=q8mi.KV_E4M3, v_scale=-1.0), dict(dtype=q8mi.KV_E4M3, v_scale=NAN), dict(dtype=q8mi.KV_E4M3, k_scale=INF)]


def append(c=None, **changed):
    a = dict(q=P, k=P, v=P, q_out=2 * P, is_bf16=0, tokens=2, q_heads=4, sqr=512, sqh=128, skr=256, svr=256, sor=512, qw=P, kw=P,
             eps=1e-6, freqs=P, rot=64, interleaved=0, positions=P, slots=P)
    a.update(changed)
    return q8mi.lib().q8mi_qk_norm_rope_append(*a.values(), cache() if c is None else c, None)


def attend(c=None, **changed):
    a = dict(q=2 * P, q_is_bf16=0, q_rows=4, sq=512, cache=cache() if c is None else c, table=P, stable=4, lens=P, starts=None, n=2, new=2, heads=4,
             max_kv=64, scale=1.0, out=P, out_is_bf16=0, so=512, scratch=P)
    a.update(changed)
    return q8mi.lib().q8mi_paged_attention(*a.values(), None)


def sample(**changed):
    a = dict(x=P, batch=2, vocab=100, stride=100, t=P, k=P, p=P, m=P, u=P, out=P, scratch=P)
    a.update(changed)
    return q8mi.lib().q8mi_sample(*a.values(), None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_cache_descriptor(bad):
    assert append(cache(**bad)) == q8mi.REJECTED
    assert attend(cache(**bad)) == q8mi.REJECTED
    assert q8mi.last_error().startswith("paged_attention")


def test_null_cache():
    none = C.POINTER(q8mi.KvCache)()
    assert append(none) == q8mi.REJECTED and attend(none) == q8mi.REJECTED


@pytest.mark.parametrize("bad", [dict(q=0), dict(k=0), dict(v=0), dict(q_out=0), dict(slots=0), dict(freqs=0), dict(positions=0),
                                 dict(rot=60), dict(rot=136), dict(q_heads=0), dict(sqh=120), dict(sqr=508), dict(skr=255),
                                 dict(svr=100), dict(sor=511), dict(q_out=P, sqh=256, sqr=1024), dict(q_out=P, sqr=1024), dict(tokens=1 << 24),
                                 dict(q_heads=65537, sqr=1 << 31)], ids=str)
def test_append(bad):
    assert append(**bad) == q8mi.REJECTED
    assert q8mi.last_error()


@pytest.mark.parametrize("bad", [dict(q=0), dict(out=0), dict(table=0), dict(lens=0), dict(scratch=0), dict(heads=0), dict(heads=5),
                                 dict(new=0), dict(new=17), dict(max_kv=65), dict(scale=NAN), dict(scale=INF), dict(q=P + 4),
                                 dict(out=P + 8), dict(scratch=P + 4), dict(sq=514), dict(so=510), dict(sq=256), dict(so=508),
                                 dict(q_is_bf16=1, sq=516), dict(n=1 << 22), dict(scale=3e38), dict(out=2 * P), dict(heads=65538, sq=1 << 24, so=1 << 24)], ids=str)
def test_attention(bad):
    assert attend(**bad) == q8mi.REJECTED
    assert q8mi.last_error()


@pytest.mark.parametrize("bad", [dict(x=0), dict(u=0), dict(out=0), dict(scratch=0), dict(vocab=0), dict(vocab=(1 << 20) + 1),
                                 dict(stride=99), dict(scratch=P + 8), dict(batch=65536)], ids=str)
def test_sample(bad):
    assert sample(**bad) == q8mi.REJECTED
    assert q8mi.last_error()


def test_nothing_to_do():
    assert append(tokens=0) == q8mi.OK
    assert attend(n=0) == q8mi.OK and attend(q_rows=0) == q8mi.OK
    assert sample(batch=0) == q8mi.OK


def test_scratch_sizes():
    L = q8mi.lib()
    assert L.q8mi_paged_attention_scratch_bytes(1, 1, 24, 4, 256, 131072) >= 16
    assert L.q8mi_paged_attention_scratch_bytes(0, 1, 24, 0, 256, 0) >= 16     # nonsense asks for a little, and does not trap
    assert L.q8mi_sample_scratch_bytes(64, 248320) >= 16
