"""The sampler against its definition with integer weights: tokens are equal, not close."""
import numpy as np
import pytest

import kv_ref as R
import q8mi
from gpu_common import NULL
from q8mi import hip, ok

pytestmark = pytest.mark.gpu
PAIR = np.dtype([("value", np.float32), ("index", np.int32)])


class Case:
    def __init__(self, z, temperature=None, top_k=None, top_p=None, min_p=None, u=None, pad=0, seed=0):
        z = np.atleast_2d(np.asarray(z, np.float32))
        self.batch, self.vocab = z.shape
        self.z = z
        self.stride = self.vocab + pad
        wide = np.full((self.batch, self.stride), 99.0, np.float32)    # larger than every logit: never to be read
        wide[:, :self.vocab] = z
        spread = lambda v, t: None if v is None else np.broadcast_to(np.asarray(v, t), (self.batch,)).copy()  # noqa: E731
        self.t, self.k = spread(temperature, np.float32), spread(top_k, np.int32)
        self.p, self.m = spread(top_p, np.float32), spread(min_p, np.float32)
        self.u = spread(u if u is not None else np.random.default_rng(seed).random(self.batch), np.float32)
        put = lambda a: None if a is None else hip.to_device(a)  # noqa: E731
        self.dev = [hip.to_device(wide)] + [put(a) for a in (self.t, self.k, self.p, self.m, self.u)]
        self.out = hip.DeviceBuffer(8 * self.batch).fill(0xff)
        self.bytes = q8mi.lib().q8mi_sample_scratch_bytes(self.batch, self.vocab)
        self.scratch = hip.DeviceBuffer(self.bytes + 64).fill(0xff)

    def launch(self, stream=NULL):
        x, t, k, p, m, u = (d.ptr if d is not None else None for d in self.dev)
        ok(q8mi.lib().q8mi_sample(x, self.batch, self.vocab, self.stride, t, k, p, m, u, self.out.ptr, self.scratch.ptr, stream), "sample")

    def want(self):
        at = lambda a, r, off: off if a is None else a[r]  # noqa: E731
        return [R.sample(self.z[r], at(self.t, r, 1.0), int(at(self.k, r, 0)), at(self.p, r, 1.0), at(self.m, r, 0.0), self.u[r])
                for r in range(self.batch)]

    def check(self):
        got = self.out.download(PAIR)
        want = self.want()
        assert got["index"].tolist() == want, [(i, g, w) for i, (g, w) in enumerate(zip(got["index"], want)) if g != w][:5]
        for r, w in enumerate(want):
            assert got["value"][r] == (self.z[r, w] if w >= 0 else -np.inf)
        assert (self.scratch.download(np.uint8)[self.bytes:] == 0xff).all(), "the scratch was overrun"


def run(*a, **k):
    c = Case(*a, **k)
    c.launch()
    hip.synchronize()
    c.check()
    return c


def logits(batch, vocab, seed, likely=48):
    rng = np.random.default_rng(seed)
    z = 2 * rng.standard_normal((batch, vocab))
    for r in range(batch):
        z[r, rng.integers(0, vocab, likely)] = 12 + 2.5 * rng.standard_normal(likely)
    return z


SETTINGS = [dict(), dict(temperature=0.7, top_k=20, top_p=0.95), dict(temperature=1.3), dict(top_k=1), dict(top_k=50), dict(top_p=0.5),
            dict(top_p=0.9999), dict(min_p=0.05), dict(temperature=0.3, min_p=0.3), dict(temperature=1.5, top_k=400, top_p=0.8, min_p=0.01),
            dict(temperature=0.0), dict(temperature=100.0, top_p=0.9), dict(temperature=100.0, top_k=3000, top_p=0.7)]


@pytest.mark.parametrize("how", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 4096, 32003])
def test_settings(gpu, vocab, how):
    run(logits(7, vocab, vocab), seed=vocab, pad=5, **how)


@pytest.mark.parametrize("how", SETTINGS, ids=str)
def test_a_vocabulary(gpu, how):
    run(logits(3, 248320, 5), seed=6, **how)


@pytest.mark.parametrize("vocab", [4095, 4097, 8192, 8193, 16384, 16385, 65536, 151936, 1 << 20])
def test_lengths(gpu, vocab):
    run(logits(2, vocab, vocab), temperature=[0.8, 1.0], top_k=[30, 0], top_p=[0.9, 0.99], seed=vocab)


def test_settings_of_each_row(gpu):
    rng = np.random.default_rng(9)
    pick = lambda v: rng.choice(v, 64)  # noqa: E731
    run(logits(64, 20000, 8), temperature=pick([0.0, -1.0, 0.5, 1.0, 2.0, np.nan, np.inf]), top_k=pick([-3, 0, 1, 5, 300, 40000]),
        top_p=pick([-0.5, 0.0, 0.3, 0.9, 1.0, 2.0, np.nan]), min_p=pick([-1.0, 0.0, 0.02, 0.5, 1.0, 3.0, np.nan]), seed=10)


def test_uniform_at_its_ends(gpu):
    z = np.tile(logits(1, 5000, 11), (9, 1))
    run(z, top_k=40, u=[0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, np.nan, np.inf, 2.0 ** -30, 0.5])


@pytest.mark.parametrize("vocab", [6, 3000, 40000])
def test_equal_logits(gpu, vocab):
    """Ties go to the lower index at every cut, and the draw is uniform over what stays."""
    z = np.zeros((6, vocab))
    run(z, top_k=[3, 0, 0, 2500, 0, 1], top_p=[1, 0.5, 1, 0.25, 0.0, 1], min_p=[0, 0, 1, 0, 0, 0],
        u=[0.7, 0.999, 0.3, 0.99, 0.9, 0.5])


def test_two_levels(gpu):
    """Cuts that end inside a run of equal logits behind larger ones; -0 and +0 are equal."""
    z = np.full((5, 9000), -1.0)
    z[:, 17::100] = 0.0
    z[:, 67::100] = -0.0
    z[:, [4000, 1]] = 2.0
    run(z, top_k=[50, 0, 100, 3, 0], top_p=[1, 0.1, 0.5, 1.0, 0.9], u=[0.95, 0.97, 0.6, 0.99, 0.999])


def test_masked_rows(gpu):
    """-inf and NaN are never drawn, a row of nothing else gives -1, +inf takes all."""
    z = logits(8, 3000, 13)
    z[0, :] = -np.inf
    z[1, :] = np.nan
    z[2, :] = -np.inf
    z[2, 2999] = -5.0
    z[3, ::2] = -np.inf
    z[4, 1::2] = np.nan
    z[5, [7, 99, 2000]] = np.inf
    z[6, :] = np.float32(-3.4e38)
    z[7, :10] = np.float32(3.4e38)
    run(z, top_k=[0, 5, 3, 0, 40, 0, 0, 0], top_p=[0.9, 1, 1, 0.9, 1, 0.9, 0.5, 1], seed=14)
    run(z, temperature=0.0)


def test_every_token_can_be_drawn(gpu):
    """u in the middle of each token's share draws that token."""
    p = np.array([0.05, 0.4, 0.15, 0.3, 0.1])
    z = np.tile(np.log(p), (5, 1))
    c = run(z, u=np.cumsum(p) - p / 2)
    assert c.out.download(PAIR)["index"].tolist() == [0, 1, 2, 3, 4]


def test_graph_and_stream(gpu):
    s = hip.Stream()
    c = Case(logits(4, 50000, 15), temperature=[0.8, 1, 0, 1.2], top_k=[40, 0, 0, 0], top_p=[0.9, 0.95, 1, 1], seed=16)
    c.launch(s.handle)
    s.synchronize()
    c.check()
    other = Case(logits(2, 9000, 17), top_p=0.8, seed=18)
    g = hip.Graph(s)
    with g:
        c.launch(s.handle)
    for rep in range(4):
        c.u = np.random.default_rng(rep).random(4).astype(np.float32)
        c.dev[5].upload(c.u)
        c.out.fill(0xff)
        hip.synchronize()
        g.launch()
        other.launch(s.handle)
        s.synchronize()
        c.check()
        other.check()


def test_token_feeds_the_embedding_lookup(gpu):
    """q8mi_get_row_from_argmax reads the pair the sampler wrote."""
    import q8mi_support as synth
    vocab, cols = 600, 256
    w = synth.q8_0_weight(vocab, cols, seed=1)
    c = run(logits(3, vocab, 19), top_k=10, seed=20)
    dw, out, want = hip.to_device(w), hip.DeviceBuffer(4 * cols), hip.DeviceBuffer(4 * cols)
    for r, token in enumerate(c.want()):
        ok(q8mi.lib().q8mi_get_row_from_argmax(dw.ptr, c.out.ptr, r, vocab, cols, out.ptr, NULL), "row of the pair")
        ok(q8mi.lib().q8mi_get_row(dw.ptr, token, vocab, cols, want.ptr, 0, NULL), "row")
        hip.synchronize()
        assert np.array_equal(out.download(np.uint32), want.download(np.uint32))


@pytest.mark.parametrize("depth", [29.45, 29.6, 29.9])
def test_a_tail_of_the_least_weights(gpu, depth):
    """2^20 logits whose weight rounds to one unit (or none) against 1 - top_p of a few units each: rounding moves the cut into
    the tail."""
    z = np.full((3, 1 << 20), -depth)
    z[:, 12345] = 0.0
    run(z, top_p=[1 - 3 * 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -20], u=1 - 2.0 ** -24)


@pytest.mark.parametrize("spread", [0.0, 1e-3])
def test_more_candidates_than_a_list_holds(gpu, spread):
    """All that top_k wants in a few chunks, whose lists overflow; and equal logits all over the row."""
    rng = np.random.default_rng(21)
    z = rng.standard_normal((4, 100000))
    z[:2, 3000:4500] = 30 + spread * rng.standard_normal((2, 1500))
    z[2:] = spread * rng.standard_normal((2, 100000))
    run(z, top_k=[60, 90, 97, 5], top_p=[0.9, 1.0, 0.5, 1.0], u=[0.3, 0.9, 0.99, 0.5])


def test_the_largest_vocabulary_by_count(gpu):
    """top_k up to the number of chunks (1024), and just above it."""
    run(logits(3, 1 << 20, 22), temperature=1.5, top_k=[1000, 1024, 1025], top_p=[0.9, 1.0, 0.99], seed=23)


@pytest.mark.parametrize("pad,shift", [(1, 0), (3, 1), (4, 0), (0, 3)])
def test_rows_on_any_boundary(gpu, pad, shift):
    """Strides and addresses that keep rows off 16-byte boundaries."""
    z = logits(5, 5003, 24)
    c = Case(z, temperature=0.9, top_k=30, top_p=0.9, pad=pad, seed=25)
    wide = np.full(5 * c.stride + shift, 99.0, np.float32)
    wide[shift:].reshape(5, c.stride)[:, :5003] = z
    big = hip.to_device(wide)
    x, t, k, p, m, u = (d.ptr if d is not None else None for d in c.dev)
    ok(q8mi.lib().q8mi_sample(big.ptr + 4 * shift, 5, 5003, c.stride, t, k, p, m, u, c.out.ptr, c.scratch.ptr, NULL), "sample")
    hip.synchronize()
    c.check()


def test_two_calls_at_once(gpu):
    """Two streams, a scratch each."""
    a, b = hip.Stream(), hip.Stream()
    c = Case(logits(16, 60000, 26), temperature=0.9, top_p=0.95, seed=27)
    d = Case(logits(8, 151936, 28), temperature=1.1, top_k=64, seed=29)
    hip.synchronize()
    for _ in range(4):
        c.launch(a.handle)
        d.launch(b.handle)
    a.synchronize()
    b.synchronize()
    c.check()
    d.check()


def test_many_rows(gpu):
    """A row each for many sequences, several chunks to a workgroup."""
    run(logits(300, 9001, 30), temperature=0.8, top_k=[5, 0, 700] * 100, top_p=[0.9, 0.95, 0.8] * 100, seed=31)


@pytest.mark.parametrize("vocab,k", [(32000, 40), (32003, 64), (32003, 65), (2000, 4), (1025, 3), (131072, 128), (65536, 128), (65536, 129)])
def test_counts_about_the_chunks(gpu, vocab, k):
    """top_k about the number of chunks of a row, and about twice that."""
    run(logits(4, vocab, vocab + k), temperature=0.9, top_k=[k - 1, k, k + 1, k], top_p=[0.95, 1.0, 0.9, 0.5], seed=k)


def test_graphs_share_a_scratch(gpu):
    """Two captured calls on one scratch, replayed in turn on one stream."""
    s = hip.Stream()
    c, d = Case(logits(3, 40000, 40), top_k=30, seed=41), Case(logits(3, 40000, 42), temperature=0.7, top_p=0.9, seed=43)
    d.scratch = c.scratch
    graphs = []
    for case in (c, d):
        case.launch(s.handle)
        g = hip.Graph(s)
        with g:
            case.launch(s.handle)
        graphs.append(g)
    for rep in range(3):
        for case in (c, d):
            case.u = np.random.default_rng(50 + rep).random(3).astype(np.float32)
            case.dev[5].upload(case.u)
            case.out.fill(0xff)
        hip.synchronize()
        for g in graphs:
            g.launch()
        s.synchronize()
        c.check()
        d.check()
