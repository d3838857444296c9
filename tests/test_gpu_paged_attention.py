"""Attention over a paged cache against its 64-bit form.

Bounds (u = 2^-24): a score is a sum of D products and a few more roundings, off by at most d = (6 sqrt(D) + 8) u of
scale * sum |q k| (probabilistic bound of D random roundings); every weight then changes by a factor within exp(+-d), their sum
likewise, the exponential and the split of a weight over matrix operands add 8 u, and n weights times values are added with
6 sqrt(n) u: below (2 d size + (6 sqrt(n) + 16) u) of sum p |v|.  bf16 outputs add half a step.

fp16 and e4m3 caches: a weight, at most 1 before the division by the sum (which is at least 1), enters the products times 2^14
as two fp16 numbers.  Its first term is off by half a step, at most 2^-11 of itself, and the second, the rest, by 2^-11 of that, 2^-22
= 4 u of the weight (part of the 8 u above), as long as their steps follow their size; fp16's smallest step is 2^-24, so that below
it a weight is off by half of that, 2^-25 / 2^14 = 2^-39 of the row's largest: where the tokens of large weight hold zeros, their sum
2^-39 sum |v| is what counts."""
import numpy as np
import pytest

import kv_ref as R
import q8mi
from gpu_common import NULL
from q8mi import hip, ok

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, lens, rows, heads, kv_heads, dim, kind="bf16", act="f32", out_act=None, page=16, order="htd", gap=0, pad=0,
                 max_q=None, starts=True, max_kv=None, far=False, seed=0, q_scale=2.0, scale=None, spare_rows=2, table_pad=1):
        rng = np.random.default_rng(seed)
        self.rng = rng
        self.lens, self.rows = list(lens), list(rows)
        self.heads, self.kv_heads, self.dim, self.kind, self.act, self.out_act = heads, kv_heads, dim, kind, act, out_act or act
        self.scale = dim ** -0.5 if scale is None else scale
        self.max_q = max_q or max(self.rows)
        self.n = len(self.lens)
        first = np.concatenate([[0], np.cumsum(self.rows)])
        self.starts = first.astype(np.int32) if starts else None
        self.q_rows = int(first[-1]) + spare_rows
        need = [max(0, (n + page - 1) // page) for n in self.lens]
        self.wide = max(need + [1]) + table_pad
        self.max_kv = max(max(self.lens), 1) if max_kv is None else max_kv
        if far:   # bounds of a long context: the cut of a large call, on the lengths of a small one
            self.wide, self.max_kv = 70000 // page + 1, 70000
        pages = sum(need) + 2
        ks, vs = (1 / 16, 1 / 8) if kind == "e4m3" else (1.0, 1.0)
        self.pools = R.Pools(kind, pages, page, kv_heads, dim, order, gap, ks, vs)     # unwritten rows are NaN in every type
        order_ = rng.permutation(pages)
        self.table = np.full((self.n, self.wide), -7, np.int32)                        # what no sequence may follow
        self.k, self.v = [], []
        at = 0
        for s, n in enumerate(self.lens):
            n = max(0, n)
            self.table[s, :need[s]] = order_[at:at + need[s]]
            at += need[s]
            k, v = rng.standard_normal((n, kv_heads, dim)), rng.standard_normal((n, kv_heads, dim))
            kb, vb = R.encode(k / ks, kind), R.encode(v / vs, kind)
            for t in range(n):
                self.pools.put("k", self.table[s, t // page], t % page, kb[t])
                self.pools.put("v", self.table[s, t // page], t % page, vb[t])
            self.k.append(R.decode(kb, kind) * ks)
            self.v.append(R.decode(vb, kind) * vs)
        self.pools.upload()
        self.width = heads * dim
        self.sq = self.so = self.width + pad
        q = (q_scale * rng.standard_normal((self.q_rows, self.sq))).astype(np.float32)
        self.q = R.act_bits(q, act)
        self.dq = hip.to_device(self.q)
        self.oes = 2 if self.out_act == "bf16" else 4
        self.dout = hip.DeviceBuffer(self.q_rows * self.so * self.oes).fill(0x5a)
        self.dt, self.dl = hip.to_device(self.table), hip.to_device(np.asarray(self.lens, np.int32))
        self.ds = hip.to_device(self.starts) if starts else None
        n = q8mi.lib().q8mi_paged_attention_scratch_bytes(self.n, self.max_q, heads, kv_heads, dim, self.max_kv)
        self.scratch = hip.DeviceBuffer(n + 64).fill(0xff)
        self.scratch_bytes = n

    def args(self, stream=NULL):
        return (self.dq.ptr, int(self.act == "bf16"), self.q_rows, self.sq, self.pools.ref, self.dt.ptr, self.wide, self.dl.ptr,
                self.ds.ptr if self.ds else None, self.n, self.max_q, self.heads, self.max_kv, self.scale, self.dout.ptr,
                int(self.out_act == "bf16"), self.so, self.scratch.ptr, stream)

    def launch(self, stream=NULL):
        ok(q8mi.lib().q8mi_paged_attention(*self.args(stream)), "paged_attention")

    def check(self, hidden=lambda s, t: False):
        """Compares what the call left with the definition; hidden(s, t): tokens behind a bad page id."""
        dt = np.uint16 if self.out_act == "bf16" else np.float32
        got = self.dout.download(dt).reshape(self.q_rows, self.so)
        raw = got.view(np.uint8).reshape(self.q_rows, -1)
        written = np.zeros(self.q_rows, bool)
        for s in range(self.n):
            first = int(self.starts[s]) if self.starts is not None else s * self.max_q
            count = int(self.starts[s + 1]) - first if self.starts is not None else self.max_q
            for i in range(min(count, self.max_q)):
                r = first + i
                if r >= self.q_rows:
                    continue
                written[r] = True
                seen = min(self.lens[s] - count + i + 1, self.max_kv)
                ts = [t for t in range(max(0, seen)) if not hidden(s, t)]
                q = R.act_value(self.q[r, :self.width], self.act).reshape(self.heads, self.dim)
                want, mag, size = R.attention(q, self.k[s][ts], self.v[s][ts], np.float64(np.float32(self.scale)), len(ts))
                u = R.U
                tol = (2 * (6 * self.dim ** 0.5 + 8) * u * size[:, None] + (6 * max(1, len(ts)) ** 0.5 + 16) * u) * mag
                if self.kind != "bf16" and ts:
                    tol = tol + 2.0 ** -39 * np.abs(self.v[s][ts]).sum(0).repeat(self.heads // self.kv_heads, 0)
                if self.out_act == "bf16":
                    tol = tol + R.HALF_STEP["bf16"] * (np.abs(want) + tol)
                g = R.act_value(got[r, :self.width], self.out_act).reshape(self.heads, self.dim)
                bad = ~(np.abs(g - want) <= tol)
                assert not bad.any(), (s, i, int(bad.sum()), np.argwhere(bad)[0], g[bad][0], want[bad][0], tol[bad][0])
        assert (raw[~written] == 0x5a).all(), "a row outside every sequence was written"
        assert (raw[:, self.width * self.oes:] == 0x5a).all(), "elements between the rows were written"
        assert (self.scratch.download(np.uint8)[self.scratch_bytes:] == 0xff).all(), "the scratch was overrun"


def run(*a, **k):
    c = Case(*a, **k)
    c.launch()
    hip.synchronize()
    c.check()
    return c


FAR = pytest.mark.parametrize("far", [False, True], ids=["near", "far"])


@FAR
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(256, 24, 4), (256, 2, 2), (128, 8, 1), (128, 10, 2), (64, 12, 12), (64, 20, 1)])
def test_types_and_heads(gpu, dim, heads, kv_heads, kind, act, far):
    run([37, 150], [1, 1], heads, kv_heads, dim, kind, act, seed=dim + heads, far=far)


@FAR
@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1023, 1025, 3001])
def test_lengths(gpu, n, kind, far):
    run([n], [1], 6, 1, 256, kind, seed=n, far=far)


@FAR
@pytest.mark.parametrize("rows", [2, 3, 5, 8, 11, 16])
@pytest.mark.parametrize("dim,heads,kv_heads", [(256, 12, 2), (128, 40, 8), (64, 7, 7)])
def test_several_rows(gpu, rows, dim, heads, kv_heads, far):
    run([rows, 3, 130, 700], [rows, min(3, rows), rows, 1], heads, kv_heads, dim, seed=rows, far=far)


def test_wide_group(gpu):
    """More query rows of a key head than one tile of any size: 80 query heads over one, 16 rows."""
    run([100, 40], [16, 7], 80, 1, 64, seed=8)


@FAR
@pytest.mark.parametrize("page", [1, 3, 8, 20, 48, 256, 1000])
def test_page_sizes(gpu, page, far):
    run([333, 1, 64], [1, 1, 2], 8, 2, 128, "f16", page=page, seed=page, far=far)


@FAR
@pytest.mark.parametrize("case", [dict(order="thd"), dict(gap=8), dict(pad=8), dict(act="bf16", out_act="f32"),
                                  dict(act="f32", out_act="bf16"), dict(starts=False), dict(starts=False, spare_rows=0), dict(scale=0.0),
                                  dict(scale=-0.3), dict(q_scale=40.0)], ids=str)
def test_strides_and_forms(gpu, case, far):
    run([90, 33], [2, 2], 8, 4, 128, seed=12, far=far, **case)


@FAR
def test_empty_and_idle(gpu, far):
    """Sequences without tokens, without rows, with fewer tokens than rows (their first rows see nothing: zeros) and a
    negative length."""
    run([0, 70, 2, -3, 5, 0], [1, 0, 4, 1, 5, 2], 4, 2, 128, seed=13, far=far)


def test_every_sequence_empty(gpu):
    run([0, 0], [1, 2], 4, 2, 256, seed=13)


def test_no_tokens_at_all(gpu):
    """A bound of no tokens: every row is zero, the cached tokens are not looked at."""
    run([5, 0], [1, 2], 4, 2, 128, max_kv=0, seed=13)


def test_bounds_of_the_host(gpu):
    """Rows beyond max_q_len and beyond q_rows are not computed, tokens from max_kv_len on not read."""
    c = Case([80, 60], [5, 2], 4, 2, 128, max_q=3, max_kv=64, seed=14, spare_rows=0)
    c.launch()
    hip.synchronize()
    c.check()
    c = Case([80, 60], [2, 3], 4, 2, 128, seed=15, spare_rows=-1)
    c.launch()
    hip.synchronize()
    c.check()


@FAR
def test_bad_pages_hide_their_tokens(gpu, far):
    """Page ids below zero and beyond the pool: nothing is read, the other tokens count."""
    c = Case([100, 50], [1, 2], 4, 2, 128, page=16, seed=16, far=far)
    bad = {(0, 1): -1, (0, 4): c.pools.pages, (1, 0): 2 ** 31 - 1, (1, 3): -2 ** 31}
    for (s, p), v in bad.items():
        c.table[s, p] = v
    c.dt.upload(c.table)
    c.launch()
    hip.synchronize()
    c.check(hidden=lambda s, t: (s, t // 16) in bad)


@FAR
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_later_tokens_do_not_leak(gpu, kind, far):
    """A draft's key or value that holds infinities or NaN reaches its own and later rows only."""
    c = Case([40], [4], 6, 2, 128, kind, seed=17, far=far)
    inf, nan = {"bf16": (0x7f80, 0x7fc0), "f16": (0x7c00, 0x7e00)}[kind]
    t = 38                                      # seen by rows 2 and 3
    for name, bits in (("v", inf), ("v", nan)):
        at = c.pools.at(c.table[0, t // 16], t % 16)
        c.pools.host[name][at[:, ::3]] = bits
    c.pools.upload()
    c.v[0][t, :, ::3] = np.nan
    c.launch()
    hip.synchronize()
    got = c.dout.download(np.float32).reshape(c.q_rows, c.so)
    for r in range(4):
        q = R.act_value(c.q[r, :c.width], c.act).reshape(c.heads, c.dim)
        want, mag, _ = R.attention(q, c.k[0], c.v[0], c.scale, 40 - 4 + r + 1)
        g = got[r, :c.width].reshape(c.heads, c.dim)
        assert np.array_equal(np.isnan(g) | np.isinf(g), np.isnan(want)), r
        fine = ~np.isnan(want)
        assert np.abs(g - want)[fine].max() < 1e-4, r


def test_long_context(gpu):
    """Long enough for every split and for the join; a late key that outweighs all before it."""
    c = Case([20011, 17], [1, 1], 6, 1, 256, "bf16", page=64, seed=18)
    c.launch()
    hip.synchronize()
    c.check()


def test_equal_scores_give_the_mean(gpu):
    """Closed form: zero queries weigh all tokens alike, whatever the split."""
    c = Case([777], [1], 4, 4, 64, "bf16", seed=19, q_scale=0.0)
    c.launch()
    hip.synchronize()
    got = c.dout.download(np.float32).reshape(c.q_rows, c.so)[0, :c.width].reshape(4, 64)
    assert np.abs(got - c.v[0].mean(0)).max() < 777 ** 0.5 * 8 * R.U * np.abs(c.v[0]).max()


def test_one_token_returns_its_value(gpu):
    c = Case([1], [1], 8, 2, 128, "e4m3", seed=20)
    c.launch()
    hip.synchronize()
    got = c.dout.download(np.float32).reshape(c.q_rows, c.so)[0, :c.width].reshape(8, 128)
    want = c.v[0][0].repeat(4, 0)
    assert np.abs(got - want).max() <= 4 * R.U * np.abs(want).max()


def test_graph_with_changing_lengths(gpu):
    """A captured call follows kv_lens and the page table as they are at the replay, between eager calls on another scratch."""
    s = hip.Stream()
    c = Case([900, 300], [2, 2], 6, 1, 256, seed=21)
    c.launch(s.handle)
    s.synchronize()
    c.check()
    other = Case([50], [1], 6, 1, 256, seed=22)
    g = hip.Graph(s)
    with g:
        c.launch(s.handle)
    for lens in ([900, 300], [3, 299], [0, 1], [640, 64]):
        c.lens = list(lens)
        c.dl.upload(np.asarray(lens, np.int32))
        c.dout.fill(0x5a)
        hip.synchronize()
        g.launch()
        other.launch(s.handle)
        s.synchronize()
        c.check()
        other.check()


def test_results_repeat(gpu):
    """The same call twice gives the same bits (nothing depends on the order in which workgroups end)."""
    c = Case([4000, 1200, 7], [3, 1, 2], 12, 2, 128, "f16", page=32, seed=23)
    c.launch()
    hip.synchronize()
    a = c.dout.download(np.uint32).copy()
    for _ in range(3):
        c.launch()
    hip.synchronize()
    assert np.array_equal(a, c.dout.download(np.uint32))


@pytest.mark.parametrize("dim,heads,kv_heads,kind", [(64, 4, 2, "e4m3"), (64, 16, 4, "f16"), (128, 4, 4, "e4m3"), (256, 6, 2, "bf16"),
                                                     (256, 12, 2, "e4m3")])
@pytest.mark.parametrize("page", [1, 4, 5, 16, 24, 64])
@pytest.mark.parametrize("rows", [1, 5])
@FAR
def test_page_sizes_of_every_type(gpu, page, dim, heads, kv_heads, kind, rows, far):
    """Pages that a transfer of several tokens fits into, and pages it does not."""
    run([203, 64, 9], [rows, 1, rows], heads, kv_heads, dim, kind, page=page, seed=page + rows, far=far)


@pytest.mark.parametrize("n", [63, 64, 65, 200])
def test_many_sequences(gpu, n):
    """More sequences than a wave has lanes: the search for a workgroup's place goes through them 64 at a time."""
    rng = np.random.default_rng(n)
    run(rng.integers(0, 90, n).tolist(), rng.integers(0, 4, n).tolist(), 4, 2, 128, "f16", seed=n, max_q=3)
    run([0] * (n - 1) + [500], [1] * n, 4, 2, 128, "f16", seed=n)


@pytest.mark.parametrize("page,dim,kind,rows", [(1, 64, "f16", 1), (1, 256, "bf16", 2), (7, 128, "e4m3", 16), (2048, 128, "bf16", 3)])
def test_runs_beyond_one_chunk(gpu, page, dim, kind, rows):
    """So many sequences (of one text: they share its pages) that one workgroup walks more than 2048 tokens of an item: its page
    ids are loaded in turns."""
    c = Case([5000], [rows], 4, 2, dim, kind, page=page, seed=rows, q_scale=1.0, spare_rows=0)
    n, lens = 600, [5000, 4999, 2049, 4097, 4096, 2048, 3001]
    kv = np.asarray([lens[s % 7] for s in range(n)], np.int32)
    dt, dl = hip.to_device(np.tile(c.table, (n, 1))), hip.to_device(kv)
    dq, out = hip.to_device(np.tile(c.q, (n, 1))), hip.DeviceBuffer(4 * n * rows * c.width).fill(0xff)
    L = q8mi.lib()
    scratch = hip.DeviceBuffer(L.q8mi_paged_attention_scratch_bytes(n, rows, 4, 2, dim, 5000)).fill(0xff)
    ok(L.q8mi_paged_attention(dq.ptr, 0, n * rows, c.width, c.pools.ref, dt.ptr, c.wide, dl.ptr, None, n, rows, 4, 5000, c.scale,
                              out.ptr, 0, c.width, scratch.ptr, NULL), "paged_attention")
    hip.synchronize()
    got = out.download(np.uint32).reshape(n, rows, c.width)
    for s in range(7):                      # the sequences of one length agree (a different cut: other roundings) with the first
        c.lens, first = [lens[s]], got[s].view(np.float32)
        c.dout.upload(first)
        c.check()
        rest = got[s::7].view(np.float32)
        assert np.abs(rest - first).max() < 1e-4 and np.isfinite(rest).all()


@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(128, 6, 1, 4), (256, 12, 1, 2), (64, 40, 1, 2), (256, 20, 1, 16)])
@FAR
def test_bad_pages_with_rows_side_by_side(gpu, dim, heads, kv_heads, rows, far):
    c = Case([300, 70], [rows, rows], heads, kv_heads, dim, "f16", page=16, seed=40 + rows, far=far)
    bad = {(0, 1): -1, (0, 9): c.pools.pages, (1, 0): 2 ** 31 - 1}
    for (s, p), v in bad.items():
        c.table[s, p] = v
    c.dt.upload(c.table)
    c.launch()
    hip.synchronize()
    c.check(hidden=lambda s, t: (s, t // 16) in bad)


@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim,heads,kv_heads,rows", [(128, 2, 2, 8), (128, 6, 2, 8), (256, 6, 1, 16), (64, 40, 1, 5)])
@FAR
def test_later_tokens_of_several_rows(gpu, dim, heads, kv_heads, rows, kind, far):
    """Every other new token holds NaN in some elements of key and value: each row is not finite exactly where a token it sees makes
    it so."""
    n = 90
    c = Case([n], [rows], heads, kv_heads, dim, kind, page=32, seed=50 + rows, far=far)
    nan = {"bf16": 0x7fc0, "f16": 0x7e00, "e4m3": 0x7f}[kind]
    for t in range(n - rows + 2, n, 2):        # value elements: those columns of rows from t's own on
        at = c.pools.at(c.table[0, t // 32], t % 32)
        c.pools.host["v"][at[:, t % 5::7]] = nan
        c.v[0][t, :, t % 5::7] = np.nan
    c.pools.host["k"][c.pools.at(c.table[0, (n - 1) // 32], (n - 1) % 32)[:, 3]] = nan
    c.k[0][n - 1, :, 3] = np.nan               # the last key: all of the last row
    c.pools.upload()
    c.launch()
    hip.synchronize()
    got = c.dout.download(np.float32).reshape(c.q_rows, c.so)
    for r in range(rows):
        q = R.act_value(c.q[r, :c.width], c.act).reshape(c.heads, c.dim)
        want, mag, _ = R.attention(q, c.k[0], c.v[0], c.scale, n - rows + r + 1)
        g = got[r, :c.width].reshape(c.heads, c.dim)
        assert np.array_equal(np.isfinite(g), np.isfinite(want)), r
        fine = np.isfinite(want)
        assert not fine.any() or np.abs(g - want)[fine].max() < 1e-4, r


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_rows_beyond_the_bound_hold_nothing_back(gpu, kind):
    """A sequence with more rows than max_q_len: the tokens of the rows that are not computed are seen by nobody, whatever they
    hold."""
    c = Case([200, 33], [60, 20], 4, 2, 128, kind, max_q=3, seed=60)
    for s, n in enumerate([200, 33]):
        for t in range(n - c.rows[s] + 3, n):
            for name in "kv":
                c.pools.host[name][c.pools.at(c.table[s, t // 16], t % 16)] = 0x7f if kind == "e4m3" else 0x7fc0
    c.pools.upload()
    c.launch()
    hip.synchronize()
    c.check()


@FAR
@pytest.mark.parametrize("page", [16, 3])
def test_a_context_behind_4_gib(gpu, page, far):
    """Pages whose bytes lie beyond 32-bit offsets of the pools, through both ways of addressing."""
    c = Case([70], [1], 4, 2, 128, "f16", page=page, seed=70, far=far)
    pages, stride = 40, (1 << 26) + 512 * page       # elements: 128 MiB a page and a little
    values = stride // 16 * 8                        # they lie half a page stride behind the keys
    big = hip.DeviceBuffer(2 * stride * pages)
    for i in range((70 + page - 1) // page):
        for name, off in (("k", 0), ("v", values)):
            src = c.pools.host[name].reshape(c.pools.pages, c.pools.sp)[c.table[0, i]]
            big.upload(src, 2 * ((pages - 1 - i) * stride + off))
        c.table[0, i] = pages - 1 - i
    c.dt.upload(c.table)
    d = c.pools.desc
    d.k, d.v, d.pages, d.stride_page = big.ptr, big.at(2 * values), pages, stride
    c.launch()
    hip.synchronize()
    c.check()
    big.free()


def test_two_calls_at_once(gpu):
    """Two streams, a scratch each."""
    a, b = hip.Stream(), hip.Stream()
    c = Case([3000, 1], [1, 1], 12, 2, 256, seed=80)
    d = Case([700] * 20, [4] * 20, 16, 4, 128, "f16", seed=81)
    hip.synchronize()
    for _ in range(4):
        c.launch(a.handle)
        d.launch(b.handle)
    a.synchronize()
    b.synchronize()
    c.check()
    d.check()


def test_graphs_share_a_scratch(gpu):
    """Two captured calls on one scratch, replayed in turn on one stream."""
    s = hip.Stream()
    c, d = Case([3000, 100], [1, 1], 6, 1, 256, seed=90), Case([500, 1800], [4, 2], 6, 1, 256, seed=91)
    big = max(c, d, key=lambda x: x.scratch_bytes)
    c.scratch = d.scratch = big.scratch
    c.scratch_bytes = d.scratch_bytes = big.scratch_bytes
    graphs = []
    for case in (c, d):
        case.launch(s.handle)
        s.synchronize()
        g = hip.Graph(s)
        with g:
            case.launch(s.handle)
        graphs.append(g)
    for _ in range(3):
        for case in (c, d):
            case.dout.fill(0x5a)
        hip.synchronize()
        for g in graphs:
            g.launch()
        s.synchronize()
        c.check()
        d.check()


@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
def test_small_weights(gpu, kind):
    """Outputs that tokens of very small weight make alone: those of large weight hold zeros there."""
    c = Case([300], [1], 4, 4, 64, kind, seed=100, q_scale=8.0)
    for t in range(300):
        at = c.pools.at(c.table[0, t // 16], t % 16)
        q = R.act_value(c.q[0, :c.width], c.act).reshape(4, 64)
        for h in range(4):
            if c.scale * (c.k[0][:, h] @ q[h]).max() - c.scale * c.k[0][t, h] @ q[h] < 15:
                c.pools.host["v"][at[h, ::2]] = 0
                c.v[0][t, h, ::2] = 0
    c.pools.upload()
    c.launch()
    hip.synchronize()
    c.check()
