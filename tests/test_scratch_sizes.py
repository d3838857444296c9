"""The scratch sizes of the paged attention and the sampler: what the largest call needs is enough for every smaller one.  No GPU needed."""
import itertools

import pytest

import q8mi

HEADS = [(24, 4, 256), (32, 8, 128), (8, 8, 256), (28, 4, 128), (20, 1, 64), (12, 12, 64), (80, 1, 64), (16, 2, 256), (64, 1, 128), (1, 1, 64)]


def attention(n_seqs, max_q_len, max_kv_len, heads):
    return q8mi.lib().q8mi_paged_attention_scratch_bytes(n_seqs, max_q_len, heads[0], heads[1], heads[2], max_kv_len)


@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention_grows_with_every_bound(heads):
    seqs, rows = [1, 2, 3, 5, 8, 17, 48, 128, 1000], [1, 2, 3, 4, 6, 8, 11, 16]
    tokens = [0, 1, 31, 32, 33, 128, 129, 500, 512, 700, 1024, 1536, 1537, 1600, 2048, 6144, 6145, 8000, 24577, 131072, 1 << 20]
    for axis, (a, b, c) in enumerate([(seqs, rows, tokens), (rows, seqs, tokens), (tokens, seqs, rows)]):
        for other in itertools.product(b, c):
            sizes = [attention(*(list(other[:axis]) + [x] + list(other[axis:])), heads) for x in a]
            assert sizes == sorted(sizes), (heads, axis, other, sizes)


def test_attention_one_token_more():
    """Every length of a range, not only chosen ones: one sequence and a few, one row and several."""
    for heads, n, rows in itertools.product(HEADS[:5], (1, 2, 3), (1, 3)):
        sizes = [attention(n, rows, t, heads) for t in range(0, 9000, 7)]
        assert sizes == sorted(sizes), (heads, n, rows)


def test_attention_stays_moderate():
    """No more than what 768 workgroups of four waves of rows leave, whatever the bounds."""
    assert attention(1 << 16, 16, (1 << 31) - 1, (80, 1, 64)) <= 16 + 2 * 768 * 64 * 66 * 4
    assert attention(128, 1, 131072, (24, 4, 256)) <= 16 + 2 * 192 * 64 * 258 * 4


def sampling(batch, vocab):
    return q8mi.lib().q8mi_sample_scratch_bytes(batch, vocab)


@pytest.mark.parametrize("vocab", [1, 1000, 1024, 1025, 15360, 15361, 32000, 50257, 61440, 65536, 151936, 248320, 1 << 20])
def test_sampling_grows_with_the_batch(vocab):
    sizes = [sampling(b, vocab) for b in list(range(1, 600)) + [1000, 4096, 65535]]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("batch", [1, 2, 7, 16, 17, 64, 300, 1000, 65535])
def test_sampling_grows_with_the_vocabulary(batch):
    sizes = [sampling(batch, v) for v in range(1, (1 << 20) + 1, 511)] + [sampling(batch, 1 << 20)]
    assert sizes == sorted(sizes)
