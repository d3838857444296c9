"""Sampling where top_k asks for more logits than can be drawn: fewer lie within reach of the maximum (about 30 temperatures), or
fewer are numbers.  Nothing is cut then, and no element is listed as a candidate."""
import numpy as np
import pytest

from test_gpu_sample import logits, run

pytestmark = pytest.mark.gpu


def within(z, temperature):
    return ((z.max(1, keepdims=True) - z) / temperature < 30).sum(1)


@pytest.mark.parametrize("vocab,k,temperature", [(100000, 400, 0.3), (248320, 1000, 0.3), (3000, 200, 0.1), (32003, 129, 0.05), (300000, 1172, 0.2)])
def test_fewer_within_reach_than_top_k(gpu, vocab, k, temperature):
    z = logits(6, vocab, vocab)
    assert (within(z, temperature) < k).all()
    run(z, temperature=temperature, top_k=k, u=[0.0, 0.2, 0.5, 0.8, 0.999, 1 - 2.0 ** -24])
    run(z, temperature=temperature, top_k=k, min_p=[0.0, 0.01, 0.1, 0.5, 1.0, 0.0], seed=vocab)
    run(z, temperature=temperature, top_k=k, top_p=[1.0, 0.9, 0.5, 0.99, 0.0, 1.0], seed=k)


@pytest.mark.parametrize("vocab", [5, 1000, 3000, 100000])
@pytest.mark.parametrize("allowed", [1, 2, 4])
def test_fewer_allowed_than_top_k(gpu, vocab, allowed):
    """Masked decoding: -inf everywhere but at a few tokens, top_k about the usual."""
    rng = np.random.default_rng(vocab + allowed)
    z = np.full((8, vocab), -np.inf)
    for r in range(8):
        z[r, rng.choice(vocab, allowed, replace=False)] = rng.standard_normal(allowed)
    run(z, temperature=0.8, top_k=[2, 3, 4, 5, 20, 50, 400, 100000], seed=allowed)
    run(z, temperature=0.8, top_k=[2, 3, 4, 5, 20, 50, 400, 100000], top_p=0.9, min_p=0.05, seed=allowed)


def test_rows_with_and_without_a_cut_within_reach(gpu):
    z = logits(64, 50000, 3)
    run(z, temperature=np.tile([0.2, 5.0], 32), top_k=np.repeat([300, 1000], 32), seed=4)
