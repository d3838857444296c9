"""A scratch that was sized once, for the largest call that a program makes, serves the smaller ones: results and the bytes behind
the scratch."""
import pytest

import q8mi
import test_gpu_paged_attention as attention
import test_gpu_sample as sampling
from q8mi import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim", [(24, 4, 256), (32, 8, 128), (20, 1, 64)])
def test_attention(gpu, heads, kv_heads, dim):
    """One sequence of any length up to the bound, then fewer sequences and rows than the bound."""
    L = q8mi.lib()
    n = L.q8mi_paged_attention_scratch_bytes(3, 4, heads, kv_heads, dim, 20000)
    scratch = hip.DeviceBuffer(n + 64)
    for i, (lens, rows) in enumerate([([1536], [1]), ([700, 700], [1, 1]), ([700] * 3, [1] * 3), ([512], [2]), ([33], [4]), ([6100], [1]),
                                      ([20000], [1]), ([1600, 5], [4, 1]), ([3000, 40, 900], [1, 4, 2])]):
        c = attention.Case(lens, rows, heads, kv_heads, dim, "f16", page=32, seed=i)
        assert c.scratch_bytes <= n, (lens, rows)     # nothing is launched on a scratch that is too small
        c.scratch, c.scratch_bytes = scratch.fill(0xff), n
        c.launch()
        hip.synchronize()
        c.check()


@pytest.mark.parametrize("most,vocab", [(32, 32000), (21, 50257), (18, 61440), (16, 65536)])
def test_sampling(gpu, most, vocab):
    """A batch from which sequences drop out, and a smaller vocabulary."""
    n = q8mi.lib().q8mi_sample_scratch_bytes(most, vocab)
    scratch = hip.DeviceBuffer(n + 64)
    for batch, v in ((most, vocab), (most - 1, vocab), (most // 2, vocab), (1, vocab), (most, vocab - 1025), (most, 1000)):
        c = sampling.Case(sampling.logits(batch, v, batch + v), temperature=0.9, top_k=[0, 40, 500, 0][batch % 4], top_p=0.9, seed=v)
        assert c.bytes <= n, (batch, v)               # nothing is launched on a scratch that is too small
        c.scratch, c.bytes = scratch.fill(0xff), n
        c.launch()
        hip.synchronize()
        c.check()
