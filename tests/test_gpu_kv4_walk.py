"""Batches of many short entries: a block's ring runs over dozens of units, some of a
single stage, and the producer steps from unit to unit while earlier ones are scored."""
import numpy as np
import pytest

from test_gpu_kv4 import check_attention, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,heads,kv,d", [(1, 8, 4, 32), (1, 4, 4, 128), (5, 4, 2, 64), (6, 8, 2, 128), (20, 4, 1, 32)])
@pytest.mark.parametrize("batch", [150, 700])
def test_many_short_entries(mri, gpu_ctx, tokens, heads, kv, d, batch):
    rng = np.random.default_rng(batch + tokens)
    cache, k, v = filled(mri, rng, batch, kv, d, 128)
    lens = rng.choice([0, 1, 31, 32, 33, 63, 64, 65, 96, 127, 128], batch)
    q = rng.normal(0, 2, (batch, tokens, heads, d)).astype(np.float32)
    got = [check_attention(mri, cache, k, v, q, lens, track=track) for track in (False, True)]
    assert np.array_equal(*got)
