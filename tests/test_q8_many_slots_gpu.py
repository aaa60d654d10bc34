"""Contexts of more than 1024 slots, and lists of many sequences without tokens."""
import numpy as np
import pytest

from leap_b200 import LeapError
from test_q8_gpu import Ragged, gpu, make, tree

pytestmark = pytest.mark.gpu


def test_slots_past_1024(cuda):
    rng = np.random.default_rng(90)
    with make("g2_64", 40, max_batch=1500) as ctx:
        slots = [1499, 0, 1024, 1023, 64]
        lens = [3, 1, 17, 0, 9]
        r = Ragged(ctx, rng, slots, [20, 0, 11, 5, 30])
        q, k, v = r.inputs(lens)
        par = np.concatenate([tree(rng, n) for n in lens])
        r.check(ctx.decode_tree(0, r.slots, r.rows, lens, par, *gpu(q, k, v)), q, k, v, lens, par)
        for bad in ([1499, 1499], [1500, 0], [3, -1]):
            with pytest.raises(LeapError, match="slot"):
                ctx.prefill_packed(0, bad, [0, 0], [1, 1], *gpu(*r.inputs([1, 1])))


@pytest.mark.parametrize("last", [0, 2, 40])
def test_many_sequences_without_tokens(cuda, last):
    """Launches that have nothing to do, and sequences without tokens at every end."""
    rng = np.random.default_rng(91)
    n = 400
    lens = [0] * n
    lens[130], lens[256], lens[399] = 3, 20, last
    with make("g2_64", 70, max_batch=n) as ctx:
        r = Ragged(ctx, rng, rng.permutation(n), [0] * 100 + [24] * 300)
        q, k, v = r.inputs(lens)
        r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)
        q, k, v = r.inputs([0] * n)
        assert ctx.prefill_packed(0, r.slots, r.rows, [0] * n, *gpu(q, k, v)).shape[0] == 0
        ctx.kv_keep(r.slots, r.rows, [0] * 399 + [1], [3])
