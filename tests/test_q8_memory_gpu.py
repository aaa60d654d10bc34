"""What an 8-bit context takes on the device: its cache, and scratch for no more
splits than it can have."""
import numpy as np
import pytest

from test_q8_gpu import ALL, Ragged, gpu, make, rnd, stored, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,max_seq,max_batch", [("l8b", 64, 1), ("g2_64", 1, 1), ("mha64", 129, 3), ("tl", 1000, 1)])
def test_a_small_context_is_small(cuda, shape, max_seq, max_batch):
    h, kv, hd = ALL[shape]
    with make(shape, max_seq, max_batch=max_batch) as ctx:
        rows = 2 * max_batch * kv * ((max_seq + 127) // 128 * 128)
        cache = rows * (hd + 4)
        # rows staged from the host, two partials a warp (a warp has two tiles of 32 rows
        # at least), partials of every query tile and key tile of 128, and 64 KB
        tiles, pairs = (max_seq + 31) // 32 + 1, (max_seq + 127) // 128 * ((max_seq * h // kv + 127) // 128)
        scratch = 8 * min(max_seq, 1024) * kv * hd + max_batch * kv * (tiles + 1) * 32 * (hd + 2) + \
            max_batch * kv * pairs * 512 * (hd + 2)
        rope = 2 * 4 * max_seq * hd // 2
        assert ctx.device_bytes() <= cache + scratch + rope + 65536


@pytest.mark.parametrize("shape", ["l8b", "tl", "mha64"])
@pytest.mark.parametrize("max_seq,max_batch", [(33, 1), (129, 2), (300, 1), (1100, 3)])
def test_every_kind_of_call_at_the_last_rows(cuda, shape, max_seq, max_batch):
    rng = np.random.default_rng(80)
    for n in (1, 2, 9, 30):
        with make(shape, max_seq, max_batch=max_batch) as ctx:
            x = rnd(rng, max_seq, ctx.n_kv_heads, ctx.head_dim)
            ctx.kv_write(0, 0, 0, x, x)
            np.testing.assert_array_equal(ctx.kv_read(0, 0, 0, max_seq)[0], stored(x))
            r = Ragged(ctx, rng, np.arange(max_batch), [max_seq - n] * max_batch)
            lens = [n] * max_batch
            q, k, v = r.inputs(lens)
            if n == 1:
                r.check(ctx.decode_batched(0, r.slots, r.rows, *gpu(q, k, v)), q, k, v, lens)
            elif n == 9:
                r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)
            else:
                par = np.concatenate([tree(rng, n) for _ in lens])
                r.check(ctx.decode_tree(0, r.slots, r.rows, lens, par, *gpu(q, k, v)), q, k, v, lens, par)
