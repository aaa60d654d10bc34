"""A context bound to a stream that is not the current one."""
import numpy as np
import pytest
import torch

from leap_b200 import AttentionContext
from test_q8_gpu import ALL, Ragged, gpu, make, near, attend, rnd, stored, tree

pytestmark = pytest.mark.gpu


def stream_of(t):
    """The stream whose pool a tensor's memory comes from."""
    p = t.untyped_storage().data_ptr()
    at = [s for s in torch.cuda.memory_snapshot() if s["address"] <= p < s["address"] + s["total_size"]]
    assert len(at) == 1
    return at[0]["stream"]


@pytest.mark.parametrize("kv", ["f32", "q8"])
def test_returned_tensors_belong_to_the_bound_stream(cuda, kv):
    """Memory of another stream's pool may still be read by what is queued there."""
    h, n_kv, hd = ALL["l8b"]
    rng = np.random.default_rng(70)
    s = torch.cuda.Stream()
    with AttentionContext(1, h, n_kv, hd, 64, max_batch=2, kv=kv) as ctx:
        q, k, v = gpu(rnd(rng, 3, h, hd), rnd(rng, 3, n_kv, hd), rnd(rng, 3, n_kv, hd))
        torch.cuda.synchronize()
        ctx.bind_torch_stream(s)
        got = [ctx.prefill(0, 0, 0, q, k, v), ctx.prefill_packed(0, [1], [0], [3], q, k, v),
               ctx.decode(0, 3, q[0], k[0], v[0]), ctx.decode_batched(0, [0, 1], [4, 3], q[:2], k[:2], v[:2]),
               *ctx.kv_read_packed(0, [1, 0], [0, 0], [3, 4])]
        if kv == "q8":
            got += [ctx.decode_tree(0, [0], [5], [3], [-1, 0, 0], q, k, v), *ctx.kv_read_device(0, 0, 0, 4)]
        assert [stream_of(t) for t in got] == [s.cuda_stream] * len(got)
        s.synchronize()
        np.testing.assert_array_equal(got[4][:3].cpu(), got[4][3:6].cpu())


def test_results_with_work_queued_on_the_current_stream(cuda):
    rng = np.random.default_rng(71)
    s = torch.cuda.Stream()
    with make("l8b", 700) as ctx:
        r = Ragged(ctx, rng, [0], [600])
        q, k, v = r.inputs([20])
        x, par = gpu(q, k, v), tree(rng, 20)
        torch.cuda.synchronize()
        ctx.bind_torch_stream(s)
        out = ctx.decode_tree(0, [0], [600], [20], par, *x)
        kk, _ = ctx.kv_read_packed(0, [0], [0], [600])
        s.synchronize()
        near(out.cpu().numpy(), attend(ctx, r.k[0], r.v[0], q, k, v, par)[0])
        np.testing.assert_array_equal(kk.cpu().numpy(), r.k[0])


def test_rows_read_on_the_contexts_own_stream(cuda):
    rng = np.random.default_rng(72)
    with make("l8b", 100, bind_torch_stream=False) as ctx:
        x = rnd(rng, 50, 8, 128)
        ctx.kv_write(0, 0, 0, x, x)
        k, v = ctx.kv_read_packed(0, [0], [0], [50])
        ctx.sync()
        np.testing.assert_array_equal(k.cpu().numpy(), stored(x))
        np.testing.assert_array_equal(v.cpu().numpy(), stored(x))
