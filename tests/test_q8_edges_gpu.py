"""Rows of the 8-bit KV cache that reach far into a query's result or not at
all: infinities and NaN that one part of a split range holds alone, and rows
whose size has nothing to do with that of the rows beside them.

Outputs are compared token by token and head by head.  A score whose terms'
magnitudes sum to S is off by S * (2^-22 + 16 * 2^-23) at most (see
test_q8_gpu; S is about 7 for N(0,1) inputs), a weight by as much of itself and
3e-5 for the split of p * s_v and the FP32 sums, so an output is off by no more
than that of the same sum with every value's magnitude in its place (in its
largest dim: the split's absolute error is relative to a row's largest code).
"""
import numpy as np
import pytest

from test_q8_gpu import ALL, attend, gpu, make, rnd, stored, tree, turned

pytestmark = pytest.mark.gpu


def check_rows(ctx, out, kc, vc, q, k, v, parents=None, terms=7):
    """One sequence's outputs: NaN where the definition says so, the rest near."""
    tol = terms * (2.0 ** -22 + 16 * 2.0 ** -23) + 3e-5
    with np.errstate(invalid="ignore"):
        ref, _, _ = attend(ctx, kc, vc, q, k, v, parents)
        mag, _, _ = attend(ctx, kc, np.abs(vc), q, k, np.abs(v), parents)
    out = np.asarray(out, np.float64)
    bad = np.isnan(ref)
    np.testing.assert_array_equal(np.isnan(out), bad)
    for t in range(ref.shape[0]):
        for h in range(ref.shape[1]):
            ok = ~bad[t, h]
            if ok.any():
                worst = np.abs(out[t, h, ok] - ref[t, h, ok]).max()
                assert worst <= tol * mag[t, h, ok].max(), (t, h, worst, mag[t, h, ok].max())


# ---- infinities and NaN alone in a part ----------------------------------------------
@pytest.mark.parametrize("shape,rows", [("l8b", 512), ("l8b", 1024), ("g8_64", 992)])
def test_decode_of_many_with_a_bad_new_key(cuda, shape, rows):
    """The new row is alone in its tile, which begins a part for some of them."""
    rng = np.random.default_rng(50)
    h, kv, hd = ALL[shape]
    n = 64 if shape == "l8b" else 160
    with make(shape, rows + 1, max_batch=n) as ctx:
        base = rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
        dev = gpu(*base)
        for s in range(n):
            ctx.kv_write(s, 0, 0, *dev)
        q, k, v = rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
        for s in range(n):  # one kv head of every sequence, the heads in turn
            k[s, s % kv, s % hd] = (np.inf, -np.inf, np.nan)[s % 3]
        out = ctx.decode_batched(0, np.arange(n), np.full(n, rows), *gpu(q, k, v)).cpu().numpy()
        kc, vc = stored(base[0]), stored(base[1])
        g = h // kv
        for s in range(n):
            assert np.isnan(out[s, s % kv * g:(s % kv + 1) * g]).all(), s
        for s in range(0, n, 9):
            check_rows(ctx, out[s:s + 1], kc, vc, q[s:s + 1], k[s:s + 1], v[s:s + 1])


def test_decode_of_long_contexts_with_a_bad_new_key(cuda):
    rng = np.random.default_rng(51)
    h, kv, hd = ALL["l8b"]
    n, rows = 16, 8192
    with make("l8b", rows + 1, max_batch=n) as ctx:
        dev = gpu(rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd))
        for s in range(n):
            ctx.kv_write(s, 0, 0, *dev)
        q, k, v = rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
        k[:, :, 5] = np.inf
        out = ctx.decode_batched(0, np.arange(n), np.full(n, rows), *gpu(q, k, v)).cpu().numpy()
        assert np.isnan(out).all()


@pytest.mark.parametrize("shape", ["l8b", "tl", "l70b"])
@pytest.mark.parametrize("bad", [1, 200])
def test_decode_with_the_last_rows_bad(cuda, shape, bad):
    """The last split of a sequence holds `bad` cached rows and the new one, or
    some of them, and they are all it holds."""
    rng = np.random.default_rng(52)
    h, kv, hd = ALL[shape]
    for rows in (129, 257, 513, 1025, 2049):
        bad_here = min(bad, rows - 1)
        with make(shape, rows + 1) as ctx:
            k0, v0 = rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
            k0[rows - bad_here:, 1, 3] = np.nan
            ctx.kv_write(0, 0, 0, k0, v0)
            q, k, v = rnd(rng, 1, h, hd), rnd(rng, 1, kv, hd), rnd(rng, 1, kv, hd)
            k[0, 1, 7] = np.inf
            out = ctx.decode_batched(0, [0], [rows], *gpu(q, k, v)).cpu().numpy()
            check_rows(ctx, out, stored(k0), stored(v0), q, k, v)


@pytest.mark.parametrize("shape,n", [("l8b", 1), ("l8b", 2), ("l8b", 40), ("mha128", 40)])
def test_bad_value_whose_weight_vanishes(cuda, shape, n):
    """A NaN in V of a row that scores 100 below the others, in another split: its
    weight underflows, and NaN times nothing is still NaN."""
    rng = np.random.default_rng(53)
    h, kv, hd = ALL[shape]
    rows = 2048
    with make(shape, rows + n) as ctx:
        u = rnd(rng, 1, 1, hd)
        q = np.broadcast_to(u, (n, h, hd)).copy()
        way = turned(u, ctx.rope_cos[rows:rows + 1], ctx.rope_sin[rows:rows + 1], False)[0, 0]
        k0, v0 = 0.01 * rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
        k0[1024:] += (way * 50 * np.sqrt(hd) / (way @ way)).astype(np.float32)
        k0[:1024] -= (way * 50 * np.sqrt(hd) / (way @ way)).astype(np.float32)
        v0[100, 1, 2] = np.nan
        ctx.kv_write(0, 0, 0, k0, v0)
        k, v = 0.01 * rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
        par = tree(rng, n, "roots")
        out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par, terms=50)
        assert np.isnan(out[:, h // kv:2 * (h // kv)]).all()


@pytest.mark.parametrize("size", [1e30, 1e33, 1e36])
@pytest.mark.parametrize("shape,n", [("l8b", 1), ("l8b", 2), ("l8b", 40), ("mha64", 120), ("tl", 3)])
def test_keys_far_beyond_the_others(cuda, shape, n, size):
    """Scores that FP32 holds (up to 1e38 here) take all the weight, or none."""
    rng = np.random.default_rng(54)
    h, kv, hd = ALL[shape]
    rows = 300
    with make(shape, rows + n) as ctx:
        k0, v0 = rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
        k0[77] *= np.float32(size)
        ctx.kv_write(0, 0, 0, k0, v0)
        q, k, v = rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
        par = tree(rng, n)
        out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par)


@pytest.mark.parametrize("shape,n", [("l8b", 2), ("l8b", 40), ("mha64", 120)])
def test_small_keys_under_large_queries(cuda, shape, n):
    """Scores of ordinary size from factors that are not."""
    rng = np.random.default_rng(55)
    h, kv, hd = ALL[shape]
    rows = 300
    for up in (1e25, 1e-25):
        with make(shape, rows + n) as ctx:
            down = np.float32(1 / up)
            k0, v0 = rnd(rng, rows, kv, hd) * down, rnd(rng, rows, kv, hd)
            ctx.kv_write(0, 0, 0, k0, v0)
            q, k, v = rnd(rng, n, h, hd) * np.float32(up), rnd(rng, n, kv, hd) * down, rnd(rng, n, kv, hd)
            par = tree(rng, n)
            out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
            check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par)
