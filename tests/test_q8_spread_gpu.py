"""Cached values whose sizes are far apart: what a query does not see, or hardly
weighs, leaves the rest of its result as exact as it is without.

Tolerances as in test_q8_edges_gpu: of a weighted sum of magnitudes, token by
token and head by head.
"""
import numpy as np
import pytest

from test_q8_edges_gpu import check_rows
from test_q8_gpu import ALL, gpu, make, rnd, stored, tree, turned

pytestmark = pytest.mark.gpu
BIG = np.float32(1e12)


@pytest.mark.parametrize("shape,n", [("l8b", 2), ("mha128", 8), ("g8_64", 1), ("l8b", 40), ("tl", 128), ("mha64", 70)])
@pytest.mark.parametrize("rows", [0, 90, 1000])
def test_a_large_sibling_changes_nothing(cuda, shape, n, rows):
    rng = np.random.default_rng(60)
    h, kv, hd = ALL[shape]
    with make(shape, rows + n) as ctx:
        k0, v0 = rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
        if rows:
            ctx.kv_write(0, 0, 0, k0, v0)
        q, k, v = rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
        v[n // 2] *= BIG
        par = tree(rng, n, "roots")
        out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par)


@pytest.mark.parametrize("shape,n", [("l8b", 2), ("mha128", 5), ("l8b", 33), ("l70b", 16), ("mha64", 200), ("tl", 150)])
@pytest.mark.parametrize("rows", [0, 200])
def test_a_large_last_token_changes_nothing_before_it(cuda, shape, n, rows):
    rng = np.random.default_rng(61)
    h, kv, hd = ALL[shape]
    with make(shape, rows + n) as ctx:
        k0, v0 = rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
        if rows:
            ctx.kv_write(0, 0, 0, k0, v0)
        q, k, v = rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
        v[n - 1] *= BIG
        out = ctx.prefill_packed(0, [0], [rows], [n], *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v)


@pytest.mark.parametrize("shape,most", [("l8b", 2), ("mha128", 8), ("g8_64", 1)])
def test_large_siblings_in_small_trees_of_many_sequences(cuda, shape, most):
    rng = np.random.default_rng(62)
    h, kv, hd = ALL[shape]
    n = 60 if shape != "g8_64" else 160
    rows = rng.integers(20, 400, n)
    lens = rng.integers(1, most + 1, n)
    with make(shape, 500, max_batch=n) as ctx:
        k0, v0 = rnd(rng, 400, kv, hd), rnd(rng, 400, kv, hd)
        dev = gpu(k0, v0)
        for s in range(n):
            ctx.kv_write(s, 0, 0, *(x[:rows[s]].contiguous() for x in dev))
        t = int(lens.sum())
        q, k, v = rnd(rng, t, h, hd), rnd(rng, t, kv, hd), rnd(rng, t, kv, hd)
        first = np.concatenate([[0], np.cumsum(lens)])
        v[first[:-1][lens > 1]] *= BIG
        par = np.concatenate([tree(rng, x, "roots") for x in lens])
        out = ctx.decode_tree(0, np.arange(n), rows, lens, par, *gpu(q, k, v)).cpu().numpy()
        kc, vc = stored(k0), stored(v0)
        for s in range(n):
            r = slice(first[s], first[s + 1])
            check_rows(ctx, out[r], kc[:rows[s]], vc[:rows[s]], q[r], k[r], v[r], par[r])


def scored(ctx, rng, n, rows, at, big, score):
    """A query shared by all heads and n nodes without parents, and cached rows of
    which those in `at` score `score` and have values `big` times as large."""
    h, kv, hd = ctx.n_heads, ctx.n_kv_heads, ctx.head_dim
    u = rnd(rng, 1, 1, hd)
    way = turned(u, ctx.rope_cos[rows:rows + 1], ctx.rope_sin[rows:rows + 1], False)[0, 0]
    k0, v0 = 0.3 * rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd)
    k0[at] = (way * score * np.sqrt(hd) / (way @ way)).astype(np.float32)
    v0[at] *= np.float32(big)
    k, v = 0.3 * rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)
    return np.broadcast_to(u, (n, h, hd)).copy(), k, v, k0, v0


@pytest.mark.parametrize("shape,n", [("l8b", 1), ("g2_64", 2), ("mha128", 8), ("l8b", 16), ("mha64", 100)])
@pytest.mark.parametrize("at", [[3], [700], [0, 130, 131, 640, 998], list(range(512, 640))])
def test_large_values_of_little_weight(cuda, shape, n, at):
    """A weight of e^-45 on values 1e12 times the others': 1e-8 of the result at
    most, while an absolute error next to the large ones would be all of it."""
    rng = np.random.default_rng(63)
    rows = 1000
    with make(shape, rows + n) as ctx:
        q, k, v, k0, v0 = scored(ctx, rng, n, rows, at, BIG, -45)
        ctx.kv_write(0, 0, 0, k0, v0)
        par = tree(rng, n, "roots")
        out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par, terms=45)


@pytest.mark.parametrize("shape,n", [("l8b", 1), ("g2_64", 2), ("mha128", 8), ("l8b", 16), ("mha64", 100)])
@pytest.mark.parametrize("at", [[0], [999], [300, 301]])
@pytest.mark.parametrize("size", [0, 1e-9])
def test_a_sink_without_a_value(cuda, shape, n, at, size):
    """Nearly all weight on a row of zeros, or next to it: the others decide."""
    rng = np.random.default_rng(64)
    rows = 1000
    with make(shape, rows + n) as ctx:
        q, k, v, k0, v0 = scored(ctx, rng, n, rows, at, size, 28)
        ctx.kv_write(0, 0, 0, k0, v0)
        par = tree(rng, n, "roots")
        out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par, terms=28)


def test_decode_of_many_with_large_values_of_little_weight(cuda):
    rng = np.random.default_rng(65)
    n, rows = 64, 1000
    with make("l8b", rows + 1, max_batch=n) as ctx:
        for size, score in ((BIG, -45), (0, 28)):
            q, k, v, k0, v0 = scored(ctx, rng, 1, rows, [5, 444, 990], size, score)
            dev = gpu(k0, v0)
            for s in range(n):
                ctx.kv_write(s, 0, 0, *dev)
            out = ctx.decode_batched(0, np.arange(n), np.full(n, rows), *gpu(*(np.repeat(x, n, 0) for x in (q, k, v))))
            out = out.cpu().numpy()
            for s in range(0, n, 9):
                check_rows(ctx, out[s:s + 1], stored(k0), stored(v0), q, k, v, terms=45)


@pytest.mark.parametrize("size", [1e-35, 1e-20, 1e20, 1e36])
@pytest.mark.parametrize("shape,n", [("l8b", 1), ("mha128", 8), ("l8b", 40), ("tl", 128)])
def test_values_all_tiny_or_all_large(cuda, shape, n, size):
    rng = np.random.default_rng(66)
    h, kv, hd = ALL[shape]
    rows = 400
    with make(shape, rows + n) as ctx:
        k0, v0 = rnd(rng, rows, kv, hd), rnd(rng, rows, kv, hd) * np.float32(size)
        ctx.kv_write(0, 0, 0, k0, v0)
        q, k, v = rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd) * np.float32(size)
        par = tree(rng, n)
        out = ctx.decode_tree(0, [0], [rows], [n], par, *gpu(q, k, v)).cpu().numpy()
        check_rows(ctx, out, stored(k0), stored(v0), q, k, v, par)
