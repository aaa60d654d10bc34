"""The 8-bit KV cache and what reads it (decode, drafted trees, packed
prompts), on the GPU against the definition in 64 bits.

Stored rows are compared bit by bit.  Attention: codes are exact in FP16, q and
the weights are carried as two FP16 (22 bits, 2^-22 relative at most), products
are summed in FP32 over at most 16 steps before they join an FP32 sum.  A score
of N(0,1) inputs (|terms| sum to about 0.64 sqrt(hd), 7 for hd 128) is so off by
at most 7 * (2^-22 + 16 * 2^-23) < 2e-5, and an output by no more, relative to
the largest value (MAX_TOL, with room for the sum over keys); errors of
different terms are independent, which leaves less than a tenth of that in the
2-norm (NORM_TOL).
"""
import ctypes

import numpy as np
import pytest
import torch

from cases import SHAPES
from leap_b200 import AttentionContext, LeapError, ModelConfig, Transformer

pytestmark = pytest.mark.gpu
MAX_TOL, NORM_TOL = 5e-5, 4e-6
HEADS = ["l8b", "tl", "l70b", "mha128", "g2_64", "mha64", "g8_64", "g2_128"]
ALL = dict(SHAPES, mha64=(4, 4, 64), g8_64=(16, 2, 64), g2_128=(4, 2, 128))


# ---- the definition ----------------------------------------------------------
def stored(x):
    """What the cache gives back for FP32 rows x[..., hd] (FP32)."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    y = np.where(np.isfinite(x), x, 0).astype(np.float32)
    s = np.abs(y).max(-1) * (np.float32(1.0) / np.float32(127.0))
    s64 = np.where(s > 0, s, 1.0).astype(np.float64)[..., None]
    c = np.clip(np.rint(y.astype(np.float64) / s64), -127, 127)
    out = (c * s[..., None].astype(np.float64)).astype(np.float32)
    out[s == 0] = 0
    out[bad] = np.nan
    return out


def turned(x, c, s, f32):
    """Interleaved pairs turned by (c, s) [tokens, hd/2]; f32: every product and
    sum rounded, as rows are before they are stored."""
    a, b = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    c, s = c[:, None].astype(np.float64), s[:, None].astype(np.float64)
    r = np.float32 if f32 else np.float64
    lo = (a * c).astype(r).astype(np.float64) - (b * s).astype(r).astype(np.float64)
    hi = (b * c).astype(r).astype(np.float64) + (a * s).astype(r).astype(np.float64)
    return np.stack([lo, hi], -1).reshape(x.shape).astype(r)


def attend(ctx, kc, vc, q, k, v, parents=None):
    """One sequence: rows kc, vc [n, kv, hd] as stored, then the run q, k, v.
    Returns the outputs in 64 bits and the run's stored rows."""
    n, t = len(kc), len(q)
    h, kv, hd = ctx.n_heads, ctx.n_kv_heads, ctx.head_dim
    sees, depth = np.tril(np.ones((t, t), bool)), np.arange(t)
    if parents is not None:
        sees, depth = np.eye(t, dtype=bool), np.zeros(t, int)
        for i, p in enumerate(parents):
            if p >= 0:
                sees[i] |= sees[p]
                depth[i] = depth[p] + 1
    c, s = ctx.rope_cos[n + depth], ctx.rope_sin[n + depth]
    kn, vn = stored(turned(k, c, s, True)), stored(v)
    qr = turned(q, c, s, False)
    keys, vals = np.concatenate([kc, kn]).astype(np.float64), np.concatenate([vc, vn]).astype(np.float64)
    vis = np.concatenate([np.ones((t, n), bool), sees], 1)
    out = np.empty((t, h, hd))
    for a in range(h if t else 0):
        sc = qr[:, a] @ keys[:, a // (h // kv)].T / np.sqrt(hd)
        for i in range(t):  # a row that is not seen takes no part, whatever it holds
            e = sc[i, vis[i]]
            p = np.exp(e - e.max())
            out[i, a] = p @ vals[vis[i], a // (h // kv)] / p.sum()
    return out, kn, vn


def near(got, ref):
    got, ref = np.asarray(got, np.float64), np.asarray(ref)
    if ref.size == 0:
        return
    assert np.abs(got - ref).max() <= MAX_TOL * np.abs(ref).max()
    assert np.linalg.norm(got - ref) <= NORM_TOL * np.linalg.norm(ref)


def rnd(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32)


def gpu(*xs):
    return [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in xs]


def make(shape, max_seq, **kw):
    h, kv, hd = ALL[shape]
    return AttentionContext(kw.pop("n_layers", 1), h, kv, hd, max_seq, kv="q8", **kw)


class Ragged:
    """Sequences in slots of one context, their rows mirrored on the host."""

    def __init__(self, ctx, rng, slots, rows, layer=0):
        self.ctx, self.rng, self.layer = ctx, rng, layer
        self.slots, self.rows = np.array(slots, np.int32), np.array(rows, np.int32)
        self.k, self.v = [], []
        for s, n in zip(self.slots, self.rows):
            k, v = rnd(rng, n, ctx.n_kv_heads, ctx.head_dim), rnd(rng, n, ctx.n_kv_heads, ctx.head_dim)
            if n:
                ctx.kv_write(int(s), layer, 0, k, v)
            self.k.append(stored(k))
            self.v.append(stored(v))

    def inputs(self, lens):
        c, t = self.ctx, int(sum(lens))
        return rnd(self.rng, t, c.n_heads, c.head_dim), rnd(self.rng, t, c.n_kv_heads, c.head_dim), \
            rnd(self.rng, t, c.n_kv_heads, c.head_dim)

    def check(self, out, q, k, v, lens, parents=None):
        """Outputs and appended rows; the mirror takes the rows on."""
        out, at = out.cpu().numpy(), 0
        for i, n in enumerate(lens):
            r = slice(at, at + n)
            ref, kn, vn = attend(self.ctx, self.k[i], self.v[i], q[r], k[r], v[r],
                                 None if parents is None else parents[r])
            near(out[r], ref)
            kk, vv = self.ctx.kv_read(int(self.slots[i]), self.layer, 0, len(self.k[i]) + n)
            self.k[i], self.v[i] = np.concatenate([self.k[i], kn]), np.concatenate([self.v[i], vn])
            np.testing.assert_array_equal(kk, self.k[i])
            np.testing.assert_array_equal(vv, self.v[i])
            at += n
        self.rows = self.rows + np.array(lens, np.int32)


def tree(rng, n, kind="random"):
    if kind == "chain":
        return np.arange(-1, n - 1, dtype=np.int32)
    if kind == "star":
        return np.array([-1] + [0] * (n - 1), np.int32)
    if kind == "roots":
        return np.full(n, -1, np.int32)
    return np.array([-1 if i == 0 or rng.random() < 0.15 else rng.integers(0, i) for i in range(n)], np.int32)


# ---- rows in and out ------------------------------------------------------------
@pytest.mark.parametrize("shape", ["l8b", "tl", "mha64", "g2_128"])
@pytest.mark.parametrize("pos0,n", [(0, 1), (3, 1), (5, 29), (0, 64), (1, 333), (700, 1300)])
def test_rows_in_and_out(cuda, shape, pos0, n):
    rng = np.random.default_rng(n)
    h, kv, hd = ALL[shape]
    k, v = rnd(rng, n, kv, hd) * 10 ** rng.uniform(-3, 3, (n, kv, 1)).astype(np.float32), rnd(rng, n, kv, hd)
    with make(shape, 2001, max_batch=3, n_layers=2) as ctx:
        ctx.kv_write(1, 1, pos0, k, v)            # from the host
        for got, x in zip(ctx.kv_read(1, 1, pos0, n), (k, v)):
            np.testing.assert_array_equal(got, stored(x))
        ctx.kv_write(2, 0, pos0, *gpu(v, k))      # from the device
        for got, x in zip(ctx.kv_read_device(2, 0, pos0, n), (v, k)):
            np.testing.assert_array_equal(got.cpu().numpy(), stored(x))
        # nothing else was touched
        for slot, layer in ((0, 0), (1, 0), (2, 1)):
            kk, vv = ctx.kv_read(slot, layer, 0, 2001)
            assert not kk.any() and not vv.any()
        kk, vv = ctx.kv_read(1, 1, 0, 2001)
        assert not kk[:pos0].any() and not kk[pos0 + n:].any() and not vv[pos0 + n:].any()
        ctx.clear_kv_cache()
        kk, vv = ctx.kv_read(1, 1, 0, 2001)
        assert not kk.any() and not vv.any()


@pytest.mark.parametrize("shape", ["l8b", "tl"])
def test_rows_at_the_edges_of_the_format(cuda, shape):
    """Ties, zeros, one large value, tiny and huge rows, infinities and NaN."""
    h, kv, hd = ALL[shape]
    rng = np.random.default_rng(0)
    x = rnd(rng, 64, kv, hd)
    x[0] = 0
    x[1] = 0
    x[1, :, 5] = -3
    x[2] = (np.arange(hd) - 63.5)                 # halves ...
    x[2, :, 0] = 127                              # ... of a scale of 1 (or next to it)
    x[3] = np.where(np.arange(hd) % 2, 126.5, 0.5) * np.float32(2.0 ** -20)
    x[3, :, 0] = 127 * 2.0 ** -20
    x[4] *= np.float32(2.0 ** 120)
    x[5] = np.float32(3.4028235e38) * np.sign(x[5])
    x[6] *= np.float32(1e-38)
    x[7] *= np.float32(1e-42)
    x[8] = np.float32(1.4e-45)                    # smaller than any scale: 0
    x[9, :, 7] = np.inf
    x[10, :, 7] = -np.inf
    x[11, :, hd - 1] = np.nan
    x[12] = np.inf
    x[13, 0, 0] = np.nan                          # one head of the row alone
    x[14] *= np.float32(2.0 ** -60)
    x[15] *= np.float32(2.0 ** -61)
    with make(shape, 64) as ctx:
        ctx.kv_write(0, 0, 0, x, -x)
        kk, vv = ctx.kv_read(0, 0, 0, 64)
    np.testing.assert_array_equal(kk, stored(x))
    np.testing.assert_array_equal(vv, stored(-x))
    assert np.isnan(kk[9]).all() and np.isnan(kk[13, 0]).all()
    assert kv == 1 or np.isfinite(kk[13, 1:]).all()


def test_many_quotients_beside_halves(cuda):
    """Values one step of FP32 around every half code: the nearest is taken."""
    rng = np.random.default_rng(3)
    x = np.zeros((400, 8, 128), np.float32)
    top = (1 + rng.random((400, 8, 1))).astype(np.float32) * np.float32(127)
    s = (top * (np.float32(1) / np.float32(127))).astype(np.float64)
    half = ((np.arange(128) - 63.5) * s).astype(np.float32)
    x[:] = half
    x[1::3] = np.nextafter(half, np.float32(np.inf))[1::3]
    x[2::3] = np.nextafter(half, np.float32(-np.inf))[2::3]
    x[..., 0:1] = top
    with make("l8b", 400) as ctx:
        ctx.kv_write(0, 0, 0, x, x)
        kk, vv = ctx.kv_read(0, 0, 0, 400)
    np.testing.assert_array_equal(kk, stored(x))
    np.testing.assert_array_equal(vv, stored(x))


@pytest.mark.parametrize("kind", ["f32", "q8"])
@pytest.mark.parametrize("shape", ["l8b", "tl"])
def test_read_packed(cuda, kind, shape):
    h, kv, hd = ALL[shape]
    rng = np.random.default_rng(1)
    with AttentionContext(2, h, kv, hd, 300, max_batch=4, kv=kind) as ctx:
        rows = [rnd(rng, 300, kv, hd) for _ in range(8)]
        for s in range(4):
            ctx.kv_write(s, 1, 0, rows[2 * s], rows[2 * s + 1])
        slots, pos0, n = [3, 0, 2], [17, 0, 299], [100, 0, 1]
        k, v = ctx.kv_read_packed(1, slots, pos0, n)
        for j, got in enumerate((k, v)):
            want = np.concatenate([rows[2 * s + j][p:p + m] for s, p, m in zip(slots, pos0, n)])
            np.testing.assert_array_equal(got.cpu().numpy(), stored(want) if kind == "q8" else want)
        k, v = ctx.kv_read_packed(0, [], [], [])
        assert tuple(k.shape) == (0, kv, hd)


# ---- decode ----------------------------------------------------------------------
@pytest.mark.parametrize("shape", HEADS)
def test_decode_lengths(cuda, shape):
    rng = np.random.default_rng(5)
    for n in (0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 1000):
        with make(shape, n + 1) as ctx:
            r = Ragged(ctx, rng, [0], [n])
            q, k, v = r.inputs([1])
            dq, dk, dv = gpu(q[0], k[0], v[0])
            r.check(ctx.decode(0, n, dq, dk, dv)[None], q, k, v, [1])
            ctx.sync()


@pytest.mark.parametrize("shape", ["l8b", "l70b", "tl"])
def test_decode_long(cuda, shape):
    rng = np.random.default_rng(6)
    with make(shape, 9000) as ctx:
        r = Ragged(ctx, rng, [0], [8190])
        for _ in range(2):
            q, k, v = r.inputs([1])
            out = ctx.decode_batched(0, [0], r.rows, *gpu(q, k, v))
            ref, kn, vn = attend(ctx, r.k[0], r.v[0], q, k, v)
            near(out.cpu().numpy(), ref)
            r.k[0], r.v[0] = np.concatenate([r.k[0], kn]), np.concatenate([r.v[0], vn])
            r.rows = r.rows + 1
        kk, vv = ctx.kv_read(0, 0, 8190, 3)
        np.testing.assert_array_equal(kk[:2], r.k[0][-2:])
        assert not kk[2].any() and not vv[2].any()


@pytest.mark.parametrize("shape", ["l8b", "tl", "l70b", "g8_64"])
def test_decode_ragged(cuda, shape):
    rng = np.random.default_rng(7)
    rows = [0, 1, 700, 33, 64, 129, 5]
    with make(shape, 1000, max_batch=9, n_layers=2) as ctx:
        r = Ragged(ctx, rng, [8, 0, 3, 5, 1, 2, 7], rows, layer=1)
        for _ in range(3):
            q, k, v = r.inputs([1] * 7)
            out = ctx.decode_batched(1, r.slots, r.rows, *gpu(q, k, v))
            r.check(out, q, k, v, [1] * 7)
        kk, _ = ctx.kv_read(4, 1, 0, 1000)
        assert not kk.any()


def test_decode_more_sequences_than_a_launch_takes(cuda):
    rng = np.random.default_rng(8)
    n = 150
    with make("g2_64", 64, max_batch=n) as ctx:
        r = Ragged(ctx, rng, rng.permutation(n), rng.integers(0, 60, n))
        q, k, v = r.inputs([1] * n)
        out = ctx.decode_batched(0, r.slots, r.rows, *gpu(q, k, v))
        r.check(out, q, k, v, [1] * n)


def test_decode_host(cuda):
    rng = np.random.default_rng(9)
    with make("l8b", 300) as ctx:
        r = Ragged(ctx, rng, [0], [200])
        for _ in range(3):
            q, k, v = r.inputs([1])
            out = ctx.decode_host(0, int(r.rows[0]), q[0], k[0], v[0])
            r.check(torch.from_numpy(out)[None], q, k, v, [1])


def test_layers_back_to_back(cuda):
    """Launches that follow one another without a wait, layers in turn and the
    same layer twice, give what they give one at a time."""
    rng = np.random.default_rng(10)
    h, kv, hd = ALL["l8b"]
    order = [0, 1, 2, 0, 0, 1, 2, 2, 1]
    ins = [gpu(rnd(rng, 1, h, hd), rnd(rng, 1, kv, hd), rnd(rng, 1, kv, hd)) for _ in order]
    base = [(rnd(rng, 900, kv, hd), rnd(rng, 900, kv, hd)) for _ in range(3)]
    outs = []
    for wait in (True, False):
        with make("l8b", 1000, n_layers=3) as ctx:
            for layer, (k, v) in enumerate(base):
                ctx.kv_write(0, layer, 0, k, v)
            pos, got = [900] * 3, []
            for layer, x in zip(order, ins):
                got.append(ctx.decode_batched(layer, [0], [pos[layer]], *x))
                pos[layer] += 1
                if wait:
                    ctx.sync()
            ctx.sync()
            outs.append(torch.stack(got).cpu())
    assert torch.equal(*outs)


# ---- trees ------------------------------------------------------------------------
@pytest.mark.parametrize("shape", HEADS)
@pytest.mark.parametrize("kind", ["random", "chain", "star", "roots"])
def test_tree_shapes(cuda, shape, kind):
    rng = np.random.default_rng(11)
    for pos, n in ((0, 1), (0, 9), (1, 2), (60, 5), (127, 16), (128, 33), (300, 64), (77, 128)):
        with make(shape, pos + n) as ctx:
            r = Ragged(ctx, rng, [0], [pos])
            q, k, v = r.inputs([n])
            par = tree(rng, n, kind)
            out = ctx.decode_tree(0, [0], r.rows, [n], par, *gpu(q, k, v))
            ctx.sync()
            r.check(out, q, k, v, [n], par)


@pytest.mark.parametrize("shape", ["l8b", "l70b", "tl", "mha128"])
@pytest.mark.parametrize("lens", [[1, 1, 1], [3, 0, 2, 1], [16, 64, 9, 31, 128], [2] * 20])
def test_tree_ragged(cuda, shape, lens):
    rng = np.random.default_rng(12)
    n = len(lens)
    with make(shape, 1600, max_batch=n + 2, n_layers=2) as ctx:
        rows = rng.integers(0, 1400, n)
        rows[0] = 0
        r = Ragged(ctx, rng, rng.permutation(n + 2)[:n], rows, layer=1)
        q, k, v = r.inputs(lens)
        par = np.concatenate([tree(rng, t) for t in lens])
        out = ctx.decode_tree(1, r.slots, r.rows, lens, par, *gpu(q, k, v))
        r.check(out, q, k, v, lens, par)


def test_tree_more_nodes_than_a_launch_takes(cuda):
    rng = np.random.default_rng(13)
    lens = [128] * 33 + [5]
    with make("mha64", 200, max_batch=34) as ctx:
        r = Ragged(ctx, rng, np.arange(34), rng.integers(0, 70, 34))
        q, k, v = r.inputs(lens)
        par = np.concatenate([tree(rng, t) for t in lens])
        r.check(ctx.decode_tree(0, r.slots, r.rows, lens, par, *gpu(q, k, v)), q, k, v, lens, par)


@pytest.mark.parametrize("shape", ["l8b", "tl"])
def test_tree_long(cuda, shape):
    rng = np.random.default_rng(14)
    for n in (1, 2, 16, 40):
        with make(shape, 8300) as ctx:
            r = Ragged(ctx, rng, [0], [8192 - n])
            q, k, v = r.inputs([n])
            par = tree(rng, n)
            r.check(ctx.decode_tree(0, [0], r.rows, [n], par, *gpu(q, k, v)), q, k, v, [n], par)


@pytest.mark.parametrize("kind", ["f32", "q8"])
@pytest.mark.parametrize("shape", ["l8b", "tl"])
def test_keep(cuda, kind, shape):
    h, kv, hd = ALL[shape]
    rng = np.random.default_rng(15)
    with AttentionContext(2, h, kv, hd, 200, max_batch=3, kv=kind) as ctx:
        rows = {(s, l): (rnd(rng, 200, kv, hd), rnd(rng, 200, kv, hd)) for s in range(3) for l in range(2)}
        for (s, l), (k, v) in rows.items():
            ctx.kv_write(s, l, 0, k, v)
        slots, pos = [2, 0], [71, 5]
        nodes = [[0, 3, 4, 9, 20, 21, 22, 50, 51, 90, 127], [2]]
        ctx.kv_keep(slots, pos, [11, 1], sum(nodes, []))
        ctx.kv_keep([1], [0], [0], [])
        for (s, l), (k, v) in rows.items():
            for got, x in zip(ctx.kv_read(s, l, 0, 200), (k, v)):
                want = x.copy()
                if s in slots:
                    p, nd = pos[slots.index(s)], nodes[slots.index(s)]
                    want[p:p + len(nd)] = x[p + np.array(nd)]
                np.testing.assert_array_equal(got, stored(want) if kind == "q8" else want)


# ---- packed prompts --------------------------------------------------------------------
@pytest.mark.parametrize("shape", HEADS)
@pytest.mark.parametrize("rows,lens", [([0], [1]), ([0], [127]), ([0], [128]), ([0], [129]), ([0], [300]),
                                       ([5, 0, 130], [17, 1, 64]), ([0, 0, 9, 0], [0, 200, 3, 33]),
                                       ([255, 256, 257], [31, 32, 33])])
def test_prefill_packed(cuda, shape, rows, lens):
    rng = np.random.default_rng(16)
    n = len(lens)
    with make(shape, max(a + b for a, b in zip(rows, lens)), max_batch=n + 1, n_layers=2) as ctx:
        r = Ragged(ctx, rng, rng.permutation(n + 1)[:n], rows, layer=1)
        q, k, v = r.inputs(lens)
        out = ctx.prefill_packed(1, r.slots, r.rows, lens, *gpu(q, k, v))
        ctx.sync()
        r.check(out, q, k, v, lens)


@pytest.mark.parametrize("shape", ["l8b", "tl"])
def test_prefill_long(cuda, shape):
    rng = np.random.default_rng(17)
    with make(shape, 4000) as ctx:
        r = Ragged(ctx, rng, [0], [1900])
        q, k, v = r.inputs([700])
        out = ctx.prefill(0, 0, 1900, *gpu(q, k, v))
        r.check(out, q, k, v, [700])


def test_prefill_more_sequences_than_a_launch_takes(cuda):
    rng = np.random.default_rng(18)
    lens = list(rng.integers(0, 40, 140))
    with make("mha64", 64, max_batch=140) as ctx:
        r = Ragged(ctx, rng, rng.permutation(140), rng.integers(0, 20, 140))
        q, k, v = r.inputs(lens)
        r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)


def test_prefill_packed_over_an_fp32_cache(cuda):
    """The FP32 cache's packed prefill is its prefill, sequence by sequence."""
    rng = np.random.default_rng(19)
    h, kv, hd = ALL["l8b"]
    lens, pos = [40, 0, 129], [3, 0, 0]
    x = gpu(rnd(rng, 169, h, hd), rnd(rng, 169, kv, hd), rnd(rng, 169, kv, hd))
    got = []
    for packed in (True, False):
        with AttentionContext(1, h, kv, hd, 200, max_batch=3) as ctx:
            if packed:
                out = ctx.prefill_packed(0, [2, 0, 1], pos, lens, *x)
            else:
                out = torch.cat([ctx.prefill(2, 0, 3, *(y[:40].contiguous() for y in x)),
                                 ctx.prefill(1, 0, 0, *(y[40:].contiguous() for y in x))])
            ctx.sync()
            got.append((out.cpu(), *ctx.kv_read(1, 0, 0, 129)))
    assert torch.equal(got[0][0], got[1][0])
    np.testing.assert_array_equal(got[0][1], got[1][1])
    np.testing.assert_array_equal(got[0][2], got[1][2])


# ---- rows that are not seen ----------------------------------------------------------------
def poison(ctx, slot, first, last):
    bad = np.full((last - first, ctx.n_kv_heads, ctx.head_dim), np.nan, np.float32)
    ctx.kv_write(slot, 0, first, bad, bad)


@pytest.mark.parametrize("shape", ["l8b", "tl"])
def test_nan_rows_behind_the_end_are_not_read(cuda, shape):
    rng = np.random.default_rng(20)
    for n in (0, 3, 33, 120, 500):
        with make(shape, 700) as ctx:
            r = Ragged(ctx, rng, [0], [n])
            poison(ctx, 0, n, 700)
            q, k, v = r.inputs([1])
            r.check(ctx.decode_batched(0, [0], [n], *gpu(q, k, v)), q, k, v, [1])
            for t in (2, 40):
                q, k, v = r.inputs([t])
                par = tree(rng, t)
                r.check(ctx.decode_tree(0, [0], r.rows, [t], par, *gpu(q, k, v)), q, k, v, [t], par)
            q, k, v = r.inputs([50])
            r.check(ctx.prefill_packed(0, [0], r.rows, [50], *gpu(q, k, v)), q, k, v, [50])


@pytest.mark.parametrize("shape", ["l8b", "tl"])
@pytest.mark.parametrize("n", [2, 6, 40])
def test_nan_in_a_node_reaches_only_what_descends_from_it(cuda, shape, n):
    rng = np.random.default_rng(21)
    par = tree(rng, n, "roots")  # no node sees another
    with make(shape, 400) as ctx:
        r = Ragged(ctx, rng, [0], [90])
        q, k, v = r.inputs([n])
        k[0, 0, 3], v[1, :, 2] = np.inf, np.nan
        out = ctx.decode_tree(0, [0], [90], [n], par, *gpu(q, k, v)).cpu().numpy()
        ref, _, _ = attend(ctx, r.k[0], r.v[0], q, k, v, par)
        g = ctx.n_heads // ctx.n_kv_heads
        assert np.isnan(out[0, :g]).all() and np.isnan(out[1]).all()
        near(out[0, g:], ref[0, g:])
        near(out[2:], ref[2:])


@pytest.mark.parametrize("t", [2, 40])
def test_nan_in_a_prompt_reaches_only_later_tokens(cuda, t):
    rng = np.random.default_rng(22)
    with make("l8b", 400) as ctx:
        r = Ragged(ctx, rng, [0], [10])
        q, k, v = r.inputs([t])
        v[t - 1, 0, 0] = np.nan
        out = ctx.prefill_packed(0, [0], [10], [t], *gpu(q, k, v)).cpu().numpy()
        ref, _, _ = attend(ctx, r.k[0], r.v[0], q, k, v)
        near(out[:t - 1], ref[:t - 1])
        g = ctx.n_heads // ctx.n_kv_heads
        assert np.isnan(out[t - 1, :g]).all()
        near(out[t - 1, g:], ref[t - 1, g:])


@pytest.mark.parametrize("t", [1, 3, 40])
def test_sizes_of_rows_far_apart(cuda, t):
    """Scales from 1e-12 to 1e6 (and zero rows) in one cache, large queries."""
    rng = np.random.default_rng(23)
    with make("l8b", 600) as ctx:
        r = Ragged(ctx, rng, [0], [0])
        k, v = rnd(rng, 500, 8, 128), rnd(rng, 500, 8, 128)
        v *= 10 ** rng.uniform(-12, 6, (500, 8, 1)).astype(np.float32)
        k *= 10 ** rng.uniform(-6, 0, (500, 8, 1)).astype(np.float32)
        k[7], v[9] = 0, 0
        ctx.kv_write(0, 0, 0, k, v)
        r.k[0], r.v[0], r.rows = stored(k), stored(v), np.array([500], np.int32)
        q, k, v = r.inputs([t])
        q *= 3
        par = tree(rng, t)
        r.check(ctx.decode_tree(0, [0], r.rows, [t], par, *gpu(q, k, v)), q, k, v, [t], par)


# ---- as they are used together -----------------------------------------------------------
@pytest.mark.parametrize("shape", ["l8b", "tl", "l70b"])
def test_prompts_then_drafts_then_decode(cuda, shape):
    rng = np.random.default_rng(24)
    with make(shape, 700, max_batch=3) as ctx:
        r = Ragged(ctx, rng, [1, 2, 0], [0, 0, 0])
        for lens in ([200, 33, 129], [65, 40, 1]):
            q, k, v = r.inputs(lens)
            r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)
        for lens in ([12, 7, 24], [2, 1, 1]):
            before = r.rows.copy()
            q, k, v = r.inputs(lens)
            par = [tree(rng, t) for t in lens]
            r.check(ctx.decode_tree(0, r.slots, r.rows, lens, np.concatenate(par), *gpu(q, k, v)), q, k, v, lens,
                    np.concatenate(par))
            paths = []
            for i, p in enumerate(par):  # the path to the last node is accepted
                path = [len(p) - 1]
                while p[path[0]] >= 0:
                    path.insert(0, int(p[path[0]]))
                paths.append(path)
                keep = list(range(before[i])) + [before[i] + x for x in path]
                r.k[i], r.v[i] = r.k[i][keep], r.v[i][keep]
            ctx.kv_keep(r.slots, before, [len(p) for p in paths], sum(paths, []))
            r.rows = before + np.array([len(p) for p in paths], np.int32)
            q, k, v = r.inputs([1, 1, 1])
            r.check(ctx.decode_batched(0, r.slots, r.rows, *gpu(q, k, v)), q, k, v, [1, 1, 1])


def test_a_chain_is_a_prompt_is_decode(cuda):
    rng = np.random.default_rng(25)
    h, kv, hd = ALL["l8b"]
    q, k, v = rnd(rng, 6, h, hd), rnd(rng, 6, kv, hd), rnd(rng, 6, kv, hd)
    base = rnd(rng, 100, kv, hd), rnd(rng, 100, kv, hd)
    outs = []
    for way in range(3):
        with make("l8b", 120) as ctx:
            ctx.kv_write(0, 0, 0, *base)
            x = gpu(q, k, v)
            if way == 0:
                o = ctx.decode_tree(0, [0], [100], [6], tree(rng, 6, "chain"), *x)
            elif way == 1:
                o = ctx.prefill(0, 0, 100, *x)
            else:
                o = torch.cat([ctx.decode_batched(0, [0], [100 + i], *(y[i:i + 1] for y in x)) for i in range(6)])
            outs.append(o.cpu().numpy())
    near(outs[0], outs[1].astype(np.float64))
    near(outs[2], outs[1].astype(np.float64))


def test_captured_and_replayed(cuda):
    rng = np.random.default_rng(26)
    h, kv, hd = ALL["l8b"]
    lens = [5, 40]
    par = np.concatenate([tree(rng, t) for t in lens])
    with make("l8b", 700, max_batch=2, n_layers=2) as ctx:
        base = [Ragged(ctx, rng, [0, 1], [300, 10], layer=i) for i in range(2)]
        s = torch.cuda.Stream()
        dec = [torch.zeros(2, n, hd, device="cuda") for n in (h, kv, kv)]
        tre = [torch.zeros(45, n, hd, device="cuda") for n in (h, kv, kv)]
        ctx.bind_torch_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            o0 = ctx.decode_batched(0, [0, 1], [300, 10], *dec)
            o1 = ctx.decode_tree(1, [0, 1], [300, 10], lens, par, *tre)
            o2 = ctx.prefill_packed(1, [0], [300], [5], *(x[:5] for x in tre))
        for _ in range(2):
            a, b = base[0].inputs([1, 1]), base[0].inputs(lens)
            for dst, src in zip(dec + tre, gpu(*a, *b)):
                dst.copy_(src)
            g.replay()
            torch.cuda.synchronize()
            for i in range(2):
                ref, _, _ = attend(ctx, base[0].k[i], base[0].v[i], *(x[i:i + 1] for x in a))
                near(o0[i:i + 1].cpu().numpy(), ref)
                r = slice(0, 5) if i == 0 else slice(5, 45)
                ref, _, _ = attend(ctx, base[1].k[i], base[1].v[i], *(x[r] for x in b), par[r])
                near(o1[r].cpu().numpy(), ref)
            ref, _, _ = attend(ctx, base[1].k[0], base[1].v[0], *(x[:5] for x in b))
            near(o2.cpu().numpy(), ref)
        ctx.sync()
        del g


def test_on_another_stream(cuda):
    rng = np.random.default_rng(27)
    s = torch.cuda.Stream()
    with make("l8b", 300) as ctx:
        r = Ragged(ctx, rng, [0], [100])
        q, k, v = r.inputs([30])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            ctx.bind_torch_stream()
            x = gpu(q, k, v)
            out = ctx.prefill_packed(0, [0], [100], [30], *x)
            kk, _ = ctx.kv_read_device(0, 0, 100, 30)
        s.synchronize()
        r.check(out, q, k, v, [30])
        np.testing.assert_array_equal(kk.cpu().numpy(), r.k[0][100:])


def test_two_contexts_on_two_streams_at_once(cuda):
    rng = np.random.default_rng(28)
    ctxs = [make("l8b", 2000) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    rs = [Ragged(c, rng, [0], [1500]) for c in ctxs]
    ins = [r.inputs([20]) for r in rs]
    par = tree(rng, 20)
    dev = [gpu(*x) for x in ins]
    torch.cuda.synchronize()
    outs = []
    for c, s, x in zip(ctxs, streams, dev):
        c.bind_torch_stream(s)
        with torch.cuda.stream(s):
            outs.append(c.decode_tree(0, [0], [1500], [20], par, *x))
    torch.cuda.synchronize()
    for r, o, x in zip(rs, outs, ins):
        r.check(o, *x, [20], par)
    for c in ctxs:
        c.close()


def test_rows_past_four_gigabytes(cuda):
    """A slot whose codes start above 2^32 bytes."""
    rng = np.random.default_rng(29)
    with make("mha128", 70016, max_batch=64) as ctx:
        assert 63 * 70016 * 8 * 128 > 2 ** 32
        r = Ragged(ctx, rng, [63, 0], [200, 40])
        q, k, v = r.inputs([1, 1])
        r.check(ctx.decode_batched(0, r.slots, r.rows, *gpu(q, k, v)), q, k, v, [1, 1])
        q, k, v = r.inputs([150, 20])
        r.check(ctx.prefill_packed(0, r.slots, r.rows, [150, 20], *gpu(q, k, v)), q, k, v, [150, 20])
        par = np.concatenate([tree(rng, 9), tree(rng, 30)])
        q, k, v = r.inputs([9, 30])
        r.check(ctx.decode_tree(0, r.slots, r.rows, [9, 30], par, *gpu(q, k, v)), q, k, v, [9, 30], par)
        x = rnd(rng, 3, 8, 128)
        ctx.kv_write(63, 0, 70013, x, x)
        np.testing.assert_array_equal(ctx.kv_read(63, 0, 70013, 3)[0], stored(x))


# ---- batches that the kernel of single warps takes ---------------------------------------
@pytest.mark.parametrize("shape", ["l8b", "l70b", "g8_64"])
def test_decode_of_many_sequences(cuda, shape):
    """More (sequence, kv head) pairs than blocks run at once, two steps."""
    rng = np.random.default_rng(31)
    n = 320 // ALL[shape][1]
    with make(shape, 1100, max_batch=n, n_layers=2) as ctx:
        rows = rng.integers(0, 1000, n)
        rows[:6] = [0, 1, 31, 32, 33, 64]
        r = Ragged(ctx, rng, rng.permutation(n), rows, layer=1)
        for _ in range(2):
            q, k, v = r.inputs([1] * n)
            r.check(ctx.decode_batched(1, r.slots, r.rows, *gpu(q, k, v)), q, k, v, [1] * n)
        kk, vv = ctx.kv_read(0, 0, 0, 1100)
        assert not kk.any() and not vv.any()


def test_decode_of_items_in_many_parts(cuda):
    """Long contexts: every item is spread over many warps and joined."""
    rng = np.random.default_rng(32)
    with make("l8b", 6200, max_batch=16) as ctx:
        r = Ragged(ctx, rng, rng.permutation(16), rng.integers(5500, 6100, 16))
        q, k, v = r.inputs([1] * 16)
        out = ctx.decode_batched(0, r.slots, r.rows, *gpu(q, k, v)).cpu().numpy()
        for i in (0, 7, 15):
            ref, kn, vn = attend(ctx, r.k[i], r.v[i], q[i:i + 1], k[i:i + 1], v[i:i + 1])
            near(out[i:i + 1], ref)
            kk, vv = ctx.kv_read(int(r.slots[i]), 0, int(r.rows[i]), 1)
            np.testing.assert_array_equal(kk, kn)
            np.testing.assert_array_equal(vv, vn)


@pytest.mark.parametrize("shape,drafted", [("l8b", True), ("l8b", False), ("mha64", True), ("l70b", False)])
def test_one_long_sequence_among_short_ones_on_tensor_cores(cuda, shape, drafted):
    """Splits of unequal sequences, with query tiles that do not see the last of them."""
    rng = np.random.default_rng(40)
    lens = [16] * 18 + [100, 70]
    with make(shape, 5000, max_batch=20) as ctx:
        rows = rng.integers(0, 400, 20)
        rows[-2:] = [0, 4900]
        r = Ragged(ctx, rng, rng.permutation(20), rows)
        q, k, v = r.inputs(lens)
        if drafted:
            parents = np.concatenate([tree(rng, n) for n in lens])
            r.check(ctx.decode_tree(0, r.slots, r.rows, lens, parents, *gpu(q, k, v)), q, k, v, lens, parents)
        else:
            r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)


def test_call_after_a_replay_that_wrote_its_layer(cuda):
    """The last eager call before the replay was on the other layer."""
    import torch
    rng = np.random.default_rng(39)
    with make("l8b", 1200, max_batch=4, n_layers=2) as ctx:
        stream = torch.cuda.Stream()
        ctx.bind_torch_stream(stream)
        rs = [Ragged(ctx, rng, range(4), [1023, 500, 31, 0], layer=x) for x in (0, 1)]
        q, k, v = rs[0].inputs([1] * 4)
        dev = gpu(q, k, v)
        with torch.cuda.stream(stream):
            ctx.decode_batched(1, rs[1].slots, rs[1].rows, *dev)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            first = ctx.decode_batched(0, rs[0].slots, rs[0].rows, *dev)
        q2, k2, v2 = rs[0].inputs([1] * 4)
        dev2 = gpu(q2, k2, v2)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            ctx.decode_batched(1, rs[1].slots, rs[1].rows, *dev)
            graph.replay()
            second = ctx.decode_batched(0, rs[0].slots, rs[0].rows + 1, *dev2)
        torch.cuda.synchronize()
        for i in range(4):
            sl = slice(i, i + 1)
            ref, kn, vn = attend(ctx, rs[0].k[i], rs[0].v[i], q[sl], k[sl], v[sl])
            near(first.cpu().numpy()[sl], ref)
            ref, _, _ = attend(ctx, np.concatenate([rs[0].k[i], kn]), np.concatenate([rs[0].v[i], vn]), q2[sl], k2[sl], v2[sl])
            near(second.cpu().numpy()[sl], ref)
        del graph


@pytest.mark.parametrize("shape", ["mha128", "mha64", "g2_64"])
@pytest.mark.parametrize("drafted", [False, True])
def test_new_rows_that_few_or_many_warps_store(cuda, shape, drafted):
    """Up to a query tile of new rows, in a block's first tiles and further on."""
    rng = np.random.default_rng(38)
    for lens in ([9, 64, 13], [17, 64, 50], [128 if shape != "g2_64" else 64, 65, 3]):
        with make(shape, 1500, max_batch=3) as ctx:
            r = Ragged(ctx, rng, [2, 0, 1], [0, 125, 1300])
            q, k, v = r.inputs(lens)
            if drafted:
                parents = np.concatenate([tree(rng, n) for n in lens])
                out = ctx.decode_tree(0, r.slots, r.rows, lens, parents, *gpu(q, k, v))
                r.check(out, q, k, v, lens, parents)
            else:
                r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)


@pytest.mark.parametrize("shape,nodes", [("l8b", 1), ("l8b", 2), ("g2_64", 1), ("l70b", 1)])
def test_one_long_sequence_among_short_ones(cuda, shape, nodes):
    """Splits of the long one, more blocks than run at once; it comes last."""
    rng = np.random.default_rng(37)
    n = 160 // ALL[shape][1] + 3
    with make(shape, 6000, max_batch=n) as ctx:
        rows = rng.integers(0, 130, n)
        rows[:3] = [0, 127, 128]
        rows[-1] = 5990
        r = Ragged(ctx, rng, rng.permutation(n), rows)
        q, k, v = r.inputs([nodes] * n)
        if nodes == 1:
            out = ctx.decode_batched(0, r.slots, r.rows, *gpu(q, k, v))
        else:
            out = ctx.prefill_packed(0, r.slots, r.rows, [nodes] * n, *gpu(q, k, v))
        r.check(out, q, k, v, [nodes] * n)


@pytest.mark.parametrize("shape,most", [("mha128", 8), ("g2_64", 4), ("l8b", 2), ("l70b", 1)])
def test_small_trees_of_many_sequences(cuda, shape, most):
    """New rows that straddle tiles of 32 rows, sequences without any, NaN behind."""
    rng = np.random.default_rng(33)
    n = 60
    lens = [int(x) for x in rng.integers(0, most + 1, n)]
    lens[0] = most
    rows = 32 * rng.integers(0, 12, n) + rng.integers(24, 34, n)
    with make(shape, 500, max_batch=n) as ctx:
        r = Ragged(ctx, rng, rng.permutation(n), rows)
        for s, c in zip(r.slots, rows):
            poison(ctx, int(s), int(c), 500)
        q, k, v = r.inputs(lens)
        par = np.concatenate([tree(rng, t) for t in lens])
        r.check(ctx.decode_tree(0, r.slots, r.rows, lens, par, *gpu(q, k, v)), q, k, v, lens, par)
        q, k, v = r.inputs(lens)
        r.check(ctx.prefill_packed(0, r.slots, r.rows, lens, *gpu(q, k, v)), q, k, v, lens)


@pytest.mark.parametrize("shape", ["l8b", "tl", "mha128"])
@pytest.mark.parametrize("pos", [127, 250, 1020, 2040, 4090])
def test_new_rows_across_tiles_and_splits(cuda, shape, pos):
    """One query tile a sequence: its blocks store the new rows themselves, each
    those of its own range."""
    rng = np.random.default_rng(34)
    with make(shape, pos + 40) as ctx:
        r = Ragged(ctx, rng, [0], [pos])
        for n in (16, 11):
            q, k, v = r.inputs([n])
            par = tree(rng, n)
            r.check(ctx.decode_tree(0, [0], r.rows, [n], par, *gpu(q, k, v)), q, k, v, [n], par)


def test_layers_back_to_back_of_every_kind(cuda):
    """Decode, trees and prompts on layers in turn without a wait between them give
    what they give with one."""
    rng = np.random.default_rng(35)
    h, kv, hd = ALL["l8b"]
    ops = [("d", 0, 1), ("t", 1, 9), ("d", 0, 1), ("p", 2, 70), ("d", 1, 1), ("t", 0, 2), ("d", 2, 1), ("t", 2, 60),
           ("d", 0, 1), ("d", 2, 1), ("p", 0, 3), ("d", 1, 1)]
    ins = [gpu(rnd(rng, n, h, hd), rnd(rng, n, kv, hd), rnd(rng, n, kv, hd)) for _, _, n in ops]
    par = [tree(rng, n) for _, _, n in ops]
    base = [(rnd(rng, 1500, kv, hd), rnd(rng, 1500, kv, hd)) for _ in range(3)]
    got = []
    for wait in (True, False):
        with make("l8b", 1800, n_layers=3) as ctx:
            for layer, (k, v) in enumerate(base):
                ctx.kv_write(0, layer, 0, k, v)
            pos, outs = [1500] * 3, []
            for (what, layer, n), x, p in zip(ops, ins, par):
                if what == "d":
                    outs.append(ctx.decode_batched(layer, [0], [pos[layer]], *x))
                elif what == "t":
                    outs.append(ctx.decode_tree(layer, [0], [pos[layer]], [n], p, *x))
                else:
                    outs.append(ctx.prefill_packed(layer, [0], [pos[layer]], [n], *x))
                pos[layer] += n
                if wait:
                    ctx.sync()
            ctx.sync()
            got.append((torch.cat(outs).cpu(), [ctx.kv_read(0, i, 1500, 300) for i in range(3)]))
    assert torch.equal(got[0][0], got[1][0])
    for a, b in zip(got[0][1], got[1][1]):
        np.testing.assert_array_equal(a[0], b[0])
        np.testing.assert_array_equal(a[1], b[1])


# ---- the engine ---------------------------------------------------------------------------
@pytest.mark.parametrize("quantized", [False, True])
def test_engine_with_an_8_bit_cache(cuda, quantized):
    """The engine's layers over either cache: the logits differ by what 8-bit
    rows cost (a row is off by half a code, 1/254 of its largest value, about
    1/80 of its length after 3-sigma maxima; attention averages that), and a
    prompt in chunks gives what it gives token by token."""
    cfg = ModelConfig(dim=512, hidden_dim=1024, n_layers=3, n_heads=8, n_kv_heads=4, vocab_size=1000, seq_len=256)
    toks = np.random.default_rng(30).integers(0, 1000, 70)
    logits, used = {}, {}
    for kv in ("f32", "q8"):
        with Transformer.synthetic(cfg, quantized, seed=3, max_chunk=32, kv=kv) as t:
            used[kv] = t.device_bytes()
            t.prefill(toks[:-1])
            chunked = t.forward(int(toks[-1]), 69)
            t.clear_kv_cache()
            for p, x in enumerate(toks):
                one = t.forward(int(x), p)
            logits[kv] = one
            assert np.linalg.norm(chunked - one) <= (2e-2 if quantized else 1e-3) * np.linalg.norm(one)
            if kv == "q8":
                t.set_kv("f32")
                for p, x in enumerate(toks):
                    one = t.forward(int(x), p)
                if not quantized:
                    np.testing.assert_array_equal(one, logits["f32"])
    assert np.linalg.norm(logits["q8"] - logits["f32"]) <= 2e-2 * np.linalg.norm(logits["f32"])


# ---- refusals --------------------------------------------------------------------------------
def test_refusals(cuda):
    h, kv, hd = ALL["tl"]
    z = lambda n, m: torch.zeros(n, m, hd, device="cuda")  # noqa: E731
    with AttentionContext(1, h, kv, hd, 64, max_batch=2) as f:
        with pytest.raises(LeapError, match="8-bit"):
            f.decode_tree(0, [0], [0], [1], [-1], z(1, h), z(1, kv), z(1, kv))
    with make("tl", 64, max_batch=2) as ctx:
        poison(ctx, 0, 0, 64)
        before = ctx.kv_read(0, 0, 0, 64)
        x = lambda n: (z(n, h), z(n, kv), z(n, kv))  # noqa: E731
        bad_trees = [([0], [0], [2], [-1, 1], 2),        # its own parent
                     ([0], [0], [2], [0, -1], 2),        # a parent that comes later
                     ([0], [0], [1], [-2], 1), ([0], [63], [2], [-1, 0], 2), ([0], [-1], [1], [-1], 1),
                     ([2], [0], [1], [-1], 1), ([0, 0], [0, 5], [1, 1], [-1, -1], 2), ([0], [0], [129], [-1] * 129, 129)]
        for slots, pos, n, par, total in bad_trees:
            with pytest.raises(LeapError):
                ctx.decode_tree(0, slots, pos, n, par, *x(total))
        for slots, pos, n, total in (([0], [60], [5], 5), ([0, 0], [0, 0], [1, 1], 2), ([-1], [0], [1], 1),
                                     ([0], [2147483647], [1], 1), ([0, 1], [0, 0], [-1, 1], 1)):
            with pytest.raises(LeapError):
                ctx.prefill_packed(0, slots, pos, n, *x(total))
            with pytest.raises(LeapError):
                ctx.kv_read_packed(0, slots, pos, n)
        for layer in (-1, 1):
            with pytest.raises(LeapError):
                ctx.prefill_packed(layer, [0], [0], [1], *x(1))
        for nodes in ([1, 1], [3, 2], [-1, 0], [0, 128], [0, 60]):
            with pytest.raises(LeapError):
                ctx.kv_keep([0], [10], [2], nodes)
        with pytest.raises(LeapError):
            ctx.decode_batched(0, [0, 0], [1, 2], *x(2))
        with pytest.raises(ValueError):
            ctx.prefill_packed(0, [0], [0], [2], *x(3))
        with pytest.raises(ValueError):
            ctx.decode_tree(0, [0], [0, 1], [1], [-1], *x(1))
        with pytest.raises(ValueError):
            ctx.decode_tree(0, [0], [0], [2], [-1], *x(2))
        q, k, v = x(2)
        with pytest.raises(TypeError):
            ctx.prefill_packed(0, [0], [0], [2], q.half(), k, v)
        with pytest.raises(TypeError):
            ctx.prefill_packed(0, [0], [0], [2], z(4, h)[::2], k, v)
        off = torch.zeros(2 * h * hd + 1, device="cuda")[1:].view(2, h, hd)
        with pytest.raises(LeapError, match="aligned"):
            ctx.prefill_packed(0, [0], [0], [2], off, k, v)
        ctx.prefill_packed(0, [], [], [], *x(0))          # nothing to do is fine
        ctx.decode_tree(0, [1], [64], [0], [], *x(0))
        ctx.sync()
        for a, b in zip(before, ctx.kv_read(0, 0, 0, 64)):
            np.testing.assert_array_equal(a, b)
        n = ctypes.c_int()
        from leap_b200 import _native
        _native.check(_native.lib().leap_ctx_kv_kind(ctx.handle, ctypes.byref(n)))
        assert n.value == _native.LEAP_KV_Q8
