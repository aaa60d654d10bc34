"""The attention operators over an 8-bit KV cache, as they are timed and checked.

Four operators, which work on one cache of codes (one byte for each value, one
scale for each row and kv head):

  cache    rows written into the cache (quantised) and read back
  decode   one new token for each of some sequences
  tree     a tree of drafted tokens behind each of some sequences
  prefill  packed prompts (or parts of prompts) of different lengths, causal

A row x of one kv head is kept as codes c and a scale s:
  s = max|x| * (1/127) in FP32,  c = x / s rounded to the nearest whole number
  (ties to even, within -127..127),  and stands for c * s.
Attention reads nothing but cached rows, the new tokens' own among them:
  k' = kept(rope(k)), v' = kept(v);  out = softmax(rope(q) . k' / sqrt(hd)) . v'
over the rows that a token sees: all rows before the run of new tokens and, of
the run, itself with its ancestors (tree) or its predecessors (prefill).  The
rotation of k is rounded product by product in FP32 (x0*c - x1*s, x1*c + x0*s),
so that codes do not depend on how it is computed.

``run`` returns the attention outputs; for ``cache`` the rows as they read back,
and for ``prefill`` the rows it appended as well, as a worker that runs prompts
for another one hands them on.  A decoded token's or node's own row is part of
what its output is computed from.
"""
import math
import random

import numpy as np
import torch

own = False

# (query heads, kv heads, head dim): the head layouts of the tests.
HEADS = {"32/8x128": (32, 8, 128), "64/8x128": (64, 8, 128), "32/4x64": (32, 4, 64),
         "8/8x128": (8, 8, 128), "16/8x64": (16, 8, 64)}


def listed():
    return [
        # one decoded token's row put away and fetched: latency only
        {"name": "cache 1 row", "op": "cache", "heads": "32/8x128", "pos0": 4095, "rows": 1},
        # a short prompt's rows at an odd place, small heads
        {"name": "cache 777 rows", "op": "cache", "heads": "32/4x64", "pos0": 131, "rows": 777},
        # a whole long prompt moved in and out
        {"name": "cache 8192 rows", "op": "cache", "heads": "32/8x128", "pos0": 0, "rows": 8192},
        # the start of a chat
        {"name": "decode 1x512", "op": "decode", "heads": "32/8x128", "seqs": 1, "lo": 512, "hi": 512, "lens": 0},
        # one long chat, the benchmark's context
        {"name": "decode 1x8192", "op": "decode", "heads": "32/8x128", "seqs": 1, "lo": 8192, "hi": 8192, "lens": 0},
        # a busy server: the ragged batch of the benchmark
        {"name": "decode 64 ragged", "op": "decode", "heads": "32/8x128", "seqs": 64, "lo": 512, "hi": 8192, "lens": 1},
        # a few drafted tokens behind a short context, small heads
        {"name": "tree 5 on 300", "op": "tree", "heads": "32/4x64", "seqs": 1, "lo": 300, "hi": 300, "tlo": 5, "thi": 5, "lens": 2},
        # one user, a usual draft tree, long context
        {"name": "tree 16 on 8192", "op": "tree", "heads": "32/8x128", "seqs": 1, "lo": 8192, "hi": 8192, "tlo": 16, "thi": 16, "lens": 3},
        # several users with trees of different sizes
        {"name": "tree 8 ragged", "op": "tree", "heads": "64/8x128", "seqs": 8, "lo": 300, "hi": 8000, "tlo": 9, "thi": 64, "lens": 4},
        # a server's prompts of different lengths, taken together
        {"name": "prefill 12 ragged", "op": "prefill", "heads": "32/8x128", "seqs": 12, "lo": 0, "hi": 0, "tlo": 1, "thi": 1500, "lens": 5},
        # the next parts of prompts whose beginnings are cached
        {"name": "prefill parts", "op": "prefill", "heads": "64/8x128", "seqs": 3, "lo": 1000, "hi": 4000, "tlo": 300, "thi": 600, "lens": 6},
        # one long document
        {"name": "prefill 1x8192", "op": "prefill", "heads": "32/8x128", "seqs": 1, "lo": 0, "hi": 0, "tlo": 8192, "thi": 8192, "lens": 7},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["cache", "decode", "decode", "tree", "tree", "prefill", "prefill"])
    heads = rng.choice(sorted(HEADS))
    lens = rng.randrange(1 << 20)
    if op == "cache":
        rows = _log(rng, 1, 8192)
        return {"op": op, "heads": heads, "pos0": rng.randrange(0, 8193 - rows), "rows": rows}
    if op == "decode":
        seqs = _log(rng, 1, 48)
        hi = _log(rng, 1, 8192)
        return {"op": op, "heads": heads, "seqs": seqs, "lo": _log(rng, 1, hi), "hi": hi, "lens": lens}
    if op == "tree":
        seqs = _log(rng, 1, 8)
        hi = _log(rng, 1, 6000)
        thi = _log(rng, 1, 64)
        return {"op": op, "heads": heads, "seqs": seqs, "lo": _log(rng, 1, hi), "hi": hi, "tlo": rng.randint(1, thi), "thi": thi, "lens": lens}
    seqs = _log(rng, 1, 12)
    thi = _log(rng, 1, 4000 // seqs)
    hi = rng.choice([0, _log(rng, 1, 2000)])
    return {"op": op, "heads": heads, "seqs": seqs, "lo": min(hi, rng.randrange(0, hi + 1)), "hi": hi, "tlo": rng.randint(1, thi), "thi": thi, "lens": lens}


def _sizes(case):
    """(rows before the run, new tokens) of each sequence, and the parents of
    all nodes in a row (-1: none): plain lists, from the case alone."""
    r = random.Random(case["lens"])
    n = case["seqs"]
    rows = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    if case["op"] == "decode":
        return [x - 1 for x in rows], [1] * n, None  # the context counts the new token
    toks = [r.randint(case["tlo"], case["thi"]) for _ in range(n)]
    if case["op"] == "prefill":
        return rows, toks, None
    # A drafted tree: most nodes continue a recent one, some branch off early.
    parents = []
    for t in toks:
        parents += [-1 if i == 0 or r.random() < 0.1 else (i - 1 if r.random() < 0.5 else r.randrange(i)) for i in range(t)]
    return rows, toks, parents


def _tables(rows, hd):
    """cos and sin of pos * 500000^(-2i/hd), the angles in 64 bits."""
    ang = np.arange(rows, dtype=np.float64)[:, None] * 500000.0 ** (-np.arange(0, hd, 2, dtype=np.float64) / hd)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def prepare(case, seed):
    h, kv, hd = HEADS[case["heads"]]
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    if case["op"] == "cache":
        rows, toks, parents = [case["pos0"]], [case["rows"]], None
    else:
        rows, toks, parents = _sizes(case)
    n, total, longest = len(rows), sum(toks), max(rows)
    max_seq = max(a + b for a, b in zip(rows, toks)) + 1
    cos, sin = _tables(max_seq, hd)
    state = {"case": case, "slots": np.arange(n, dtype=np.int32), "rows": np.array(rows, np.int32), "toks": np.array(toks, np.int32),
             "parents": None if parents is None else np.array(parents, np.int32), "k": _randn(gen, total, kv, hd), "v": _randn(gen, total, kv, hd)}
    # keys and values of trained models differ in size from channel to channel
    size = 0.25 + 1.5 * torch.rand(2, kv, hd, device="cuda", generator=gen)
    state["k"] *= size[0]
    state["v"] *= size[1]
    if case["op"] != "cache":
        state["q"] = _randn(gen, total, h, hd)
    if own:
        from leap_b200 import AttentionContext
        state["ctx"] = AttentionContext(1, h, kv, hd, max_seq, max_batch=n, rope_cos=cos, rope_sin=sin, kv="q8")
    else:
        state["cos"], state["sin"] = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        state["codes"] = torch.zeros(2, n, kv, longest, hd, dtype=torch.int8, device="cuda")
        state["scales"] = torch.zeros(2, n, kv, longest, device="cuda")
    if case["op"] != "cache":  # the rows that are cached already (keys as they are after the rotation)
        for i, c in enumerate(rows):
            k, v = (_randn(gen, c, kv, hd) * s for s in size)
            if own:
                state["ctx"].kv_write(i, 0, 0, k, v)
            else:
                for j, x in enumerate((k, v)):
                    codes, scales = _keep(x)
                    state["codes"][j, i, :, :c] = codes.transpose(0, 1).to(torch.int8)
                    state["scales"][j, i, :, :c] = scales.transpose(0, 1)
    return state


def _keep(x):
    """Codes (whole numbers) and scales of rows x [..., hd]; the quotients in
    64 bits, since a code depends on which side of a half they lie."""
    s = x.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)
    c = torch.round(x.double() / torch.where(s > 0, s, 1.0).double()[..., None]).clamp(-127, 127)
    return c, s


def _kept(x):
    c, s = _keep(x)
    return c.float() * s[..., None]


def _turn(x, c, s):
    """Interleaved pairs of x [tokens, heads, hd] turned by (c, s) [tokens, hd/2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = c[:, None], s[:, None]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def run(state):
    op = state["case"]["op"]
    if own:
        ctx, slots, rows, toks = state["ctx"], state["slots"], state["rows"], state["toks"]
        if op == "cache":
            ctx.kv_write(0, 0, int(rows[0]), state["k"], state["v"])
            return ctx.kv_read_device(0, 0, int(rows[0]), int(toks[0]))
        if op == "decode":
            return ctx.decode_batched(0, slots, rows, state["q"], state["k"], state["v"])
        if op == "tree":
            return ctx.decode_tree(0, slots, rows, toks, state["parents"], state["q"], state["k"], state["v"])
        out = ctx.prefill_packed(0, slots, rows, toks, state["q"], state["k"], state["v"])
        return (out, *ctx.kv_read_packed(0, slots, rows, toks))
    if op == "cache":
        return _kept(state["k"]), _kept(state["v"])
    dev = state["q"].device
    rows, toks = (torch.from_numpy(state[x]).to(dev).long() for x in ("rows", "toks"))
    n, (total, h, hd), kv = len(toks), state["q"].shape, state["k"].shape[1]
    longest, width = int(state["rows"].max()), int(state["toks"].max())
    first = torch.cumsum(toks, 0) - toks
    of = torch.repeat_interleave(torch.arange(n, device=dev), toks, output_size=total)  # the sequence of each token,
    at = torch.arange(total, device=dev) - first[of]                                    # and its place in the run
    i = torch.arange(width, device=dev)
    sees = (i[None, :] <= i[:, None]).expand(n, width, width)  # of the run: a token sees those up to itself
    turn = rows[of] + at                                       # its angle: that of its row
    if op == "tree":
        up = torch.eye(width, dtype=torch.float64, device=dev).repeat(n, 1, 1)
        parents = torch.from_numpy(state["parents"]).to(dev).long()
        up[of, at, torch.where(parents < 0, at, parents)] = 1.0
        sees = torch.linalg.matrix_power(up, width) > 0        # itself and its ancestors
        turn = rows[of] + sees[of, at].sum(-1) - 1             # its angle: that of its depth
    q = _turn(state["q"], state["cos"][turn], state["sin"][turn])
    new = torch.stack([_kept(_turn(state["k"], state["cos"][turn], state["sin"][turn])), _kept(state["v"])])
    # keys and values [2, n, kv, longest + width, hd]: the cached rows, then the run
    all_ = torch.zeros(2, n, kv, longest + width, hd, device=dev)
    all_[:, :, :, :longest] = state["codes"].float() * state["scales"][..., None]
    all_[:, of, :, longest + at] = new.transpose(0, 1)
    sees = torch.cat([(torch.arange(longest, device=dev) < rows[:, None])[:, None, :].expand(n, width, longest), sees], -1)
    qs = torch.zeros(n, width, h, hd, device=dev)
    qs[of, at] = q
    qs = qs.view(n, width, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)
    s = (qs @ all_[0].transpose(-1, -2)).view(n, kv, h // kv, width, -1) * (1.0 / math.sqrt(hd))
    s = s.masked_fill_(~sees[:, None, None], float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (s.view(n, kv, -1, s.shape[-1]) @ all_[1]).view(n, kv, h // kv, width, hd) / s.sum(-1, keepdim=True)
    out = o.permute(0, 3, 1, 2, 4).reshape(n, width, h, hd)[of, at]
    return (out, new[0], new[1]) if op == "prefill" else out


def work(case):
    h, kv, hd = HEADS[case["heads"]]
    row = 2 * kv * (hd + 4)     # a cached row: codes and scales of k and v
    fresh = 2 * kv * hd * 4     # the same before it is quantised, or read back
    if case["op"] == "cache":
        return {"bytes": case["rows"] * (fresh + row + row + fresh), "flops": 0}
    rows, toks, parents = _sizes(case)
    total = sum(toks)
    moved = sum(rows) * row + total * (row + fresh + 2 * h * hd * 4)
    if case["op"] == "prefill":
        moved += total * (row + fresh)
        pairs = sum(r * t + t * (t + 1) // 2 for r, t in zip(rows, toks))
    elif case["op"] == "decode":
        pairs = sum(r + 1 for r in rows)
    else:
        depth, seen = [], 0
        for r, t in zip(rows, toks):
            mine = parents[seen:seen + t]
            d = []
            for p in mine:
                d.append(1 if p < 0 else d[p] + 1)
            depth.append(sum(d))
            seen += t
        pairs = sum(r * t + d for r, t, d in zip(rows, toks, depth))
    return {"bytes": moved, "flops": 4 * h * hd * pairs}


def exact(case, seed):
    """From the definition, sequence by sequence in 64 bits; the stored rows'
    scales and the rotated keys are rounded to FP32, as they are defined to be."""
    kept_own = globals()["own"]
    globals()["own"] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()["own"] = kept_own

    def stored(x):  # x in FP32, [rows, kv, hd]
        top = x.abs().max(-1, keepdim=True).values
        s = (top.double() * float(np.float32(1.0) / np.float32(127.0))).float().double()
        return torch.where(s > 0, torch.round(x.double() / s.clamp_min(1e-300)), 0.0).clamp(-127, 127) * s

    if case["op"] == "cache":
        return stored(st["k"]), stored(st["v"])
    h, kv, hd = HEADS[case["heads"]]
    rows, toks, parents = _sizes(case)
    outs, ks, vs, seen = [], [], [], 0
    for i, (r, t) in enumerate(zip(rows, toks)):
        mine = slice(seen, seen + t)
        vis = torch.tril(torch.ones(t, t, dtype=torch.bool))
        place = list(range(t))
        if parents is not None:
            vis, place = torch.eye(t, dtype=torch.bool), []
            for a, p in enumerate(parents[mine]):
                if p >= 0:
                    vis[a] |= vis[p]
                place.append(0 if p < 0 else place[p] + 1)
        seen += t
        ang = [r + p for p in place]
        c, s = (st[x][ang].double()[:, None] for x in ("cos", "sin"))
        k, q = st["k"][mine].double(), st["q"][mine].double()
        k0, k1, q0, q1 = k[..., ::2], k[..., 1::2], q[..., ::2], q[..., 1::2]
        k = torch.empty_like(k, dtype=torch.float32)
        k[..., ::2] = ((k0 * c).float().double() - (k1 * s).float().double()).float()
        k[..., 1::2] = ((k1 * c).float().double() + (k0 * s).float().double()).float()
        qr = torch.empty_like(q)
        qr[..., ::2], qr[..., 1::2] = q0 * c - q1 * s, q1 * c + q0 * s
        ks.append(stored(k))
        vs.append(stored(st["v"][mine]))
        old = st["codes"][:, i, :, :r].double() * st["scales"][:, i, :, :r, None].double()
        keys, vals = (torch.cat([o, x.transpose(0, 1)], 1) for o, x in zip(old, (ks[-1], vs[-1])))
        hide = torch.cat([torch.zeros(t, r, dtype=torch.bool), ~vis], 1).cuda()
        o = torch.empty(t, h, hd, dtype=torch.float64, device="cuda")
        for a in range(h):
            for b in range(0, t, 2048):
                e = qr[b:b + 2048, a] @ keys[a // (h // kv)].T / math.sqrt(hd)
                o[b:b + 2048, a] = torch.softmax(e.masked_fill(hide[b:b + 2048], -math.inf), -1) @ vals[a // (h // kv)]
        outs.append(o)
    out = torch.cat(outs)
    return (out, torch.cat(ks), torch.cat(vs)) if case["op"] == "prefill" else out
