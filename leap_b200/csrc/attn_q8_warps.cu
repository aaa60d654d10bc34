// attn_q8_warps.cu — attention of a few query rows for each kv head over the
// 8-bit KV cache, for batches with much cached (decode of many sequences): every
// warp on its own.
//
// What bounds it: the cache's bytes, 2*(HD + 4) a row and kv head.  All tiles (32
// rows) of all (sequence, kv head) items are one list, cut in equal parts for all
// warps of the GPU (two blocks of 8 an SM).  A warp streams its tiles through its
// own two buffers (K's is free for the next copy while V is worked on), and where
// an item ends it stages the next item's queries and leaves its part of the sums,
// or the output, alone: no block ever waits for its warps, so the other 15 of an
// SM keep the copies going.  64 sequences of 512 to 8192 rows, 8 kv heads of 128:
// 106 us one launch after another, 112 to 114 us where nothing is in the L2 (5.1 TB/s); blocks
// that walked such a list together lost about 9 us an item to their joins (141 us).  The parts of an item are joined by the warp that is last (atomic
// ticket).  The products are those of q8_tile.cuh.
//
// New rows are appended by the warp that reads the tile they fall in, before it
// asks for the tile: the tile then comes back with them.
#include <algorithm>

#include "q8_tile.cuh"

namespace leap {
namespace {

constexpr int kWarps = 8;       // of a block; two blocks an SM
constexpr int kTile = 32;
constexpr int kPad = 1;         // an item's cost besides its tiles, in tiles

template <int HD>
struct Warps {
    static constexpr int kHalf = kTile * HD + kTile * 4;     // codes and scales of K or of V
    static constexpr int kQBytes = 2 * kQ8Rows * HD * 2;
    static constexpr int kWarp = 2 * kHalf + kQBytes;
    static constexpr size_t kSmem = size_t(kWarps) * kWarp;
};

// Where a warp's range of units meets an item.
struct Segment {
    int seq, h;
    int item0, tiles;  // the item's first unit, and how many tiles it has
    int a, b;          // its tiles that are this warp's (none in its padding)
    __device__ __forceinline__ int next() const { return item0 + tiles + kPad; }
};

// A unit is a tile of one (sequence, kv head), an item; units are numbered through
// all items, kPad empty ones behind each, and warp w of the grid has `chunk` of
// them from w * chunk on.  Row r of an item's up to 8 query rows is new token
// r / G, head h*G + r % G.
template <int HD, int G, bool TREE>
__global__ void __launch_bounds__(32 * kWarps, 2)
q8_warps_kernel(const __grid_constant__ RowsArgs a, const __grid_constant__ Q8Seqs tab,
                const __grid_constant__ Q8Units plan, const __grid_constant__ Q8See<TREE> see) {
    using C = Warps<HD>;
    using M = TileMath<HD, kTile, 2>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bars[kWarps][2];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int self = blockIdx.x * kWarps + warp;
    const int u0 = min(self * plan.chunk, plan.unit0[tab.n_seq]), u1 = min(u0 + plan.chunk, plan.unit0[tab.n_seq]);
    unsigned char *buf = smem + warp * C::kWarp;  // K, V
    __half *s_q = reinterpret_cast<__half *>(buf + 2 * C::kHalf);

    auto segment_at = [&](int u) {
        Segment s;
        int lo = 0, hi = tab.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (plan.unit0[mid] <= u) lo = mid; else hi = mid - 1;
        }
        s.seq = lo;
        s.tiles = (tab.pos[lo] + tab.tok0[lo + 1] - tab.tok0[lo] + kTile - 1) / kTile;
        s.h = (u - plan.unit0[lo]) / (s.tiles + kPad);
        s.item0 = plan.unit0[lo] + s.h * (s.tiles + kPad);
        s.a = min(u - s.item0, s.tiles);
        s.b = min(s.tiles, u1 - s.item0);
        return s;
    };
    auto first_row = [&](const Segment &s) { return tab.slot[s.seq] * a.L.slot_rows + s.h * a.L.head_rows; };
    // the next tile's first row in the cache, and how many rows of it to copy: whole
    // groups of 8 (the cache has room for 128 at a time); rows past the end are read
    // as they are and masked
    size_t ask_row = 0;
    int ask_n = 0;
    auto aim = [&](const Segment &s, int ti) {
        const int end = tab.pos[s.seq] + tab.tok0[s.seq + 1] - tab.tok0[s.seq];
        ask_row = first_row(s) + ti * kTile;
        ask_n = min(kTile, (end - ti * kTile + 7) & ~7);
    };
    auto ask = [&](int v) {  // into the K (0) or V (1) buffer
        if (lane == 0) {
            unsigned char *st = buf + v * C::kHalf;
            uint64_t *bar = &bars[warp][v];
            mbar_arrive_expect_tx(bar, ask_n * (HD + 4));
            bulk_g2s(st, (v ? a.L.v : a.L.k) + ask_row * HD, ask_n * HD, bar);
            bulk_g2s(st + kTile * HD, (v ? a.L.vs : a.L.ks) + ask_row, ask_n * 4, bar);
        }
    };
    // the new rows that fall in tile ti, before it is asked for
    auto append = [&](const Segment &s, int ti) {
        const int pos = tab.pos[s.seq], t0 = tab.tok0[s.seq], n_new = tab.tok0[s.seq + 1] - t0;
        const size_t r0 = first_row(s);
        for (int i = max(ti * kTile - pos, 0); i < min((ti + 1) * kTile - pos, n_new); ++i) {
            const size_t src = (size_t(t0 + i) * a.L.n_kv + s.h) * HD;
            const int at = pos + see.depth(t0, i);
            uint32_t codes;
            q8_append_row<HD>(a.k_new + src, true, a.rope_cos, a.rope_sin, at, a.L.k + r0 * HD, a.L.ks + r0, pos + i, codes);
            q8_append_row<HD>(a.v_new + src, false, a.rope_cos, a.rope_sin, at, a.L.v + r0 * HD, a.L.vs + r0, pos + i, codes);
        }
        fence_proxy_async_global();  // the copy reads what was stored here
        __syncwarp();
    };
    auto has_new = [&](const Segment &s, int ti) { return (ti + 1) * kTile > tab.pos[s.seq]; };

    if (lane == 0) {
        mbar_init(&bars[warp][0], 1);
        mbar_init(&bars[warp][1], 1);
    }
    fence_mbar_init();
    __syncwarp();
    // the next tile to ask for
    Segment as = {};
    int at = 0;
    bool more = false;
    auto settle = [&](int u) {  // to the first tile of this warp from unit u on
        more = false;
        while (u < u1) {
            as = segment_at(u);
            if (as.a < as.b) {
                at = as.a;
                more = true;
                return;
            }
            u = as.next();
        }
    };
    settle(u0);
    Segment sg = as;
    int ti = at;
    bool on = more;
    const bool early = on && !has_new(sg, ti);
    if (on) aim(sg, ti);
    if (early) {
        ask(0);
        ask(1);
    }
    // Only cached rows of this layer were asked for so far, which the previous
    // kernel of the stream never writes (the host allows the overlap only then).
    grid_dependency_wait();
    grid_launch_dependents();
    if (on && !early) {
        append(sg, ti);
        ask(0);
        ask(1);
    }

    uint32_t phase = 0;
    bool ok = true;
    while (on && ok) {
        const int t0 = tab.tok0[sg.seq], n_new = tab.tok0[sg.seq + 1] - t0, pos = tab.pos[sg.seq];
        // ---- the item's queries --------------------------------------------------
        float fac = 0.f;
        {
            QueryRow<HD> row[kQ8Rows / 2];
#pragma unroll
            for (int r0 = 0; r0 < kQ8Rows; r0 += kQ8Rows / 2) {
                if (r0 >= n_new * G) break;  // rows without a query: whatever is there
#pragma unroll
                for (int r = 0; r < kQ8Rows / 2; ++r) {
                    const int i = min((r0 + r) / G, n_new - 1);  // rows past the last repeat it
                    row[r].load(a.q + (size_t(t0 + i) * a.L.n_kv * G + sg.h * G + (r0 + r) % G) * HD, a.rope_cos,
                                a.rope_sin, pos + see.depth(t0, i));
                }
#pragma unroll
                for (int r = 0; r < kQ8Rows / 2; ++r) {
                    const float f = row[r].stage(a.scale_log2, s_q, r0 + r);
                    if (g == r0 + r) fac = f;
                }
            }
        }
        __syncwarp();
        float m = -INFINITY, l = 0.f, o[M::NT][2];
#pragma unroll
        for (int i = 0; i < M::NT; ++i) o[i][0] = o[i][1] = 0.f;

        for (;; ++ti) {
            // what comes after this tile
            if (ti + 1 < sg.b) {
                at = ti + 1;
                more = true;
                ask_row += kTile;
                if (at + 1 == sg.tiles) aim(sg, at);  // the item's last may be short
            } else {
                settle(sg.next());
                if (more) aim(as, at);
            }
            const int k0 = ti * kTile, n = pos - k0;  // keys below n are cached
            float s[kTile / 8][2];
            ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][0], phase));
            if (!ok) break;
            M::scores(buf, reinterpret_cast<const float *>(buf + kTile * HD), s_q, fac, s);
            __syncwarp();
            if (more) {
                if (has_new(as, at)) append(as, at);
                ask(0);
            }
            if (n < kTile) {
                const int mine = g / G;  // token of row g
#pragma unroll
                for (int j = 0; j < kTile / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int i = 8 * j + 2 * t + e - n;  // new token, if not negative
                        if (i >= 0 && (i >= n_new || mine >= n_new || !see.sees(t0, mine, i))) s[j][e] = -INFINITY;
                    }
            }
            ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][1], phase));
            if (!ok) break;
            const float *svs = reinterpret_cast<const float *>(buf + C::kHalf + kTile * HD);
            M::absorb(buf + C::kHalf, svs, s, m, l, o);
            __syncwarp();
            if (more) ask(1);
            phase ^= 1;
            if (ti + 1 >= sg.b) break;
        }
        if (!ok) break;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        // ---- this warp's part: warps w0 .. w0 + ns - 1 have the item; a warp leaves two
        // partials at most, of an item that it begins (odd) and of one that it goes on
        const int n_rows = n_new * G;
        const int w0 = sg.item0 / plan.chunk, ns = (sg.item0 + sg.tiles - 1) / plan.chunk - w0 + 1;
        // thread (g, t) has dims 2t*HD/8 + i and (2t+1)*HD/8 + i: HD/4 in a row
        const size_t p = size_t(2 * self + (sg.a == 0)) * kQ8Rows + g;
        if (g < n_rows) {
            const float by = ns == 1 ? 1.f / l : 1.f;
            float *d = (ns == 1 ? a.out + (size_t(t0 + g / G) * a.L.n_kv * G + sg.h * G + g % G) * HD : a.part_o + p * HD) +
                       t * (HD / 4);
#pragma unroll
            for (int i = 0; i < M::NT; i += 4) {
                *reinterpret_cast<float4 *>(d + i) =
                    make_float4(o[i][0] * by, o[i + 1][0] * by, o[i + 2][0] * by, o[i + 3][0] * by);
                *reinterpret_cast<float4 *>(d + HD / 8 + i) =
                    make_float4(o[i][1] * by, o[i + 1][1] * by, o[i + 2][1] * by, o[i + 3][1] * by);
            }
            if (ns > 1 && t == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * p) = make_float2(part_max(m, l), l);
        }
        if (ns > 1) {
            __threadfence();
            __syncwarp();
            int last = 0;
            if (lane == 0) {
                unsigned *c = a.counters + sg.seq * a.L.n_kv + sg.h;
                last = atom_add_acq_rel_gpu(c, 1u) == unsigned(ns - 1);
                if (last) *c = 0;  // for the next launch
            }
            if (__shfl_sync(0xffffffffu, last, 0)) {
                __threadfence();
                for (int f = lane; f < n_rows * (HD / 4); f += 32) {
                    const int r = f / (HD / 4), d = (f % (HD / 4)) * 4;
                    float mx = -INFINITY, sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int U = 8;
                    for (int s0 = 0; s0 < ns; s0 += U) {
                        float4 z[U];
                        float2 y[U];
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            const int w = min(s0 + k, ns - 1);
                            const size_t q = size_t(2 * (w0 + w) + (w == 0)) * kQ8Rows + r;
                            z[k] = __ldcg(reinterpret_cast<const float4 *>(a.part_o + q * HD + d));
                            y[k] = __ldcg(reinterpret_cast<const float2 *>(a.part_ml + 2 * q));
                            if (s0 + k >= ns) y[k].x = -INFINITY;
                        }
                        float top = mx;
#pragma unroll
                        for (int k = 0; k < U; ++k) top = fmaxf(top, y[k].x);
                        const float back = mx == -INFINITY ? 0.f : fast_exp2(mx - top);
                        mx = top;
                        sum *= back;
                        v.x *= back; v.y *= back; v.z *= back; v.w *= back;
#pragma unroll
                        for (int k = 0; k < U; ++k) {
                            if (y[k].x == -INFINITY) continue;
                            const float e = fast_exp2(y[k].x - top);
                            sum += y[k].y * e;
                            v.x += z[k].x * e; v.y += z[k].y * e; v.z += z[k].z * e; v.w += z[k].w * e;
                        }
                    }
                    const float inv = 1.f / sum;
                    *reinterpret_cast<float4 *>(a.out + (size_t(t0 + r / G) * a.L.n_kv * G + sg.h * G + r % G) * HD + d) =
                        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                }
            }
        }
        on = more;
        sg = as;
        ti = at;
    }
    if (!ok) {
        // a wait gave up: wait, bounded again, for what may still be on its way
        for (int v = 0; v < 2; ++v)
            for (int k = 0; k < 2; ++k) (void)mbar_wait(&bars[warp][v], phase ^ k);
        if (lane == 0) report_error(a.err, a.err_host, kDevWaitTimeout);
    }
}

template <int HD, int G, bool TREE>
int launch(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Units &plan, const Q8See<TREE> &see, bool overlap) {
    auto fn = q8_warps_kernel<HD, G, TREE>;
    if (int st = set_kernel_smem(reinterpret_cast<const void *>(fn), Warps<HD>::kSmem, "cudaFuncSetAttribute(q8_warps)"))
        return st;
    const int warps = (plan.unit0[tab.n_seq] + plan.chunk - 1) / plan.chunk;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((warps + kWarps - 1) / kWarps);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = Warps<HD>::kSmem;
    cfg.stream = c->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, fn, a, tab, plan, see), "q8_warps_kernel launch");
}

template <int HD, int G>
int launch_g(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Units &plan, const Q8Tree *tree, bool overlap) {
    return tree ? launch<HD, G, true>(c, a, tab, plan, q8_see(*tree), overlap)
                : launch<HD, G, false>(c, a, tab, plan, Q8See<false>(), overlap);
}

// Units of all items, and of a warp: equal parts, two tiles at least.
void plan_units(const leap_ctx *c, const Q8Seqs &tab, Q8Units &plan, int *longest) {
    long n = 0;
    *longest = 0;
    for (int i = 0; i < tab.n_seq; ++i) {
        plan.unit0[i] = int(n);
        const int n_new = tab.tok0[i + 1] - tab.tok0[i];
        if (n_new == 0) continue;
        const int tiles = (tab.pos[i] + n_new + kTile - 1) / kTile;
        *longest = std::max(*longest, tiles);
        n += long(tiles + kPad) * c->n_kv;
    }
    plan.unit0[tab.n_seq] = int(n);
    const long warps = long(2 * kWarps) * c->num_sms;
    plan.chunk = int(std::max((n + warps - 1) / warps, 2L));
}

}  // namespace

// Two partials a warp, of those that a batch of the longest sequences has work for.
int q8_warps_parts(const leap_ctx *c) {
    const long units = long(std::min(c->max_batch, kMaxSeqPerLaunch)) * c->n_kv * ((c->max_seq + kTile - 1) / kTile + kPad);
    return 2 * int(std::min((units + 1) / 2, long(2 * kWarps) * c->num_sms));  // plan_units: two units a warp at least
}

// What a batch costs here, in the unit of the rows kernel's plan (1/140 us with 128
// dims): a warp's tiles, and one warp's join of the item in most parts, 8 of a row at a
// time (1x8192 of 8 kv heads, 129 parts: 45 us with 4 rows, 80 with 8).
long q8_warps_cost(const leap_ctx *c, const Q8Seqs &tab) {
    Q8Units plan;
    int longest;
    plan_units(c, tab, plan, &longest);
    int rows = 0;
    for (int i = 0; i < tab.n_seq; ++i) rows = std::max(rows, (tab.tok0[i + 1] - tab.tok0[i]) * c->group);
    return 1080 + 450L * plan.chunk + 9L * rows * ((longest + plan.chunk - 1) / plan.chunk);
}

int q8_warps_launch(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Tree *tree, bool overlap) {
    Q8Units plan;
    int longest;
    plan_units(c, tab, plan, &longest);
    switch (c->hd * 100 + c->group) {
        case 12801: return launch_g<128, 1>(c, a, tab, plan, tree, overlap);
        case 12802: return launch_g<128, 2>(c, a, tab, plan, tree, overlap);
        case 12804: return launch_g<128, 4>(c, a, tab, plan, tree, overlap);
        case 12808: return launch_g<128, 8>(c, a, tab, plan, tree, overlap);
        case 6401: return launch_g<64, 1>(c, a, tab, plan, tree, overlap);
        case 6402: return launch_g<64, 2>(c, a, tab, plan, tree, overlap);
        case 6404: return launch_g<64, 4>(c, a, tab, plan, tree, overlap);
        case 6408: return launch_g<64, 8>(c, a, tab, plan, tree, overlap);
        default:
            set_error("unsupported head_dim %d / kv_mul %d", c->hd, c->group);
            return LEAP_ERR_INVALID;
    }
}

}  // namespace leap
