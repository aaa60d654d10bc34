// attn_q8_rows.cu — attention of a few query rows for each kv head (decode;
// drafted trees and prompt ends of up to 8 rows = tokens x heads of a group)
// over the 8-bit KV cache, fused with the rotation, quantisation and append of
// the new rows.
//
//   s_j = s_kj * (rope(q) . c_kj) / sqrt(hd),  out = sum_j p_j s_vj c_vj / sum_j p_j
//
// What bounds it: 2*(HD + 4) bytes a cached row and kv head must come from HBM,
// a quarter of the FP32 cache's.  At that rate the FP32 kernel's CUDA-core sums
// (2*G*HD multiply-adds a row, plus the conversion of 2*HD codes) take longer
// than the bytes, so the products run on mma.sync (q8_tile.cuh).  tcgen05 has
// nothing to give here: its 128-row tiles would be 16 times empty.
//
// This kernel is for little work (see q8_rows_attend): splits of a sequence, a block
// each, in one wave where that is best.
//  * A warp works alone: it streams its own tiles of 32 rows (K and V codes and
//    scales, one bulk copy each) through its own ring of shared-memory buffers
//    and keeps its own running maximum, sum and output.  No barrier is shared
//    until the block joins its warps.
//  * Splits of one (sequence, kv head) are joined by the block that is last
//    (atomic ticket).
#include <algorithm>

#include "q8_tile.cuh"

namespace leap {
namespace {

constexpr int kTile = 32;       // rows a warp takes at a time
constexpr int kNew = 16;        // rows of the new tokens' tile (at most 8 used)

constexpr int W = 8;            // warps of a block
template <int HD>
struct Rows {
    static constexpr int kStageBytes = 2 * kTile * HD + 2 * kTile * 4;
    static constexpr int kStages = HD == 128 ? 3 : 5;
    static constexpr int kRing = W * kStages * kStageBytes;
    static constexpr int kNewBytes = 2 * kNew * HD + 2 * kNew * 4;
    static constexpr int kQBytes = 2 * kQ8Rows * HD * 2;
    static constexpr size_t kSmem = size_t(kRing) + kNewBytes + kQBytes;
    static_assert(W * kQ8Rows * HD * 4 <= kRing, "the warps' outputs are joined in the ring");
};

// Block (x, y): split x of the batch's plan, kv head y.  Row r of the up to 8
// query rows is new token r / G, head y*G + r % G.
template <int HD, int G, bool TREE>
__global__ void __launch_bounds__(32 * W, 1)
q8_rows_kernel(const RowsArgs a, const __grid_constant__ Q8Seqs tab,
               const __grid_constant__ Q8Splits plan, const __grid_constant__ Q8See<TREE> see) {
    using C = Rows<HD>;
    using M = TileMath<HD, kTile, 1>;
    constexpr int E = HD / 32;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bars[W][C::kStages];
    __shared__ float s_fac[kQ8Rows], s_m[W][kQ8Rows], s_l[W][kQ8Rows];
    __shared__ int s_fail, s_last;
    unsigned char *s_new = smem + C::kRing;
    __half *s_q = reinterpret_cast<__half *>(s_new + C::kNewBytes);  // [hi, lo][8][HD]
    float *s_nks = reinterpret_cast<float *>(s_new + 2 * kNew * HD), *s_nvs = s_nks + kNew;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.y;
    int seq = 0;
    {
        int hi = tab.n_seq - 1;
        while (seq < hi) {
            const int mid = (seq + hi + 1) >> 1;
            if (plan.split0[mid] <= int(blockIdx.x)) seq = mid; else hi = mid - 1;
        }
    }
    const int nsplit = plan.split0[seq + 1] - plan.split0[seq];
    const int split = blockIdx.x - plan.split0[seq];
    const int t0 = tab.tok0[seq], n_new = tab.tok0[seq + 1] - t0, pos = tab.pos[seq];
    const int n_rows = n_new * G;
    const int row0 = split * plan.chunk, row1 = min(row0 + plan.chunk, pos);
    const bool last_split = split == nsplit - 1;
    const size_t r0 = tab.slot[seq] * a.L.slot_rows + h * a.L.head_rows;
    uint8_t *gk = a.L.k + r0 * HD, *gv = a.L.v + r0 * HD;
    float *gks = a.L.ks + r0, *gvs = a.L.vs + r0;

    // ---- this warp's tiles: warp, warp + W, ... of the split -----------------
    unsigned char *ring = smem + warp * C::kStages * C::kStageBytes;
    const int n_all = row1 > row0 ? (row1 - row0 + kTile - 1) / kTile : 0;
    const int n_tiles = n_all > warp ? (n_all - warp + W - 1) / W : 0;
    if (lane == 0)
        for (int i = 0; i < C::kStages; ++i) mbar_init(&bars[warp][i], 1);
    if (tid == 0) s_fail = 0;
    fence_mbar_init();
    __syncwarp();
    auto request = [&](int i) {
        // whole groups of 8 rows (the cache has room for 128 at a time): rows
        // past the end are read as they are and masked
        const int first = row0 + (warp + i * W) * kTile;
        const int n = min(kTile, (row1 - first + 7) & ~7);
        unsigned char *st = ring + (i % C::kStages) * C::kStageBytes;
        uint64_t *bar = &bars[warp][i % C::kStages];
        mbar_arrive_expect_tx(bar, 2 * n * HD + 2 * n * 4);
        bulk_g2s(st, gk + size_t(first) * HD, n * HD, bar);
        bulk_g2s(st + 2 * kTile * HD, gks + first, n * 4, bar);
        bulk_g2s(st + kTile * HD, gv + size_t(first) * HD, n * HD, bar);
        bulk_g2s(st + 2 * kTile * HD + kTile * 4, gvs + first, n * 4, bar);
    };
    int asked = 0;
    if (lane == 0)
        for (; asked < min(C::kStages, n_tiles); ++asked) request(asked);
    asked = min(C::kStages, n_tiles);
    // Only cached rows of this layer were asked for so far, which the previous
    // kernel of the stream never writes (the host allows the overlap only then).
    grid_dependency_wait();
    grid_launch_dependents();

    // ---- queries ---------------------------------------------------------------
    for (int r = warp; r < kQ8Rows; r += W) {
        const int i = min(r / G, n_new - 1);  // rows past the last repeat it (not stored)
        QueryRow<HD> row;
        row.load(a.q + (size_t(t0 + i) * a.L.n_kv * G + h * G + r % G) * HD, a.rope_cos, a.rope_sin,
                 pos + see.depth(t0, i));
        const float f = row.stage(a.scale_log2, s_q, r);
        if (lane == 0) s_fac[r] = f;
    }
    // ---- the last split's block appends the new rows, and keeps them as a tile -
    if (last_split) {
        for (int w = warp; w < 2 * kNew; w += W) {
            const int i = w >> 1;
            const bool is_v = w & 1;
            uint32_t codes = E == 4 ? 0x80808080u : 0x8080u;
            float s = 0.f;
            if (i < n_new)
                s = q8_append_row<HD>((is_v ? a.v_new : a.k_new) + (size_t(t0 + i) * a.L.n_kv + h) * HD, !is_v,
                                      a.rope_cos, a.rope_sin, pos + see.depth(t0, i), is_v ? gv : gk,
                                      is_v ? gvs : gks, pos + i, codes);
            q8_store_codes<HD>(s_new + (is_v ? kNew * HD : 0), i, lane, codes);
            if (lane == 0) (is_v ? s_nvs : s_nks)[i] = s;
        }
    }
    __syncthreads();

    const int g = lane >> 2, t = lane & 3;
    const float fac = s_fac[g];
    float m = -INFINITY, l = 0.f, o[M::NT][2];
#pragma unroll
    for (int i = 0; i < M::NT; ++i) o[i][0] = o[i][1] = 0.f;

    bool ok = true;
    int tile = 0;
    for (; tile < n_tiles; ++tile) {
        const int b = tile % C::kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][b], (tile / C::kStages) & 1));
        if (!ok) break;
        const unsigned char *st = ring + b * C::kStageBytes;
        const float *sks = reinterpret_cast<const float *>(st + 2 * kTile * HD), *svs = sks + kTile;
        const int n = row1 - (row0 + (warp + tile * W) * kTile);  // rows of it that are cached
        float s[kTile / 8][2];
        M::scores(st, sks, s_q, fac, s);
        if (n < kTile) {
#pragma unroll
            for (int j = 0; j < kTile / 8; ++j) {
                if (8 * j + 2 * t >= n) s[j][0] = -INFINITY;
                if (8 * j + 2 * t + 1 >= n) s[j][1] = -INFINITY;
            }
        }
        M::absorb(st + kTile * HD, svs, s, m, l, o);
        __syncwarp();  // the buffer is free
        if (asked < n_tiles) {
            if (lane == 0) request(asked);
            ++asked;
        }
    }
    if (!ok) {  // wait, bounded again, for what is still on its way
        for (int i = tile + 1; i < asked; ++i) (void)mbar_wait(&bars[warp][i % C::kStages], (i / C::kStages) & 1);
        if (lane == 0) atomicExch(&s_fail, 1);
    } else if (last_split && warp == W - 1) {  // (the warp with the fewest tiles)
        using N = TileMath<HD, kNew, 1>;
        float s[kNew / 8][2];
        N::scores(s_new, s_nks, s_q, fac, s);
        const int mine = g / G;  // token of row g; rows past n_rows see nothing here
#pragma unroll
        for (int j = 0; j < kNew / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = 8 * j + 2 * t + e;
                if (mine >= n_new || !see.sees(t0, mine, key)) s[j][e] = -INFINITY;
            }
        N::absorb(s_new + kNew * HD, s_nvs, s, m, l, o);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();  // every warp is done with its ring (or gave up)
    if (s_fail) {
        if (tid == 0) report_error(a.err, a.err_host, kDevWaitTimeout);
        return;
    }

    // ---- join the warps: thread f of 8*HD/4 holds 4 dims of one row -------------
    float *s_o = reinterpret_cast<float *>(smem);  // [W][8][HD]
    if (t == 0) {
        s_m[warp][g] = m;
        s_l[warp][g] = l;
    }
    // thread (g, t) has dims 2t*HD/8 + i and (2t+1)*HD/8 + i: HD/4 in a row
#pragma unroll
    for (int i = 0; i < M::NT; i += 4) {
        float *d = s_o + (warp * kQ8Rows + g) * HD + t * (HD / 4) + i;
        *reinterpret_cast<float4 *>(d) = make_float4(o[i][0], o[i + 1][0], o[i + 2][0], o[i + 3][0]);
        *reinterpret_cast<float4 *>(d + HD / 8) = make_float4(o[i][1], o[i + 1][1], o[i + 2][1], o[i + 3][1]);
    }
    __syncthreads();
    const size_t part0 = size_t(h) * plan.split0[tab.n_seq] + plan.split0[seq];  // this (sequence, head)'s first
    for (int f = tid; f < n_rows * (HD / 4); f += 32 * W) {
        const int r = f / (HD / 4), d = (f % (HD / 4)) * 4;
        float mx = s_m[0][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < W; ++w) mx = fmaxf(mx, s_m[w][r]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float e = s_m[w][r] == -INFINITY ? 0.f : fast_exp2(s_m[w][r] - mx);
            const float4 x = *reinterpret_cast<const float4 *>(s_o + (w * kQ8Rows + r) * HD + d);
            sum += s_l[w][r] * e;
            v.x += x.x * e; v.y += x.y * e; v.z += x.z * e; v.w += x.w * e;
        }
        if (nsplit == 1) {
            const float inv = 1.f / sum;
            const size_t at = (size_t(t0 + r / G) * a.L.n_kv * G + h * G + r % G) * HD + d;
            *reinterpret_cast<float4 *>(a.out + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        } else {
            const size_t p = (part0 + split) * kQ8Rows + r;
            *reinterpret_cast<float4 *>(a.part_o + p * HD + d) = v;
            if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * p) = make_float2(part_max(mx, sum), sum);
        }
    }
    if (nsplit == 1) return;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        unsigned *c = a.counters + seq * a.L.n_kv + h;
        s_last = atom_add_acq_rel_gpu(c, 1u) == unsigned(nsplit - 1);
        if (s_last) *c = 0;  // for the next launch
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    // ---- join the splits: the threads' groups take every ng-th --------------------
    const int items = n_rows * (HD / 4);  // at most 256
    const int ng = 32 * W / items, grp = tid / items;
    float mx = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const int f = tid - grp * items, r = f / (HD / 4), d = (f % (HD / 4)) * 4;
    if (grp < ng) {
        constexpr int U = 8;
        for (int s0 = grp; s0 < nsplit; s0 += U * ng) {
            float4 z[U];
            float2 y[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int s = min(s0 + k * ng, nsplit - 1);
                const size_t p = (part0 + s) * kQ8Rows + r;
                z[k] = __ldcg(reinterpret_cast<const float4 *>(a.part_o + p * HD + d));
                y[k] = __ldcg(reinterpret_cast<const float2 *>(a.part_ml + 2 * p));
                if (s0 + k * ng >= nsplit) y[k].x = -INFINITY;
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
    }
    if (ng > 1) {  // through the ring's place
        float4 *s_v = reinterpret_cast<float4 *>(smem);
        float2 *s_y = reinterpret_cast<float2 *>(smem + 32 * W * 16);
        if (grp < ng) {
            s_v[tid] = v;
            s_y[tid] = make_float2(part_max(mx, sum), sum);
        }
        __syncthreads();
        if (grp == 0)
            for (int k = 1; k < ng; ++k) {
                const float4 z = s_v[k * items + f];
                const float2 y = s_y[k * items + f];
                if (y.x == -INFINITY) continue;
                const float top = fmaxf(mx, y.x);
                const float e0 = mx == -INFINITY ? 0.f : fast_exp2(mx - top), e1 = fast_exp2(y.x - top);
                mx = top;
                sum = sum * e0 + y.y * e1;
                v.x = v.x * e0 + z.x * e1; v.y = v.y * e0 + z.y * e1;
                v.z = v.z * e0 + z.z * e1; v.w = v.w * e0 + z.w * e1;
            }
        __syncthreads();
    }
    if (grp == 0) {
        const float inv = 1.f / sum;
        const size_t to = (size_t(t0 + r / G) * a.L.n_kv * G + h * G + r % G) * HD + d;
        *reinterpret_cast<float4 *>(a.out + to) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

template <int HD, int G, bool TREE>
int launch_rows(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Splits &plan,
                const Q8See<TREE> &see, bool overlap) {
    auto fn = q8_rows_kernel<HD, G, TREE>;
    if (int st = set_kernel_smem(reinterpret_cast<const void *>(fn), Rows<HD>::kSmem,
                                 "cudaFuncSetAttribute(q8_rows)"))
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.split0[tab.n_seq], c->n_kv);
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = Rows<HD>::kSmem;
    cfg.stream = c->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, fn, a, tab, plan, see), "q8_rows_kernel launch");
}

template <int HD, int G>
int launch_rows_g(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Splits &plan,
                  const Q8Tree *tree, bool overlap) {
    return tree ? launch_rows<HD, G, true>(c, a, tab, plan, q8_see(*tree), overlap)
                : launch_rows<HD, G, false>(c, a, tab, plan, Q8See<false>(), overlap);
}

// Rows of a split, at least kMinChunk.  What a batch costs, in rows that a block
// streams (140 a us with 128 dims, 220 with 64): a block besides its rows kBlock, the
// joins at the end kJoin (8 kv heads of 128 on the device, sequences x cached rows:
// 1x128, one block each, 5.4 us; 1x512 in 4 splits 8.2; 16x8192, one each, 61;
// 32x2048, two waves, 40).
constexpr int kMinChunk = 128;
constexpr long kBlock = 512, kJoin = 320;

// Splits with the least cost; returns it.  One wave of a block an SM takes as long as
// its longest, more take about all work / SMs and half the longest block at the end.
long plan_splits(const leap_ctx *c, const Q8Seqs &tab, Q8Splits &plan) {
    long total = 0;
    unsigned longest = 0, n_any = 0;
    for (int i = 0; i < tab.n_seq; ++i)
        if (tab.tok0[i + 1] > tab.tok0[i]) {
            total += tab.pos[i];
            longest = std::max(longest, unsigned(tab.pos[i]));
            ++n_any;
        }
    auto splits = [&](int i, unsigned ch) {
        return tab.tok0[i + 1] == tab.tok0[i] ? 0u : std::max((unsigned(tab.pos[i]) + ch - 1) / ch, 1u);
    };
    long best = -1;
    unsigned ch = unsigned(std::max(((total * c->n_kv + c->num_sms - 1) / c->num_sms + 63) / 64 * 64, long(kMinChunk)));
    // finer steps where one wave can be had
    const int step = long(n_any) * c->n_kv <= c->num_sms ? 16 : 2;
    for (;; ch += std::max(ch / step / 64 * 64, 64u)) {
        long n = 0;
        for (int i = 0; i < tab.n_seq; ++i) n += splits(i, ch);
        const bool split = longest > ch, wave = n * c->n_kv <= c->num_sms;
        const long last = std::min(ch, longest) + kBlock;
        const long cost = (wave ? last : std::max((total + n * kBlock) * c->n_kv / c->num_sms, last) + last / 2) +
                          (split ? kJoin : 0);
        if ((!split || n * c->n_kv <= c->q8_parts) && (best < 0 || cost < best)) {
            best = cost;
            plan.chunk = int(ch);
        }
        if (wave || !split) break;
    }
    int n = 0;
    for (int i = 0; i < tab.n_seq; ++i) {
        plan.split0[i] = n;
        n += int(splits(i, unsigned(plan.chunk)));
    }
    plan.split0[tab.n_seq] = n;
    return best;
}

}  // namespace

int q8_rows_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
                   const float *k, const float *v, float *out) {
    RowsArgs a;
    a.q = q;
    a.k_new = k;
    a.v_new = v;
    a.out = out;
    a.L = q8_layer(c, layer);
    a.rope_cos = c->rope_cos;
    a.rope_sin = c->rope_sin;
    a.part_o = c->q8_part_o;
    a.part_ml = c->q8_part_ml;
    a.counters = c->q8_counters;
    a.err = c->d_err;
    a.err_host = c->err_host;
    a.scale_log2 = kLog2e / sqrtf(float(c->hd));
    // as launch_decode: only if the previous operation did not write this layer
    const bool overlap = c->overlap && c->last_written_layer != leap_ctx::kWroteAll &&
                         c->last_written_layer != layer;
    Q8Splits plan;
    // Measured against expected (device us of the rows, warps kernel; 8 kv heads of 128,
    // 4 query heads each): 1x8192 10.1, 44.8; 8x8192 35.4, 41.0; 16x8192 60.6, 58.5;
    // 20x2048 35.6, 26.5; 64x512 33.2, 23.6; 64x8192 239, 180; one of 32768 among 20
    // short ones 34, 90, among 64 65, 68; 4x32768 63, 73; 8x32768 118, 105.  Of 222
    // batches (heads 32/8, 32/32, 16/2 and 8/1 of 128, 32/8 and 32/4 of 64) the taken one
    // was within 10% of the other in all but one (36x1024 of 32/8x64: 18.5, 15.2).
    if (q8_warps_cost(c, tab) < plan_splits(c, tab, plan)) return q8_warps_launch(c, a, tab, tree, overlap);
    switch (c->hd * 100 + c->group) {
        case 12801: return launch_rows_g<128, 1>(c, a, tab, plan, tree, overlap);
        case 12802: return launch_rows_g<128, 2>(c, a, tab, plan, tree, overlap);
        case 12804: return launch_rows_g<128, 4>(c, a, tab, plan, tree, overlap);
        case 12808: return launch_rows_g<128, 8>(c, a, tab, plan, tree, overlap);
        case 6401: return launch_rows_g<64, 1>(c, a, tab, plan, tree, overlap);
        case 6402: return launch_rows_g<64, 2>(c, a, tab, plan, tree, overlap);
        case 6404: return launch_rows_g<64, 4>(c, a, tab, plan, tree, overlap);
        case 6408: return launch_rows_g<64, 8>(c, a, tab, plan, tree, overlap);
        default:
            set_error("unsupported head_dim %d / kv_mul %d", c->hd, c->group);
            return LEAP_ERR_INVALID;
    }
}

}  // namespace leap
