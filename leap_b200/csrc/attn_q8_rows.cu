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
// than the bytes, so the products run on mma.sync (m16n8k16, FP16 operands,
// FP32 sums).  A query row needs 2 x 11 bits for FP32-like results, and the 16
// rows of the A operand are filled with 8 query rows' high halves and the same
// 8 rows' low halves: hi and lo come out in the same thread's c0/c1 and c2/c3
// and are added there.  Codes are exact in FP16.  tcgen05 has nothing to give
// here: its 128-row tiles would be 16 times empty.
//
//  * A warp works alone: it streams its own tiles of 32 rows (K and V codes and
//    scales, one bulk copy each) through its own ring of shared-memory buffers
//    and keeps its own running maximum, sum and output.  No barrier is shared
//    until the block joins its warps.
//  * The contraction index may be permuted freely as long as both operands
//    agree, so a thread's K operands are whole 16-byte chunks of one row, and
//    its V operands 16-byte chunks of four rows: no transposition, one
//    permute per 2 codes for K and 1.5 for V (half pairs are 0x6400 | code,
//    minus 1152).  q8.cuh's chunk order keeps both reads free of conflicts.
//  * Tensor-core sums are truncated, and a long run of them drifts towards
//    zero; each 32-row tile is summed from zero and joins the FP32 output by an
//    ordinary multiply-add.
//  * p*s_v is scaled by a power of two for each tile so that FP16's range holds
//    it whatever the scales are; the same for each q row.
//  * Splits of one (sequence, kv head) are joined by the block that is last
//    (atomic ticket).
#include "q8.cuh"

namespace leap {
namespace {

constexpr int kTile = 32;       // rows a warp takes at a time
constexpr int kNew = 16;        // rows of the new tokens' tile (at most 8 used)

template <int HD, int W>
struct Rows {
    static constexpr int kStageBytes = 2 * kTile * HD + 2 * kTile * 4;
    static constexpr int kStages = W == 8 ? (HD == 128 ? 3 : 5) : (HD == 128 ? 3 : 5);
    static constexpr int kRing = W * kStages * kStageBytes;
    static constexpr int kNewBytes = 2 * kNew * HD + 2 * kNew * 4;
    static constexpr int kQBytes = 2 * kQ8Rows * HD * 2;
    static constexpr size_t kSmem = size_t(kRing) + kNewBytes + kQBytes;
    static_assert(W * kQ8Rows * HD * 4 <= kRing, "the warps' outputs are joined in the ring");
};

struct RowsArgs {
    const float *q, *k_new, *v_new;
    float *out;
    Q8Layer L;
    const float *rope_cos, *rope_sin;
    float *part_o, *part_ml;
    unsigned *counters;
    int *err, *err_host;
    float scale_log2;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two of four bytes x (codes + 128) as FP16 values code, code.
template <int SEL>
__device__ __forceinline__ uint32_t half_pair(uint32_t x) {
    const uint32_t y = __byte_perm(x, 0x64646464u, SEL);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), __float2half2_rn(1152.f));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// One warp's work on a tile of NK (16 or 32) rows in shared memory.
template <int HD, int NK>
struct TileMath {
    static constexpr int KS = HD / 16;  // 16-dim steps of the score product
    static constexpr int NT = HD / 8;   // 8-dim column tiles of the output

    static __device__ __forceinline__ void scores(const unsigned char *sk, const float *skv,
                                                  const uint32_t (&qa)[KS][4], float fac,
                                                  float (&s)[NK / 8][2]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < HD / 64; ++j) {
                const uint4 w = *reinterpret_cast<const uint4 *>(sk + q8_chunk<HD>(n * 8 + g, t + 4 * j));
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t(&a)[4] = qa[4 * j + u];
                    mma_f16(c, a[0], a[1], a[2], a[3], half_pair<0x5140>(ww[u]), half_pair<0x5342>(ww[u]));
                }
            }
            const float2 f = *reinterpret_cast<const float2 *>(skv + n * 8 + 2 * t);
            s[n][0] = (c[0] + c[2]) * (f.x * fac);
            s[n][1] = (c[1] + c[3]) * (f.y * fac);
        }
    }

    // o, m, l of row g take the tile's rows; s is -inf where a row is not seen.
    static __device__ __forceinline__ void absorb(const unsigned char *sv, const float *svv, float top,
                                                  const float (&s)[NK / 8][2], float &m, float &l,
                                                  float (&o)[NT][2]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m, mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen so far
        const float alpha = fast_exp2(m - ref);
        m = mn;
        // p * s_v in units of 2^(e-14), 2^e just above the tile's largest scale
        const int e = max(int(__float_as_uint(top) >> 23), 15);
        const float vup = __uint_as_float(uint32_t(268 - e) << 23), vdown = __uint_as_float(uint32_t(e - 14) << 23);
        uint32_t hi[NK / 8], lo[NK / 8];
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) {
            const float2 f = *reinterpret_cast<const float2 *>(svv + n * 8 + 2 * t);
            const float p0 = fast_exp2(s[n][0] - ref), p1 = fast_exp2(s[n][1] - ref);
            sum += p0 + p1;
            // a row that is not seen takes no part, whatever its scale
            const float w0 = s[n][0] == -INFINITY ? 0.f : p0 * (f.x * vup);
            const float w1 = s[n][1] == -INFINITY ? 0.f : p1 * (f.y * vup);
            const __half2 h = __floats2half2_rn(w0, w1);
            const float2 b = __half22float2(h);
            const __half2 r = __floats2half2_rn(w0 - b.x, w1 - b.y);
            hi[n] = *reinterpret_cast<const uint32_t *>(&h);
            lo[n] = *reinterpret_cast<const uint32_t *>(&r);
        }
        l = l * alpha + sum;
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < NK / 16; ++kk) {
            uint32_t w[4][HD / 32];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = kk * 16 + 2 * t + (r & 1) + (r >> 1) * 8;
                if (HD == 128) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(sv + q8_chunk<HD>(row, g));
                    w[r][0] = x.x; w[r][1] = x.y; w[r][HD / 32 - 2] = x.z; w[r][HD / 32 - 1] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(sv + q8_chunk<HD>(row, g >> 1) + (g & 1) * 8);
                    w[r][0] = x.x; w[r][1] = x.y;
                }
            }
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const uint32_t ab0 = __byte_perm(w[0][j], w[1][j], 0x5140), ab1 = __byte_perm(w[0][j], w[1][j], 0x7362);
                const uint32_t cd0 = __byte_perm(w[2][j], w[3][j], 0x5140), cd1 = __byte_perm(w[2][j], w[3][j], 0x7362);
                mma_f16(acc[4 * j + 0], hi[2 * kk], lo[2 * kk], hi[2 * kk + 1], lo[2 * kk + 1],
                        half_pair<0x5140>(ab0), half_pair<0x5140>(cd0));
                mma_f16(acc[4 * j + 1], hi[2 * kk], lo[2 * kk], hi[2 * kk + 1], lo[2 * kk + 1],
                        half_pair<0x5342>(ab0), half_pair<0x5342>(cd0));
                mma_f16(acc[4 * j + 2], hi[2 * kk], lo[2 * kk], hi[2 * kk + 1], lo[2 * kk + 1],
                        half_pair<0x5140>(ab1), half_pair<0x5140>(cd1));
                mma_f16(acc[4 * j + 3], hi[2 * kk], lo[2 * kk], hi[2 * kk + 1], lo[2 * kk + 1],
                        half_pair<0x5342>(ab1), half_pair<0x5342>(cd1));
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            o[i][0] = o[i][0] * alpha + (acc[i][0] + acc[i][2]) * vdown;
            o[i][1] = o[i][1] * alpha + (acc[i][1] + acc[i][3]) * vdown;
        }
    }
};

// The largest scale of a tile as FP32 bits (scales are never negative; NaN
// counts as 0).
__device__ __forceinline__ float top_scale(float x) {
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, b < 0x7f800000u ? b : 0u));
}

// Block (x, y): split x of the batch's plan, kv head y.  Row r of the up to 8
// query rows is new token r / G, head y*G + r % G.
template <int HD, int G, int W, bool TREE>
__global__ void __launch_bounds__(32 * W, 8 / W)
q8_rows_kernel(const RowsArgs a, const __grid_constant__ Q8Seqs tab,
               const __grid_constant__ Q8Splits plan, const __grid_constant__ Q8See<TREE> see) {
    using C = Rows<HD, W>;
    using M = TileMath<HD, kTile>;
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

    // ---- queries: rotated, scaled by a power of two, split in two halves ------
    for (int r = warp; r < kQ8Rows; r += W) {
        float x[E];
        const bool on = r < n_rows;
        const int i = on ? r / G : 0;
        const int at = pos + (on ? see.depth(t0, i) : 0);
        const float *qr = a.q + (size_t(t0 + i) * a.L.n_kv * G + h * G + r % G) * HD + E * lane;
        const float *rc = a.rope_cos + size_t(at) * (HD / 2) + lane * (E / 2);
        const float *rs = a.rope_sin + size_t(at) * (HD / 2) + lane * (E / 2);
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 z = on ? rope_pair(qr[e], qr[e + 1], rc[e / 2], rs[e / 2]) : make_float2(0.f, 0.f);
            x[e] = z.x;
            x[e + 1] = z.y;
            top = fmaxf(top, fmaxf(fabsf(z.x), fabsf(z.y)));
        }
        // largest value to [2^14, 2^15); an infinite or NaN query gives NaN
        const int ex = min(max(int(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23), 15), 254);
        const float up = __uint_as_float(uint32_t(268 - ex) << 23);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = x[e] * up;
            const __half b = __float2half_rn(y);
            s_q[r * HD + E * lane + e] = b;
            s_q[(kQ8Rows + r) * HD + E * lane + e] = __float2half_rn(y - __half2float(b));
        }
        if (lane == 0) s_fac[r] = __uint_as_float(uint32_t(ex - 14) << 23) * a.scale_log2;
    }
    // ---- the last split's block appends the new rows, and keeps them as a tile -
    if (last_split) {
        for (int w = warp; w < 2 * kNew; w += W) {
            const int i = w >> 1;
            const bool is_v = w & 1;
            uint32_t codes = E == 4 ? 0x80808080u : 0x8080u;
            float s = 0.f;
            if (i < n_new) {
                const float *src = (is_v ? a.v_new : a.k_new) + (size_t(t0 + i) * a.L.n_kv + h) * HD + E * lane;
                float x[E];
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = src[e];
                if (!is_v) {
                    const int at = pos + see.depth(t0, i);
                    const float *rc = a.rope_cos + size_t(at) * (HD / 2) + lane * (E / 2);
                    const float *rs = a.rope_sin + size_t(at) * (HD / 2) + lane * (E / 2);
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const float2 z = rope_pair(x[e], x[e + 1], rc[e / 2], rs[e / 2]);
                        x[e] = z.x;
                        x[e + 1] = z.y;
                    }
                }
                s = q8_quantize<E>(x, codes);
                q8_store_codes<HD>(is_v ? gv : gk, pos + i, lane, codes);
                if (lane == 0) (is_v ? gvs : gks)[pos + i] = s;
            }
            q8_store_codes<HD>(s_new + (is_v ? kNew * HD : 0), i, lane, codes);
            if (lane == 0) (is_v ? s_nvs : s_nks)[i] = s;
        }
    }
    __syncthreads();

    // ---- the warp's query operand: hi in rows 0-7, lo in rows 8-15 --------------
    const int g = lane >> 2, t = lane & 3;
    uint32_t qa[M::KS][4];
#pragma unroll
    for (int ks = 0; ks < M::KS; ++ks) {
        const int d = 16 * (t + 4 * (ks >> 2)) + 4 * (ks & 3);
        const uint2 a0 = *reinterpret_cast<const uint2 *>(s_q + g * HD + d);
        const uint2 a1 = *reinterpret_cast<const uint2 *>(s_q + (kQ8Rows + g) * HD + d);
        qa[ks][0] = a0.x;
        qa[ks][1] = a1.x;
        qa[ks][2] = a0.y;
        qa[ks][3] = a1.y;
    }
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
        M::scores(st, sks, qa, fac, s);
        float sv = svs[lane];
        if (n < kTile) {
            if (lane >= n) sv = 0.f;
#pragma unroll
            for (int j = 0; j < kTile / 8; ++j) {
                if (8 * j + 2 * t >= n) s[j][0] = -INFINITY;
                if (8 * j + 2 * t + 1 >= n) s[j][1] = -INFINITY;
            }
        }
        M::absorb(st + kTile * HD, svs, top_scale(sv), s, m, l, o);
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
        using N = TileMath<HD, kNew>;
        float s[kNew / 8][2];
        N::scores(s_new, s_nks, qa, fac, s);
        const int mine = g / G;  // token of row g; rows past n_rows see nothing here
#pragma unroll
        for (int j = 0; j < kNew / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = 8 * j + 2 * t + e;
                if (mine >= n_new || !see.sees(t0, mine, key)) s[j][e] = -INFINITY;
            }
        N::absorb(s_new + kNew * HD, s_nvs, top_scale(lane < kNew ? s_nvs[lane] : 0.f), s, m, l, o);
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
            if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * p) = make_float2(mx, sum);
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
    // ---- join the splits ----------------------------------------------------------
    for (int f = tid; f < n_rows * (HD / 4); f += 32 * W) {
        const int r = f / (HD / 4), d = (f % (HD / 4)) * 4;
        const float *po = a.part_o + (part0 * kQ8Rows + r) * HD + d;
        const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + part0 * kQ8Rows + r;
        float mx = -INFINITY, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int U = 8;
        for (int s0 = 0; s0 < nsplit; s0 += U) {
            float4 x[U];
            float2 y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = min(s0 + u, nsplit - 1);
                x[u] = __ldcg(reinterpret_cast<const float4 *>(po + size_t(s) * kQ8Rows * HD));
                y[u] = __ldcg(ml + size_t(s) * kQ8Rows);
            }
            float top = mx;
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, y[u].x);
            const float back = mx == -INFINITY ? 0.f : fast_exp2(mx - top);
            mx = top;
            sum *= back;
            v.x *= back; v.y *= back; v.z *= back; v.w *= back;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float e = (s0 + u < nsplit && y[u].x != -INFINITY) ? fast_exp2(y[u].x - top) : 0.f;
                if (s0 + u < nsplit) {
                    sum += y[u].y * e;
                    v.x += x[u].x * e; v.y += x[u].y * e; v.z += x[u].z * e; v.w += x[u].w * e;
                }
            }
        }
        const float inv = 1.f / sum;
        const size_t at = (size_t(t0 + r / G) * a.L.n_kv * G + h * G + r % G) * HD + d;
        *reinterpret_cast<float4 *>(a.out + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

template <int HD, int G, int W, bool TREE>
int launch_rows(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Splits &plan,
                const Q8See<TREE> &see, bool overlap) {
    auto fn = q8_rows_kernel<HD, G, W, TREE>;
    if (int st = set_kernel_smem(reinterpret_cast<const void *>(fn), Rows<HD, W>::kSmem,
                                 "cudaFuncSetAttribute(q8_rows)"))
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.split0[tab.n_seq], c->n_kv);
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = Rows<HD, W>::kSmem;
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
    return tree ? launch_rows<HD, G, 8, true>(c, a, tab, plan, q8_see(*tree), overlap)
                : launch_rows<HD, G, 8, false>(c, a, tab, plan, Q8See<false>(), overlap);
}

// Rows of a split: one wave of one block an SM where the work is that little,
// at least kMinChunk (a partial costs as much as some rows) and at most
// kMaxChunk (so that long sequences of a large batch do not finish late).
constexpr int kMinChunk = 128, kMaxChunk = 2048;

}  // namespace

int q8_rows_parts(const leap_ctx *c) {
    const long nb = c->max_batch < kMaxSeqPerLaunch ? c->max_batch : kMaxSeqPerLaunch;
    return int(nb * c->n_kv * (c->max_seq / kMaxChunk + 2) + 2 * c->num_sms);
}

static void plan_rows(const leap_ctx *c, const Q8Seqs &tab, Q8Splits &plan) {
    long total = 0;
    for (int i = 0; i < tab.n_seq; ++i) total += tab.pos[i];
    long chunk = (total * c->n_kv + c->num_sms - 1) / c->num_sms;
    chunk = (chunk + 63) / 64 * 64;
    if (chunk < kMinChunk) chunk = kMinChunk;
    auto count = [&](long ch) {
        long n = 0;
        for (int i = 0; i < tab.n_seq; ++i)
            if (tab.tok0[i + 1] > tab.tok0[i]) n += tab.pos[i] > 0 ? (tab.pos[i] + ch - 1) / ch : 1;
        return n * c->n_kv;
    };
    // one wave, if the sequences' last splits do not push past it
    while (chunk < kMaxChunk && count(chunk) > c->num_sms) chunk += 64;
    if (chunk > kMaxChunk) chunk = kMaxChunk;
    plan.chunk = int(chunk);
    int n = 0;
    for (int i = 0; i < tab.n_seq; ++i) {
        plan.split0[i] = n;
        if (tab.tok0[i + 1] > tab.tok0[i]) n += tab.pos[i] > 0 ? int((tab.pos[i] + chunk - 1) / chunk) : 1;
    }
    plan.split0[tab.n_seq] = n;
}

int q8_rows_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
                   const float *k, const float *v, float *out) {
    Q8Splits plan;
    plan_rows(c, tab, plan);
    if (long(plan.split0[tab.n_seq]) * c->n_kv > c->q8_parts) {
        set_error("8-bit decode plan needs %d partials, scratch holds %d",
                  plan.split0[tab.n_seq] * c->n_kv, c->q8_parts);
        return LEAP_ERR_INVALID;
    }
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
    int st;
    switch (c->hd * 100 + c->group) {
        case 12801: st = launch_rows_g<128, 1>(c, a, tab, plan, tree, overlap); break;
        case 12802: st = launch_rows_g<128, 2>(c, a, tab, plan, tree, overlap); break;
        case 12804: st = launch_rows_g<128, 4>(c, a, tab, plan, tree, overlap); break;
        case 12808: st = launch_rows_g<128, 8>(c, a, tab, plan, tree, overlap); break;
        case 6401: st = launch_rows_g<64, 1>(c, a, tab, plan, tree, overlap); break;
        case 6402: st = launch_rows_g<64, 2>(c, a, tab, plan, tree, overlap); break;
        case 6404: st = launch_rows_g<64, 4>(c, a, tab, plan, tree, overlap); break;
        case 6408: st = launch_rows_g<64, 8>(c, a, tab, plan, tree, overlap); break;
        default:
            set_error("unsupported head_dim %d / kv_mul %d", c->hd, c->group);
            return LEAP_ERR_INVALID;
    }
    return st;
}

}  // namespace leap
