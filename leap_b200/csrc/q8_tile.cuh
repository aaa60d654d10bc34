// q8_tile.cuh — one warp's work on a tile of cached 8-bit rows for up to 8 query
// rows, on mma.sync (m16n8k16, FP16 operands, FP32 sums).
//
// A query row needs 2 x 11 bits for FP32-like results, and the 16 rows of the A
// operand are 8 query rows' high halves and the same 8 rows' low halves: hi and lo
// come out in the same thread's c0/c1 and c2/c3 and are added there.  Codes are
// exact in FP16.
//
//  * The contraction index may be permuted freely as long as both operands
//    agree, so a thread's K operands are whole 16-byte chunks of one row, and
//    its V operands 16-byte chunks of four rows: no transposition, one
//    permute per 2 codes for K and 1.5 for V (half pairs are 0x6400 | code,
//    minus 1152).  q8.cuh's chunk order keeps both reads free of conflicts.
//  * Tensor-core sums are truncated, and a long run of them drifts towards
//    zero; each tile is summed from zero and joins the FP32 output by an
//    ordinary multiply-add.
//  * p*s_v is scaled by a power of two for each query row and tile, so that FP16
//    holds the row's largest to 22 bits, whatever the scales are of what it does
//    not see or hardly weighs; the same for each q row.
#pragma once

#include "q8.cuh"

namespace leap {

// What the kernels of a few query rows get.
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

// attn_q8_warps.cu: what a batch costs there, and its launch.
long q8_warps_cost(const leap_ctx *c, const Q8Seqs &tab);
int q8_warps_launch(leap_ctx *c, const RowsArgs &a, const Q8Seqs &tab, const Q8Tree *tree, bool overlap);

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Two of four bytes x (codes + 128) as FP16 values code, code.
template <int SEL>
__device__ __forceinline__ uint32_t half_pair(uint32_t x) {
    const uint32_t y = __byte_perm(x, 0x64646464u, SEL);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), __float2half2_rn(1152.f));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// One warp's work on a tile of NK (16 or 32) rows in shared memory; the output's
// columns in PARTS parts, one after another, which bounds the registers.
template <int HD, int NK, int PARTS>
struct TileMath {
    static constexpr int NT = HD / 8;   // 8-dim column tiles of the output

    // sq: the queries' hi, then lo halves [8][HD] (hi in operand rows 0-7, lo in 8-15).
    static __device__ __forceinline__ void scores(const unsigned char *sk, const float *skv, const __half *sq,
                                                  float fac, float (&s)[NK / 8][2]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        float cc[NK / 8][4];
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
            // this thread's 16 dims of the query's rows: 4 steps
            const uint4 *h = reinterpret_cast<const uint4 *>(sq + g * HD + 16 * (t + 4 * j));
            const uint4 *e = reinterpret_cast<const uint4 *>(sq + (kQ8Rows + g) * HD + 16 * (t + 4 * j));
            const uint4 h0 = h[0], h1 = h[1], e0 = e[0], e1 = e[1];
            const uint32_t qh[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
            const uint32_t ql[8] = {e0.x, e0.y, e0.z, e0.w, e1.x, e1.y, e1.z, e1.w};
#pragma unroll
            for (int n = 0; n < NK / 8; ++n) {
                const uint4 w = *reinterpret_cast<const uint4 *>(sk + q8_chunk<HD>(n * 8 + g, t + 4 * j));
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t b0 = half_pair<0x5140>(ww[u]), b1 = half_pair<0x5342>(ww[u]);
                    if (j + u == 0) mma_f16_first(cc[n], qh[0], ql[0], qh[1], ql[1], b0, b1);
                    else mma_f16(cc[n], qh[2 * u], ql[2 * u], qh[2 * u + 1], ql[2 * u + 1], b0, b1);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) {
            const float(&c)[4] = cc[n];
            const float2 f = *reinterpret_cast<const float2 *>(skv + n * 8 + 2 * t);
            s[n][0] = (c[0] + c[2]) * (f.x * fac);
            s[n][1] = (c[1] + c[3]) * (f.y * fac);
        }
    }

    // o, m, l of row g take the tile's rows; s is -inf where a row is not seen.
    static __device__ __forceinline__ void absorb(const unsigned char *sv, const float *svv, const float (&s)[NK / 8][2],
                                                  float &m, float &l, float (&o)[NT][2]) {
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
        float w[NK / 8][2], sum = 0.f, most = 0.f;
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) {
            const float2 f = *reinterpret_cast<const float2 *>(svv + n * 8 + 2 * t);
            const float p0 = fast_exp2(s[n][0] - ref), p1 = fast_exp2(s[n][1] - ref);
            sum += p0 + p1;
            // a row that is not seen takes no part, whatever its scale
            w[n][0] = s[n][0] == -INFINITY ? 0.f : p0 * f.x;
            w[n][1] = s[n][1] == -INFINITY ? 0.f : p1 * f.y;
            most = fmaxf(most, fmaxf(w[n][0], w[n][1]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the row's largest weight to [2^14, 2^15)
        const int e = max(int(__float_as_uint(most) >> 23), 15);
        const float vup = __uint_as_float(uint32_t(268 - e) << 23), vdown = __uint_as_float(uint32_t(e - 14) << 23);
        uint32_t hi[NK / 8], lo[NK / 8];
#pragma unroll
        for (int n = 0; n < NK / 8; ++n) {
            const float w0 = w[n][0] * vup, w1 = w[n][1] * vup;
            const __half2 h = __floats2half2_rn(w0, w1);
            const float2 b = __half22float2(h);
            const __half2 r = __floats2half2_rn(w0 - b.x, w1 - b.y);
            hi[n] = *reinterpret_cast<const uint32_t *>(&h);
            lo[n] = *reinterpret_cast<const uint32_t *>(&r);
        }
        l = l * alpha + sum;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            float acc[NT / PARTS][4];
#pragma unroll
            for (int kk = 0; kk < NK / 16; ++kk) {
                constexpr int NW = HD / 32 / PARTS;  // words of a row
                uint32_t w[4][NW];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = kk * 16 + 2 * t + (r & 1) + (r >> 1) * 8;
                    const unsigned char *src = HD == 128 ? sv + q8_chunk<HD>(row, g) + 4 * NW * part
                                                         : sv + q8_chunk<HD>(row, g >> 1) + (g & 1) * 8 + 4 * NW * part;
                    if constexpr (NW == 4) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(src);
                        w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
                    } else if constexpr (NW == 2) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(src);
                        w[r][0] = x.x; w[r][1] = x.y;
                    } else {
                        w[r][0] = *reinterpret_cast<const uint32_t *>(src);
                    }
                }
                const uint32_t a0 = hi[2 * kk], a1 = lo[2 * kk], a2 = hi[2 * kk + 1], a3 = lo[2 * kk + 1];
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    const uint32_t ab0 = __byte_perm(w[0][j], w[1][j], 0x5140), ab1 = __byte_perm(w[0][j], w[1][j], 0x7362);
                    const uint32_t cd0 = __byte_perm(w[2][j], w[3][j], 0x5140), cd1 = __byte_perm(w[2][j], w[3][j], 0x7362);
                    auto mma = [&](float (&d)[4], uint32_t b0, uint32_t b1) {
                        if (kk == 0) mma_f16_first(d, a0, a1, a2, a3, b0, b1);
                        else mma_f16(d, a0, a1, a2, a3, b0, b1);
                    };
                    mma(acc[4 * j + 0], half_pair<0x5140>(ab0), half_pair<0x5140>(cd0));
                    mma(acc[4 * j + 1], half_pair<0x5342>(ab0), half_pair<0x5342>(cd0));
                    mma(acc[4 * j + 2], half_pair<0x5140>(ab1), half_pair<0x5140>(cd1));
                    mma(acc[4 * j + 3], half_pair<0x5342>(ab1), half_pair<0x5342>(cd1));
                }
            }
#pragma unroll
            for (int i = 0; i < NT / PARTS; ++i) {
                float(&z)[2] = o[part * (NT / PARTS) + i];
                z[0] = z[0] * alpha + (acc[i][0] + acc[i][2]) * vdown;
                z[1] = z[1] * alpha + (acc[i][1] + acc[i][3]) * vdown;
            }
        }
    }
};

// A query row on its way: E = HD / 32 dims a lane, with its rotation.
template <int HD>
struct QueryRow {
    static constexpr int E = HD / 32;
    float x[E], rc[E / 2], rs[E / 2];
    __device__ __forceinline__ void load(const float *q, const float *rope_cos, const float *rope_sin, int at) {
        const int lane = threadIdx.x & 31;
        const size_t c = size_t(at) * (HD / 2) + lane * (E / 2);
        load_vec<E>(x, q + E * lane);
        load_vec<E / 2>(rc, rope_cos + c);
        load_vec<E / 2>(rs, rope_sin + c);
    }
    // Rotates it, scales it by a power of two and stores its two FP16 halves (row r
    // of sq [hi, lo][8][HD]); returns what scores of it are to be multiplied by.
    __device__ __forceinline__ float stage(float scale_log2, __half *sq, int r) {
        const int lane = threadIdx.x & 31;
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 z = rope_pair(x[e], x[e + 1], rc[e / 2], rs[e / 2]);
            x[e] = z.x;
            x[e + 1] = z.y;
            top = fmaxf(top, fmaxf(fabsf(z.x), fabsf(z.y)));
        }
        // largest value to [2^14, 2^15); an infinite or NaN query gives NaN
        const int ex = min(max(int(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23), 15), 254);
        const float up = __uint_as_float(uint32_t(268 - ex) << 23);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float y0 = x[e] * up, y1 = x[e + 1] * up;
            const __half2 b = __floats2half2_rn(y0, y1);
            const float2 back = __half22float2(b);
            *reinterpret_cast<__half2 *>(sq + r * HD + E * lane + e) = b;
            *reinterpret_cast<__half2 *>(sq + (kQ8Rows + r) * HD + E * lane + e) =
                __floats2half2_rn(y0 - back.x, y1 - back.y);
        }
        return __uint_as_float(uint32_t(ex - 14) << 23) * scale_log2;
    }
};

}  // namespace leap
