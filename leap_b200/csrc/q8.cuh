// q8.cuh — the 8-bit KV cache: row format, batch tables, device helpers.
//
// A row x[HD] of one kv head is stored as HD codes of one byte and one FP32
// scale:  s = max|x| * (1/127),  c = x / s rounded to the nearest integer
// (ties to even, within -127..127); it stands for c * s.  Codes are stored
// plus 128 (1..255), so that one byte permute per two codes builds FP16 pairs
// (0x6400 | u is 1024 + u).  A row that holds an infinity or a NaN gets codes
// 0 and a NaN scale: it reads back as NaN, and what attends to it is NaN.
//
// Layout: codes [slot][layer][kv_head][max_seq_pad][HD], scales
// [slot][layer][kv_head][max_seq_pad], so a run of rows is one contiguous
// bulk copy of each.  Inside a 128-byte line (one row of 128, two rows of 64)
// the 16-byte chunks are permuted by the row index (q8_chunk below): a linear
// copy into shared memory then serves both fragment patterns of mma.sync
// without bank conflicts (eight consecutive rows read at two chunk halves for
// K, rows 2t / 2t+1 read at neighbouring chunks for V).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "ctx.h"

namespace leap {

template <int N>
__device__ __forceinline__ void load_vec(float (&v)[N], const float *p) {
    if constexpr (N == 4) {
        const float4 x = *reinterpret_cast<const float4 *>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else if constexpr (N == 2) {
        const float2 x = *reinterpret_cast<const float2 *>(p);
        v[0] = x.x; v[1] = x.y;
    } else {
        v[0] = *p;
    }
}

// Byte offset, from the first row of a head, of 16-byte chunk `c` of row `r`.
template <int HD>
__host__ __device__ __forceinline__ size_t q8_chunk(int r, int c) {
    if (HD == 128)
        return size_t(r) * 128 + (unsigned(c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2))) << 4);
    const int line = r >> 1;
    return size_t(line) * 128 + (unsigned((((r & 1) << 2) | c) ^ ((line & 3) << 1)) << 4);
}

// Sequence of packed token `t`: the last i with tok0[i] <= t (sequences
// without tokens are stepped over, since their tok0 equals the next one's).
__device__ __forceinline__ int q8_seq_of(const Q8Seqs &tab, int t) {
    int lo = 0, hi = tab.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.tok0[mid] <= t) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// How the tokens of a run see one another.  Causal: token i sees 0..i, at
// position pos + i.  Tree: i sees itself and its ancestors, at pos + depth.
template <bool TREE>
struct Q8See;
template <>
struct Q8See<false> {
    __device__ __forceinline__ int depth(int, int i) const { return i; }
    __device__ __forceinline__ bool sees(int, int i, int j) const { return j <= i; }
};
template <>
struct Q8See<true> {
    Q8Tree tree;
    // t0: the sequence's first packed token.  Parents come before children.
    __device__ __forceinline__ int depth(int t0, int i) const { return tree.depth[t0 + i]; }
    __device__ __forceinline__ bool sees(int t0, int i, int j) const {
        while (i > j) i = tree.parent[t0 + i];
        return i == j;
    }
};
inline const Q8See<true> &q8_see(const Q8Tree &tree) {
    static_assert(sizeof(Q8See<true>) == sizeof(Q8Tree), "one is the other");
    return reinterpret_cast<const Q8See<true> &>(tree);
}

// The code nearest to x / s (ties to even), `s` normal and inv near 1 / s:
// the rounded product is at most one off, and the residual x - q*s, exact in
// one fused multiply-add, tells on which side of the half x lies.
__device__ __forceinline__ int q8_code(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x);
    const float a = fabsf(r), half = 0.5f * s;
    if (a > half || (a == half && (int(q) & 1))) q += r > 0.f ? 1.f : -1.f;
    return int(fminf(fmaxf(q, -127.f), 127.f));
}

// The larger of a and |b|; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
    return d;
}

// One warp quantises one row, lane l holding x[E] = dims E*l .. E*l+E-1.
// Returns the scale (the same in every lane) and this lane's codes + 128, the
// lowest dim in the lowest byte.
template <int E>
__device__ __forceinline__ float q8_quantize(const float (&x)[E], uint32_t &codes) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) most = max_nan(most, x[i]);
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    codes = E == 4 ? 0x80808080u : 0x8080u;
    if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const float s = __fmul_rn(__uint_as_float(top), 1.0f / 127.0f);
    if (s == 0.f) return 0.f;
    // tiny rows: x and s by 2^64 (exact), so that 1/s stays finite
    const bool tiny = top < 0x21800000u;  // 2^-60
    const float up = tiny ? 18446744073709551616.f : 1.f, su = s * up, inv = 1.0f / su;
    // x*inv + 128 + 1.5*2^23 has the rounded sum's integer in its low bits.  Where no
    // residual reaches half a step this is the code: |x| <= 127.5 s then, unless s has
    // lost bits (tiny).  Instructions bound the append, and the exact test of every
    // value takes three times as many.
    constexpr float kMagic = 12582912.f + 128.f;
    float off = 0.f;
    uint32_t t[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float m = fmaf(x[i] * up, inv, kMagic);
        off = fmaxf(off, fabsf(fmaf(kMagic - m, su, x[i] * up)));
        t[i] = __float_as_uint(m);
    }
    if (off < 0.5f * su && !tiny) {
        if constexpr (E == 4) codes = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
        else codes = __byte_perm(t[0], t[1], 0x0040) & 0xffffu;
    } else {
        codes = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) codes |= uint32_t(q8_code(x[i] * up, su, inv) + 128) << (8 * i);
    }
    return s;
}

// Store / load a lane's codes (E = HD / 32 of them) of row r.
template <int HD>
__device__ __forceinline__ void q8_store_codes(uint8_t *head, int r, int lane, uint32_t codes) {
    if (HD == 128)
        *reinterpret_cast<uint32_t *>(head + q8_chunk<HD>(r, lane >> 2) + (lane & 3) * 4) = codes;
    else
        *reinterpret_cast<uint16_t *>(head + q8_chunk<HD>(r, lane >> 3) + (lane & 7) * 2) =
            uint16_t(codes);
}
template <int HD>
__device__ __forceinline__ uint32_t q8_load_codes(const uint8_t *head, int r, int lane) {
    if (HD == 128)
        return *reinterpret_cast<const uint32_t *>(head + q8_chunk<HD>(r, lane >> 2) + (lane & 3) * 4);
    return *reinterpret_cast<const uint16_t *>(head + q8_chunk<HD>(r, lane >> 3) + (lane & 7) * 2);
}

// The maximum that a part of a split range leaves for the join, which leaves out
// parts with -inf (nothing seen).  A running maximum passes NaN over, so a part that
// saw nothing but NaN has -inf too: its sum says so, and the maximum becomes NaN.
// (A join that takes every part in, by a weight of zero, costs 2.5% of a batch of 64.)
__device__ __forceinline__ float part_max(float m, float l) { return fmaf(l, 0.f, m); }

// A new row as a warp takes it: the lane's dims, and for k what rotates them.
template <int HD>
struct Q8NewRow {
    static constexpr int E = HD / 32;
    float x[E], rc[E / 2], rs[E / 2];

    __device__ __forceinline__ void load(const float *src, bool is_k, const float *rope_cos, const float *rope_sin, int at) {
        const int lane = threadIdx.x & 31;
        load_vec<E>(x, src + E * lane);
        if (is_k) {
            const size_t c = size_t(at) * (HD / 2) + lane * (E / 2);
            load_vec<E / 2>(rc, rope_cos + c);
            load_vec<E / 2>(rs, rope_sin + c);
        }
    }
    // Rotates (k), quantises and stores it as row `row` of its head; `codes` and the
    // scale (every lane's) come back.
    __device__ __forceinline__ float store(bool is_k, uint8_t *head, float *scales, int row, uint32_t &codes) {
        const int lane = threadIdx.x & 31;
        if (is_k) {
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 z = rope_pair(x[e], x[e + 1], rc[e / 2], rs[e / 2]);
                x[e] = z.x;
                x[e + 1] = z.y;
            }
        }
        const float s = q8_quantize<E>(x, codes);
        q8_store_codes<HD>(head, row, lane, codes);
        if (lane == 0) scales[row] = s;
        return s;
    }
};
template <int HD>
__device__ __forceinline__ float q8_append_row(const float *src, bool is_k, const float *rope_cos, const float *rope_sin,
                                               int at, uint8_t *head, float *scales, int row, uint32_t &codes) {
    Q8NewRow<HD> r;
    r.load(src, is_k, rope_cos, rope_sin, at);
    return r.store(is_k, head, scales, row, codes);
}

}  // namespace leap
