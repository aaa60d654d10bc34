// attn_q8_tc.cu — attention of many query rows for each kv head (packed
// prompts, drafted trees) over the 8-bit KV cache, on tcgen05 tensor cores.
//
//   out = softmax(rope(q) . (c_k s_k) / sqrt(hd)) . (c_v s_v)
//
// The run's own rows are stored first (by the append kernel of kv_q8.cu, or where a
// sequence has one query tile by the block that reads them) and read as they are
// kept.  A block takes 128 query rows (row r is token r / G of its
// tile, head r % G of the kv head's group) and a range of key tiles of 128.
//
// Arithmetic: codes are exact in FP16.  Queries (scaled by a power of two for
// each row) and weights p*s_v (by one for each tile, or row and tile) are split into two FP16,
// hi + lo, 22 bits: two FP16 products in place of one give FP32-like results,
// and are what bounds the kernel (twice the FLOPs of one FP16 product; 32
// tcgen05.mma of 128x128x16 a tile, about 2048 cycles).  Tensor-core sums are
// truncated and would drift over a long context, so O is summed from zero for
// every tile and joins FP32 registers by ordinary multiply-adds, with the
// running maximum's correction: nothing is rescaled in TMEM.
//
// Roles (16 warps; registers moved to where O lives by setmaxnreg, 200 + 200 +
// 72 + 40 = 4 x 128):
//   warps 0-7        softmax, two threads a row (64 keys and half of O's columns
//                    each): S(j) from TMEM, p, hi/lo back over S in place; O(j-1),
//                    whose product ran meanwhile, into registers.
//   warps 8-11       codes -> FP16 operand tiles (128-byte swizzle; V is used
//                    N-major, so nothing is transposed), a tile ahead in
//                    registers, and the tile's scales.
//   warps 13-15      store the block's new rows, where that is left to it (with the
//                    softmax warps' help, where its first tiles have them).
//   warp 12          issues the products: S(j+1) = Q K^T, then O(j) = P V.
// TMEM: two buffers of S/P (128 columns each), O (HD) and Q hi/lo (HD): both
// products take their A operand from TMEM, since two operands in shared memory
// would fill its 128 bytes a cycle and starve everything else.  Shared memory:
// two buffers each of K and V, and Q on its way to TMEM.
// Long ranges are split over blocks when a launch has few tiles; partials are
// joined by a second kernel.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "q8.cuh"
#include "tc.cuh"

namespace leap {
namespace {

constexpr int kBM = 128;        // query rows of a block = TMEM lanes
constexpr int kBN = 128;        // keys of a tile
constexpr int kThreads = 512;
constexpr int kLaunchRegs = 65536 / kThreads;
constexpr int kRegsSoftmax = 200, kRegsConvert = 72, kRegsIssue = 40;  // of each group of 4 warps
static_assert(2 * kRegsSoftmax + kRegsConvert + kRegsIssue == 4 * kLaunchRegs, "register split");
constexpr int kSlots = 4;       // tiles whose scales are held

template <int HD>
struct Tc {
    static constexpr uint32_t kOp = kBN * HD * 2;           // one operand tile
    static constexpr uint32_t kChunk = 128 * 128;           // 64 dims of 128 rows
    static constexpr uint32_t kK = 0, kV = 2 * kOp, kQ = 4 * kOp;
    static constexpr uint32_t kQRow = HD * 2 + 16;          // a staged query row, hi or lo
    static constexpr size_t kSmem = 4 * size_t(kOp) + 2 * kBM * kQRow + 1024;
    static constexpr uint32_t kCols = 512;                  // TMEM columns (a power of two)
    static constexpr uint32_t kColS(int b) { return b * 128; }
    static constexpr uint32_t kColO = 256;
    static constexpr uint32_t kColQ(int u) { return 384 + u * (HD / 2); }
};

struct TcArgs {
    const float *q;
    const float *k_new, *v_new;  // not null: the blocks append the run's rows themselves
    float *out;
    Q8Layer L;
    const float *rope_cos, *rope_sin;
    float *part_o, *part_ml;  // [parts][128][HD], [parts][128][2]
    int *err;
    float scale;  // 2^-14 log2(e) / sqrt(HD), taken into the scales of K
};

struct TcBars {
    uint64_t q_ready;    // Q in TMEM (8 softmax warps)
    uint64_t new_full;   // the block's new rows are stored (n_app warps)
    uint64_t k_full[2], v_full[2];  // operand tile in place (4 converter warps)
    uint64_t sc_full[kSlots];       // scales of a tile in place (4 converter warps)
    uint64_t s_full[2];  // S(j) done: K buffer free (commit)
    uint64_t p_full[2];  // P(j) in TMEM (8 softmax warps)
    uint64_t o_full[2];  // O(j) done: V buffer and S/P columns free (commit)
};

__device__ __forceinline__ uint32_t par(int j) { return uint32_t(j >> 1) & 1u; }

// Which (sequence, query tile, split, kv head) a block has.
struct Item {
    int seq, qt, split, h, part;
};
__device__ __forceinline__ Item item_of(const Q8TcPlan &plan, int n_kv, int block) {
    Item it;
    const int x = block / n_kv;
    it.h = block - x * n_kv;
    int lo = 0, hi = plan.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (plan.item0[mid] <= x) lo = mid; else hi = mid - 1;
    }
    it.seq = plan.seq[lo];
    const int i = x - plan.item0[lo];
    it.split = i % plan.nsplit[lo];
    it.qt = plan.n_qt[lo] - 1 - i / plan.nsplit[lo];  // the longest first
    it.part = plan.nsplit[lo] > 1 ? (plan.part0[lo] + i) * n_kv + it.h : -1;
    return it;
}

// How far apart the V scales lie of the rows that a block has taken so far, as
// FP32 bits (scales are never negative; NaN counts for nothing).  FP16 hi + lo
// of p * s_v have an absolute error of 2^-25 where the unit puts the tile's
// largest scale into [2^14, 2^15).  While all scales are within 2^kSpan that is
// 2^-27 of any weight's row at most, less than FP32 sums cost.  Past it (`wide`)
// the unit has to be that of what a query row weighs: a large row that it does
// not see, or next to nothing of, would take the others' bits.  Rows of zeros count
// as far apart, since one can hold nearly all of a query's weight.  That costs an
// exchange between the two threads of a row (prompt of 8192: 1116 us a call narrow,
// 1617 wide; 8 ragged trees 93, 142).
struct ScaleSpan {
    static constexpr uint32_t kSpan = 12;
    uint32_t top = 0u, low = 0x7f7fffffu;

    // A lane's scale of the next tile, into `t` (largest) and `l` (smallest).
    static __device__ __forceinline__ void look(float x, bool counts, uint32_t &t, uint32_t &l) {
        const uint32_t b = __float_as_uint(x);
        if (counts && b < 0x7f800000u) {
            t = max(t, b);
            l = min(l, b);
        }
    }
    // The tile's largest, every lane's t and l taken in.
    __device__ __forceinline__ float take(uint32_t t, uint32_t l) {
        t = __reduce_max_sync(0xffffffffu, t);
        top = max(top, t);
        low = min(low, __reduce_min_sync(0xffffffffu, l));
        return __uint_as_float(t);
    }
    __device__ __forceinline__ bool wide() const { return (top >> 23) > (low >> 23) + kSpan; }
};

// Eight codes as FP16 values (a 16-byte granule).
__device__ __forceinline__ uint4 expand(uint32_t a, uint32_t b) {
    auto two = [](uint32_t x, uint32_t sel) {
        const uint32_t y = __byte_perm(x, 0x64646464u, sel);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), __float2half2_rn(1152.f));
        return *reinterpret_cast<const uint32_t *>(&h);
    };
    return make_uint4(two(a, 0x5140), two(a, 0x5342), two(b, 0x5140), two(b, 0x5342));
}

// The largest of three (NaN counts as absent), one instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Barrier of the 256 softmax threads (named barrier 1): true if `ok` everywhere.
__device__ __forceinline__ bool group_and(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, 1, 256, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(uint32_t(ok))
        : "memory");
    return r != 0;
}

template <int HD, int G, bool TREE>
__global__ void __launch_bounds__(kThreads, 1)
q8_tc_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ Q8Seqs tab, const __grid_constant__ Q8TcPlan plan,
             const __grid_constant__ Q8See<TREE> see) {
    using C = Tc<HD>;
    constexpr int BT = kBM / G;  // tokens of a block
    extern __shared__ unsigned char smem_raw[];
    __shared__ TcBars bars;
    __shared__ __align__(16) float s_ks[kSlots][kBN], s_vs[kSlots][kBN];
    __shared__ float s_vdown[kSlots];  // negative: wide (ScaleSpan)
    __shared__ float s_fac[kBM], s_mx[2][2][kBM], s_most[2][2][kBM], s_l[2][kBM];
    __shared__ int8_t s_parent[TREE ? kMaxTreeNodes : 1];
    __shared__ uint32_t s_anc[TREE ? 4 : 1][kBM];  // TREE: what each row sees of the run
    __shared__ uint32_t tmem_sh;
    __shared__ int s_fail;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char *base = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_addr(base);

    const Item it = item_of(plan, a.L.n_kv, blockIdx.x);
    const int seq = it.seq, h = it.h;
    const int pos = tab.pos[seq], tok0 = tab.tok0[seq], n_new = tab.tok0[seq + 1] - tok0;
    const int t0 = it.qt * BT;                       // first token of the tile, within the run
    const int t_end = min(t0 + BT, n_new);
    const int kv_end = TREE ? pos + n_new : pos + t_end;
    const int n_all = (kv_end + kBN - 1) / kBN;
    const int j0 = it.split * plan.chunk;
    const int n_kt = max(min(n_all - j0, plan.chunk), 0);  // tiles j0 .. j0 + n_kt - 1

    // The run's rows that this block reads, where it stores them: i0 .. i1 - 1.  Warps
    // 13-15 do it beside the first tiles; where these need the rows, the softmax warps help.
    const int i0 = max(j0 * kBN - pos, 0), i1 = a.k_new ? max(min((j0 + n_kt) * kBN - pos, n_new), i0) : i0;
    const int n_app = i1 - i0 > 6 * (max(pos - j0 * kBN, 0) / kBN) ? 11 : 3;

    if (tid == 0) {
        mbar_init(&bars.q_ready, 8);
        mbar_init(&bars.new_full, n_app);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars.k_full[b], 4);
            mbar_init(&bars.v_full[b], 4);
            mbar_init(&bars.s_full[b], 1);
            mbar_init(&bars.p_full[b], 8);
            mbar_init(&bars.o_full[b], 1);
        }
        for (int i = 0; i < kSlots; ++i) mbar_init(&bars.sc_full[i], 4);
        s_fail = 0;
        fence_mbar_init();
    }
    if (warp == 12) {
        tc::alloc(&tmem_sh, C::kCols);
        tc::relinquish();
    }
    if constexpr (TREE)
        if (tid < n_new) s_parent[tid] = see.tree.parent[tok0 + tid];
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = tmem_sh;
    // Warp w's part of the new rows, U of them (k or v) in flight at a time.
    auto append = [&](auto u_, int w) {
        constexpr int U = decltype(u_)::value;
        const size_t r0 = tab.slot[seq] * a.L.slot_rows + h * a.L.head_rows;
        for (int x = 2 * i0 + w; x < 2 * i1; x += U * n_app) {
            Q8NewRow<HD> r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int y = x + u * n_app, i = y >> 1;
                if (y < 2 * i1)
                    r[u].load((y & 1 ? a.v_new : a.k_new) + (size_t(tok0 + i) * a.L.n_kv + h) * HD, !(y & 1), a.rope_cos,
                              a.rope_sin, pos + see.depth(tok0, i));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int y = x + u * n_app;
                uint32_t codes;
                if (y < 2 * i1)
                    r[u].store(!(y & 1), (y & 1 ? a.L.v : a.L.k) + r0 * HD, (y & 1 ? a.L.vs : a.L.ks) + r0, pos + (y >> 1), codes);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.new_full);
    };

    if (warp < 8) {
        // ================= softmax groups =====================================
        regs_up<kRegsSoftmax>();
        // Two threads a row: half 0 has keys 0-63 of a tile and the lower half of
        // O's columns, half 1 the rest.
        const int half = warp >> 2;
        const int row = tid & 127;           // TMEM lane
        const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
        // Q was written before the append kernel began, so it needs no wait
        {
            // A warp's 16 rows with all their loads in flight at once.  Rows past
            // the last token repeat it (no branch; what they give is not stored).
            constexpr int E = HD / 32, U = kBM / 8;
            float x[U][E], rc[U][E / 2], rs[U][E / 2];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = warp + 8 * u, t = min(t0 + r / G, t_end - 1);
                const size_t c = size_t(pos + see.depth(tok0, t)) * (HD / 2) + lane * (E / 2);
                load_vec<E>(x[u], a.q + (size_t(tok0 + t) * a.L.n_kv * G + h * G + r % G) * HD + E * lane);
                load_vec<E / 2>(rc[u], a.rope_cos + c);
                load_vec<E / 2>(rs[u], a.rope_sin + c);
            }
            // while they are on their way: what a row sees of the run, itself and its
            // ancestors (the barrier below makes it known)
            if (TREE && half == 0) {
                uint32_t anc[4] = {0u, 0u, 0u, 0u};
                for (int p = min(t0 + row / G, t_end - 1); p >= 0; p = s_parent[p]) {
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        if ((p >> 5) == w) anc[w] |= 1u << (p & 31);
                }
#pragma unroll
                for (int w = 0; w < 4; ++w) s_anc[w][row] = anc[w];
            }
            float fac_of_lane = 0.f;  // lane u: of row u
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = warp + 8 * u;
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 z = rope_pair(x[u][e], x[u][e + 1], rc[u][e / 2], rs[u][e / 2]);
                    x[u][e] = z.x;
                    x[u][e + 1] = z.y;
                    top = fmaxf(top, fmaxf(fabsf(z.x), fabsf(z.y)));
                }
                // largest value to [2^14, 2^15); an infinite or NaN query gives NaN
                const int ex = min(max(int(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23), 15), 254);
                const float up = __uint_as_float(uint32_t(268 - ex) << 23);
                uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float y0 = x[u][e] * up, y1 = x[u][e + 1] * up;
                    const __half2 a2 = __floats2half2_rn(y0, y1);
                    const float2 back = __half22float2(a2);
                    const __half2 b2 = __floats2half2_rn(y0 - back.x, y1 - back.y);
                    hi[e / 2] = *reinterpret_cast<const uint32_t *>(&a2);
                    lo[e / 2] = *reinterpret_cast<const uint32_t *>(&b2);
                }
                unsigned char *qs = base + C::kQ + r * C::kQRow + E * lane * 2;
                if constexpr (E == 4) {
                    *reinterpret_cast<uint2 *>(qs) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2 *>(qs + kBM * C::kQRow) = make_uint2(lo[0], lo[1]);
                } else {
                    *reinterpret_cast<uint32_t *>(qs) = hi[0];
                    *reinterpret_cast<uint32_t *>(qs + kBM * C::kQRow) = lo[0];
                }
                // A power of two, so that score * fac is exact and the largest key's
                // exponent is 0, however large the scores are.
                fac_of_lane = lane == u ? __uint_as_float(uint32_t(ex) << 23) : fac_of_lane;
            }
            if (lane < U) s_fac[warp + 8 * lane] = fac_of_lane;
        }
        // The staged rows into TMEM, a thread its row's half of the dims; dims
        // 64-127 in the converters' order (neighbouring 8-dim granules swapped).
        bool ok = group_and(true);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {  // 32 dims: 16 columns
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int gr = half * (HD / 16) + 4 * c + i;
                    const uint4 x = *reinterpret_cast<const uint4 *>(
                        base + C::kQ + (u * kBM + row) * C::kQRow + 16 * (gr < 8 ? gr : gr ^ 1));
                    w[4 * i] = x.x;
                    w[4 * i + 1] = x.y;
                    w[4 * i + 2] = x.z;
                    w[4 * i + 3] = x.w;
                }
                tc::st16u(tmem + lane_off + C::kColQ(u) + half * (HD / 4) + 16 * c, w);
            }
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_ready);
        if (n_app > 3) append(std::integral_constant<int, 4>(), 3 + warp);

        // What this row sees: keys below `lim`, or (TREE) keys below pos and
        // those of the run whose bit is set (itself and its ancestors).
        const int tok = t0 + row / G;
        const int lim = pos + min(tok, t_end - 1) + 1;
        // bit i: whether key k0 + i is seen
        auto seen = [&](int k0) -> uint32_t {
            if (!TREE) {
                const int n = lim - k0;
                return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u);
            }
            const int rel = k0 - pos, w = rel >> 5;  // bits below 0 are all ones, from 128 on zeros
            const uint32_t lo = w < 0 ? ~0u : (w > 3 ? 0u : s_anc[w][row]);
            const uint32_t hi = w < -1 ? ~0u : (w > 2 ? 0u : s_anc[w + 1][row]);
            return __funnelshift_r(lo, hi, rel & 31);
        };

        const float fac = s_fac[row];
        constexpr int OC = HD / 2;           // O columns of a thread
        float m = -INFINITY, l = 0.f;
        float o[OC];
#pragma unroll
        for (int i = 0; i < OC; ++i) o[i] = 0.f;

        // o = o * alpha + O(j) * vdown, in FP32; most tiles move no row's maximum
        auto absorb = [&](int j, float alpha, float vdown, float (&x)[4][16]) -> bool {
            const bool there = __all_sync(0xffffffffu, mbar_wait(&bars.o_full[j & 1], par(j)));
            if (!there) return false;
            tc::fence_after_sync();
            const uint32_t ocol = tmem + lane_off + C::kColO + half * OC;
            const float2 al2 = make_float2(alpha, alpha), vd2 = make_float2(vdown, vdown);
#pragma unroll
            for (int c = 0; c < OC / 16; ++c) tc::ld16_async(ocol + 16 * c, x[c]);
            if (!__all_sync(0xffffffffu, alpha == 1.f)) {
#pragma unroll
                for (int i = 0; i < OC; i += 2) {
                    const float2 z = __fmul2_rn(make_float2(o[i], o[i + 1]), al2);
                    o[i] = z.x;
                    o[i + 1] = z.y;
                }
            }
#pragma unroll
            for (int c = 0; c < OC / 16; ++c) {
                tc::wait_ld16(x[c]);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float2 z = __ffma2_rn(make_float2(x[c][i], x[c][i + 1]), vd2,
                                                make_float2(o[16 * c + i], o[16 * c + i + 1]));
                    o[16 * c + i] = z.x;
                    o[16 * c + i + 1] = z.y;
                }
            }
            return true;
        };

        float alpha = 1.f, vdown = 0.f;      // of the tile whose O is still to come
        float s[4][16];                      // scores, weights, then a part of O
        for (int j = 0; j < n_kt; ++j) {
            const int b = j & 1, slot = j & (kSlots - 1);
            ok = ok && mbar_wait(&bars.sc_full[slot], uint32_t(j / kSlots) & 1u) &&
                 mbar_wait(&bars.s_full[b], par(j));
            ok = __all_sync(0xffffffffu, ok);
            tc::fence_after_sync();
            const int k0 = (j0 + j) * kBN + 64 * half;
            const uint32_t scol = tmem + lane_off + C::kColS(b) + 64 * half;
            const float4 *ks = reinterpret_cast<const float4 *>(s_ks[slot]) + 16 * half;
            const float4 *vs = reinterpret_cast<const float4 *>(s_vs[slot]) + 16 * half;
            const bool full = __all_sync(0xffffffffu, (TREE ? pos : lim) >= k0 + 64);
            const uint2 vis = full ? make_uint2(~0u, ~0u) : make_uint2(seen(k0), seen(k0 + 32));
            // scores in units of 1/fac, and the largest of the thread's half
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 4; ++c) tc::ld16_async(scol + 16 * c, s[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                tc::wait_ld16(s[c]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 f = ks[4 * c + i];
                    const float2 y = __fmul2_rn(make_float2(s[c][4 * i], s[c][4 * i + 1]), make_float2(f.x, f.y));
                    const float2 z = __fmul2_rn(make_float2(s[c][4 * i + 2], s[c][4 * i + 3]), make_float2(f.z, f.w));
                    s[c][4 * i] = y.x;
                    s[c][4 * i + 1] = y.y;
                    s[c][4 * i + 2] = z.x;
                    s[c][4 * i + 3] = z.y;
                }
            }
            if (!full) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!((c < 2 ? vis.x : vis.y) >> ((16 * c + i) & 31) & 1)) s[c][i] = -INFINITY;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 16; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], s[c][i], s[c][i + 1]);
            const float mine = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
            // The row's other half; the barrier also carries a wait that gave up,
            // so that all leave together.  (s_mx alternates: a slow thread may
            // still read the tile before.)
            s_mx[b][half][row] = mine;
            ok = group_and(ok);
            if (!ok) break;
            const float mn = fmaxf(m, fmaxf(mine, s_mx[b][half ^ 1][row]) * fac);
            const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen so far
            const float al = fast_exp2(m - ref);
            m = mn;
            float vd = s_vdown[slot];
            float2 up2 = make_float2(1.f, 1.f);
            const float2 fac2 = make_float2(fac, fac), nref2 = make_float2(-ref, -ref);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            // s becomes p a step of 16 keys (one of the PV product) ahead of the
            // split into halves, so that exponentials and the rest overlap.
            auto weights = [&](auto all_seen) {
                constexpr bool FULL = decltype(all_seen)::value;
                uint32_t off[4] = {0u, 0u, 0u, 0u};  // !FULL: keys that are not seen
                auto exps = [&](int c) {
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 e = __ffma2_rn(make_float2(s[c][i], s[c][i + 1]), fac2, nref2);
                        if (!FULL) {
                            off[c] |= (s[c][i] == -INFINITY ? 1u << i : 0u) | (s[c][i + 1] == -INFINITY ? 2u << i : 0u);
                        }
                        s[c][i] = fast_exp2(e.x);
                        s[c][i + 1] = fast_exp2(e.y);
                    }
                };
                exps(0);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c + 1 < 4) exps(c + 1);
                    uint32_t hl[16];  // 8 words hi, 8 words lo: over the scores they come from
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float4 g = vs[4 * c + i / 2];
                        const float2 p = make_float2(s[c][2 * i], s[c][2 * i + 1]);
                        float2 w = __fmul2_rn(FULL ? p : __fmul2_rn(p, up2), i & 1 ? make_float2(g.z, g.w) : make_float2(g.x, g.y));
                        if (!FULL) {  // what is not seen (p = 0) takes no part, whatever its scale
                            if (off[c] >> (2 * i) & 1) w.x = 0.f;
                            if (off[c] >> (2 * i + 1) & 1) w.y = 0.f;
                        }
                        sum[i & 1] = __fadd2_rn(sum[i & 1], p);
                        // hi: the top 11 bits (exact in FP16), cheaper than to round and convert back
                        const float2 top = make_float2(tc::tf32_hi(w.x), tc::tf32_hi(w.y));
                        const __half2 hi = __floats2half2_rn(top.x, top.y);
                        const float2 r = __fadd2_rn(w, make_float2(-top.x, -top.y));
                        const __half2 lo = __floats2half2_rn(r.x, r.y);
                        hl[i] = *reinterpret_cast<const uint32_t *>(&hi);
                        hl[8 + i] = *reinterpret_cast<const uint32_t *>(&lo);
                    }
                    tc::st16u_free(scol + 16 * c, hl);
                }
            };
            if (full && vd > 0.f) {
                weights(std::true_type());
            } else {
                if (vd < 0.f) {
                    // Scales far apart (every thread's vd says so): the unit is that of the
                    // row's largest weight, known to a factor of two from its scores and
                    // the scales' exponents.
                    float most = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 g = vs[4 * c + i / 4];
                            const float gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (gs[e] > 0.f)
                                    most = fmaxf(most, fmaf(s[c][i + e], fac, float(int(__float_as_uint(gs[e]) >> 23) - 127)));
                        }
                    s_most[b][half][row] = most;
                    (void)group_and(true);
                    most = fmaxf(most, s_most[b][half ^ 1][row]);
                    const int u = most == -INFINITY ? 0 : int(fminf(fmaxf(14.f - ceilf(most - ref), -1.f), 120.f));
                    up2.x = up2.y = __uint_as_float(uint32_t(127 + u) << 23);
                    vd *= -__uint_as_float(uint32_t(127 - u) << 23);
                }
                weights(std::false_type());
            }
            l = l * al + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
            tc::wait_st();
            // O(j-1), whose product ran beside this softmax; then PV(j) may start
            if (j > 0) ok = absorb(j - 1, alpha, vdown, s);
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[b]);
            alpha = al;
            vdown = vd;
        }
        if (ok && n_kt > 0) ok = absorb(n_kt - 1, alpha, vdown, s);
        if (!ok && lane == 0) atomicExch(&s_fail, 1);
        s_l[half][row] = l;
        ok = group_and(ok);
        if (ok) {
            // through shared memory (where Q was staged), so that a warp stores whole rows
            constexpr int RS = HD * 4 + 16;
            static_assert(kBM * RS <= 2 * kBM * C::kQRow, "output staging");
            const float sum = s_l[0][row] + s_l[1][row], by = it.part < 0 ? 1.f / sum : 1.f;
            if (it.part >= 0 && half == 0 && tok < t_end)
                reinterpret_cast<float2 *>(a.part_ml)[size_t(it.part) * kBM + row] = make_float2(m, sum);
#pragma unroll
            for (int i = 0; i < OC / 4; ++i)  // columns 64-127 have neighbouring 8-dim granules swapped
                *reinterpret_cast<float4 *>(base + C::kQ + row * RS + half * OC * 4 + 16 * (HD == 128 && half ? i ^ 2 : i)) =
                    make_float4(o[4 * i] * by, o[4 * i + 1] * by, o[4 * i + 2] * by, o[4 * i + 3] * by);
            (void)group_and(true);
            constexpr int LPR = HD / 4;  // lanes of a row
#pragma unroll 4
            for (int r = warp * (32 / LPR) + lane / LPR; r < kBM; r += 8 * (32 / LPR)) {
                const int t = t0 + r / G;
                float *dst = it.part < 0 ? a.out + (size_t(tok0 + t) * a.L.n_kv * G + h * G + r % G) * HD
                                         : a.part_o + (size_t(it.part) * kBM + r) * HD;
                if (t < t_end)
                    *reinterpret_cast<float4 *>(dst + 4 * (lane % LPR)) =
                        *reinterpret_cast<const float4 *>(base + C::kQ + r * RS + 16 * (lane % LPR));
            }
        }
    } else if (warp < 12) {
        // ================= converters: codes -> FP16 operand tiles =============
        regs_down<kRegsConvert>();
        constexpr int N = kBN * HD / 16 / 128;  // 16-byte chunks of a tile a thread takes
        const int ct = tid - 256;
        const size_t r0 = tab.slot[seq] * a.L.slot_rows + h * a.L.head_rows;
        const uint8_t *gk = a.L.k + r0 * HD, *gv = a.L.v + r0 * HD;
        const float *gks = a.L.ks + r0, *gvs = a.L.vs + r0;
        grid_dependency_wait();  // the append kernel has stored the run's rows
        grid_launch_dependents();
        // Half an operand tile is in flight while the half before it is stored:
        // K's two halves, V's two, the next tile's K, ... in two register sets.
        constexpr int N2 = N / 2;
        uint4 w[2][N2];
        auto load = [&](const uint8_t *g, int j, int half) {
            const uint4 *src = reinterpret_cast<const uint4 *>(g + size_t(j0 + j) * kBN * HD) + ct + half * 128 * N2;
#pragma unroll
            for (int i = 0; i < N2; ++i) w[half][i] = src[128 * i];
        };
        // Chunk ct + 128 i (16 bytes each) of a tile: its line is (ct >> 3) + 16 i,
        // so its dims and its place in an 8-row swizzle group are the same for
        // every i.  Chunks 4-7 have their two 8-dim granules swapped, so that
        // eight neighbouring threads meet eight different bank groups; Q's dims
        // 64-127 and O's columns 64-127 are in that order too.
        int row, ch;
        if (HD == 128) {
            row = ct >> 3;
            ch = (ct & 7) ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2));
        } else {
            const int x = (ct & 7) ^ (((ct >> 3) & 3) << 1);
            row = 2 * (ct >> 3) + (x >> 2);
            ch = x & 3;
        }
        constexpr uint32_t kStep = HD == 128 ? 2048 : 4096;  // 16 or 32 rows on
        const bool upper = ch & 4;
        const uint32_t g0 = (ch >> 2) * C::kChunk + (row >> 3) * 1024 + (row & 7) * 128 +
                            (((2 * (ch & 3) + upper) ^ (row & 7)) << 4);
        auto store = [&](uint32_t dst, int half) {
            unsigned char *d0 = base + dst + g0 + half * N2 * kStep, *d1 = base + dst + (g0 ^ 16) + half * N2 * kStep;
#pragma unroll
            for (int i = 0; i < N2; ++i) {
                const uint4 x = w[half][i];
                *reinterpret_cast<uint4 *>(d0 + i * kStep) = expand(x.x, x.y);
                *reinterpret_cast<uint4 *>(d1 + i * kStep) = expand(x.z, x.w);
            }
        };
        ScaleSpan span;
        bool ok = true, awaited = a.k_new == nullptr;
        // before the first load of a tile that has rows of the run
        auto settle = [&](int j) {
            if (awaited || (j0 + j + 1) * kBN <= pos) return;
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.new_full, 0));
            awaited = true;
        };
        if (n_kt > 0) {
            settle(0);
            load(gk, 0, 0);
            load(gk, 0, 1);
        }
        for (int j = 0; j < n_kt && ok; ++j) {
            const int b = j & 1, slot = j & (kSlots - 1);
            if (j >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[b], par(j - 2)));
            if (!ok) break;
            store(C::kK + b * C::kOp, 0);
            load(gv, j, 0);
            store(C::kK + b * C::kOp, 1);
            load(gv, j, 1);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.k_full[b]);
            // Scales (of rows the block may see; the others count as 0).  Slot
            // j % 4 was last read for tile j - 4: S(j-2) was issued after
            // PV(j-4), that after the softmax of tile j-4.
            {
                const int first = (j0 + j) * kBN, n = kv_end - first;
                uint32_t t = 0u, l = 0x7f7fffffu;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 32 * i + lane;
                    ScaleSpan::look(r < n ? gvs[first + r] : 0.f, r < n, t, l);
                }
                const int e = max(int(__float_as_uint(span.take(t, l)) >> 23), 15);
                const float vup = __uint_as_float(uint32_t(268 - e) << 23);
                s_ks[slot][ct] = ct < n ? gks[first + ct] * a.scale : 0.f;
                s_vs[slot][ct] = ct < n ? gvs[first + ct] * vup : 0.f;
                if (ct == 0) s_vdown[slot] = __uint_as_float(uint32_t(e - 14) << 23 | (span.wide() ? 0x80000000u : 0u));
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.sc_full[slot]);
            }
            if (j >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full[b], par(j - 2)));
            if (!ok) break;
            if (j + 1 < n_kt) settle(j + 1);
            if (!ok) break;
            store(C::kV + b * C::kOp, 0);
            if (j + 1 < n_kt) load(gk, j + 1, 0);
            store(C::kV + b * C::kOp, 1);
            if (j + 1 < n_kt) load(gk, j + 1, 1);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.v_full[b]);
        }
        if (!ok && lane == 0) atomicExch(&s_fail, 1);
    } else {
        regs_down<kRegsIssue>();
        if (warp > 12 && a.k_new) {
            // ================= the run's rows that this block reads =============
            append(std::integral_constant<int, 1>(), warp - 13);
        }
        if (warp == 12) {
            // ================= MMA issuer ======================================
            const bool leader = tc::elect_one_sync();
            constexpr uint32_t idesc_s = tc::idesc_f16(kBM, kBN, false);
            constexpr uint32_t idesc_o = tc::idesc_f16(kBM, HD, true);
            const uint64_t dk = tc::sw128_kmajor_desc(sbase + C::kK);
            const uint64_t dv = tc::sw128_nmajor_desc(sbase + C::kV, C::kChunk);
            int s_issued = 0, pv_issued = 0;
            auto wait_all = [](uint64_t *bar, uint32_t parity) {
                return bool(__all_sync(0xffffffffu, mbar_wait(bar, parity)));
            };
            bool ok = wait_all(&bars.q_ready, 0);
            // S(j) = (Q hi + Q lo) K^T.  Its columns hold P(j-2) until PV(j-2) is done.
            auto issue_s = [&](int j) {
                const int b = j & 1;
                ok = ok && wait_all(&bars.k_full[b], par(j));
                if (ok && j >= 2) ok = wait_all(&bars.o_full[b], par(j - 2));
                if (!ok) return;
                tc::fence_after_sync();
                if (leader) {
                    const uint64_t k = dk + uint64_t(b) * (C::kOp >> 4);
#pragma unroll 1
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            const uint64_t off = ((kk >> 2) * C::kChunk + (kk & 3) * 32) >> 4;
                            tc::mma_f16_ts(tmem + C::kColS(b), tmem + C::kColQ(u) + 8 * kk, k + off, idesc_s,
                                            u + kk > 0 ? 1u : 0u);
                        }
                    tc::commit(&bars.s_full[b]);
                }
                __syncwarp();
                ++s_issued;
            };
            // O(j) = (P hi + P lo) V, from zero.
            auto issue_pv = [&](int j) {
                const int b = j & 1;
                ok = ok && wait_all(&bars.v_full[b], par(j)) && wait_all(&bars.p_full[b], par(j));
                if (!ok) return;
                tc::fence_after_sync();
                if (leader) {
                    const uint64_t v = dv + uint64_t(b) * (C::kOp >> 4);
#pragma unroll
                    for (int kk = 0; kk < kBN / 16; ++kk)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            tc::mma_f16_ts(tmem + C::kColO, tmem + C::kColS(b) + 16 * kk + 8 * u,
                                            v + uint64_t(kk * 2048 >> 4), idesc_o, u + kk > 0 ? 1u : 0u);
                    tc::commit(&bars.o_full[b]);
                }
                __syncwarp();
                ++pv_issued;
            };
            if (n_kt > 0) issue_s(0);
            for (int j = 0; j < n_kt && ok; ++j) {
                if (j + 1 < n_kt) issue_s(j + 1);
                if (ok) issue_pv(j);
            }
            if (!ok && leader) atomicExch(&s_fail, 1);
            // nothing may be in flight when shared memory and TMEM go: wait
            // (bounded) for the last product of either kind in either buffer
            for (int b = 0; b < 2; ++b) {
                const int ls = s_issued - 1 - ((s_issued - 1 - b) & 1);
                if (ls >= 0) (void)mbar_wait(&bars.s_full[b], par(ls));
                const int lp = pv_issued - 1 - ((pv_issued - 1 - b) & 1);
                if (lp >= 0) (void)mbar_wait(&bars.o_full[b], par(lp));
            }
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (tid == 0 && s_fail) report_error(a.err, kDevWaitTimeout);
    if (warp == 12) tc::dealloc(tmem, C::kCols);
}

// Join the splits: one warp for each query row of a tile that was split.
template <int HD, int G>
__global__ void __launch_bounds__(256)
q8_tc_join_kernel(const TcArgs a, const __grid_constant__ Q8Seqs tab, const __grid_constant__ Q8TcPlan plan) {
    grid_launch_dependents();
    // where things are, while the kernel before runs
    const int lane = threadIdx.x & 31;
    const int n_kv = a.L.n_kv;
    // block: 8 rows of a (query tile, kv head); tiles numbered as in the plan
    const int tile = blockIdx.x / (kBM / 8), row = (blockIdx.x % (kBM / 8)) * 8 + (threadIdx.x >> 5);
    const int x = tile / n_kv, h = tile - x * n_kv;
    int lo = 0, hi = plan.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (plan.tile0[mid] <= x) lo = mid; else hi = mid - 1;
    }
    const int ns = plan.nsplit[lo], seq = plan.seq[lo];
    const int i = x - plan.tile0[lo], qt = plan.n_qt[lo] - 1 - i;
    const int tok = qt * (kBM / G) + row / G;
    const int tok0 = tab.tok0[seq], n_new = tab.tok0[seq + 1] - tok0;
    const size_t p0 = size_t(plan.part0[lo] + i * ns) * n_kv + h;  // splits n_kv apart
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + p0 * kBM + row;
    const float4 *po = reinterpret_cast<const float4 *>(a.part_o) + (p0 * kBM + row) * (HD / 4) + lane % (HD / 4);
    grid_dependency_wait();
    if (ns == 1 || tok >= n_new) return;
    // 32 splits at a time: lane s has split s's maximum and sum, the row's dims
    // are spread over the lanes; 16 splits' loads in flight, the first before the
    // weights are known
    constexpr int U = 16;
    float mx = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f), z[U];
    for (int s0 = 0; s0 < ns; s0 += 32) {
        const float2 y = s0 + lane < ns ? ml[size_t(s0 + lane) * n_kv * kBM] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < U; ++k) z[k] = po[size_t(min(s0 + k, ns - 1)) * n_kv * kBM * (HD / 4)];
        float top = y.x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        top = fmaxf(top, mx);
        const float back = mx == -INFINITY ? 0.f : fast_exp2(mx - top);
        // a split that had nothing this row sees weighs nothing; its sums are taken in
        // all the same (zeros, or the NaN that it saw)
        const float e = y.x == -INFINITY ? 0.f : fast_exp2(y.x - top);
        float part = y.y * e;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) part += __shfl_xor_sync(0xffffffffu, part, off);
        mx = top;
        sum = sum * back + part;
        v.x *= back; v.y *= back; v.z *= back; v.w *= back;
        for (int s1 = s0;;) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const float w = __shfl_sync(0xffffffffu, e, (s1 + k - s0) & 31);
                if (s1 + k >= ns) continue;
                v.x += z[k].x * w; v.y += z[k].y * w; v.z += z[k].z * w; v.w += z[k].w * w;
            }
            s1 += U;
            if (s1 >= min(s0 + 32, ns)) break;
#pragma unroll
            for (int k = 0; k < U; ++k) z[k] = po[size_t(min(s1 + k, ns - 1)) * n_kv * kBM * (HD / 4)];
        }
    }
    const float inv = 1.f / sum;
    if (lane < HD / 4)
        *reinterpret_cast<float4 *>(a.out + (size_t(tok0 + tok) * n_kv * G + h * G + row % G) * HD + 4 * lane) =
            make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
}

template <int HD, int G, bool TREE>
int launch_tc(leap_ctx *c, const TcArgs &a, const Q8Seqs &tab, const Q8TcPlan &plan, const Q8See<TREE> &see) {
    // behind the append kernel it may start early: it waits before it reads the cache
    const int early = a.k_new ? 0 : 1;
    auto fn = q8_tc_kernel<HD, G, TREE>;
    if (int st = set_kernel_smem(reinterpret_cast<const void *>(fn), Tc<HD>::kSmem, "cudaFuncSetAttribute(q8_tc)"))
        return st;
    // The register split adds up to 128 a thread; a build that launches with
    // fewer would wait for registers that never come.
    static std::atomic<bool> checked{false};
    if (!checked.load(std::memory_order_relaxed)) {
        cudaFuncAttributes fa;
        if (int st = cuda_status(cudaFuncGetAttributes(&fa, fn), "cudaFuncGetAttributes(q8_tc)")) return st;
        if (fa.numRegs != kLaunchRegs) {
            set_error("q8_tc_kernel was built with %d registers a thread, not %d", fa.numRegs, kLaunchRegs);
            return LEAP_ERR_CUDA;
        }
        checked.store(true, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(plan.item0[plan.n]) * c->n_kv);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Tc<HD>::kSmem;
    cfg.stream = c->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = early;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int st = cuda_status(cudaLaunchKernelEx(&cfg, fn, a, tab, plan, see), "q8_tc_kernel launch");
    if (st != LEAP_OK || plan.n_parts == 0) return st;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(unsigned(plan.tile0[plan.n]) * c->n_kv * (kBM / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, q8_tc_join_kernel<HD, G>, a, tab, plan), "q8_tc_join_kernel launch");
}

template <int HD, int G>
int launch_tc_g(leap_ctx *c, const TcArgs &a, const Q8Seqs &tab, const Q8TcPlan &plan, const Q8Tree *tree) {
    return tree ? launch_tc<HD, G, true>(c, a, tab, plan, q8_see(*tree))
                : launch_tc<HD, G, false>(c, a, tab, plan, Q8See<false>());
}

// A block's work apart from its tiles (queries, first loads, output) costs
// about as much as kOverhead tiles, the join of splits as two and one for every 16
// of a tile, whose loads are in flight together.
constexpr long kOverhead = 5, kJoinSplits = 16;

// Blocks as the hardware hands them out, in order, each to the SM that is free first:
// how long all take.  Loads are kept as counts of SMs; those of a ring differ by one
// block at most.
struct Schedule {
    static constexpr int kRing = 1024;
    int free_at[kRing] = {};  // SMs that fall free at a time, modulo kRing
    long now = 0, end = 0;
    int unit;                 // tiles of a time step

    Schedule(int sms, int longest) : unit((longest + int(kOverhead)) / (kRing - 8) + 1) { free_at[0] = sms; }
    void put(long blocks, int tiles) {
        const int t = (tiles + int(kOverhead) + unit - 1) / unit;
        while (blocks > 0) {
            while (free_at[now % kRing] == 0) ++now;
            const int k = int(std::min(blocks, long(free_at[now % kRing])));
            free_at[now % kRing] -= k;
            free_at[(now + t) % kRing] += k;
            blocks -= k;
            end = std::max(end, now + t);
        }
    }
    long time() const { return end * unit; }
};
constexpr int kScheduleTiles = 128;  // query tiles up to which it is worked out (host time)

// Sequences longest first, and the tiles of a split: the chunk that takes least, by
// Schedule, or for many query tiles by all work / SMs and part of a block at the end,
// among those whose partials fit the scratch.  Device us with all work / SMs alone and
// so: 8 ragged trees (64/8x128) 97, 87; 16 nodes each on one of 32768 and 19 of 300 rows
// 71, 61; 16 nodes on 2048 rows 19.1, 15.5; of 75 batches one lost (6%).
void plan_tc(const leap_ctx *c, const Q8Seqs &tab, bool tree, Q8TcPlan &plan) {
    const int bt = kBM / c->group;
    plan.n = 0;
    for (int i = 0; i < tab.n_seq; ++i)
        if (tab.tok0[i + 1] > tab.tok0[i]) plan.seq[plan.n++] = i;
    auto rows = [&](int i) { return tab.pos[i] + tab.tok0[i + 1] - tab.tok0[i]; };
    std::sort(plan.seq, plan.seq + plan.n, [&](int x, int y) { return rows(x) != rows(y) ? rows(x) > rows(y) : x < y; });
    unsigned all[kMaxSeqPerLaunch], mean[kMaxSeqPerLaunch];  // tiles of a sequence, of a query tile on average
    for (int i = 0; i < plan.n; ++i) {
        const int s = plan.seq[i];
        plan.n_qt[i] = (tab.tok0[s + 1] - tab.tok0[s] + bt - 1) / bt;
        all[i] = unsigned(rows(s) + kBN - 1) / kBN;
        // causal tiles see from pos + bt rows on to all of them
        mean[i] = tree ? all[i] : (all[i] + unsigned(tab.pos[s] + bt + kBN - 1) / kBN + 1) / 2;
    }
    const int longest = plan.n ? int(all[0]) : 1;
    long n_tiles = 0;
    for (int i = 0; i < plan.n; ++i) n_tiles += plan.n_qt[i];
    long best = -1;
    plan.chunk = longest;
    for (int chunk = longest; chunk >= 1; chunk -= std::max(chunk / 16, 1)) {
        long work = 0, parts = 0, items = 0;
        for (int i = 0; i < plan.n; ++i) {
            const unsigned ns = (all[i] + chunk - 1) / chunk;
            work += plan.n_qt[i] * (mean[i] + ns * kOverhead);
            if (ns > 1) parts += plan.n_qt[i] * long(ns);
            items += plan.n_qt[i] * long(ns);
        }
        if (parts * c->n_kv > c->q8_tc_parts) break;
        const long block = chunk + kOverhead, sms = c->num_sms;
        const long splits = (longest + chunk - 1) / chunk;
        const long join = parts ? 2 + (splits + kJoinSplits - 1) / kJoinSplits : 0, mean_load = work * c->n_kv / sms;
        long cost = join + block;
        if (items * c->n_kv > sms) {
            if (n_tiles > kScheduleTiles) {
                cost = join + std::max(mean_load + block / 4, block);
            } else {
                if (best >= 0 && join + std::max(mean_load, block) >= best) continue;
                Schedule when(c->num_sms, longest);
                for (int i = 0; i < plan.n; ++i) {
                    const int s = plan.seq[i], n = tab.tok0[s + 1] - tab.tok0[s];
                    const int ns = int(all[i] + chunk - 1) / chunk;
                    for (int qt = plan.n_qt[i] - 1; qt >= 0; --qt) {
                        const int tiles = tree ? int(all[i]) : (tab.pos[s] + std::min((qt + 1) * bt, n) + kBN - 1) / kBN;
                        const int full = tiles / chunk, rest = full < ns;
                        when.put(long(full) * c->n_kv, chunk);
                        if (rest) when.put(c->n_kv, tiles - full * chunk);
                        when.put(long(ns - full - rest) * c->n_kv, 0);  // splits that this tile does not see
                    }
                }
                cost = join + when.time();
            }
        }
        if (best < 0 || cost < best) {
            best = cost;
            plan.chunk = chunk;
        }
    }
    int items = 0, tiles = 0, parts = 0;
    for (int i = 0; i < plan.n; ++i) {
        const int ns = int(all[i] + plan.chunk - 1) / plan.chunk;
        plan.nsplit[i] = ns;
        plan.item0[i] = items;
        plan.tile0[i] = tiles;
        plan.part0[i] = parts;
        items += plan.n_qt[i] * ns;
        tiles += plan.n_qt[i];
        if (ns > 1) parts += plan.n_qt[i] * ns;
    }
    plan.item0[plan.n] = items;
    plan.tile0[plan.n] = tiles;
    plan.n_parts = parts;
}

}  // namespace

// Partials of 128 rows: four an SM, or every query tile of the longest runs in splits
// of one key tile where that is less (plan_tc keeps to what there is).
int q8_tc_parts_needed(const leap_ctx *c) {
    const long splits = (long(c->max_seq) + kBN - 1) / kBN;
    if (splits < 2) return 0;
    const long tiles = (long(c->max_seq) * c->group + kBM - 1) / kBM;
    const long all = std::min(c->max_batch, kMaxSeqPerLaunch) * c->n_kv * std::min(tiles, 1L << 20) * std::min(splits, 1L << 20);
    return int(std::min(all, 4L * c->num_sms));
}

int q8_tc_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q, const float *k,
                 const float *v, float *out) {
    Q8TcPlan plan;
    plan_tc(c, tab, tree != nullptr, plan);
    // One query tile a sequence: every new row is read by one block, which can store
    // it itself (a launch less: 5 nodes on 300 rows, 13.2 -> 11.6 us on the device and
    // 4 us less to issue), unless there are many (32 kv heads, device us of appended
    // by the blocks and by the kernel: 16 rows 11.8, 10.9; 64 rows 15.7, 11.9; 128 rows
    // 20.8, 13.0; 4 x 64 behind 2000 43.9, 46.1).  Otherwise several blocks read it.
    constexpr int kMostFused = 64;
    bool fused = true;
    for (int i = 0; i < plan.n; ++i)
        fused = fused && plan.n_qt[i] == 1 && tab.tok0[plan.seq[i] + 1] - tab.tok0[plan.seq[i]] <= kMostFused;
    if (!fused)
        if (int st = q8_append(c, layer, tab, tree, k, v)) return st;
    TcArgs a;
    a.q = q;
    a.k_new = fused ? k : nullptr;
    a.v_new = fused ? v : nullptr;
    a.out = out;
    a.L = q8_layer(c, layer);
    a.rope_cos = c->rope_cos;
    a.rope_sin = c->rope_sin;
    a.part_o = c->q8_tc_part_o;
    a.part_ml = c->q8_tc_part_ml;
    a.err = c->d_err;
    a.scale = kLog2e / (16384.f * sqrtf(float(c->hd)));
    switch (c->hd * 100 + c->group) {
        case 12801: return launch_tc_g<128, 1>(c, a, tab, plan, tree);
        case 12802: return launch_tc_g<128, 2>(c, a, tab, plan, tree);
        case 12804: return launch_tc_g<128, 4>(c, a, tab, plan, tree);
        case 12808: return launch_tc_g<128, 8>(c, a, tab, plan, tree);
        case 6401: return launch_tc_g<64, 1>(c, a, tab, plan, tree);
        case 6402: return launch_tc_g<64, 2>(c, a, tab, plan, tree);
        case 6404: return launch_tc_g<64, 4>(c, a, tab, plan, tree);
        case 6408: return launch_tc_g<64, 8>(c, a, tab, plan, tree);
        default:
            set_error("unsupported head_dim %d / kv_mul %d", c->hd, c->group);
            return LEAP_ERR_INVALID;
    }
}

}  // namespace leap
