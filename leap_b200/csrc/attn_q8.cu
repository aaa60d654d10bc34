// attn_q8.cu — attention over the 8-bit KV cache.
#include "q8.cuh"

namespace leap {
namespace {

// One block for each (new token, kv head), its warps on every fourth row: a
// lane holds HD/32 dims of the G query heads, scores are warp sums, each warp
// keeps a running maximum and sum, and the block joins them at the end.
template <int HD, int G, bool TREE>
__global__ void __launch_bounds__(128)
q8_attn_kernel(const float *__restrict__ q, float *__restrict__ out, const Q8Layer L,
               const float *__restrict__ rope_cos, const float *__restrict__ rope_sin,
               const __grid_constant__ Q8Seqs tab, const __grid_constant__ Q8Tree tree,
               float scale_log2) {
    constexpr int E = HD / 32, W = 4;
    __shared__ float s_m[W][G], s_l[W][G], s_o[W][G][HD];
    const int t = blockIdx.x, h = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seq = q8_seq_of(tab, t);
    const int t0 = tab.tok0[seq], i = t - t0, pos = tab.pos[seq];
    int at = pos + i;
    if (TREE) {
        at = pos;
        for (int p = tree.parent[t]; p >= 0; p = tree.parent[t0 + p]) ++at;
    }
    float qr[G][E], m[G], l[G], o[G][E];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float *x = q + (size_t(t) * L.n_kv * G + h * G + g) * HD + E * lane;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const size_t a = size_t(at) * (HD / 2) + (E * lane + e) / 2;
            const float2 r = rope_pair(x[e], x[e + 1], rope_cos[a], rope_sin[a]);
            qr[g][e] = r.x;
            qr[g][e + 1] = r.y;
            o[g][e] = o[g][e + 1] = 0.f;
        }
        m[g] = -INFINITY;
        l[g] = 0.f;
    }
    const size_t r0 = tab.slot[seq] * L.slot_rows + h * L.head_rows;
    for (int row = warp; row <= pos + i; row += W) {
        if (TREE && row >= pos) {  // a node: itself or an ancestor?
            int p = i;
            while (p > row - pos) p = tree.parent[t0 + p];
            if (p != row - pos) continue;
        }
        const uint32_t ck = q8_load_codes<HD>(L.k + r0 * HD, row, lane);
        const uint32_t cv = q8_load_codes<HD>(L.v + r0 * HD, row, lane);
        const float sk = L.ks[r0 + row] * scale_log2, sv = L.vs[r0 + row];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s += qr[g][e] * float(int((ck >> (8 * e)) & 255u) - 128);
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            s *= sk;
            const float mn = fmaxf(m[g], s);
            const float alpha = exp2f(m[g] - mn), p = exp2f(s - mn);
            m[g] = mn;
            l[g] = l[g] * alpha + p;
#pragma unroll
            for (int e = 0; e < E; ++e)
                o[g][e] = o[g][e] * alpha + p * (float(int((cv >> (8 * e)) & 255u) - 128) * sv);
        }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        s_m[warp][g] = m[g];
        s_l[warp][g] = l[g];
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[warp][g][E * lane + e] = o[g][e];
    }
    __syncthreads();
    for (int f = threadIdx.x; f < G * HD; f += 128) {
        const int g = f / HD, d = f % HD;
        float mx = s_m[0][g], sum = 0.f, acc = 0.f;
        for (int w = 1; w < W; ++w) mx = fmaxf(mx, s_m[w][g]);
        for (int w = 0; w < W; ++w) {
            if (s_l[w][g] == 0.f) continue;  // no row came to this warp
            const float a = exp2f(s_m[w][g] - mx);
            sum += s_l[w][g] * a;
            acc += s_o[w][g][d] * a;
        }
        out[(size_t(t) * L.n_kv * G + h * G + g) * HD + d] = acc / sum;
    }
}

template <int HD, int G>
int launch(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
           float *out) {
    static const Q8Tree none = {};
    const dim3 grid(tab.tok0[tab.n_seq], c->n_kv);
    const float scale = kLog2e / sqrtf(float(HD));
    if (tree)
        q8_attn_kernel<HD, G, true><<<grid, 128, 0, c->stream>>>(
            q, out, q8_layer(c, layer), c->rope_cos, c->rope_sin, tab, *tree, scale);
    else
        q8_attn_kernel<HD, G, false><<<grid, 128, 0, c->stream>>>(
            q, out, q8_layer(c, layer), c->rope_cos, c->rope_sin, tab, none, scale);
    return cuda_status(cudaGetLastError(), "q8_attn_kernel launch");
}

}  // namespace

int q8_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
              const float *k, const float *v, float *out) {
    if (tab.tok0[tab.n_seq] == 0) return LEAP_OK;
    int most = 0;
    for (int i = 0; i < tab.n_seq; ++i)
        if (tab.tok0[i + 1] - tab.tok0[i] > most) most = tab.tok0[i + 1] - tab.tok0[i];
    if (most * c->group <= kQ8Rows) return q8_rows_attend(c, layer, tab, tree, q, k, v, out);
    if (int st = q8_append(c, layer, tab, tree, k, v)) return st;
    switch (c->hd * 100 + c->group) {
        case 12801: return launch<128, 1>(c, layer, tab, tree, q, out);
        case 12802: return launch<128, 2>(c, layer, tab, tree, q, out);
        case 12804: return launch<128, 4>(c, layer, tab, tree, q, out);
        case 12808: return launch<128, 8>(c, layer, tab, tree, q, out);
        case 6401: return launch<64, 1>(c, layer, tab, tree, q, out);
        case 6402: return launch<64, 2>(c, layer, tab, tree, q, out);
        case 6404: return launch<64, 4>(c, layer, tab, tree, q, out);
        case 6408: return launch<64, 8>(c, layer, tab, tree, q, out);
        default:
            set_error("unsupported head_dim %d / kv_mul %d", c->hd, c->group);
            return LEAP_ERR_INVALID;
    }
}

}  // namespace leap
