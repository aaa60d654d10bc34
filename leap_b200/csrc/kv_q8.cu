// kv_q8.cu — rows into and out of the 8-bit KV cache: quantise (with or
// without the rotation), read back, and the compaction after a verified tree.
//
// All of it is bound by HBM: a row of K and V of one kv head is 8*HD bytes of
// FP32 on one side and 2*(HD + 4) bytes on the other.  One warp takes two
// (token, kv head) pairs, all their loads in flight together: a lane holds HD/32 neighbouring dims of k and of v (a
// rotation pair never leaves a lane), the row's maximum is one warp reduction,
// and each row is stored as one 128-byte (or 64-byte) line.
#include <algorithm>

#include "q8.cuh"

namespace leap {
namespace {

constexpr int kWarps = 8;  // warps of a block
constexpr int kItems = 2;  // (token, kv head) pairs of a warp

enum { kRaw = 0, kCausal = 1, kTree = 2 };  // what the append kernel rotates by

template <int HD>
struct Vec;
template <> struct Vec<128> { using T = float4; };
template <> struct Vec<64> { using T = float2; };

// MODE kRaw: rows as they are; kCausal: k rotated for its row's position;
// kTree: k rotated for position pos + depth.
template <int HD, int MODE>
__global__ void __launch_bounds__(32 * kWarps)
q8_append_kernel(const float *__restrict__ k, const float *__restrict__ v, const __grid_constant__ Q8Layer L,
                 const float *__restrict__ rope_cos, const float *__restrict__ rope_sin,
                 const __grid_constant__ Q8Seqs tab,
                 const __grid_constant__ Q8See<MODE == kTree> see) {
    constexpr int E = HD / 32;
    grid_launch_dependents();  // what follows waits for this grid before it reads
    const int lane = threadIdx.x & 31;
    const int first = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kItems;
    const int items = tab.tok0[tab.n_seq] * L.n_kv;
    float x[kItems][E], y[kItems][E];
#pragma unroll
    for (int u = 0; u < kItems; ++u)
        if (first + u < items) {
            load_vec<E>(x[u], k + size_t(first + u) * HD + E * lane);
            load_vec<E>(y[u], v + size_t(first + u) * HD + E * lane);
        }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        if (first + u >= items) return;
        const int t = (first + u) / L.n_kv, h = first + u - t * L.n_kv;
        const int seq = q8_seq_of(tab, t);
        const int i = t - tab.tok0[seq];
        const int row = tab.pos[seq] + i;
        if (MODE != kRaw) {
            const size_t c = size_t(tab.pos[seq] + see.depth(tab.tok0[seq], i)) * (HD / 2) + lane * (E / 2);
            float rc[E / 2], rs[E / 2];
            load_vec<E / 2>(rc, rope_cos + c);
            load_vec<E / 2>(rs, rope_sin + c);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 r = rope_pair(x[u][e], x[u][e + 1], rc[e / 2], rs[e / 2]);
                x[u][e] = r.x;
                x[u][e + 1] = r.y;
            }
        }
        const size_t r0 = tab.slot[seq] * L.slot_rows + h * L.head_rows;
        uint32_t c;
        const float sk = q8_quantize<E>(x[u], c);
        q8_store_codes<HD>(L.k + r0 * HD, row, lane, c);
        const float sv = q8_quantize<E>(y[u], c);
        q8_store_codes<HD>(L.v + r0 * HD, row, lane, c);
        if (lane == 0) {
            L.ks[r0 + row] = sk;
            L.vs[r0 + row] = sv;
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(32 * kWarps)
q8_read_kernel(float *__restrict__ k, float *__restrict__ v, const __grid_constant__ Q8Layer L,
               const __grid_constant__ Q8Seqs tab) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    const int first = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kItems;
    const int items = tab.tok0[tab.n_seq] * L.n_kv;
    uint32_t ck[kItems], cv[kItems];
    float sk[kItems], sv[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u)
        if (first + u < items) {
            const int t = (first + u) / L.n_kv, h = first + u - t * L.n_kv;
            const int seq = q8_seq_of(tab, t);
            const int row = tab.pos[seq] + t - tab.tok0[seq];
            const size_t r0 = tab.slot[seq] * L.slot_rows + h * L.head_rows;
            ck[u] = q8_load_codes<HD>(L.k + r0 * HD, row, lane);
            cv[u] = q8_load_codes<HD>(L.v + r0 * HD, row, lane);
            sk[u] = L.ks[r0 + row];
            sv[u] = L.vs[r0 + row];
        }
    using V = typename Vec<HD>::T;
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
        if (first + u >= items) return;
        V x, y;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            reinterpret_cast<float *>(&x)[e] = float(int((ck[u] >> (8 * e)) & 255u) - 128) * sk[u];
            reinterpret_cast<float *>(&y)[e] = float(int((cv[u] >> (8 * e)) & 255u) - 128) * sv[u];
        }
        *reinterpret_cast<V *>(k + size_t(first + u) * HD + E * lane) = x;
        *reinterpret_cast<V *>(v + size_t(first + u) * HD + E * lane) = y;
    }
}

// The same from an FP32 cache.
__global__ void __launch_bounds__(256)
f32_read_kernel(float *__restrict__ k, float *__restrict__ v, const float *__restrict__ kc,
                const float *__restrict__ vc, size_t head_stride, size_t slot_stride, int n_kv,
                int hd4, const __grid_constant__ Q8Seqs tab) {
    const long n = long(tab.tok0[tab.n_seq]) * n_kv * hd4;
    const long f = blockIdx.x * 256L + threadIdx.x;
    if (f >= n) return;
    const int item = int(f / hd4), d = int(f % hd4);
    const int t = item / n_kv, h = item - t * n_kv;
    const int seq = q8_seq_of(tab, t);
    const size_t src = tab.slot[seq] * slot_stride + h * head_stride +
                       (size_t(tab.pos[seq] + t - tab.tok0[seq]) * hd4 + d) * 4;
    reinterpret_cast<float4 *>(k)[f] = *reinterpret_cast<const float4 *>(kc + src);
    reinterpret_cast<float4 *>(v)[f] = *reinterpret_cast<const float4 *>(vc + src);
}

// Keep rows pos + node[j] as pos + j.  A thread moves the same dims of every
// row, in order of j; node[] increases strictly, so a row is read before
// anything is written to it (node[j] >= j), also when kBatch rows are read
// ahead of their writes.  Block: (sequence, layer, kv head); T: what a thread
// moves of a K or V row (RowOff: where that lies in row r).
constexpr int kBatch = 8;
template <typename T, typename RowOff>
__device__ __forceinline__ void keep_rows(T *head, int n, int pos, const int8_t *node, RowOff off) {
    for (int j0 = 0; j0 < n; j0 += kBatch) {
        T x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (j0 + u < n) x[u] = head[off(pos + node[j0 + u])];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (j0 + u < n) head[off(pos + j0 + u)] = x[u];
    }
}

template <int HD>
__global__ void __launch_bounds__(96)
q8_keep_kernel(const Q8Layer L, size_t layer_rows, const __grid_constant__ Q8Seqs tab,
               const __grid_constant__ Q8Nodes nodes) {
    const int seq = blockIdx.x, h = blockIdx.z;
    const int t0 = tab.tok0[seq], n = tab.tok0[seq + 1] - t0, pos = tab.pos[seq];
    const int8_t *node = nodes.at + t0;
    const size_t r0 = tab.slot[seq] * L.slot_rows + blockIdx.y * layer_rows + h * L.head_rows;
    const int lane = threadIdx.x & 31, what = threadIdx.x >> 5;
    using T = typename std::conditional<HD == 128, uint32_t, uint16_t>::type;
    if (what < 2) {  // a warp each for the codes of K and of V
        keep_rows(reinterpret_cast<T *>((what ? L.v : L.k) + r0 * HD), n, pos, node, [lane](int r) {
            return HD == 128 ? q8_chunk<HD>(r, lane >> 2) / 4 + (lane & 3)
                             : q8_chunk<HD>(r, lane >> 3) / 2 + (lane & 7);
        });
    } else if (lane < 2) {  // a thread each for the scales
        keep_rows((lane ? L.vs : L.ks) + r0, n, pos, node, [](int r) { return size_t(r); });
    }
}

__global__ void __launch_bounds__(64)
f32_keep_kernel(float *kc, float *vc, size_t head_stride, size_t layer_stride, size_t slot_stride,
                int hd4, const __grid_constant__ Q8Seqs tab, const __grid_constant__ Q8Nodes nodes) {
    const int seq = blockIdx.x;
    const int t0 = tab.tok0[seq], n = tab.tok0[seq + 1] - t0;
    const int lane = threadIdx.x & 31;
    float *head = ((threadIdx.x >> 5) ? vc : kc) + tab.slot[seq] * slot_stride +
                  blockIdx.y * layer_stride + blockIdx.z * head_stride;
    if (lane < hd4)
        keep_rows(reinterpret_cast<float4 *>(head), n, tab.pos[seq], nodes.at + t0,
                  [lane, hd4](int r) { return size_t(r) * hd4 + lane; });
}

template <int HD, int MODE>
int launch_append(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8See<MODE == kTree> &see,
                  const float *k, const float *v) {
    const int items = tab.tok0[tab.n_seq] * c->n_kv;
    if (items == 0) return LEAP_OK;
    q8_append_kernel<HD, MODE><<<(items + kWarps * kItems - 1) / (kWarps * kItems), 32 * kWarps, 0, c->stream>>>(
        k, v, q8_layer(c, layer), c->rope_cos, c->rope_sin, tab, see);
    return cuda_status(cudaGetLastError(), "q8_append_kernel launch");
}

int launch_read(leap_ctx *c, int layer, const Q8Seqs &tab, float *k, float *v) {
    const int items = tab.tok0[tab.n_seq] * c->n_kv;
    if (items == 0) return LEAP_OK;
    const int grid = (items + kWarps * kItems - 1) / (kWarps * kItems);
    if (c->hd == 128)
        q8_read_kernel<128><<<grid, 32 * kWarps, 0, c->stream>>>(k, v, q8_layer(c, layer), tab);
    else
        q8_read_kernel<64><<<grid, 32 * kWarps, 0, c->stream>>>(k, v, q8_layer(c, layer), tab);
    return cuda_status(cudaGetLastError(), "q8_read_kernel launch");
}

Q8Seqs one_run(int slot, int pos0, int n) {
    Q8Seqs tab;
    tab.n_seq = 1;
    tab.slot[0] = slot;
    tab.pos[0] = pos0;
    tab.tok0[0] = 0;
    tab.tok0[1] = n;
    return tab;
}

int write_rows(leap_ctx *c, int layer, const Q8Seqs &tab, const float *k, const float *v) {
    return c->hd == 128 ? launch_append<128, kRaw>(c, layer, tab, {}, k, v)
                        : launch_append<64, kRaw>(c, layer, tab, {}, k, v);
}

}  // namespace

Q8Layer q8_layer(const leap_ctx *c, int layer) {
    const size_t r = layer * c->layer_rows;
    return {c->k8 + r * c->hd, c->v8 + r * c->hd, c->ks8 + r, c->vs8 + r,
            c->head_rows,      c->slot_rows,      c->n_kv};
}

int q8_create(leap_ctx *c) {
    c->head_rows = (c->max_seq + 127) / 128 * 128;  // whole tiles can be read
    c->layer_rows = c->n_kv * c->head_rows;
    c->slot_rows = c->n_layers * c->layer_rows;
    const size_t rows = c->max_batch * c->slot_rows;
    c->q8_parts = q8_warps_parts(c);  // the rows kernel keeps to as many
    c->q8_tc_parts = q8_tc_parts_needed(c);
    c->stage_rows = std::min(c->max_seq, kQ8StageRows);
    // two allocations (each costs a good part of a context's making): the cache, and
    // everything else; every piece a multiple of 256 bytes
    const size_t cache = 2 * rows * (c->hd + sizeof(float));
    char *p = nullptr, *q = nullptr;
    struct Piece {
        void **at;
        size_t bytes;
    };
    const size_t f = sizeof(float);
    const Piece pieces[] = {
        {reinterpret_cast<void **>(&c->q8_counters), size_t(kMaxSeqPerLaunch) * c->n_kv * sizeof(unsigned)},
        {reinterpret_cast<void **>(&c->d_rows), 2 * f * c->stage_rows * c->n_kv * c->hd},
        {reinterpret_cast<void **>(&c->q8_part_o), f * c->q8_parts * kQ8Rows * c->hd},
        {reinterpret_cast<void **>(&c->q8_part_ml), f * c->q8_parts * kQ8Rows * 2},
        {reinterpret_cast<void **>(&c->q8_tc_part_o), f * c->q8_tc_parts * 128 * c->hd},
        {reinterpret_cast<void **>(&c->q8_tc_part_ml), f * c->q8_tc_parts * 128 * 2},
    };
    size_t scratch = 0;
    for (const Piece &x : pieces) scratch += (x.bytes + 255) / 256 * 256;
    cudaError_t e = cudaMalloc(&p, cache);
    if (e == cudaSuccess) {
        c->k8 = reinterpret_cast<uint8_t *>(p);
        c->v8 = c->k8 + rows * c->hd;
        c->ks8 = reinterpret_cast<float *>(c->v8 + rows * c->hd);
        c->vs8 = c->ks8 + rows;
        e = cudaMalloc(&q, scratch);
    }
    if (e == cudaSuccess) {
        for (const Piece &x : pieces) {
            *x.at = q;
            q += (x.bytes + 255) / 256 * 256;
        }
        e = cudaMemset(c->q8_counters, 0, pieces[0].bytes);
    }
    if (e != cudaSuccess) return cuda_status(e, "cudaMalloc(8-bit cache)");
    c->device_bytes += cache + scratch;
    return q8_clear(c);
}

void q8_free(leap_ctx *c) {
    cudaFree(c->k8);           // the cache
    cudaFree(c->q8_counters);  // the rest
}

int q8_clear(leap_ctx *c) {
    // code 128 stands for 0; with scale 0 every row reads as zeros
    const size_t rows = c->max_batch * c->slot_rows;
    cudaError_t e = cudaMemsetAsync(c->k8, 128, 2 * rows * c->hd, c->stream);  // v8 follows
    if (e == cudaSuccess) e = cudaMemsetAsync(c->ks8, 0, 2 * rows * sizeof(float), c->stream);
    return cuda_status(e, "clear the 8-bit cache");
}

int q8_write(leap_ctx *c, int slot, int layer, int pos0, int n, const float *k, const float *v,
             bool from_host) {
    if (!from_host) return write_rows(c, layer, one_run(slot, pos0, n), k, v);
    const size_t row = size_t(c->n_kv) * c->hd;
    float *dk = c->d_rows, *dv = dk + c->stage_rows * row;
    for (int r = 0; r < n; r += c->stage_rows) {
        const int m = std::min(n - r, c->stage_rows);
        const size_t bytes = m * row * sizeof(float);
        cudaError_t e = cudaMemcpyAsync(dk, k + r * row, bytes, cudaMemcpyHostToDevice, c->stream);
        if (e == cudaSuccess)
            e = cudaMemcpyAsync(dv, v + r * row, bytes, cudaMemcpyHostToDevice, c->stream);
        if (int st = cuda_status(e, "kv_write copy")) return st;
        if (int st = write_rows(c, layer, one_run(slot, pos0 + r, m), dk, dv)) return st;
    }
    return cuda_status(cudaStreamSynchronize(c->stream), "kv_write sync");
}

int q8_read(leap_ctx *c, int slot, int layer, int pos0, int n, float *k, float *v, bool to_host) {
    if (!to_host) return launch_read(c, layer, one_run(slot, pos0, n), k, v);
    const size_t row = size_t(c->n_kv) * c->hd;
    float *dk = c->d_rows, *dv = dk + c->stage_rows * row;
    for (int r = 0; r < n; r += c->stage_rows) {
        const int m = std::min(n - r, c->stage_rows);
        const size_t bytes = m * row * sizeof(float);
        if (int st = launch_read(c, layer, one_run(slot, pos0 + r, m), dk, dv)) return st;
        cudaError_t e = cudaMemcpyAsync(k + r * row, dk, bytes, cudaMemcpyDeviceToHost, c->stream);
        if (e == cudaSuccess)
            e = cudaMemcpyAsync(v + r * row, dv, bytes, cudaMemcpyDeviceToHost, c->stream);
        if (int st = cuda_status(e, "kv_read copy")) return st;
    }
    return cuda_status(cudaStreamSynchronize(c->stream), "kv_read sync");
}

int q8_append(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *k,
              const float *v) {
    if (c->hd == 128)
        return tree ? launch_append<128, kTree>(c, layer, tab, q8_see(*tree), k, v)
                    : launch_append<128, kCausal>(c, layer, tab, {}, k, v);
    return tree ? launch_append<64, kTree>(c, layer, tab, q8_see(*tree), k, v)
                : launch_append<64, kCausal>(c, layer, tab, {}, k, v);
}

int kv_read_packed(leap_ctx *c, int layer, const Q8Seqs &tab, float *k, float *v) {
    if (c->kv_kind == LEAP_KV_Q8) return launch_read(c, layer, tab, k, v);
    const long n = long(tab.tok0[tab.n_seq]) * c->n_kv * (c->hd / 4);
    if (n == 0) return LEAP_OK;
    f32_read_kernel<<<unsigned((n + 255) / 256), 256, 0, c->stream>>>(
        k, v, k_head_ptr(c, 0, layer, 0), v_head_ptr(c, 0, layer, 0), c->head_stride,
        c->slot_stride, c->n_kv, c->hd / 4, tab);
    return cuda_status(cudaGetLastError(), "f32_read_kernel launch");
}

int kv_keep(leap_ctx *c, const Q8Seqs &tab, const Q8Nodes &nodes) {
    const dim3 grid(tab.n_seq, c->n_layers, c->n_kv);
    if (c->kv_kind != LEAP_KV_Q8) {
        f32_keep_kernel<<<grid, 64, 0, c->stream>>>(c->k_cache, c->v_cache, c->head_stride,
                                                    c->layer_stride, c->slot_stride, c->hd / 4,
                                                    tab, nodes);
        return cuda_status(cudaGetLastError(), "f32_keep_kernel launch");
    }
    if (c->hd == 128)
        q8_keep_kernel<128><<<grid, 96, 0, c->stream>>>(q8_layer(c, 0), c->layer_rows, tab, nodes);
    else
        q8_keep_kernel<64><<<grid, 96, 0, c->stream>>>(q8_layer(c, 0), c->layer_rows, tab, nodes);
    return cuda_status(cudaGetLastError(), "q8_keep_kernel launch");
}

}  // namespace leap
