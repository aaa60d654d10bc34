// ctx.h — host-side definition of the opaque leap_ctx and shared helpers.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <string>

#include "leap_b200.h"

struct leap_ctx {
    // shape (reference Config fields, src/inference/Config.h:5-13)
    int device = 0;
    int n_layers = 0, layer0 = 0;
    int n_heads = 0, n_kv = 0, hd = 0, group = 0;
    int max_seq = 0, max_seq_pad = 0, max_batch = 0;
    int num_sms = 148;

    cudaStream_t own_stream = nullptr;
    cudaStream_t stream = nullptr;

    // KV cache [slot][layer][kv_head][max_seq_pad][hd] (floats)
    float *k_cache = nullptr, *v_cache = nullptr;
    size_t head_stride = 0, layer_stride = 0, slot_stride = 0;
    size_t cache_bytes = 0;  // per tensor (K or V)

    // 8-bit cache (kv_kind LEAP_KV_Q8; format in q8.cuh): codes in the layout
    // of the FP32 cache with one byte a value, one scale for each row; the
    // strides below count rows
    int kv_kind = LEAP_KV_F32;
    uint8_t *k8 = nullptr, *v8 = nullptr;
    float *ks8 = nullptr, *vs8 = nullptr;
    size_t head_rows = 0, layer_rows = 0, slot_rows = 0;
    float *d_rows = nullptr;  // FP32 rows on their way from or to host memory,
    int stage_rows = 0;       // so many of k and of v
    // its split-KV scratch, no more than the context can use: partials of up to 8
    // rows, and tickets
    float *q8_part_o = nullptr, *q8_part_ml = nullptr;  // [q8_parts][8][hd], [q8_parts][8][2]
    unsigned *q8_counters = nullptr;                    // [kMaxSeqPerLaunch][n_kv]
    int q8_parts = 0;
    float *q8_tc_part_o = nullptr, *q8_tc_part_ml = nullptr;  // of 128 rows
    int q8_tc_parts = 0;

    // RoPE table [max_seq][hd/2]
    float *rope_cos = nullptr, *rope_sin = nullptr;

    // split-KV scratch, two sets: consecutive decode launches alternate so
    // that a launch overlapping the previous one's tail never shares it
    float *part_o[2] = {nullptr, nullptr};      // [max_parts][group*hd]
    float *part_ml[2] = {nullptr, nullptr};     // [max_parts][2*max(group,2)]
    unsigned *counters[2] = {nullptr, nullptr}; // [kMaxSeqPerLaunch][n_kv]
    int max_parts = 0;
    int parity = 0;

    // Launch overlap (programmatic dependent launch): a decode kernel may
    // start streaming its layer's K/V while the previous kernel finishes,
    // unless the previous op of this context wrote that layer.
    int overlap = 1;
    int last_written_layer = kWroteAll;  // layer the previous op wrote
    static constexpr int kWroteAll = -2;
    static constexpr int kWroteNone = -1;  // the previous grid wrote no cache row

    // decode kernel choice: 0 auto, 1 split-KV (global combine),
    // 2 cluster (distributed-shared-memory combine)
    int decode_impl = 0;
    int cluster_capacity = 0;  // co-resident 16-CTA decode clusters

    // device error word (kernels report bounded-wait timeouts here)
    int *d_err = nullptr;
    // set only inside leap_attn_decode_host: the decode kernels also store an
    // error code to this host-mapped word (the caller waits on the host)
    int *err_host = nullptr;

    // host-pointer entry points: pinned staging and device mirrors
    float *h_stage = nullptr;  // pinned: q | k | v | out for one token
    float *h_stage_dev = nullptr;  // the same pinned buffer as device code addresses it
    float *d_stage = nullptr;

    // prefill scratch (rotated q), grown on demand
    float *d_qrot = nullptr;
    size_t qrot_cap = 0;  // floats
    int prefill_impl = 3;  // see leap_set_prefill_impl

    size_t device_bytes = 0;
};

namespace leap {

constexpr int kMaxDevices = 64;

// Device error word codes (bounded waits use small positive codes).
constexpr int kDevErrBadToken = 0x70;  // a device-side token id outside [0, vocab)

// thread-local last error
void set_error(const char *fmt, ...);
void clear_error();

// Convert a CUDA error into a LEAP status (sets the message).
int cuda_status(cudaError_t e, const char *what);

// Opt kernel `fn` into `bytes` of dynamic shared memory on the current
// device (and, with `nonportable_cluster`, into clusters above 8 CTAs).
// Done once per (kernel, device) under a lock, so launches from several host
// threads do not race.
int set_kernel_smem(const void *fn, size_t bytes, const char *what,
                    bool nonportable_cluster = false);

inline float *k_head_ptr(const leap_ctx *c, int slot, int layer, int kvh) {
    return c->k_cache + slot * c->slot_stride + layer * c->layer_stride +
           kvh * c->head_stride;
}
inline float *v_head_ptr(const leap_ctx *c, int slot, int layer, int kvh) {
    return c->v_cache + slot * c->slot_stride + layer * c->layer_stride +
           kvh * c->head_stride;
}

// ---- decode attention (decode_attn.cu) -----------------------------------
constexpr int kMaxSeqPerLaunch = 128;

struct DecodeSeq {
    int n_seq;
    int chunk;                         // rows per split
    int pos[kMaxSeqPerLaunch];
    int slot[kMaxSeqPerLaunch];
    int split0[kMaxSeqPerLaunch + 1];  // prefix sum of splits per sequence
};

// Launch one batch of decode work (n_seq <= kMaxSeqPerLaunch; only n_seq,
// pos and slot of `seqs` need to be set: the split plan is made here).
// q/k_new/v_new/out point at the first sequence of the batch.
int launch_decode(leap_ctx *c, int layer, const DecodeSeq &tab, const float *q,
                  const float *k_new, const float *v_new, float *out);

// Fill tab.chunk / tab.split0 for the given positions; returns total splits.
int plan_decode(const leap_ctx *c, DecodeSeq &tab, int shape);

// decode_cluster.cu: co-resident 16-CTA clusters, and the launch.
int decode_cluster_capacity(leap_ctx *c, int *n);
// Host-pointer staging kernel (stage_host.cu): n4 float4s pinned host ->
// device after everything before on the stream.
int launch_stage_in(cudaStream_t st, const float *h_src, float *d_dst, int n4);

int launch_decode_cluster(leap_ctx *c, int layer, const DecodeSeq &tab, const float *q,
                          const float *k_new, const float *v_new, float *out, bool overlap);

// Upper bound on split-KV partials one decode launch can need.
int max_decode_parts(int hd, int n_kv, int max_batch, int max_seq_pad, int num_sms);

// ---- prefill attention (prefill_attn.cu) ---------------------------------
int launch_prefill(leap_ctx *c, int slot, int layer, int pos0, int n_tok,
                   const float *q, const float *k, const float *v, float *out);

// ---- 8-bit KV cache (kv_q8.cu, attn_q8*.cu) --------------------------------
constexpr int kMaxTreeNodes = 128;     // nodes of one sequence's tree
constexpr int kMaxNodesPerLaunch = 1024;  // (parameters of 2 KB)
constexpr int kQ8StageRows = 1024;     // rows of k and v that d_rows holds at most

// A ragged batch of new tokens, by value in kernel parameters: sequence i has
// packed tokens tok0[i] .. tok0[i+1]-1 behind pos[i] cached rows of its slot.
struct Q8Seqs {
    int n_seq;
    int slot[kMaxSeqPerLaunch];
    int pos[kMaxSeqPerLaunch];
    int tok0[kMaxSeqPerLaunch + 1];
};
// Parent of each packed token, counted from its sequence's first (-1: none),
// and its depth.
struct Q8Tree {
    int8_t parent[kMaxNodesPerLaunch], depth[kMaxNodesPerLaunch];
};
struct Q8Nodes {
    int8_t at[kMaxNodesPerLaunch];
};

// Splits of the rows kernel: `chunk` cached rows each, sequence i's are split0[i]
// .. split0[i+1]-1 (none without new tokens).
struct Q8Splits {
    int chunk;
    int split0[kMaxSeqPerLaunch + 1];
};
// The warps kernel's work list: sequence i has units unit0[i] .. unit0[i+1]-1
// (tiles of 32 rows, kv head by kv head; none without new tokens), a warp `chunk`
// of them.
struct Q8Units {
    int chunk;
    int unit0[kMaxSeqPerLaunch + 1];
};
// Blocks of the tensor-core kernel: entry i is sequence seq[i] (those without
// tokens left out, longest first), n_qt[i] query tiles of 128 rows, each over
// nsplit[i] splits of `chunk` key tiles.
struct Q8TcPlan {
    int n, chunk, n_parts;
    int seq[kMaxSeqPerLaunch], n_qt[kMaxSeqPerLaunch], nsplit[kMaxSeqPerLaunch];
    int part0[kMaxSeqPerLaunch];      // partials of split tiles, before this one
    int item0[kMaxSeqPerLaunch + 1];  // (tile, split) pairs before it
    int tile0[kMaxSeqPerLaunch + 1];  // tiles before it
};
constexpr int kQ8Rows = 8;  // query rows (tokens x heads of a group) of the rows kernel

// One layer of the cache as kernels see it.
struct Q8Layer {
    uint8_t *k, *v;    // codes of (slot 0, this layer, kv head 0)
    float *ks, *vs;    // scales
    size_t head_rows, slot_rows;
    int n_kv;
};
Q8Layer q8_layer(const leap_ctx *c, int layer);

int q8_create(leap_ctx *c);
void q8_free(leap_ctx *c);
int q8_clear(leap_ctx *c);
int q8_write(leap_ctx *c, int slot, int layer, int pos0, int n, const float *k, const float *v,
             bool from_host);
int q8_read(leap_ctx *c, int slot, int layer, int pos0, int n, float *k, float *v, bool to_host);
// Rotate (tree: by depth), quantise and append every token's k and v.
int q8_append(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *k,
              const float *v);
int kv_read_packed(leap_ctx *c, int layer, const Q8Seqs &tab, float *k, float *v);
// Move rows pos + at[j] to pos + j (j counted from each sequence's first).
int kv_keep(leap_ctx *c, const Q8Seqs &tab, const Q8Nodes &nodes);
int q8_warps_parts(const leap_ctx *c);
int q8_tc_parts_needed(const leap_ctx *c);
int q8_rows_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
                   const float *k, const float *v, float *out);
int q8_tc_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
                 const float *k, const float *v, float *out);
// Append and attend: causal, or a tree of each sequence's tokens.
int q8_attend(leap_ctx *c, int layer, const Q8Seqs &tab, const Q8Tree *tree, const float *q,
              const float *k, const float *v, float *out);

}  // namespace leap
