// Internal launch API of the operators that serve a packed batch of requests of different lengths (device pointers,
// caller stream): page tables, the 4-bit paged cache and its attention, the chunked delta rule.
#pragma once

#include "gdn.h"

namespace fn {

struct PagePlan {
    int B, T, max_blocks, npages;
    const int32_t *past, *nnew;         // [B] tokens in the cache, new tokens
    const int32_t *free_list;           // [npages] free pages, a stack
    const int32_t *free_top;            // [1] entries of the stack
    int32_t *free_left;                 // [1] entries after the call (may be free_top)
    int32_t *table;                     // [B][max_blocks] in/out
    int32_t *cu, *slot, *seq;           // [B + 1], [T], [T]
};

struct PageRelease {
    int B, max_blocks, npages;
    const int32_t *done;                // [B] nonzero: the request has ended
    int32_t *past, *free_list, *free_top, *table;
};

struct Kv4Rows {                        // rows in and out of the 4-bit cache
    int n, nkv, hd, npages;
    const int32_t *slot;                // [n]
    float *k, *v;                       // [n][nkv][hd]
    uint8_t *cache;
};

struct Kv4Attn {
    int B, T, nq, nkv, hd, nrot, max_blocks, npages, nsplit;
    float theta, eps;
    const int32_t *past, *cu, *table, *slot, *seq;
    const float *qg, *k, *v, *wq, *wk;
    uint8_t *cache;
    void *work;
    size_t work_bytes;
    float *og;
};

struct GdnChunk {
    int B, T, nkh, nvh, dk, dv, head_map;
    const int32_t *cu;                  // [B + 1]
    const float *q, *k;                 // [T][nkh][dk]
    const float *v;                     // [T][nvh][dv]
    const float *beta, *g;              // [T][nvh]
    float *S;                           // [B][nvh][dk][dv]
    float *o;                           // [T][nvh][dv]
    void *work;
    size_t work_bytes;
    // the fused block: conv1d + SiLU + L2-norm and gates in front, gated RMSNorm behind
    bool block = false;
    int gate_act = 0, ring = 0;
    float eps = 0.0f;
    const int32_t *pos = nullptr;       // [B]
    const float *qkv = nullptr, *conv_w = nullptr;
    float *conv_ring = nullptr;         // [B][ring][C]
    const float *ab = nullptr, *dt_bias = nullptr, *ssm_a = nullptr, *z = nullptr, *norm_w = nullptr;
};

int page_plan_launch(const PagePlan &p, hipStream_t st);
int page_release_launch(const PageRelease &p, hipStream_t st);
size_t kv4_page_bytes(int nkv, int hd);
int kv4_pack_launch(const Kv4Rows &p, hipStream_t st);
int kv4_unpack_launch(const Kv4Rows &p, hipStream_t st);
size_t kv4_work_bytes(int B, int T, int nq, int nkv, int hd, int nsplit);
int kv4_pick_nsplit(int B, int T, int nq, int nkv, int ctx);
int kv4_attn_launch(const Kv4Attn &p, hipStream_t st);
size_t gdn_chunk_work_bytes(int B, int T, int nkh, int nvh);
int gdn_chunk_launch(const GdnChunk &p, hipStream_t st);

}  // namespace fn
