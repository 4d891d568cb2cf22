// C ABI of libfaie2fn.so, section 3c (include/faie2fn.h): the operators that serve a packed batch.
#include "../../include/faie2fn.h"
#include "serve.h"

#define FN_API extern "C" __attribute__((visibility("default")))

FN_API int fn_page_plan_dev(int B, int T, int max_blocks, int npages, const int32_t *past, const int32_t *nnew,
                            const int32_t *free_list, const int32_t *free_top, int32_t *free_left, int32_t *table,
                            int32_t *cu, int32_t *slot, int32_t *seq, void *stream) {
    fn::PagePlan p{B, T, max_blocks, npages, past, nnew, free_list, free_top, free_left, table, cu, slot, seq};
    return fn::page_plan_launch(p, (hipStream_t) stream);
}

FN_API int fn_page_release_dev(int B, int max_blocks, int npages, const int32_t *done, int32_t *past,
                               int32_t *free_list, int32_t *free_top, int32_t *table, void *stream) {
    fn::PageRelease p{B, max_blocks, npages, done, past, free_list, free_top, table};
    return fn::page_release_launch(p, (hipStream_t) stream);
}

FN_API size_t fn_kv4_page_bytes(int nkv, int hd) { return fn::kv4_page_bytes(nkv, hd); }

FN_API int fn_kv4_pack_dev(int n, int nkv, int hd, int npages, const int32_t *slot, const float *k, const float *v,
                           uint8_t *cache, void *stream) {
    fn::Kv4Rows p{n, nkv, hd, npages, slot, const_cast<float *>(k), const_cast<float *>(v), cache};
    return fn::kv4_pack_launch(p, (hipStream_t) stream);
}

FN_API int fn_kv4_unpack_dev(int n, int nkv, int hd, int npages, const int32_t *slot, const uint8_t *cache, float *k,
                             float *v, void *stream) {
    fn::Kv4Rows p{n, nkv, hd, npages, slot, k, v, const_cast<uint8_t *>(cache)};
    return fn::kv4_unpack_launch(p, (hipStream_t) stream);
}

FN_API size_t fn_attn_kv4_work_bytes(int B, int T, int nq, int nkv, int hd, int nsplit) {
    if (B < 1 || T < 1 || nq < 1 || nkv < 1 || nq % nkv || nsplit < 1) return 0;
    return fn::kv4_work_bytes(B, T, nq, nkv, hd, nsplit);
}

FN_API int fn_attn_kv4_nsplit(int B, int T, int nq, int nkv, int ctx) {
    if (B < 1 || T < 1 || nq < 1 || nkv < 1 || nq % nkv) return 1;
    return fn::kv4_pick_nsplit(B, T, nq, nkv, ctx);
}

FN_API int fn_attn_kv4_dev(int B, int T, int nq, int nkv, int hd, int nrot, float theta, float eps, int max_blocks,
                           int npages, const int32_t *past, const int32_t *cu, const int32_t *table,
                           const int32_t *slot, const int32_t *seq, const float *qg, const float *k, const float *v,
                           const float *wq, const float *wk, uint8_t *cache, int nsplit, void *work, size_t work_bytes,
                           float *og, void *stream) {
    fn::Kv4Attn p{B, T, nq, nkv, hd, nrot, max_blocks, npages, nsplit, theta, eps, past, cu, table, slot, seq, qg, k, v,
                  wq, wk, cache, work, work_bytes, og};
    return fn::kv4_attn_launch(p, (hipStream_t) stream);
}

FN_API size_t fn_gdn_chunk_work_bytes(int B, int T, int nkh, int nvh) {
    if (B < 1 || T < 1 || nkh < 1 || nvh < 1) return 0;
    return fn::gdn_chunk_work_bytes(B, T, nkh, nvh);
}

FN_API int fn_gdn_core_chunk_dev(int B, int T, int nkh, int nvh, int dk, int dv, int head_map, const int32_t *cu,
                                 const float *q, const float *k, const float *v, const float *beta, const float *g,
                                 float *S, float *o, void *work, size_t work_bytes, void *stream) {
    fn::GdnChunk p{B, T, nkh, nvh, dk, dv, head_map, cu, q, k, v, beta, g, S, o, work, work_bytes};
    return fn::gdn_chunk_launch(p, (hipStream_t) stream);
}

FN_API int fn_gdn_block_chunk_dev(int B, int T, int nkh, int nvh, int dk, int dv, int head_map, int gate_act, int ring,
                                  const int32_t *cu, const int32_t *pos, const float *qkv, const float *conv_w,
                                  float *conv_ring, const float *ab, const float *dt_bias, const float *ssm_a, float *S,
                                  const float *z, const float *norm_w, float eps, float *out, void *work,
                                  size_t work_bytes, void *stream) {
    fn::GdnChunk p{B, T, nkh, nvh, dk, dv, head_map, cu, nullptr, nullptr, nullptr, nullptr, nullptr, S, out, work,
                   work_bytes, true, gate_act, ring, eps, pos, qkv, conv_w, conv_ring, ab, dt_bias, ssm_a, z, norm_w};
    return fn::gdn_chunk_launch(p, (hipStream_t) stream);
}
