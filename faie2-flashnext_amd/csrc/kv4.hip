// Rows into and out of the 4-bit paged cache: what moves an fp32 cache into it and reads it back.  One wave a row of
// one head; a row is read or written as 16 bytes a lane, its page bytes as the layout has them (136 bytes a row and head).
#include "kv4.cuh"

namespace fn {

namespace {

using namespace kv4;

// grid (n, nkv), two waves: K and V
__global__ void __launch_bounds__(128) k_kv4_pack(const Kv4Rows p, unsigned *status) {
    const int i = blockIdx.x, g = blockIdx.y, lane = threadIdx.x & 63;
    const bool is_v = threadIdx.x >= 64;
    const int slot = p.slot[i];
    if (slot < 0 || slot / PG >= p.npages) {
        if (slot >= 0 && threadIdx.x == 0) atomicOr(status, FN_STATUS_PAGE);
        return;
    }
    uint8_t *page = p.cache + ((size_t) (slot / PG) * p.nkv + g) * HEAD_BYTES;
    const float4 x = reinterpret_cast<const float4 *>((is_v ? p.v : p.k) + ((size_t) i * p.nkv + g) * HD)[lane];
    const double y[4] = {x.x, x.y, x.z, x.w};
    if (is_v) store_row<false>(page, slot % PG, y, lane, status);
    else store_row<true>(page, slot % PG, y, lane, status);
}

__global__ void __launch_bounds__(128) k_kv4_unpack(const Kv4Rows p, unsigned *status) {
    const int i = blockIdx.x, g = blockIdx.y, lane = threadIdx.x & 63, grp = lane >> 3, sub = lane & 7;
    const bool is_v = threadIdx.x >= 64;
    const int slot = p.slot[i];
    if (slot < 0 || slot / PG >= p.npages) {
        if (slot >= 0 && threadIdx.x == 0) atomicOr(status, FN_STATUS_PAGE);
        return;
    }
    const uint8_t *page = p.cache + ((size_t) (slot / PG) * p.nkv + g) * HEAD_BYTES;
    const int r = slot % PG;
    uint32_t c;
    int s;
    if (is_v) {
        c = page[v_code(r, grp, 2 * sub)] | (uint32_t) page[v_code(r, grp, 2 * sub + 1)] << 8;
        s = page[v_scale(r, grp)];
    } else {
        c = *reinterpret_cast<const uint16_t *>(page + k_code(r, grp) + sub * 2);
        s = page[k_scale(r, grp)];
    }
    reinterpret_cast<float4 *>((is_v ? p.v : p.k) + ((size_t) i * p.nkv + g) * HD)[lane] =
        make_float4(value_of(c & 15, s), value_of(c >> 4 & 15, s), value_of(c >> 8 & 15, s), value_of(c >> 12, s));
}

int check(const Kv4Rows &p) {
    if (p.n < 1 || p.nkv < 1) FN_FAIL("kv4: n and nkv must be >= 1");
    if (p.nkv > 65535) FN_FAIL("kv4: nkv must be <= 65535");
    if (p.n > (1 << 25) - 1) FN_FAIL("kv4: n must be <= 33554431 (a launch has below 2^32 threads)");
    if (p.hd != HD) FN_FAIL("kv4: only head_dim 256 is built");
    if (p.npages < 1 || p.npages > INT_MAX / PG) FN_FAIL("kv4: npages must be in 1..33554431 (slots are 32-bit)");
    if (!p.slot || !p.k || !p.v || !p.cache) FN_FAIL("kv4: null pointer");
    if (((uintptr_t) p.k | (uintptr_t) p.v | (uintptr_t) p.cache) & 15) FN_FAIL("kv4: k, v and cache must be 16-byte aligned");
    return 0;
}

}  // namespace

size_t kv4_page_bytes(int nkv, int hd) { return nkv < 1 || hd != HD ? 0 : (size_t) nkv * HEAD_BYTES; }

int kv4_pack_launch(const Kv4Rows &p, hipStream_t st) {
    if (check(p)) return -1;
    unsigned *status;
    if (status_word(&status)) return -1;
    hipLaunchKernelGGL(k_kv4_pack, dim3(p.n, p.nkv), dim3(128), 0, st, p, status);
    FN_CK(hipGetLastError());
    return 0;
}

int kv4_unpack_launch(const Kv4Rows &p, hipStream_t st) {
    if (check(p)) return -1;
    unsigned *status;
    if (status_word(&status)) return -1;
    hipLaunchKernelGGL(k_kv4_unpack, dim3(p.n, p.nkv), dim3(128), 0, st, p, status);
    FN_CK(hipGetLastError());
    return 0;
}

}  // namespace fn
