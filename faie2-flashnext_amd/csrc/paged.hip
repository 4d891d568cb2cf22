// Page tables of a paged cache, built on the GPU from request lengths: which pages the new tokens of a packed batch
// need, where each token's row goes (slot = page * 64 + row of the page), and pages given back by ended requests.
//
// All of it is integer prefix sums: cu = exclusive sum of the new tokens, and the pages a request needs beyond those it
// has are taken from the end of a stack of free pages at the exclusive sum of the page counts, so the result does not
// depend on the order in which threads run.  What bounds a call is a chain of a few memory latencies: on the device 4.0 us
// for 16 requests and 6.9 us for 512 with 66,000 tokens (5.8 + 3.3 us in two launches); a call among others takes 7.8 us.
// A workgroup does the sums, the table entries of the new pages and the tokens; in a longer batch each of many workgroups
// does the sums for itself and maps its own tokens, whose new pages it takes from the stack as the first workgroup does, so
// that none waits for another.  Only where the count that is left goes into the count that is read does a second launch
// map them, from the table.
#include "serve.h"

namespace fn {

namespace {

constexpr int PG = 64;             // tokens a page
constexpr int MAXB = 8000;         // requests a call: two words of LDS a request, in 64 KiB
constexpr int PAST_LDS = 5000;     // requests up to which a third word, the past, fits
constexpr int ONE_WG = 4096;       // tokens one workgroup maps (four a thread)

struct PlanArgs {
    PagePlan p;
    unsigned *status;
};

// exclusive prefix sums over the workgroup of each of N values; totals to every thread.  tmp: N words for each wave.
template <int N> __device__ __forceinline__ void wg_scan(long long (&v)[N], long long *tmp, long long (&total)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    long long x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const long long y = __shfl_up(x[i], d);
            if (lane >= d) x[i] += y;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane == 63) tmp[wave * N + i] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        long long before = 0, all = 0;
        for (int w = 0; w < waves; ++w) {
            if (w < wave) before += tmp[w * N + i];
            all += tmp[w * N + i];
        }
        total[i] = all;
        v[i] = before + x[i] - v[i];
    }
}
__device__ __forceinline__ long long wg_scan(long long v, long long *tmp, long long &total) {
    long long x[1] = {v}, t[1];
    wg_scan<1>(x, tmp, t);
    total = t[0];
    return x[0];
}

// the last i < n with a[i] <= x (a not decreasing, a[0] <= x)
__device__ __forceinline__ int last_le(const int32_t *a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int blocks_of(int tokens) { return tokens / PG + (tokens % PG > 0); }

// what page (of the table or, from block `have` on, of the stack) token t of request b at position `at` lies in
template <typename F> __device__ __forceinline__ void map_token(const PlanArgs &a, int t, int b, long long at, F page_of) {
    const PagePlan &p = a.p;
    int slot = -1;
    if (b >= 0 && at >= 0 && at / PG < p.max_blocks) {
        const int page = page_of((int) (at / PG));
        if (page >= 0 && page < p.npages) slot = page * PG + (int) (at % PG);
        else atomicOr(a.status, FN_STATUS_PAGE);
    }
    p.slot[t] = slot;
    p.seq[t] = b;
}

// tokens: none (0), all by the one workgroup (1), or by the workgroups behind the first, one a thread (2)
__global__ void __launch_bounds__(1024) k_page_plan(const PlanArgs a, int tokens) {
    extern __shared__ int32_t plan_lds[];
    __shared__ long long tmp[32];
    const PagePlan &p = a.p;
    int32_t *cu = plan_lds, *bef = plan_lds + p.B + 1, *had = bef + p.B;
    const bool past_lds = p.B <= PAST_LDS, first = blockIdx.x == 0;
    const int tid = threadIdx.x, nth = blockDim.x;
    const int top = max(0, min(p.free_top[0], p.npages));
    long long rows = 0, pages = 0;
    unsigned bits = 0;
    for (int b0 = 0; b0 < p.B; b0 += nth) {
        const int b = b0 + tid;
        const long long past = b < p.B ? p.past[b] : 0;
        long long n = b < p.B ? p.nnew[b] : 0;
        if (n < 0) {
            n = 0;
            bits |= FN_STATUS_ROWS;
        }
        // pages that m new tokens need beyond those of the past
        const auto pages_for = [&](long long m) {
            const long long want = min((past + m + PG - 1) / PG, (long long) p.max_blocks);
            return past < 0 ? 0 : max(0ll, want - (past + PG - 1) / PG);
        };
        long long both[2] = {n, pages_for(n)}, sum[2];
        wg_scan(both, tmp, sum);
        const long long r0 = rows + both[0], start = min(r0, (long long) p.T), end = min(r0 + n, (long long) p.T);
        if (rows + sum[0] > p.T) both[1] = wg_scan(pages_for(end - start), tmp, sum[1]);  // some tokens are cut off
        if (r0 + n > p.T) bits |= FN_STATUS_ROWS;
        if (past < 0 || (past + end - start + PG - 1) / PG > p.max_blocks) bits |= FN_STATUS_POS;
        const long long f0 = pages + both[1];
        rows += sum[0];
        pages += sum[1];
        if (b < p.B) {
            cu[b] = (int32_t) start;
            bef[b] = (int32_t) min(f0, (long long) INT_MAX);
            if (past_lds) had[b] = (int32_t) past;
            if (first) p.cu[b] = (int32_t) start;
        }
    }
    const int total = (int) min(rows, (long long) p.T);
    // the stack is read up to `pages`, all of it at most: what it does not hold is no page
    const int need = (int) min(pages, (long long) INT_MAX);
    if (need > top) bits |= FN_STATUS_PAGE;
    __syncthreads();  // every thread has read free_top, which may be free_left; what the LDS holds is there
    auto past_of = [&](int b) { return past_lds ? had[b] : p.past[b]; };
    auto fresh_page = [&](int i) { return i >= 0 && i < top ? p.free_list[top - 1 - i] : -1; };
    if (first) {
        if (tid == 0) {
            p.cu[p.B] = total;
            p.free_left[0] = top - min(need, top);
        }
        for (int i = tid; i < need; i += nth) {
            const int b = last_le(bef, p.B, i);
            int page = fresh_page(i);
            if (page < 0 || page >= p.npages) {
                page = -1;
                bits |= FN_STATUS_PAGE;
            }
            p.table[(size_t) b * p.max_blocks + blocks_of(past_of(b)) + (i - bef[b])] = page;
        }
        if (bits) atomicOr(a.status, bits);
    }
    if (tokens == 0 || (tokens == 2 && first)) return;
    for (int t = tokens == 1 ? tid : (blockIdx.x - 1) * nth + tid; t < p.T; t += tokens == 1 ? nth : p.T) {
        const int b = t < total ? last_le(cu, p.B, t) : -1;
        const int past = b < 0 ? -1 : past_of(b), have = blocks_of(past);
        map_token(a, t, b, past < 0 ? -1 : (long long) past + (t - cu[b]), [&](int blk) {
            return blk < have ? p.table[(size_t) b * p.max_blocks + blk] : fresh_page(bef[b] + (blk - have));
        });
    }
}

__global__ void __launch_bounds__(256) k_page_slots(const PlanArgs a) {
    extern __shared__ int32_t plan_lds[];
    const PagePlan &p = a.p;
    for (int b = threadIdx.x; b <= p.B; b += 256) plan_lds[b] = p.cu[b];
    __syncthreads();
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= p.T) return;
    const int b = t < plan_lds[p.B] ? last_le(plan_lds, p.B, t) : -1, past = b < 0 ? -1 : p.past[b];
    map_token(a, t, b, past < 0 ? -1 : (long long) past + (t - plan_lds[b]),
              [&](int blk) { return p.table[(size_t) b * p.max_blocks + blk]; });
}

// One workgroup: the pages of the ended requests go back on the stack in request order, then page order.
__global__ void __launch_bounds__(256) k_page_release(const PageRelease p, unsigned *status) {
    extern __shared__ int32_t plan_lds[];
    __shared__ long long tmp[16];
    const int tid = threadIdx.x, nth = blockDim.x;
    long long pages = 0, sum;
    for (int b0 = 0; b0 < p.B; b0 += nth) {
        const int b = b0 + tid;
        long long n = 0;
        if (b < p.B && p.done[b]) n = max(0ll, min(((long long) p.past[b] + PG - 1) / PG, (long long) p.max_blocks));
        const long long f0 = pages + wg_scan(n, tmp, sum);
        pages += sum;
        if (b < p.B) plan_lds[b] = (int32_t) min(f0, (long long) INT_MAX);
    }
    long long top = max(0, min(p.free_top[0], p.npages));
    __syncthreads();
    const int need = (int) min(pages, (long long) INT_MAX);
    for (int i0 = 0; i0 < need; i0 += nth) {
        const int i = i0 + tid;
        int page = -1;
        if (i < need) {
            const int b = last_le(plan_lds, p.B, i);
            int32_t *e = p.table + (size_t) b * p.max_blocks + (i - plan_lds[b]);
            page = *e;
            *e = -1;
        }
        const bool ok = page >= 0 && page < p.npages;  // a block that got no page has none to give back
        const long long at = top + wg_scan(ok, tmp, sum);
        top += sum;
        if (ok && at < p.npages) p.free_list[at] = page;
    }
    if (tid == 0) {
        if (top > p.npages) atomicOr(status, FN_STATUS_PAGE);
        p.free_top[0] = (int32_t) min(top, (long long) p.npages);
    }
    for (int b = tid; b < p.B; b += nth)
        if (p.done[b]) p.past[b] = 0;
}

int check(int B, int max_blocks, int npages) {
    if (B < 1 || B > MAXB) FN_FAIL("page: B must be in 1..8000");
    if (max_blocks < 1) FN_FAIL("page: max_blocks must be >= 1");
    if (npages < 1 || npages > INT_MAX / PG) FN_FAIL("page: npages must be in 1..33554431 (slots are 32-bit)");
    return 0;
}

}  // namespace

int page_plan_launch(const PagePlan &p, hipStream_t st) {
    if (check(p.B, p.max_blocks, p.npages)) return -1;
    if (p.T < 1 || p.T > 1 << 30) FN_FAIL("page_plan: T must be in 1..1073741824");
    if (!p.past || !p.nnew || !p.free_list || !p.free_top || !p.free_left || !p.table || !p.cu || !p.slot || !p.seq)
        FN_FAIL("page_plan: null pointer");
    PlanArgs a{p, nullptr};
    if (status_word(&a.status)) return -1;
    const int tokens = p.T <= ONE_WG ? 1 : p.free_left == p.free_top ? 0 : 2;
    const int nth = p.B <= 256 && p.T <= 256 ? 256 : 1024;
    const size_t word = (size_t) p.B * sizeof(int32_t), lds = (p.B <= PAST_LDS ? 3 : 2) * word + sizeof(int32_t);
    const int wgs = tokens == 2 ? 1 + (p.T - 1) / nth + 1 : 1;
    hipLaunchKernelGGL(k_page_plan, dim3(wgs), dim3(nth), lds, st, a, tokens);
    if (!tokens) hipLaunchKernelGGL(k_page_slots, dim3((p.T - 1) / 256 + 1), dim3(256), word + sizeof(int32_t), st, a);
    FN_CK(hipGetLastError());
    return 0;
}

int page_release_launch(const PageRelease &p, hipStream_t st) {
    if (check(p.B, p.max_blocks, p.npages)) return -1;
    if (!p.done || !p.past || !p.free_list || !p.free_top || !p.table) FN_FAIL("page_release: null pointer");
    unsigned *status;
    if (status_word(&status)) return -1;
    hipLaunchKernelGGL(k_page_release, dim3(1), dim3(256), (size_t) p.B * sizeof(int32_t), st, p, status);
    FN_CK(hipGetLastError());
    return 0;
}

}  // namespace fn
