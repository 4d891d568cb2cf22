// GQA attention of a packed ragged batch over the 4-bit paged cache: q/k RMSNorm + partial RoPE, append, online softmax,
// sigmoid gate.  One call takes requests of one new token (decode), a few (verify) and whole prompts together.
#include "kv4.cuh"
#include "serve.cuh"

#include <algorithm>
#include <cmath>

namespace fn {

namespace {

using namespace kv4;

constexpr int MAXROT = 128;
constexpr int NPART = 5;                               // fp6 parts of a query value
constexpr int FRAG = 64 * 24;                          // a part's operand: 16 bytes, then 8 bytes a lane
constexpr int QBLK = 2 * NPART * FRAG + 2 * 64 * 8;    // 16 query rows: [half][part] operands, [half] scales: 16 KiB
static_assert(QBLK == 16384, "1 KiB a query row");
constexpr int WAVES = 4;
constexpr int OS = 68;                                 // floats a row of the merge buffer (64 dims; rows 4 banks apart)

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v32f __attribute__((ext_vector_type(32)));
typedef unsigned v6u __attribute__((ext_vector_type(6)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Kv4Args {
    int B, T, nq, nkv, grp, mb, npages, nsplit, nrot, items;
    float eps;
    const int32_t *past, *cu, *table, *slot, *seq;
    const float *qg, *k, *v, *wq, *wk;
    uint8_t *cache;
    uint8_t *Q;                 // [nkv][items][rows / 16] query blocks of QBLK bytes
    float *part_o;              // [items][nkv][nsplit][rows][HD]
    float *part_ml;             // [items][nkv][nsplit][rows][2]
    float *og;
    unsigned *status;
    double freq[MAXROT / 2];
};

// One token: sines and cosines of its position, its keys and values into their page, its queries as operands.
template <int RT>
__global__ void __launch_bounds__(256) k_kv4_prep(const Kv4Args a) {
    __shared__ double cs[MAXROT / 2], sn[MAXROT / 2];
    __shared__ double krow[WAVES][HD];
    __shared__ float qrow[WAVES][8][MAXROT + 4];
    const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int total = min(a.cu[a.B], a.T);
    if (t >= total) return;
    const int b = a.seq[t];
    if (b < 0 || b >= a.B || t < a.cu[b] || t >= a.cu[b + 1] || a.cu[b] < 0) {
        if (threadIdx.x == 0) atomicOr(a.status, FN_STATUS_ROWS);
        return;
    }
    const long long P = (long long) a.past[b] + (t - a.cu[b]);
    if ((a.past[b] < 0 || P >= (long long) a.mb * PG) && threadIdx.x == 0) atomicOr(a.status, FN_STATUS_POS);
    const int half = a.nrot / 2;
    // the angle in 64 bits: a float product is off by up to half a radian at a million tokens
    if (threadIdx.x < half) sincos((double) P * a.freq[threadIdx.x], &sn[threadIdx.x], &cs[threadIdx.x]);
    __syncthreads();
    const int slot = a.slot[t];
    const bool put = slot >= 0 && slot / PG < a.npages;
    if (slot >= 0 && !put && threadIdx.x == 0) atomicOr(a.status, FN_STATUS_PAGE);
    const int octets = (a.nq + 7) / 8;
    for (int task = wave; task < 2 * a.nkv + octets; task += WAVES) {
        if (task < 2 * a.nkv) {
            if (!put) continue;
            const int g = task >> 1;
            uint8_t *page = a.cache + ((size_t) (slot / PG) * a.nkv + g) * HEAD_BYTES;
            const bool is_v = task & 1;
            const float4 x = reinterpret_cast<const float4 *>((is_v ? a.v : a.k) + ((size_t) t * a.nkv + g) * HD)[lane];
            double y[4] = {x.x, x.y, x.z, x.w};
            if (is_v) {
                store_row<false>(page, slot % PG, y, lane, a.status);
                continue;
            }
            const float4 w = reinterpret_cast<const float4 *>(a.wk)[lane];
            double ss = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) ss += __shfl_xor(ss, d);
            const double r = 1.0 / sqrt(ss / HD + (double) a.eps);
            y[0] *= r * w.x, y[1] *= r * w.y, y[2] *= r * w.z, y[3] *= r * w.w;
#pragma unroll
            for (int i = 0; i < 4; ++i) krow[wave][4 * lane + i] = y[i];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 4 * lane + i;
                if (d < a.nrot) {
                    const int j = d < half ? d : d - half;
                    const double x0 = krow[wave][j], x1 = krow[wave][j + half];
                    y[i] = d < half ? x0 * cs[j] - x1 * sn[j] : x1 * cs[j] + x0 * sn[j];
                }
            }
            store_row<true>(page, slot % PG, y, lane, a.status);
            __builtin_amdgcn_wave_barrier();
            continue;
        }
        // eight query heads a wave, a lane holds one 32-dim group of one
        const int h = (task - 2 * a.nkv) * 8 + (lane >> 3), gi = lane & 7;
        const bool on = h < a.nq;
        const float4 *src = reinterpret_cast<const float4 *>(a.qg + ((size_t) t * a.nq + min(h, a.nq - 1)) * 2 * HD + 32 * gi);
        const float4 *wsrc = reinterpret_cast<const float4 *>(a.wq + 32 * gi);
        float x[32];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 f = src[i];
            x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
            ss += sumsq4(f);
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) ss += __shfl_xor(ss, d);
        const float r = rsqrtf(ss / HD + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 w = wsrc[i];
            x[4 * i] *= r * w.x, x[4 * i + 1] *= r * w.y, x[4 * i + 2] *= r * w.z, x[4 * i + 3] *= r * w.w;
        }
        if (32 * gi < a.nrot) {  // the rotated dims meet in the LDS
#pragma unroll
            for (int i = 0; i < 32; ++i) qrow[wave][lane >> 3][32 * gi + i] = x[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (32 * gi < a.nrot) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int d = 32 * gi + i;
                if (d < a.nrot) {
                    const int j = d < half ? d : d - half;
                    const float x0 = qrow[wave][lane >> 3][j], x1 = qrow[wave][lane >> 3][j + half];
                    const float c = (float) cs[j], s = (float) sn[j];
                    x[i] = d < half ? x0 * c - x1 * s : x1 * c + x0 * s;
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        // Five fp6 (e2m3) parts under one power-of-two scale each: the first part's is the least that reaches the
        // group's largest value without saturating, and what a part leaves is at most 1/4 of its scale (1/8 from the
        // second on, whose values are at most 4), so the following scales are 2^-4, 2^-9, 2^-14 and 2^-19 of the
        // first.  What is left of a value is at most 2^-24.9 of the group's largest.
        float am = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            am = fmaxf(am, fabsf(x[i]));
            bad |= !(fabsf(x[i]) < INFINITY);
        }
        const uint32_t u = __float_as_uint(am);
        int e0 = (int) (u >> 23) - 127 - 2 + ((u & 0x7fffffu) > 0x700000u);
        e0 = max(e0, EMIN);
        const int g = h / a.grp, row = (t - a.cu[b]) * a.grp + (h - g * a.grp);
        const int item = first_item(a.cu, b, a.grp, RT) + row / RT;
        uint8_t *dst = a.Q + (((size_t) g * a.items + item) * (RT / 16) + row % RT / 16) * QBLK;
        const int uh = gi >> 2, ln = (gi & 3) * 16 + row % 16;
        const bool st = on && item < a.items;
        v16f lo, hi;
#pragma unroll
        for (int i = 0; i < 16; ++i) lo[i] = x[2 * i], hi[i] = x[2 * i + 1];
        int e = e0;
#pragma unroll
        for (int p = 0; p < NPART; ++p) {
            const float sc = __uint_as_float((uint32_t) (e + 127) << 23);
            const v6u part = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(lo, hi, sc);
            // (this compiler lets the conversions' results overlap their operands, which they read in passes: the
            // operands are kept in use past each of them)
            asm volatile("" ::"v"(lo), "v"(hi), "v"(sc), "v"(part));
            if (st) {
                *reinterpret_cast<v4u *>(dst + (uh * NPART + p) * FRAG + ln * 16) = v4u{part[0], part[1], part[2], part[3]};
                *reinterpret_cast<v2u *>(dst + (uh * NPART + p) * FRAG + 1024 + ln * 8) = v2u{part[4], part[5]};
            }
            if (p + 1 < NPART) {
                const v32f back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(part, sc);
                asm volatile("" ::"v"(part), "v"(sc), "v"(back));
#pragma unroll
                for (int i = 0; i < 16; ++i) lo[i] -= back[2 * i], hi[i] -= back[2 * i + 1];
            }
            e -= p == 0 ? 4 : 5;
        }
        // fp6 has no infinity or NaN: such a query group gets the NaN scale, so that its row's scores are NaN
        const uint32_t s0 = e0 + 127;
        const v2u sc = bad ? v2u{~0u, ~0u}
                           : v2u{s0 | (s0 - 4) << 8 | (s0 - 9) << 16 | (s0 - 14) << 24, s0 - 19};
        if (st) *reinterpret_cast<v2u *>(dst + 2 * NPART * FRAG + uh * 512 + ln * 8) = sc;
    }
}

template <int OA, int OB> __device__ __forceinline__ v4f mma_k(v4u k, int ks, const v6u &q, int qs, v4f c) {
    const v8i A = {(int) k[0], (int) k[1], (int) k[2], (int) k[3], 0, 0, 0, 0};
    const v8i Bq = {(int) q[0], (int) q[1], (int) q[2], (int) q[3], (int) q[4], (int) q[5], 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, Bq, c, 4, 2, OA, ks, OB, qs);
}
__device__ __forceinline__ v4f mma_v(const v4u &a, const v4u &b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), bf16x2));
}
constexpr float SM_SCALE = 0.0625f * 1.4426950408889634f;  // 1 / sqrt(HD), and the softmax in powers of two
constexpr float SLACK = 8.0f * 16.0f;                      // growth of a row's largest raw score that moves its reference
constexpr float PUP = 16.0f;                               // probabilities times 2^16: the parts of the least ones stay normal

struct KvBlock {  // 32 keys of one head in registers
    v4u k[2][2];  // [16-key block][half of the row]
    uint32_t ks;
    v4u v[4], vs[4];
};

// grid (nsplit, nkv, items), 256 threads: the RT = 16 NRB rows of an item against the keys of a split; the waves take
// 32-key blocks in turn, each with its own softmax state, and meet at the end.
template <int NRB>
__global__ void __launch_bounds__(WAVES * 64) k_attn_kv4(const Kv4Args a) {
    constexpr int RT = 16 * NRB;
    constexpr int QB = NRB * QBLK, MB = WAVES * RT * OS * 4;
    __shared__ __align__(16) uint8_t lds[QB > MB ? QB : MB];
    __shared__ float wm[WAVES][RT], wl[WAVES][RT];
    const int sp = blockIdx.x, g = blockIdx.y, item = a.items - 1 - (int) blockIdx.z;  // the longest rows first
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int b = request_of(a.cu, a.B, item, a.grp, RT);
    const int c0 = a.cu[b], n = min(a.cu[b + 1], a.T) - c0, r0 = (item - first_item(a.cu, b, a.grp, RT)) * RT;
    const int rows = n * a.grp;
    if (c0 < 0 || r0 < 0 || r0 >= rows) return;
    const int past = a.past[b], cap = a.mb * PG;
    auto visible = [&](int t) { return past < 0 ? 0 : (int) min((long long) past + t + 1, (long long) cap); };
    const int kvalid = visible(n - 1), kmax = visible((min(r0 + RT, rows) - 1) / a.grp);
    const int tiles = (kmax + PG - 1) / PG, per = (tiles + a.nsplit - 1) / a.nsplit;
    const int k0 = min(sp * per, tiles) * PG, k1 = min(min((sp + 1) * per, tiles) * PG, kmax);

    // the item's query operands into the LDS
    const v4u *Q = reinterpret_cast<const v4u *>(a.Q + ((size_t) g * a.items + item) * NRB * QBLK);
    for (int i = threadIdx.x; i < QB / 16; i += WAVES * 64) reinterpret_cast<v4u *>(lds)[i] = Q[i];
    __syncthreads();
    int lim[NRB];
    v2u qs[NRB][2];
#pragma unroll
    for (int j = 0; j < NRB; ++j) {
        lim[j] = min(visible(min((r0 + 16 * j + (lane & 15)) / a.grp, n - 1)), k1);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            qs[j][u] = *reinterpret_cast<const v2u *>(lds + j * QBLK + 2 * NPART * FRAG + u * 512 + lane * 8);
    }
    v4f o[NRB][16];
    float m[NRB], l[NRB];
#pragma unroll
    for (int j = 0; j < NRB; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int t = 0; t < 16; ++t) o[j][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int32_t *table = a.table + (size_t) b * a.mb;
    auto page_of = [&](int kb) { return kb * 32 < k1 ? table[kb >> 1] : 0; };
    auto load = [&](int kb, int page, KvBlock &x) {
        if (page < 0 || page >= a.npages) page = 0;  // in bounds; the block is skipped
        const uint8_t *p = a.cache + ((size_t) page * a.nkv + g) * HEAD_BYTES;
        const int kk = kb & 1;
#pragma unroll
        for (int hb = 0; hb < 2; ++hb)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                x.k[hb][u] = *reinterpret_cast<const v4u *>(p + (((kk * 2 + hb) * 2 + u) * 64 + lane) * 16);
        x.ks = *reinterpret_cast<const uint32_t *>(p + KS + (kk * 64 + lane) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = *reinterpret_cast<const v4u *>(p + VC + ((kk * 4 + i) * 64 + lane) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x.vs[i] = *reinterpret_cast<const v4u *>(p + VS + (kk * 4 + (lane >> 4)) * 64 + i * 16);
    };
    int kb = k0 / 32 + wave;
    int page = page_of(kb), next_page = page_of(kb + WAVES);
    KvBlock cur, nxt;
    if (kb * 32 < k1) load(kb, page, cur);
    for (; kb * 32 < k1; kb += WAVES) {
        const int here = page;
        page = next_page;
        next_page = page_of(kb + 2 * WAVES);
        load((kb + WAVES) * 32 < k1 ? kb + WAVES : kb, (kb + WAVES) * 32 < k1 ? page : here, nxt);
        if (here < 0 || here >= a.npages) {
            if (lane == 0) atomicOr(a.status, FN_STATUS_PAGE);
            cur = nxt;
            continue;
        }
        if (kb * 32 + 32 > kvalid) {  // rows of the page that hold no token: their value scales may be anything
            const int base = kb * 32 + 4 * (lane >> 4);
            uint32_t keep[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) keep[j / 4] |= base + 16 * (j / 4) + j % 4 < kvalid ? 0xffu << (8 * (j % 4)) : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) cur.vs[i] &= v4u{keep[0], keep[1], keep[0], keep[1]};
        }
        // scores
        v4f S[2][NRB];
        {
            v4f big[2][NRB], small[2][NRB];
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int j = 0; j < NRB; ++j) big[hb][j] = small[hb][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#define FN_KV4_PART(U, P)                                                                                            \
    do {                                                                                                            \
        _Pragma("unroll") for (int j = 0; j < NRB; ++j) {                                                            \
            const uint8_t *f = lds + j * QBLK + ((U) * NPART + (P)) * FRAG;                                          \
            const v4u qa = *reinterpret_cast<const v4u *>(f + lane * 16);                                            \
            const v2u qb = *reinterpret_cast<const v2u *>(f + 1024 + lane * 8);                                      \
            const v6u q = {qa[0], qa[1], qa[2], qa[3], qb[0], qb[1]};                                                \
            v4f(&acc)[2][NRB] = (P) == 0 ? big : small;                                                              \
            acc[0][j] = mma_k<(U), (P) % 4>(cur.k[0][U], (int) cur.ks, q, (int) qs[j][U][(P) / 4], acc[0][j]);       \
            acc[1][j] = mma_k<2 + (U), (P) % 4>(cur.k[1][U], (int) cur.ks, q, (int) qs[j][U][(P) / 4], acc[1][j]);   \
        }                                                                                                           \
    } while (0)
            FN_KV4_PART(0, 0);
            FN_KV4_PART(0, 1);
            FN_KV4_PART(0, 2);
            FN_KV4_PART(0, 3);
            FN_KV4_PART(0, 4);
            FN_KV4_PART(1, 0);
            FN_KV4_PART(1, 1);
            FN_KV4_PART(1, 2);
            FN_KV4_PART(1, 3);
            FN_KV4_PART(1, 4);
#undef FN_KV4_PART
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int j = 0; j < NRB; ++j) S[hb][j] = big[hb][j] + small[hb][j];
        }
        // online softmax of the lane's row (lane % 16) over the 32 keys; the probabilities in three bf16 parts
        v4u P[NRB][3];
        float corr[NRB];
        bool rescale = false;
        const int key = kb * 32 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NRB; ++j) {
            float sc[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sc[i] = key + 16 * (i / 4) + i % 4 < lim[j] ? S[i / 4][j][i % 4] : -INFINITY;
                mx = fmaxf(mx, sc[i]);
            }
            mx = max_quarters(mx);
            const bool first = m[j] == -INFINITY, moved = !first && mx > m[j] + SLACK;
            const float mn = first || moved ? mx : m[j];
            corr[j] = moved ? __builtin_amdgcn_exp2f((m[j] - mn) * SM_SCALE) : 1.0f;
            rescale |= moved;
            float ps = 0.0f;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = sc[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(sc[i] - mn, SM_SCALE, PUP));
                ps += p[i];
            }
            l[j] = fmaf(l[j], corr[j], ps);
            m[j] = mn;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = p[2 * i], y = p[2 * i + 1];
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    const uint32_t h = bf16_pair(x, y);
                    P[j][q][i] = h;
                    x -= __uint_as_float(h << 16);
                    y -= __uint_as_float(h & 0xffff0000u);
                }
            }
        }
        if (__ballot(rescale)) {
#pragma unroll
            for (int j = 0; j < NRB; ++j)
#pragma unroll
                for (int t = 0; t < 16; ++t) o[j][t] *= corr[j];
        }
        // o += V^T P^T, 32 dims at a time: one conversion gives two dims of a key, a permute two keys of a dim
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            uint32_t pr[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t w = cur.v[t / 2][t % 2 * 2 + j / 4], s4 = cur.vs[t / 2][t % 2 * 2 + j / 4];
                // the instruction takes the scale from bits 30:23 of a float and looks at no other
                const float s = __uint_as_float(j % 4 == 3 ? s4 >> 1 : s4 << (23 - 8 * (j % 4)));
                const auto cv = [&](auto sel) {
                    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, decltype(sel)::value));
                };
                pr[j] = j % 4 == 0   ? cv(std::integral_constant<int, 0>{})
                        : j % 4 == 1 ? cv(std::integral_constant<int, 1>{})
                        : j % 4 == 2 ? cv(std::integral_constant<int, 2>{})
                                     : cv(std::integral_constant<int, 3>{});
            }
            v4u even, odd;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                even[i] = __builtin_amdgcn_perm(pr[2 * i + 1], pr[2 * i], 0x05040100u);
                odd[i] = __builtin_amdgcn_perm(pr[2 * i + 1], pr[2 * i], 0x07060302u);
            }
#pragma unroll
            for (int q = 2; q >= 0; --q)
#pragma unroll
                for (int j = 0; j < NRB; ++j) {
                    o[j][2 * t] = mma_v(even, P[j][q], o[j][2 * t]);
                    o[j][2 * t + 1] = mma_v(odd, P[j][q], o[j][2 * t + 1]);
                }
        }
        cur = nxt;
    }
    // the waves meet: reference of every row, then the sums, 64 dims at a time
#pragma unroll
    for (int j = 0; j < NRB; ++j) {
        const float ls = sum_quarters(l[j]);
        if (lane < 16) {
            wm[wave][16 * j + lane] = m[j];
            wl[wave][16 * j + lane] = ls;
        }
    }
    float *mo = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        __syncthreads();  // the query operands, or the last 64 dims, have been read
#pragma unroll
        for (int j = 0; j < NRB; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) {  // the lane's row, dims 8 (lane / 16) .. + 7 of the group
                float *d = mo + (wave * RT + 16 * j + (lane & 15)) * OS + 32 * t + 8 * (lane >> 4);
                const v4f e = o[j][4 * c + 2 * t], f = o[j][4 * c + 2 * t + 1];
                *reinterpret_cast<float4 *>(d) = make_float4(e[0], f[0], e[1], f[1]);
                *reinterpret_cast<float4 *>(d + 4) = make_float4(e[2], f[2], e[3], f[3]);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < RT * 16; i += WAVES * 64) {
            const int row = i >> 4, r = r0 + row, d = (i & 15) * 4;
            if (r >= rows) continue;
            float M = wm[0][row];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) M = fmaxf(M, wm[w][row]);
            float L = 0.0f;
            float4 s = f4(0.0f);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float mw = wm[w][row];
                const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw - M) * SM_SCALE);
                L = fmaf(wl[w][row], f, L);
                s = add_scaled(s, *reinterpret_cast<const float4 *>(mo + (w * RT + row) * OS + d), f);
            }
            if (a.nsplit == 1) {
                const int t = r / a.grp;
                const size_t at = (size_t) (c0 + t) * a.nq + g * a.grp + (r - t * a.grp);
                const float4 z = *reinterpret_cast<const float4 *>(a.qg + (at * 2 + 1) * HD + 64 * c + d);
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // a row that sees no key: zeros
                *reinterpret_cast<float4 *>(a.og + at * HD + 64 * c + d) =
                    make_float4(s.x * inv * sigmoidf_(z.x), s.y * inv * sigmoidf_(z.y), s.z * inv * sigmoidf_(z.z),
                                s.w * inv * sigmoidf_(z.w));
            } else {
                const size_t at = (((size_t) item * a.nkv + g) * a.nsplit + sp) * RT + row;
                *reinterpret_cast<float4 *>(a.part_o + at * HD + 64 * c + d) = s;
                if (c == 0 && d == 0) {
                    a.part_ml[2 * at] = M;
                    a.part_ml[2 * at + 1] = L;
                }
            }
        }
    }
}

// grid (items RT / 4, nkv), a wave a row, lane = 4 dims: the splits of a row joined, and the gate
template <int RT>
__global__ void __launch_bounds__(256) k_kv4_combine(const Kv4Args a) {
    const int item = blockIdx.x / (RT / 4), g = blockIdx.y, lane = threadIdx.x & 63;
    const int row = blockIdx.x % (RT / 4) * 4 + (threadIdx.x >> 6);
    const int b = request_of(a.cu, a.B, item, a.grp, RT);
    const int c0 = a.cu[b], n = min(a.cu[b + 1], a.T) - c0, r = (item - first_item(a.cu, b, a.grp, RT)) * RT + row;
    if (c0 < 0 || r < 0 || r >= n * a.grp) return;
    const size_t at0 = ((size_t) item * a.nkv + g) * a.nsplit * RT + row;
    float M = -INFINITY;
    for (int s = lane; s < a.nsplit; s += 64) M = fmaxf(M, a.part_ml[2 * (at0 + (size_t) s * RT)]);
    M = wave_max(M);
    float L = 0.0f;
    float4 o = f4(0.0f);
    for (int s = 0; s < a.nsplit; ++s) {
        const size_t at = at0 + (size_t) s * RT;
        const float ms = a.part_ml[2 * at], ls = a.part_ml[2 * at + 1];
        const float f = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ms - M) * SM_SCALE);
        L = fmaf(ls, f, L);
        o = add_scaled(o, reinterpret_cast<const float4 *>(a.part_o + at * HD)[lane], f);
    }
    const int t = r / a.grp;
    const size_t at = (size_t) (c0 + t) * a.nq + g * a.grp + (r - t * a.grp);
    const float4 z = reinterpret_cast<const float4 *>(a.qg + (at * 2 + 1) * HD)[lane];
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    reinterpret_cast<float4 *>(a.og + at * HD)[lane] = make_float4(
        o.x * inv * sigmoidf_(z.x), o.y * inv * sigmoidf_(z.y), o.z * inv * sigmoidf_(z.z), o.w * inv * sigmoidf_(z.w));
}

// 16-row blocks an item: one where the requests have few rows (decode), two otherwise
int row_blocks(int B, int T, int grp) { return (long long) T * grp <= 16ll * B ? 1 : 2; }

}  // namespace

size_t kv4_work_bytes(int B, int T, int nq, int nkv, int hd, int nsplit) {
    const int grp = nq / nkv, rt = 16 * row_blocks(B, T, grp);
    const size_t rows = item_count(B, T, grp, rt) * nkv * rt;
    return rows * 1024 + (nsplit > 1 ? rows * nsplit * (HD + 2) * sizeof(float) : 0);
}

int kv4_pick_nsplit(int B, int T, int nq, int nkv, int ctx) {
    const int grp = nq / nkv;
    const long long groups = (long long) item_count(B, T, grp, 16 * row_blocks(B, T, grp)) * nkv;
    const int most = std::max(1, (ctx + 127) / 128);  // a 32-key block for each wave
    const long long want = std::max(1ll, 2ll * device_cus() / groups);
    return (int) std::min<long long>(want, most);
}

int kv4_attn_launch(const Kv4Attn &p, hipStream_t st) {
    if (p.B < 1 || p.T < 1 || p.nq < 1 || p.nkv < 1) FN_FAIL("attn_kv4: B, T, nq and nkv must be >= 1");
    if (p.hd != HD) FN_FAIL("attn_kv4: only head_dim 256 is built");
    if (p.nq % p.nkv) FN_FAIL("attn_kv4: nq must be a multiple of nkv");
    if (p.nrot < 0 || p.nrot > MAXROT || (p.nrot & 1)) FN_FAIL("attn_kv4: nrot must be even and <= 128");
    if (p.nsplit < 1 || p.nsplit > 65535) FN_FAIL("attn_kv4: nsplit must be in 1..65535");
    if (p.max_blocks < 1 || p.max_blocks > 1 << 24) FN_FAIL("attn_kv4: max_blocks must be in 1..16777216");
    if (p.npages < 1 || p.npages > INT_MAX / PG) FN_FAIL("attn_kv4: npages must be in 1..33554431 (slots are 32-bit)");
    if (!p.past || !p.cu || !p.table || !p.slot || !p.seq || !p.qg || !p.k || !p.v || !p.wq || !p.wk || !p.cache ||
        !p.work || !p.og)
        FN_FAIL("attn_kv4: null pointer");
    if (((uintptr_t) p.qg | (uintptr_t) p.k | (uintptr_t) p.v | (uintptr_t) p.wq | (uintptr_t) p.wk | (uintptr_t) p.cache |
         (uintptr_t) p.work | (uintptr_t) p.og) & 15)
        FN_FAIL("attn_kv4: qg, k, v, wq, wk, cache, work and og must be 16-byte aligned");
    const int grp = p.nq / p.nkv, nrb = row_blocks(p.B, p.T, grp);
    if ((long long) p.T * grp > INT_MAX - 64) FN_FAIL("attn_kv4: too many query rows");
    const size_t items = item_count(p.B, p.T, grp, 16 * nrb);
    if (p.nkv > 65535 || items > 65535) FN_FAIL("attn_kv4: batch too large (at most 65535 items of 32 query rows)");
    if (p.work_bytes < kv4_work_bytes(p.B, p.T, p.nq, p.nkv, p.hd, p.nsplit)) FN_FAIL("attn_kv4: workspace too small");
    Kv4Args a{};
    a.B = p.B; a.T = p.T; a.nq = p.nq; a.nkv = p.nkv; a.grp = grp; a.mb = p.max_blocks; a.npages = p.npages;
    a.nsplit = p.nsplit; a.nrot = p.nrot; a.items = (int) items; a.eps = p.eps; a.past = p.past; a.cu = p.cu;
    a.table = p.table; a.slot = p.slot; a.seq = p.seq; a.qg = p.qg; a.k = p.k; a.v = p.v; a.wq = p.wq; a.wk = p.wk;
    a.cache = p.cache; a.og = p.og;
    if (status_word(&a.status)) return -1;
    const size_t rows = items * p.nkv * 16 * nrb;
    a.Q = static_cast<uint8_t *>(p.work);
    a.part_o = reinterpret_cast<float *>(a.Q + rows * 1024);
    a.part_ml = a.part_o + rows * p.nsplit * HD;
    for (int i = 0; i < p.nrot / 2; ++i) a.freq[i] = std::pow((double) p.theta, -(2.0 * i) / p.nrot);
    const dim3 grid(p.nsplit, p.nkv, (unsigned) items);
    if (nrb == 1) {
        hipLaunchKernelGGL(k_kv4_prep<16>, dim3(p.T), dim3(256), 0, st, a);
        hipLaunchKernelGGL(k_attn_kv4<1>, grid, dim3(WAVES * 64), 0, st, a);
        if (p.nsplit > 1) hipLaunchKernelGGL(k_kv4_combine<16>, dim3((unsigned) items * 4, p.nkv), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL(k_kv4_prep<32>, dim3(p.T), dim3(256), 0, st, a);
        hipLaunchKernelGGL(k_attn_kv4<2>, grid, dim3(WAVES * 64), 0, st, a);
        if (p.nsplit > 1) hipLaunchKernelGGL(k_kv4_combine<32>, dim3((unsigned) items * 8, p.nkv), dim3(256), 0, st, a);
    }
    FN_CK(hipGetLastError());
    return 0;
}

}  // namespace fn
