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
constexpr int QBLK = 2 * NPART * FRAG + 2 * 64 * 8;    // 16 query rows: [half][part] operands, [half] scales
constexpr int HSLOT = 3;                               // 8 query rows: columns 0..7 hold parts 0..2, 8..15 parts 3, 4, zero
constexpr int HBLK = 2 * HSLOT * FRAG + 2 * 64 * 4;    // [half][slot] operands, [half] scales
constexpr int NRB = 2;                                 // blocks of 16 rows an item that is not one of 8
template <int RT> constexpr int item_bytes = RT == 8 ? HBLK : NRB * QBLK;  // RT: query rows an item
constexpr int WAVES = 4;

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
    uint8_t *Q;                 // [nkv][items] query operands of item_bytes
    float *part_o;              // [items][nkv][nsplit][rows][HD]
    float *part_ml;             // [items][nkv][nsplit][rows][2]
    float *og;
    unsigned *status;
    double freq[MAXROT / 2];
};

// Sine and cosine in 64 bits of 0 <= x < 2^30: x less the nearest multiple of pi / 2, which is kept in two parts (the
// first product is exact in the fused multiply-add), then the Taylor series to r^17, whose rest is below 2^-60 for
// |r| <= pi / 4.
__device__ __forceinline__ void sin_cos(double x, double &s, double &c) {
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.5707963267948966192, x);
    r = fma(-n, 6.123233995736766036e-17, r);
    const double z = r * r;
    double a = 2.8114572543455206e-15, b = 4.7794773323873853e-14;  // 1/17!, 1/16!
    a = fma(a, z, -7.6471637318198164e-13);
    b = fma(b, z, -1.1470745597729725e-11);
    a = fma(a, z, 1.6059043836821613e-10);
    b = fma(b, z, 2.0876756987868099e-09);
    a = fma(a, z, -2.5052108385441719e-08);
    b = fma(b, z, -2.7557319223985893e-07);
    a = fma(a, z, 2.7557319223985893e-06);
    b = fma(b, z, 2.4801587301587302e-05);
    a = fma(a, z, -1.9841269841269841e-04);
    b = fma(b, z, -1.3888888888888889e-03);
    a = fma(a, z, 8.3333333333333333e-03);
    b = fma(b, z, 4.1666666666666667e-02);
    a = fma(a, z, -1.6666666666666667e-01);
    b = fma(b, z, -0.5);
    const double sr = fma(r * z, a, r), cr = fma(z, b, 1.0);
    const int q = (int) n & 3;
    s = q & 1 ? cr : sr;
    c = q & 1 ? sr : cr;
    if (q & 2) s = -s;
    if (q == 1 || q == 2) c = -c;
}

// One token: sines and cosines of its position, its keys and values into their page, its queries as operands.  A wave takes
// one row of keys or values, or eight query heads.  What bounds it is the way through one token (a load, 64-bit sines, the
// norm, five conversions one after the other): 6 us.  So a small batch gets workgroups for all of a token's tasks at once
// (7.4 -> 6.4 us at one token of 2 + 2 + 16 heads, 9.0 -> 6.7 us at 64), and a large one two launches (PART 1: keys and
// values, 2: queries): the keys' share in a kernel of its own has room for three times the waves.
enum { PREP_ALL, PREP_KEYS, PREP_QUERIES };
template <int RT, int PART>
__global__ void __launch_bounds__(256, PART == PREP_KEYS ? 6 : 2) k_kv4_prep(const Kv4Args a) {
    __shared__ double cs[MAXROT], sn[MAXROT];  // of each rotated dim; the sine with the sign that its pair's other value gets
    __shared__ float cf[MAXROT], sf[MAXROT];
    __shared__ double krow[PART == PREP_QUERIES ? 1 : WAVES][MAXROT];
    __shared__ float qrow[PART == PREP_KEYS ? 1 : WAVES][8][MAXROT + 4];
    const int t = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // the wave's first rows, and what else depends on no other load, are requested before anything that waits
    const int slot = a.slot[t], b = a.seq[t], begin = a.cu[0], total = min(a.cu[a.B], a.T), half = a.nrot / 2;
    auto freq = [&](int d) { return a.freq[d < half ? d : d < a.nrot ? d - half : 0]; };
    double fr = freq(threadIdx.x);
    const int waves = blockDim.x >> 6, octets = (a.nq + 7) / 8;
    const int from = PART == PREP_QUERIES ? 2 * a.nkv : 0, tasks = 2 * a.nkv + (PART == PREP_KEYS ? 0 : octets);
    const int first = from + wave + waves * blockIdx.y;
    float4 row[8];
    auto request = [&](int task) __attribute__((always_inline)) {
        if (PART == PREP_KEYS || (PART == PREP_ALL && task < 2 * a.nkv)) {
            row[0] = reinterpret_cast<const float4 *>((task & 1 ? a.v : a.k) + ((size_t) t * a.nkv + (task >> 1)) * HD)[lane];
        } else {
            const int h = min((task - 2 * a.nkv) * 8 + (lane >> 3), a.nq - 1);
            const float4 *src = reinterpret_cast<const float4 *>(a.qg + ((size_t) t * a.nq + h) * 2 * HD + 32 * (lane & 7));
#pragma unroll
            for (int i = 0; i < 8; ++i) row[i] = src[i];
        }
    };
    if (first < tasks) request(first);
    if (t < begin || t >= total) return;
    // (three loads at once, of some request where seq names none)
    const int sb = min(max(b, 0), a.B - 1), c0 = a.cu[sb], c1 = a.cu[sb + 1], past = a.past[sb];
    if (b != sb || t < c0 || t >= c1 || c0 < 0) {
        if (threadIdx.x == 0) atomicOr(a.status, FN_STATUS_ROWS);
        return;
    }
    const long long P = (long long) past + (t - c0);
    if ((past < 0 || P >= (long long) a.mb * PG) && threadIdx.x == 0) atomicOr(a.status, FN_STATUS_POS);
    // the angle in 64 bits: a float product is off by up to half a radian at a million tokens
    for (int d = threadIdx.x; d < MAXROT; d += blockDim.x) {
        double sv = 0.0, cv = 1.0;
        if (d != threadIdx.x) fr = freq(d);
        if (d < a.nrot) sin_cos((double) P * fr, sv, cv);
        if (d < half) sv = -sv;
        cs[d] = cv, sn[d] = sv;
        cf[d] = (float) cv, sf[d] = (float) sv;
    }
    __syncthreads();
    const bool put = slot >= 0 && slot / PG < a.npages;
    if (PART != PREP_QUERIES && slot >= 0 && !put && threadIdx.x == 0) atomicOr(a.status, FN_STATUS_PAGE);
    for (int task = first; task < tasks; task += waves * gridDim.y) {
        if (task != first) request(task);
        if (PART == PREP_KEYS || (PART == PREP_ALL && task < 2 * a.nkv)) {
            if (!put) continue;
            const int g = task >> 1;
            uint8_t *page = a.cache + ((size_t) (slot / PG) * a.nkv + g) * HEAD_BYTES;
            const bool is_v = task & 1;
            double y[4] = {row[0].x, row[0].y, row[0].z, row[0].w};
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
            if (4 * lane < a.nrot) {
#pragma unroll
                for (int i = 0; i < 4; ++i) krow[wave][4 * lane + i] = y[i];
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            if (4 * lane < a.nrot) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 4 * lane + i, o = d < half ? d + half : d < a.nrot ? d - half : d;
                    y[i] = y[i] * cs[d] + krow[wave][o] * sn[d];
                }
            }
            store_row<true>(page, slot % PG, y, lane, a.status);
            __builtin_amdgcn_wave_barrier();
            continue;
        }
        // eight query heads a wave, a lane holds one 32-dim group of one
        const int h = (task - 2 * a.nkv) * 8 + (lane >> 3), gi = lane & 7;
        const bool on = h < a.nq;
        const float4 *wsrc = reinterpret_cast<const float4 *>(a.wq + 32 * gi);
        float x[32];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 f = row[i];
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
            if (i == 3) __builtin_amdgcn_sched_barrier(0);
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
                const int d = 32 * gi + i, o = d < half ? d + half : d < a.nrot ? d - half : d;
                x[i] = fmaf(qrow[wave][lane >> 3][o], sf[d], x[i] * cf[d]);
                if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // (reads of eight at a time)
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
        const int g = h / a.grp, row = (t - c0) * a.grp + (h - g * a.grp);
        const int item = first_item(a.cu, b, a.grp, RT) + row / RT;
        uint8_t *dst = a.Q + ((size_t) g * a.items + item) * item_bytes<RT> + (RT == 8 ? 0 : row % RT / 16 * QBLK);
        const int uh = gi >> 2, ln = (gi & 3) * 16 + row % (RT == 8 ? 8 : 16);
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
                uint8_t *f = dst + (RT == 8 ? uh * HSLOT + p % HSLOT : uh * NPART + p) * FRAG;
                const int l = ln + (RT == 8 && p >= HSLOT ? 8 : 0);
                *reinterpret_cast<v4u *>(f + l * 16) = v4u{part[0], part[1], part[2], part[3]};
                *reinterpret_cast<v2u *>(f + 1024 + l * 8) = v2u{part[4], part[5]};
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
        if (RT == 8) {
            if (st) {
                uint8_t *f = dst + (uh * HSLOT + 2) * FRAG;
                *reinterpret_cast<v4u *>(f + (ln + 8) * 16) = v4u{0, 0, 0, 0};
                *reinterpret_cast<v2u *>(f + 1024 + (ln + 8) * 8) = v2u{0, 0};
                uint32_t *d = reinterpret_cast<uint32_t *>(dst + 2 * HSLOT * FRAG + uh * 256) + ln;
                d[0] = sc[0];
                d[8] = sc[0] >> 24 | (sc[1] & 0xff) << 8;  // parts 3, 4
            }
        } else if (st) {
            *reinterpret_cast<v2u *>(dst + 2 * NPART * FRAG + uh * 512 + ln * 8) = sc;
        }
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
constexpr float SLACK = 8.0f;                              // growth of a row's largest score, in powers of two, that moves its reference
// Probabilities times 2^PUP, so that the sums hold every value of the format: the largest, 6 2^125, times probabilities of up
// to 2^(SLACK + 1/2) over 2^19 keys stays below 2^128, and of the least, 2^-101, a product keeps 2^-149 (the matrix
// instructions hold denormals), 20 bits of it.  (With 2^16 values from 2^103 on gave infinities.)
constexpr float PUP = -28.0f;

// 64 dims of the lane's eight keys as bf16 pairs: dims 32 t + 2 (l % 16), + 1
__device__ __forceinline__ void values_of(const v4u &v, const v4u &vs, int t, uint32_t (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t w = v[t * 2 + j / 4], s4 = vs[t * 2 + j / 4];
        // the instruction takes the scale from bits 30:23 of a float and looks at no other
        const float s = __uint_as_float(j % 4 == 3 ? s4 >> 1 : s4 << (23 - 8 * (j % 4)));
        const auto cv = [&](auto sel) {
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, decltype(sel)::value));
        };
        x[j] = j % 4 == 0   ? cv(std::integral_constant<int, 0>{})
               : j % 4 == 1 ? cv(std::integral_constant<int, 1>{})
               : j % 4 == 2 ? cv(std::integral_constant<int, 2>{})
                            : cv(std::integral_constant<int, 3>{});
    }
}

// A 32-key block of one head in 49 registers.  What a wave has used up it requests of its next block at once (K behind the
// scores, V behind each pair of its groups).
struct KvBlock {
    v4u k[2][2];  // [16-key block][half of the row]
    uint32_t ks;
    v4u v[4], vs[4];
    __device__ __forceinline__ void load_k(const uint8_t *p, int kk, int lane) {
#pragma unroll
        for (int hb = 0; hb < 2; ++hb)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                k[hb][u] = *reinterpret_cast<const v4u *>(p + kk * 4096 + (hb * 2 + u) * 1024 + lane * 16);
        ks = *reinterpret_cast<const uint32_t *>(p + KS + kk * 256 + lane * 4);
    }
    __device__ __forceinline__ void load_v(int i, const uint8_t *p, int kk, int lane) {
        v[i] = *reinterpret_cast<const v4u *>(p + VC + kk * 4096 + i * 1024 + lane * 16);
        vs[i] = *reinterpret_cast<const v4u *>(p + VS + kk * 256 + i * 16 + (lane >> 4) * 64);
    }
    __device__ __forceinline__ void values(int t, uint32_t (&x)[8]) const { values_of(v[t / 2], vs[t / 2], t % 2, x); }
};

// The state of one row (the lane's column) of an online softmax.  The reference m is a whole power of two near the row's
// largest: a probability is then one fused multiply-add and one exponential away from its score, and every factor between
// references (of keys before, of other waves and splits) is a power of two, exact.  MASK: keys from lim on count for nothing.
struct Softmax {
    float m = -INFINITY, l = 0.0f;
    // eight raw scores (key + 16 (i / 4) + i % 4), those behind the mask -infinity; returns the largest of the lane's row
    template <bool MASK> static __device__ __forceinline__ float largest(float (&s)[8], int key, int lim) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (MASK) s[i] = key + 16 * (i / 4) + i % 4 < lim ? s[i] : -INFINITY;
            mx = fmaxf(mx, s[i]);
        }
        return max_quarters(mx);
    }
    // -> probabilities 2^PUP p; returns the factor of what was summed before
    template <bool MASK> __device__ __forceinline__ float step(const float (&s)[8], float mx, float (&p)[8]) {
        const float top = rintf(mx * SM_SCALE);
        const bool first = m == -INFINITY, moved = !first && top > m + SLACK;
        const float mn = first || moved ? top : m, up = PUP - mn;
        const float corr = moved ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
        float ps = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], SM_SCALE, up));
            if (MASK && s[i] == -INFINITY) p[i] = 0.0f;
            ps += p[i];
        }
        l = fmaf(l, corr, ps);
        m = mn;
        return corr;
    }
};

// grid (nsplit, nkv, items), four waves: the eight rows of an item (a decode step of up to 8 query heads a kv head) against
// the keys of a split; the waves take 32-key blocks in turn, each with its own softmax state, and meet at the end.
// Eight rows use both halves of the products' 16 columns.  Scores:
// columns 0..7 take parts 0..2 of the queries and 8..15 parts 3, 4, so three products do for five, and a rotation by
// eight lanes adds the halves.  P.V: the conversion leaves dims 2m, 2m + 1 of a key in one register, which as it stands
// is two contraction slots; the columns 0..7 hold a probability in the first of them and 0 in the second, which gives
// the even dims, and 8..15 the other way round.  So nothing is permuted and the sums take half the registers.
// What bounds it: the cache's bytes at long contexts (64 requests of 8k keys: 289 MB in 69 us, 4.2 TB/s, while vector and
// matrix instructions take half and two fifths of the cycles), latency at short ones (one request of 4k keys: 5.3 us).
__global__ void __launch_bounds__(WAVES * 64, 3) k_attn_kv4(const Kv4Args a) {
    constexpr int RT = 8, MS = HD + 4;  // rows, floats a row of the merge
    constexpr int MB = WAVES * RT * MS * 4;
    __shared__ __align__(16) uint8_t lds[HBLK > MB ? HBLK : MB];
    __shared__ float wm[WAVES][RT], wl[WAVES][RT];
    const int sp = blockIdx.x, g = blockIdx.y, item = a.items - 1 - (int) blockIdx.z;  // the longest rows first
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int b = request_of(a.cu, a.B, item, a.grp, RT);
    const int c0 = a.cu[b], n = min(a.cu[b + 1], a.T) - c0, r0 = (item - first_item(a.cu, b, a.grp, RT)) * RT;
    const int rows = n * a.grp;
    if (c0 < 0 || r0 < 0 || r0 >= rows) return;
    const int past = a.past[b], cap = a.mb * PG;
    auto visible = [&](int t) { return past < 0 ? 0 : (int) min((long long) past + t + 1, (long long) cap); };
    const int kvalid = visible(n - 1), kmax = visible((min(r0 + RT, rows) - 1) / a.grp);
    const int tiles = (kmax + PG - 1) / PG, per = (tiles + a.nsplit - 1) / a.nsplit;
    const int k0 = min(sp * per, tiles) * PG, k1 = min(min((sp + 1) * per, tiles) * PG, kmax);
    const int all = min(visible(r0 / a.grp), k1);  // keys that every row of the item sees

    // through the scalar cache: a vector load's wait would wait for every key block in flight, too
    typedef const __attribute__((address_space(4))) int32_t *scalar_i32;
    const scalar_i32 table = (scalar_i32) (uintptr_t) (a.table + (size_t) b * a.mb);
    const size_t stride = (size_t) a.nkv * HEAD_BYTES;
    const uint8_t *cache = a.cache + (size_t) g * HEAD_BYTES;
    auto page_of = [&](int kb) { return kb * 32 < k1 ? table[kb >> 1] : 0; };
    auto ok = [&](int page) { return page >= 0 && page < a.npages; };
    auto base_of = [&](int page) { return cache + (ok(page) ? page : 0) * stride; };  // in bounds; the block is passed over
    int kb = k0 / 32 + wave;
    int page = page_of(kb), next = page_of(kb + WAVES);
    KvBlock x;
    if (kb * 32 < k1) {
        const uint8_t *p = base_of(page);
        x.load_k(p, kb & 1, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.load_v(i, p, kb & 1, lane);
    }
    // the item's query operands into the LDS
    const v4u *Q = reinterpret_cast<const v4u *>(a.Q + ((size_t) g * a.items + item) * HBLK);
    for (int i = threadIdx.x; i < HBLK / 16; i += WAVES * 64) reinterpret_cast<v4u *>(lds)[i] = Q[i];
    __syncthreads();
    uint32_t hs[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) hs[u] = *reinterpret_cast<const uint32_t *>(lds + 2 * HSLOT * FRAG + u * 256 + lane * 4);
    auto operand = [&](int at) __attribute__((always_inline)) {
        const v4u qa = *reinterpret_cast<const v4u *>(lds + at + lane * 16);
        const v2u qb = *reinterpret_cast<const v2u *>(lds + at + 1024 + lane * 8);
        return v6u{qa[0], qa[1], qa[2], qa[3], qb[0], qb[1]};
    };
    const int lim = min(visible(min((r0 + (lane & 7)) / a.grp, n - 1)), k1);
    v4f o[8];
    Softmax sm;
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < 8; ++t) o[t] = zero;
    for (; kb * 32 < k1; kb += WAVES) {
        // what takes the place of this block: the wave's next (at the end, this one again)
        const bool more = (kb + WAVES) * 32 < k1;
        const int here = page, kn = more ? kb + WAVES : kb;
        page = more ? next : here;
        const uint8_t *p = base_of(page);
        next = page_of(kb + 2 * WAVES);
        const bool in = ok(here);  // a block outside the cache counts for nothing
        if (!in && lane == 0) atomicOr(a.status, FN_STATUS_PAGE);
        // scores, the small parts of the queries first
        float S[8];
        v4f acc[2] = {zero, zero};
#define FN_KV4_SLOT(U, P)                                                                              \
    do {                                                                                              \
        const v6u q = operand(((U) * HSLOT + (P)) * FRAG);                                             \
        acc[0] = mma_k<(U), (P)>(x.k[0][U], (int) x.ks, q, (int) hs[U], acc[0]);                       \
        acc[1] = mma_k<2 + (U), (P)>(x.k[1][U], (int) x.ks, q, (int) hs[U], acc[1]);                   \
    } while (0)
        FN_KV4_SLOT(0, 2);
        FN_KV4_SLOT(1, 2);
        FN_KV4_SLOT(0, 1);
        FN_KV4_SLOT(1, 1);
        FN_KV4_SLOT(0, 0);
        FN_KV4_SLOT(1, 0);
#undef FN_KV4_SLOT
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float s = acc[i / 4][i % 4];
            S[i] = s + dpp_ror<8>(s);
        }
        x.load_k(p, kn & 1, lane);
        if (!in || kb * 32 + 32 > kvalid) {  // rows of the page that hold no token: their value scales may be anything
            const int at = kb * 32 + 4 * (lane >> 4), end = in ? kvalid : 0;
            uint32_t keep[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) keep[j / 4] |= at + 16 * (j / 4) + j % 4 < end ? 0xffu << (8 * (j % 4)) : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) x.vs[i] &= v4u{keep[0], keep[1], keep[0], keep[1]};
        }
        float pr[8];
        const int key = kb * 32 + 4 * (lane >> 4);
        const float corr = in && kb * 32 + 32 <= all ? sm.step<false>(S, Softmax::largest<false>(S, key, lim), pr)
                                                     : sm.step<true>(S, Softmax::largest<true>(S, key, in ? lim : 0), pr);
        if (__ballot(corr != 1.0f)) {
#pragma unroll
            for (int t = 0; t < 8; ++t) o[t] *= corr;
        }
        // o += V^T P^T, 32 dims at a time, the probabilities in three bf16 parts
        v4u P[2][3];  // [16-key block][part]; parts by truncation (8 bits each: exact), in the half of the register that
                      // the column takes
        const int sh = lane & 8 ? 0 : 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float f = pr[i];
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const uint32_t h = __float_as_uint(f) & 0xffff0000u;
                P[i / 4][q][i % 4] = h >> sh;
                f -= __uint_as_float(h);
            }
        }
        uint32_t w[2][8];
        x.values(0, w[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 8; ++t) {  // the next 32 dims are converted between the products
            if (t < 7) x.values(t + 1, w[(t + 1) & 1]);
            if (t % 2 == 0 && t < 6) x.load_v(t / 2, p, kn & 1, lane);
            if (t == 7) x.load_v(3, p, kn & 1, lane);
#pragma unroll
            for (int q = 2; q >= 0; --q)
#pragma unroll
                for (int hb = 0; hb < 2; ++hb) {
                    const uint32_t *y = w[t & 1] + 4 * hb;
                    o[t] = mma_v(v4u{y[0], y[1], y[2], y[3]}, P[hb][q], o[t]);
                }
#pragma unroll
            for (int i = 0; i < 6; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // the waves meet: reference of every row, then the sums
    const float ls = sum_quarters(sm.l);
    if (lane < RT) {
        wm[wave][lane] = sm.m;
        wl[wave][lane] = ls;
    }
    float *mo = reinterpret_cast<float *>(lds);
    __syncthreads();  // the query operands have been read
    float *d0 = mo + (wave * RT + (lane & 7)) * MS + 8 * (lane >> 4) + ((lane >> 3) & 1);
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) d0[32 * t + 2 * i] = o[t][i];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * HD / 4; i += WAVES * 64) {
        const int row = i / (HD / 4), r = r0 + row, d = i % (HD / 4) * 4;
        if (r >= rows) continue;
        float M = wm[0][row];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) M = fmaxf(M, wm[w][row]);
        float L = 0.0f;
        float4 s = f4(0.0f);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float mw = wm[w][row];
            const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - M);
            L = fmaf(wl[w][row], f, L);
            s = add_scaled(s, *reinterpret_cast<const float4 *>(mo + (w * RT + row) * MS + d), f);
        }
        if (a.nsplit == 1) {
            const int t = r / a.grp;
            const size_t at = (size_t) (c0 + t) * a.nq + g * a.grp + (r - t * a.grp);
            const float4 z = *reinterpret_cast<const float4 *>(a.qg + (at * 2 + 1) * HD + d);
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // a row that sees no key: zeros
            *reinterpret_cast<float4 *>(a.og + at * HD + d) =
                make_float4(s.x * inv * gate_of(z.x), s.y * inv * gate_of(z.y), s.z * inv * gate_of(z.z),
                            s.w * inv * gate_of(z.w));
        } else {
            const size_t at = (((size_t) item * a.nkv + g) * a.nsplit + sp) * RT + row;
            *reinterpret_cast<float4 *>(a.part_o + at * HD + d) = s;
            if (d == 0) {
                a.part_ml[2 * at] = M;
                a.part_ml[2 * at + 1] = L;
            }
        }
    }
}

// The item of workgroup z, and its request (-1: none): the requests with the most keys first, each from its last rows on.
// The workgroups of a call last as long as their keys; in the order of the items the last round of a mixed batch is begun
// late by its longest (24 requests of 1 or 300 tokens over 0.8k to 8k keys: 689 us, in this order 573 us).  A wave ranks up
// to 64 requests, one a lane; beyond that a call has many rounds, and the order is that of the items.
__device__ __forceinline__ int longest_first(const Kv4Args &a, int rt, int z, int &item) {
    const int lane = threadIdx.x & 63;
    if (a.B > 64) {
        item = a.items - 1 - z;
        return request_of(a.cu, a.B, item, a.grp, rt);
    }
    const int lb = min(lane, a.B - 1), c0 = a.cu[lb], n = max(0, min(a.cu[lb + 1], a.T) - c0), past = a.past[lb];
    const int keys = past < 0 ? 0 : min(past, a.mb * PG) + n;
    const int cnt = lane < a.B && c0 >= 0 ? (n * a.grp + rt - 1) / rt : 0;
    int before = 0;
    for (int i = 0; i < a.B; ++i) {
        const int k = __builtin_amdgcn_readlane(keys, i), c = __builtin_amdgcn_readlane(cnt, i);
        before += k > keys || (k == keys && i < lane) ? c : 0;
    }
    const uint64_t hit = __ballot(z >= before && z < before + cnt);
    if (!hit) return -1;
    const int b = __ffsll((unsigned long long) hit) - 1;
    item = first_item(a.cu, b, a.grp, rt) + __builtin_amdgcn_readlane(cnt, b) - 1 - (z - __builtin_amdgcn_readlane(before, b));
    return b;
}

// grid (nsplit, nkv, items), four waves: the 32 rows of an item against the keys of a split, 128 keys at a time.  For the
// scores a wave takes 32 of the keys, for the values a quarter of the dims: so each value is converted once for all rows,
// the sums of a wave are 32 registers and not 128 (which left one wave a SIMD: 463 us for what now takes 323), and nothing
// is left to be joined at the end.  The waves share the rows' references (a row's largest score goes through the LDS) and
// the probabilities.
// What bounds it: 136 matrix instructions of 16 cycles and some 570 vector instructions of 4 a wave and step, which two
// waves a SIMD overlap in part, and 240 KB a step through the LDS: 8,100 to 8,700 cycles a step of two workgroups a CU, of
// which the scores take 2,000, the largest scores 700, the probabilities 1,900 and the values 3,400.  A prompt of 4001
// tokens, 16 + 2 heads: 323 us, the matrix instructions alone 113 us; 24 requests of 1 or 300 tokens over 0.8k to 8k keys:
// 534 us, 197 us.
__global__ void __launch_bounds__(WAVES * 64, 2) k_attn_kv4_rows(const Kv4Args a) {
    constexpr int RT = 16 * NRB, STEP = WAVES * 32;
    __shared__ __align__(16) uint8_t lq[NRB * QBLK];
    __shared__ v4u lp[WAVES][NRB][3][64];  // probabilities of 32 keys: [row block][part]
    __shared__ float lm[WAVES][RT], ll[WAVES][RT];
    const int sp = blockIdx.x, g = blockIdx.y;
    int item;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15;
    const int b = longest_first(a, RT, blockIdx.z, item);
    if (b < 0 || item < 0 || item >= a.items) return;
    const int c0 = a.cu[b], n = min(a.cu[b + 1], a.T) - c0, r0 = (item - first_item(a.cu, b, a.grp, RT)) * RT;
    const int rows = n * a.grp;
    if (c0 < 0 || r0 < 0 || r0 >= rows) return;
    const int past = a.past[b], cap = a.mb * PG;
    auto visible = [&](int t) { return past < 0 ? 0 : (int) min((long long) past + t + 1, (long long) cap); };
    const int kvalid = visible(n - 1), kmax = visible((min(r0 + RT, rows) - 1) / a.grp);
    const int tiles = (kmax + PG - 1) / PG, per = (tiles + a.nsplit - 1) / a.nsplit;
    const int k0 = min(sp * per, tiles) * PG, k1 = min(min((sp + 1) * per, tiles) * PG, kmax);
    const int all = min(visible(r0 / a.grp), k1);  // keys that every row of the item sees

    // through the scalar cache: a vector load's wait would wait for every key block in flight, too
    typedef const __attribute__((address_space(4))) int32_t *scalar_i32;
    const scalar_i32 table = (scalar_i32) (uintptr_t) (a.table + (size_t) b * a.mb);
    const size_t stride = (size_t) a.nkv * HEAD_BYTES;
    const uint8_t *cache = a.cache + (size_t) g * HEAD_BYTES;
    auto page_of = [&](int k) { return k < k1 ? table[k / PG] : -1; };
    auto ok = [&](int page) { return page >= 0 && page < a.npages; };
    auto base_of = [&](int page) { return cache + (ok(page) ? page : 0) * stride; };  // in bounds; the block is passed over
    int page[2] = {page_of(k0), page_of(k0 + PG)}, next[2] = {page_of(k0 + STEP), page_of(k0 + STEP + PG)};
    v4u k[2][2], v[WAVES], vs[WAVES];  // keys of the wave's 32: [16][half of the row]; its dims of each 32 keys
    uint32_t ks;
    auto load_k = [&](const int (&pg)[2]) __attribute__((always_inline)) {
        const uint8_t *p = base_of(wave < 2 ? pg[0] : pg[1]);
        const int kk = wave & 1;
#pragma unroll
        for (int hb = 0; hb < 2; ++hb)
#pragma unroll
            for (int u = 0; u < 2; ++u) k[hb][u] = *reinterpret_cast<const v4u *>(p + kk * 4096 + (hb * 2 + u) * 1024 + lane * 16);
        ks = *reinterpret_cast<const uint32_t *>(p + KS + kk * 256 + lane * 4);
    };
    auto load_v = [&](int c, const int (&pg)[2]) __attribute__((always_inline)) {
        const uint8_t *p = base_of(pg[c / 2]);
        v[c] = *reinterpret_cast<const v4u *>(p + VC + c % 2 * 4096 + wave * 1024 + lane * 16);
        vs[c] = *reinterpret_cast<const v4u *>(p + VS + c % 2 * 256 + wave * 16 + (lane >> 4) * 64);
    };
    // in the order of the loop's requests: its waits count them as both ways into it have them
    load_k(page);
#pragma unroll
    for (int c = 0; c < WAVES; ++c) {
        __builtin_amdgcn_sched_barrier(0);
        load_v(c, page);
    }
    __builtin_amdgcn_sched_barrier(0);
    // the item's query operands into the LDS
    const v4u *Q = reinterpret_cast<const v4u *>(a.Q + ((size_t) g * a.items + item) * item_bytes<RT>);
    for (int i = threadIdx.x; i < NRB * QBLK / 16; i += WAVES * 64) reinterpret_cast<v4u *>(lq)[i] = Q[i];
    __syncthreads();
    v2u qs[NRB][2];
    int lim[NRB];
    v4f o[NRB][2][2];  // [32 dims of the wave's 64][even, odd]: lane = row, dims 8 (lane / 16) + 2 i
    Softmax sm[NRB];
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NRB; ++j) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            qs[j][u] = *reinterpret_cast<const v2u *>(lq + j * QBLK + 2 * NPART * FRAG + u * 512 + lane * 8);
            o[j][u][0] = o[j][u][1] = zero;
        }
        lim[j] = min(visible(min((r0 + 16 * j + col) / a.grp, n - 1)), k1);
    }
    auto operand = [&](int at) __attribute__((always_inline)) {
        const v4u qa = *reinterpret_cast<const v4u *>(lq + at + lane * 16);
        const v2u qb = *reinterpret_cast<const v2u *>(lq + at + 1024 + lane * 8);
        return v6u{qa[0], qa[1], qa[2], qa[3], qb[0], qb[1]};
    };
    for (int at = k0; at < k1; at += STEP) {
        const int kb = at + 32 * wave;  // the wave's first key
        const int own = wave < 2 ? page[0] : page[1];
        const bool in = kb < k1 && ok(own);  // a block outside the cache counts for nothing
        if (kb < k1 && !in && lane == 0) atomicOr(a.status, FN_STATUS_PAGE);
        // scores, the small parts of the queries first
        float S[NRB][8];
        {
            v4f acc[2][NRB];
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int j = 0; j < NRB; ++j) acc[hb][j] = zero;
#define FN_KV4_PART(U, P)                                                                                            \
    do {                                                                                                            \
        _Pragma("unroll") for (int j = 0; j < NRB; ++j) {                                                            \
            const v6u q = operand(j * QBLK + ((U) * NPART + (P)) * FRAG);                                            \
            acc[0][j] = mma_k<(U), (P) % 4>(k[0][U], (int) ks, q, (int) qs[j][U][(P) / 4], acc[0][j]);               \
            acc[1][j] = mma_k<2 + (U), (P) % 4>(k[1][U], (int) ks, q, (int) qs[j][U][(P) / 4], acc[1][j]);           \
        }                                                                                                           \
    } while (0)
            FN_KV4_PART(0, 4);
            FN_KV4_PART(1, 4);
            FN_KV4_PART(0, 3);
            FN_KV4_PART(1, 3);
            FN_KV4_PART(0, 2);
            FN_KV4_PART(1, 2);
            FN_KV4_PART(0, 1);
            FN_KV4_PART(1, 1);
            FN_KV4_PART(0, 0);
            FN_KV4_PART(1, 0);
#undef FN_KV4_PART
            // (here, and not behind the branches of the first row block, where the compiler would move half of the products)
#pragma unroll
            for (int j = 0; j < NRB; ++j) asm volatile("" : "+v"(acc[0][j]), "+v"(acc[1][j]));
#pragma unroll
            for (int j = 0; j < NRB; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) S[j][i] = acc[i / 4][j][i % 4];
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        const bool whole = in && kb + 32 <= all;
        const int key = kb + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < NRB; ++j) {
            const float mx = whole ? Softmax::largest<false>(S[j], key, lim[j]) : Softmax::largest<true>(S[j], key, in ? lim[j] : 0);
            if (lane < 16) lm[wave][16 * j + lane] = mx;
        }
        lds_barrier();  // the largest scores are there, and the last probabilities have been read
        bool moved = false;
        float corr[NRB];
#pragma unroll
        for (int j = 0; j < NRB; ++j) {
            float p[8];
            const float mx = fmaxf(fmaxf(lm[0][16 * j + col], lm[1][16 * j + col]), fmaxf(lm[2][16 * j + col], lm[3][16 * j + col]));
            corr[j] = whole ? sm[j].template step<false>(S[j], mx, p) : sm[j].template step<true>(S[j], mx, p);
            moved |= corr[j] != 1.0f;
            v4u parts[3];  // three bf16 parts of each
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float f = p[2 * i], h = p[2 * i + 1];
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    const uint32_t w = bf16_pair(f, h);
                    parts[q][i] = w;
                    f -= __uint_as_float(w << 16);
                    h -= __uint_as_float(w & 0xffff0000u);
                }
            }
#pragma unroll
            for (int q = 0; q < 3; ++q) lp[wave][j][q][lane] = parts[q];
        }
        if (__ballot(moved)) {
#pragma unroll
            for (int j = 0; j < NRB; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) o[j][t / 2][t % 2] *= corr[j];
        }
        if (at + STEP > k1 || !ok(page[0]) || !ok(page[1])) {  // rows of pages that hold no token: their scales may be anything
#pragma unroll
            for (int c = 0; c < WAVES; ++c) {
                const int first = at + 32 * c + 4 * (lane >> 4), end = at + 32 * c < k1 && ok(page[c / 2]) ? kvalid : 0;
                uint32_t keep[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) keep[j / 4] |= first + 16 * (j / 4) + j % 4 < end ? 0xffu << (8 * (j % 4)) : 0u;
                vs[c] &= v4u{keep[0], keep[1], keep[0], keep[1]};
            }
        }
        // o += V^T P^T, 32 keys and 32 dims at a time; the next ones are converted between the products
        v4u ve[2], vo[2];  // one dim of two keys
        auto values = [&](int s) __attribute__((always_inline)) {
            const int c = s / 2;
            uint32_t w[8];
            values_of(v[c], vs[c], s % 2, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ve[s & 1][i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
                vo[s & 1][i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
            }
        };
        values(0);
        lds_barrier();  // the probabilities are there
        v4u P[2][NRB][3];
        auto load_p = [&](int c) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NRB; ++j)
#pragma unroll
                for (int q = 0; q < 3; ++q) P[c & 1][j][q] = lp[c][j][q][lane];
        };
        load_p(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2 * WAVES; ++s) {
            const int c = s / 2, t = s % 2;
            if (s + 1 < 2 * WAVES) values(s + 1);
            if (t == 0 && c + 1 < WAVES) load_p(c + 1);
            if (t == 1 || s + 1 == 2 * WAVES) load_v(c, next);
#pragma unroll
            for (int q = 2; q >= 0; --q)
#pragma unroll
                for (int j = 0; j < NRB; ++j) {
                    o[j][t][0] = mma_v(ve[s & 1], P[c & 1][j][q], o[j][t][0]);
                    o[j][t][1] = mma_v(vo[s & 1], P[c & 1][j][q], o[j][t][1]);
                }
#pragma unroll
            for (int i = 0; i < 6 * NRB; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 4 / NRB, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            page[i] = next[i];
            next[i] = page_of(at + 2 * STEP + PG * i);
        }
    }
    // The rows' sums; the references are the same in all waves.  A wave passes its 64 dims of 16 rows at a time through its
    // part of the query operands' LDS, so that 16 lanes load and store a row's 256 bytes.
    constexpr int MS = 64 + 4;
    float *mo = reinterpret_cast<float *>(lq) + wave * 16 * MS;
    const int dim = 64 * wave + 4 * col;
    size_t at[NRB][4];   // the lane's rows 16 j + 4 k + lane / 16: row of og
    float4 z[NRB][4];    // and their gates, all requested before the first store
#pragma unroll
    for (int j = 0; j < NRB; ++j) {
        const float ls = sum_quarters(sm[j].l);
        if (lane < 16) ll[wave][16 * j + lane] = ls;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = min(r0 + 16 * j + 4 * k + (lane >> 4), rows - 1), tok = r / a.grp;
            at[j][k] = (size_t) (c0 + tok) * a.nq + g * a.grp + (r - tok * a.grp);
            if (a.nsplit == 1) z[j][k] = *reinterpret_cast<const float4 *>(a.qg + (at[j][k] * 2 + 1) * HD + dim);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NRB; ++j) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const v4f e = o[j][u / 2][0], f = o[j][u / 2][1];
            const int i = u % 2 * 2;
            *reinterpret_cast<float4 *>(mo + col * MS + 32 * (u / 2) + 8 * (lane >> 4) + 4 * (u % 2)) =
                make_float4(e[i], f[i], e[i + 1], f[i + 1]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int row = 16 * j + 4 * k + (lane >> 4);
            const float4 x = *reinterpret_cast<const float4 *>(mo + (row - 16 * j) * MS + 4 * col);
            if (r0 + row >= rows) continue;
            const float L = (ll[0][row] + ll[1][row]) + (ll[2][row] + ll[3][row]);
            if (a.nsplit == 1) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // a row that sees no key: zeros
                const float4 y = z[j][k];
                *reinterpret_cast<float4 *>(a.og + at[j][k] * HD + dim) =
                    make_float4(x.x * inv * gate_of(y.x), x.y * inv * gate_of(y.y), x.z * inv * gate_of(y.z),
                                x.w * inv * gate_of(y.w));
            } else {
                const size_t part = (((size_t) item * a.nkv + g) * a.nsplit + sp) * RT + row;
                *reinterpret_cast<float4 *>(a.part_o + part * HD + dim) = x;
                if (dim == 0) a.part_ml[2 * part + 1] = L;
            }
        }
        if (a.nsplit > 1 && wave == 0 && lane < 16 && r0 + 16 * j + lane < rows)
            a.part_ml[2 * ((((size_t) item * a.nkv + g) * a.nsplit + sp) * RT + 16 * j + lane)] = sm[j].m;
    }
}

// grid (items RT, nkv), four waves a row, lane = 4 dims: the splits of a row joined, and the gate.  A chain of latencies:
// 2.8 us for 32 splits (3.6 us with the sums requested behind the references).
template <int RT>
__global__ void __launch_bounds__(256) k_kv4_combine(const Kv4Args a) {
    __shared__ float4 part[WAVES][HD / 4];
    __shared__ float pl[WAVES];
    const int item = blockIdx.x / RT, g = blockIdx.y, row = blockIdx.x % RT, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = request_of(a.cu, a.B, item, a.grp, RT);
    const int c0 = a.cu[b], n = min(a.cu[b + 1], a.T) - c0, r = (item - first_item(a.cu, b, a.grp, RT)) * RT + row;
    if (c0 < 0 || r < 0 || r >= n * a.grp) return;
    // the gate and the sums of the wave's first splits are requested before the references are there
    const int t = r / a.grp;
    const size_t at = (size_t) (c0 + t) * a.nq + g * a.grp + (r - t * a.grp);
    const float4 z = reinterpret_cast<const float4 *>(a.qg + (at * 2 + 1) * HD)[lane];
    const size_t at0 = ((size_t) item * a.nkv + g) * a.nsplit * RT + row;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml);
    constexpr int AHEAD = 8;
    float4 po[AHEAD];
    float2 pm[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        if (wave + i * WAVES >= a.nsplit) break;
        const size_t p = at0 + (size_t) (wave + i * WAVES) * RT;
        pm[i] = ml[p];
        po[i] = reinterpret_cast<const float4 *>(a.part_o + p * HD)[lane];
    }
    float M = -INFINITY;
    for (int s = lane; s < a.nsplit; s += 64) M = fmaxf(M, ml[at0 + (size_t) s * RT].x);
    M = wave_max(M);
    float L = 0.0f;
    float4 o = f4(0.0f);
    auto join = [&](const float2 &x, const float4 &y) {
        const float f = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - M);
        L = fmaf(x.y, f, L);
        o = add_scaled(o, y, f);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (wave + i * WAVES < a.nsplit) join(pm[i], po[i]);
#pragma unroll 4
    for (int s = wave + AHEAD * WAVES; s < a.nsplit; s += WAVES) {
        const size_t p = at0 + (size_t) s * RT;
        join(ml[p], reinterpret_cast<const float4 *>(a.part_o + p * HD)[lane]);
    }
    part[wave][lane] = o;
    if (lane == 0) pl[wave] = L;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        o = add_scaled(o, part[w][lane], 1.0f);
        L += pl[w];
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    reinterpret_cast<float4 *>(a.og + at * HD)[lane] = make_float4(
        o.x * inv * gate_of(z.x), o.y * inv * gate_of(z.y), o.z * inv * gate_of(z.z), o.w * inv * gate_of(z.w));
}

template <int RT> void launch(const Kv4Args &a, hipStream_t st) {
    const int octets = (a.nq + 7) / 8, groups = (2 * a.nkv + octets + WAVES - 1) / WAVES;
    if ((long long) a.T * groups <= 2 * device_cus()) {  // one round
        hipLaunchKernelGGL((k_kv4_prep<RT, PREP_ALL>), dim3(a.T, groups), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((k_kv4_prep<8, PREP_KEYS>), dim3(a.T), dim3(64 * std::min(2 * a.nkv, WAVES)), 0, st, a);
        hipLaunchKernelGGL((k_kv4_prep<RT, PREP_QUERIES>), dim3(a.T), dim3(64 * std::min(octets, WAVES)), 0, st, a);
    }
    hipLaunchKernelGGL(RT == 8 ? k_attn_kv4 : k_attn_kv4_rows, dim3(a.nsplit, a.nkv, a.items), dim3(WAVES * 64), 0, st, a);
    if (a.nsplit > 1) hipLaunchKernelGGL(k_kv4_combine<RT>, dim3(a.items * RT, a.nkv), dim3(256), 0, st, a);
}

// Query rows an item.  A request of up to 24 rows is cheaper as up to three items of eight, which read its keys one behind
// the other, than as one of 32 in which rows are left empty.  8 query heads a kv head, 8k keys, us with 8 | 32 rows an item:
// 16 requests of 1, 2, 3, 4 tokens 51 | 56, 51 | 56, 65 | 58, 72 | 62; 64 requests of 1, 2, 3 tokens 131 | 146, 158 | 184,
// 172 | 182; 24 requests, 4 kv heads, 20k keys, of 1, 2, 3 tokens 195 | 218, 197 | 217, 218 | 299.  (16 rows an item won
// by 9% at one of these and lost at the others.)
int item_rows(int B, int T, int grp) { return (long long) T * grp <= 24ll * B ? 8 : 32; }
size_t query_bytes(int rt) { return rt == 8 ? item_bytes<8> : item_bytes<32>; }

}  // namespace

size_t kv4_work_bytes(int B, int T, int nq, int nkv, int hd, int nsplit) {
    const int grp = nq / nkv, rt = item_rows(B, T, grp);
    const size_t n = item_count(B, T, grp, rt) * nkv;
    return n * query_bytes(rt) + (nsplit > 1 ? n * rt * nsplit * (HD + 2) * sizeof(float) : 0);
}

int kv4_pick_nsplit(int B, int T, int nq, int nkv, int ctx) {
    const int grp = nq / nkv, rt = item_rows(B, T, grp);
    // One round of workgroups, two a CU (k_attn_kv4 has room for three; what that gives was measured for one request only,
    // below): items of an average request times requests.  All requests of a call get as many splits, so a long one among
    // short ones or beside prompts is the call's time.
    const long long avg = ((long long) T * grp + B - 1) / B, groups = std::max(1ll, (avg + rt - 1) / rt) * B * nkv;
    const long long want = std::max(1ll, 2ll * device_cus() / groups);
    // A split costs a row of sums that is written and read again, so the time is about u keys / nsplit + w nsplit, least at
    // a multiple of sqrt(keys).  One token, 2 kv heads, us at 16, 32, 64, 128, 256 splits: 4k keys 25.0, 24.1, 24.7, 27.0,
    // 32.6; 32k keys 43.4, 34.4, 30.6, 32.2, 38.9; 100k keys 86.5, 58.4, 45.4, 45.0, 52.1.
    const int most = std::max(1, (int) (std::sqrt((double) std::max(ctx, 1)) * 0.5));
    return (int) std::min<long long>(want, most);
}

int kv4_attn_launch(const Kv4Attn &p, hipStream_t st) {
    if (p.B < 1 || p.T < 1 || p.nq < 1 || p.nkv < 1) FN_FAIL("attn_kv4: B, T, nq and nkv must be >= 1");
    if (p.hd != HD) FN_FAIL("attn_kv4: only head_dim 256 is built");
    if (p.nq % p.nkv) FN_FAIL("attn_kv4: nq must be a multiple of nkv");
    if (p.nrot < 0 || p.nrot > MAXROT || (p.nrot & 1)) FN_FAIL("attn_kv4: nrot must be even and <= 128");
    if (!(p.theta >= 1.0f)) FN_FAIL("attn_kv4: theta must be >= 1");
    if (p.nsplit < 1 || p.nsplit > 65535) FN_FAIL("attn_kv4: nsplit must be in 1..65535");
    if (p.max_blocks < 1 || p.max_blocks > 1 << 24) FN_FAIL("attn_kv4: max_blocks must be in 1..16777216");
    if (p.npages < 1 || p.npages > INT_MAX / PG) FN_FAIL("attn_kv4: npages must be in 1..33554431 (slots are 32-bit)");
    if (!p.past || !p.cu || !p.table || !p.slot || !p.seq || !p.qg || !p.k || !p.v || !p.wq || !p.wk || !p.cache ||
        !p.work || !p.og)
        FN_FAIL("attn_kv4: null pointer");
    if (((uintptr_t) p.qg | (uintptr_t) p.k | (uintptr_t) p.v | (uintptr_t) p.wq | (uintptr_t) p.wk | (uintptr_t) p.cache |
         (uintptr_t) p.work | (uintptr_t) p.og) & 15)
        FN_FAIL("attn_kv4: qg, k, v, wq, wk, cache, work and og must be 16-byte aligned");
    const int grp = p.nq / p.nkv, rt = item_rows(p.B, p.T, grp);
    if ((long long) p.T * grp > INT_MAX - 64) FN_FAIL("attn_kv4: too many query rows");
    const size_t items = item_count(p.B, p.T, grp, rt);
    if (p.nkv > 65535 || items > 65535) FN_FAIL("attn_kv4: batch too large (at most 65535 requests and pieces of their query rows)");
    if (p.work_bytes < kv4_work_bytes(p.B, p.T, p.nq, p.nkv, p.hd, p.nsplit)) FN_FAIL("attn_kv4: workspace too small");
    Kv4Args a{};
    a.B = p.B; a.T = p.T; a.nq = p.nq; a.nkv = p.nkv; a.grp = grp; a.mb = p.max_blocks; a.npages = p.npages;
    a.nsplit = p.nsplit; a.nrot = p.nrot; a.items = (int) items; a.eps = p.eps; a.past = p.past; a.cu = p.cu;
    a.table = p.table; a.slot = p.slot; a.seq = p.seq; a.qg = p.qg; a.k = p.k; a.v = p.v; a.wq = p.wq; a.wk = p.wk;
    a.cache = p.cache; a.og = p.og;
    if (status_word(&a.status)) return -1;
    a.Q = static_cast<uint8_t *>(p.work);
    a.part_o = reinterpret_cast<float *>(a.Q + items * p.nkv * query_bytes(rt));
    a.part_ml = a.part_o + items * p.nkv * rt * p.nsplit * HD;
    for (int i = 0; i < p.nrot / 2; ++i) a.freq[i] = std::pow((double) p.theta, -(2.0 * i) / p.nrot);
    if (rt == 8) launch<8>(a, st);
    else launch<32>(a, st);
    FN_CK(hipGetLastError());
    return 0;
}

}  // namespace fn
