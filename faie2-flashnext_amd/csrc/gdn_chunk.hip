// The gated delta rule over whole prompts of a packed batch, chunk by chunk.
//
// A token does S <- g S, d = beta (v - S^T k), S <- S + k d^T, o = S^T q / sqrt(dk).  Within a chunk of 64 tokens, with
// G_i the sum of the log decays up to token i and S the state before the chunk, the updates d (rows of U) solve a
// unit lower triangular system:
//   U = M X,  X_i = beta_i (v_i - e^G_i S^T k_i),  M = (I + A)^-1,  A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i)
//   o_i = (e^G_i S^T q_i + sum_(j <= i) e^(G_i - G_j) q_i.k_j u_j) / sqrt(dk)
//   S' = e^G_63 S + sum_j e^(G_63 - G_j) k_j u_j^T
// so that only S -> S' is sequential, in steps of 64 tokens.  Two launches:
//   k_chunk_intra, one workgroup a (chunk, key head), everything that does not need S: M and P_ij = e^(G_i - G_j) q_i.k_j of
//     each value head that reads the key head, and q, k as matrix operands;
//   k_chunk_scan, one workgroup a (request, value head, 32 columns of S), which walks the request's chunks with its
//     columns of S in registers: five small products a chunk.
// Products: an fp32 operand is two f16 values (hi and lo, 11 bits each) under a power-of-two scale, and a product is hi
// hi + hi lo + lo hi on v_mfma_f32_16x16x32_f16: what is left out is 2^-22 of a product at the worst and 2^-24 in the
// mean, in half the instructions of six bf16 products and a fifth of the time of fp32 ones.  f16's range is met by
// scales: one a row of q, k, M and P (they are factors of output rows, folded into the gates' factors), one a column
// and 32 rows for S (from its largest value there), and bounds for X and U: |X| <= max beta max|v| + max(beta e^G |k|)
// sqrt(128) max|S| in its column, |U| <= (largest row sum of |M|) of that.  A bound too large by a factor of up to 2^15
// costs no bit of a value as large as the column's largest: f16 reaches 2^-24 and lo goes down to there.
// Decays: G is summed in 64 bits, because differences of far sums are taken; all exponents are then <= 0 for decays < 1.
#include "serve.cuh"

namespace fn {

namespace {

constexpr int D = 128;                        // dk = dv
constexpr int C = 64;                         // tokens a chunk
constexpr int RS = D + 4;                     // floats a row of q, k in the LDS
constexpr int AS = C + 4, MS = 20;            // floats a row of A, of the diagonal blocks of M
constexpr int FRAG = 1024;                    // an operand of one 16 x 16 x 32 product: 16 bytes a lane
constexpr int KF = 0, QF = 32 * FRAG, KT = 64 * FRAG, KEY_BYTES = 96 * FRAG;    // a (chunk, key head)
constexpr int MF = 0, PF = 16 * FRAG, GATES = 32 * FRAG, HEAD_BYTES = 34 * FRAG;  // a (chunk, value head)
// GATES: [6][64] floats beta, beta e^G 2^ek, e^G 2^eq / sqrt(dk), e^(G63 - G) 2^ek, 2^ep / sqrt(dk), 2^em; then scalars
constexpr int G_BETA = 0, G_KS = 64, G_QS = 128, G_UP = 192, G_P = 256, G_M = 320, G_SC = 384;
constexpr float RSQRT_D = 0.08838834764831845f;

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

struct ChunkArgs {
    GdnChunk p;
    uint8_t *keys, *heads;  // the two parts of the workspace
    int items;
};

__device__ __forceinline__ v4f mma(const v4u &a, const v4u &b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// Two values as f16 hi and lo pairs.  (The values are taken as they are in fp32: a product folded into the conversion
// is rounded once for the hi that is kept and twice for the one that is subtracted, and where the two differ lo is
// wrong by a unit of hi: one element in some thousands, by 2^-11.)
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    asm("" : "+v"(a), "+v"(b));
    const h2 h = {(_Float16) a, (_Float16) b};
    const h2 l = {(_Float16) (a - (float) h.x), (_Float16) (b - (float) h.y)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}
__device__ __forceinline__ void split8(const float (&x)[8], v4u &hi, v4u &lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h, l;
        split2(x[2 * i], x[2 * i + 1], h, l);
        hi[i] = h;
        lo[i] = l;
    }
}
// exponent k of 2^k <= x < 2^(k + 1); 14 - k and k - 14 as powers of two: x up to 2^15 (f16: 65504), and back
__device__ __forceinline__ int exp_of(float x) { return x > 0.0f ? max(-100, min(126, (int) (__float_as_uint(x) >> 23) - 127)) : 0; }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t) (e + 127) << 23); }

__device__ __forceinline__ float silu_(float x) { return x * __builtin_amdgcn_rcpf(1.0f + expf(-x)); }

__device__ __forceinline__ float4 lds4(const float *p) { return *reinterpret_cast<const float4 *>(p); }

template <bool BLOCK>
__global__ void __launch_bounds__(256, 2) k_chunk_intra(const ChunkArgs a) {
    __shared__ __align__(16) float rows[2][C * RS];            // q, k; later K operands | A, diagonal blocks of M
    __shared__ float mul[2][C], back[2][C], kn[C], bet[C];     // row factors to f16's range and back, |k|, beta
    __shared__ double G[C];
    const GdnChunk &p = a.p;
    const int item = blockIdx.x, kh = blockIdx.y;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q4 = lane >> 4;
    const int b = request_of(p.cu, p.B, item, 1, C);
    const int c0 = p.cu[b], t0 = (item - first_item(p.cu, b, 1, C)) * C, n = min(C, min(p.cu[b + 1], p.T) - c0 - t0);
    if (c0 < 0 || t0 < 0 || n <= 0) return;
    const size_t row0 = (size_t) c0 + t0;
    uint8_t *kd = a.keys + ((size_t) item * p.nkh + kh) * KEY_BYTES;

    // 1. q, k rows
    if (BLOCK) {
        const int ch = tid & (D - 1), part = tid >> 7, Cc = 2 * p.nkh * D + p.nvh * D, col = (part * p.nkh + kh) * D + ch;
        const float4 w = *reinterpret_cast<const float4 *>(p.conv_w + 4 * col);
        const float *x = p.qkv + row0 * Cc + col;
        float h[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int t = t0 - 3 + j;
            h[j] = t >= 0 ? x[(ptrdiff_t) (j - 3) * Cc]
                          : p.conv_ring[((size_t) b * p.ring + ((p.pos[b] + t) & (p.ring - 1))) * Cc + col];
        }
        for (int t = 0; t < C; t += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = t + i < n ? x[(size_t) (t + i) * Cc] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float y = w.x * h[0];
                y = fmaf(w.y, h[1], y);
                y = fmaf(w.z, h[2], y);
                y = fmaf(w.w, v[i], y);
                rows[part][(t + i) * RS + ch] = t + i < n ? silu_(y) : 0.0f;
                h[0] = h[1];
                h[1] = h[2];
                h[2] = v[i];
            }
        }
    } else {
        for (int i = tid; i < 2 * C * (D / 4); i += 256) {
            const int part = i >> 11, t = (i >> 5) & (C - 1), d = (i & 31) * 4;
            const float *src = (part ? p.k : p.q) + ((row0 + t) * p.nkh + kh) * D + d;
            *reinterpret_cast<float4 *>(&rows[part][t * RS + d]) = t < n ? *reinterpret_cast<const float4 *>(src) : f4(0.0f);
        }
    }
    __syncthreads();
    {  // the row's norm and largest value, by two threads
        const int part = tid >> 7, t = (tid >> 1) & (C - 1);
        const float *x = &rows[part][t * RS + (tid & 1) * (D / 2)];
        float ss = 0.0f, am = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const float4 v = lds4(x + 4 * i);
            ss += sumsq4(v);
            am = fmaxf(am, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        ss += __shfl_xor(ss, 1);
        am = fmaxf(am, __shfl_xor(am, 1));
        const float nr = BLOCK ? rsqrtf(ss + 1e-6f) : 1.0f;
        const int e = exp_of(am * nr) - 14;
        if ((tid & 1) == 0) {
            mul[part][t] = nr * pow2(-e);
            back[part][t] = pow2(e);
            if (part) kn[t] = sqrtf(ss) * nr;
        }
    }
    __syncthreads();
    // 2. operands.  Row operand (q, k): lane = row 16 wave + l%16, slot j of step s = dim 32 s + 16 (j / 4) + 4 (l / 16) + j % 4
    v4u qh[4], ql[4], kh_[4], kl[4];
    {
        const int t = 16 * wave + r;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const float m = mul[part][t];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float4 x = lds4(&rows[part][t * RS + 32 * s + 4 * q4]), y = lds4(&rows[part][t * RS + 32 * s + 16 + 4 * q4]);
                const float v[8] = {x.x * m, x.y * m, x.z * m, x.w * m, y.x * m, y.y * m, y.z * m, y.w * m};
                v4u hi, lo;
                split8(v, hi, lo);
                uint8_t *d = kd + (part ? KF : QF) + ((wave * 4 + s) * 2) * FRAG + lane * 16;
                *reinterpret_cast<v4u *>(d) = hi;
                *reinterpret_cast<v4u *>(d + FRAG) = lo;
                if (part) kh_[s] = hi, kl[s] = lo;
                else qh[s] = hi, ql[s] = lo;
            }
        }
        // Column operand (k^T): lane = dim 32 wave + 16 c + l%16, slot j of step s = token 32 s + 16 (j / 4) + 4 (l / 16) + j % 4
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int u = 32 * s + 16 * (j / 4) + 4 * q4 + j % 4;
                    v[j] = rows[1][u * RS + 32 * wave + 16 * c + r] * mul[1][u];
                }
                v4u hi, lo;
                split8(v, hi, lo);
                uint8_t *d = kd + KT + (((wave * 2 + c) * 2 + s) * 2) * FRAG + lane * 16;
                *reinterpret_cast<v4u *>(d) = hi;
                *reinterpret_cast<v4u *>(d + FRAG) = lo;
            }
    }
    __syncthreads();
    v4u *kop = reinterpret_cast<v4u *>(rows[0]);  // [tile][step][hi, lo][lane]
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        kop[((wave * 4 + s) * 2) * 64 + lane] = kh_[s];
        kop[((wave * 4 + s) * 2 + 1) * 64 + lane] = kl[s];
    }
    __syncthreads();
    // 3. k_j.k_i and k_j.q_i of the wave's 16 rows i (lane: i = 16 wave + l%16, j = 16 tile + 4 (l / 16) + e)
    v4f kk[4], qk[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk[j] = qk[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (j <= wave) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const v4u h = kop[((j * 4 + s) * 2) * 64 + lane], l = kop[((j * 4 + s) * 2 + 1) * 64 + lane];
                kk[j] = mma(h, kl[s], kk[j]);
                qk[j] = mma(h, ql[s], qk[j]);
                kk[j] = mma(l, kh_[s], kk[j]);
                qk[j] = mma(l, qh[s], qk[j]);
                kk[j] = mma(h, kh_[s], kk[j]);
                qk[j] = mma(h, qh[s], qk[j]);
            }
            const float4 f = lds4(&back[1][16 * j + 4 * q4]);
            const float fk = back[1][16 * wave + r], fq = back[0][16 * wave + r];
            const float g[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kk[j][e] *= g[e] * fk;
                qk[j][e] *= g[e] * fq;
            }
        }
    }
    // 4. each value head of the key head
    float *A = rows[1], *Md = rows[1] + C * AS;
    const int per = p.nvh / p.nkh;
    for (int hi_ = 0; hi_ < per; ++hi_) {
        const int h = p.head_map == 0 ? kh + hi_ * p.nkh : kh * per + hi_;
        float be = 0.0f, g = 0.0f;
        if (lane < n) {
            const size_t t = row0 + lane;
            if (BLOCK) {
                const float ga = p.ab[t * 2 * p.nvh + h] + p.dt_bias[h];
                be = sigmoidf_(p.ab[t * 2 * p.nvh + p.nvh + h]);
                g = (ga > 20.0f ? ga : log1pf(expf(ga))) * p.ssm_a[h];
            } else {
                be = p.beta[t * p.nvh + h];
                g = p.g[t * p.nvh + h];
            }
        }
        double gs = fmax((double) g, -200.0);  // a decay below e^-200 is 0 in fp32 (and -infinity would cancel to NaN)
        if (g != g) gs = g;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double y = __shfl_up(gs, d);
            if (lane >= d) gs += y;
        }
        __syncthreads();  // the last head's A, Md, G and beta have been read (and K's operands)
        if (wave == 0) {
            G[lane] = gs;
            bet[lane] = be;
        }
        uint8_t *hd = a.heads + ((size_t) item * p.nvh + h) * HEAD_BYTES;
        float *gd = reinterpret_cast<float *>(hd + GATES);
        if (wave == 0) {
            const double g63 = __shfl(gs, 63);
            const float eg = expf((float) gs), up = expf((float) (g63 - gs)) * back[1][lane];
            gd[G_BETA + lane] = be;
            gd[G_KS + lane] = be * eg * back[1][lane];
            gd[G_QS + lane] = eg * back[0][lane] * RSQRT_D;
            gd[G_UP + lane] = up;
            const float bb = wave_max(fabsf(be)), bk = wave_max(fabsf(be) * eg * kn[lane]), um = wave_max(up);
            if (lane == 0) {
                gd[G_SC] = bb;
                gd[G_SC + 1] = bk * 11.3138f;  // sqrt(128), rounded up
                gd[G_SC + 2] = um;
                gd[G_SC + 3] = expf((float) g63);
            }
        }
        __syncthreads();
        const double gi = G[16 * wave + r];
        const float bi = bet[16 * wave + r];
        float pv[4][4], pm = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float av[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int jt = 16 * j + 4 * q4 + e, it = 16 * wave + r;
                const float dec = j <= wave && jt <= it ? expf((float) (gi - G[jt])) : 0.0f;
                av[e] = j <= wave && jt < it ? bi * dec * kk[j][e] : 0.0f;
                pv[j][e] = j <= wave && jt <= it ? dec * qk[j][e] : 0.0f;
                pm = fmaxf(pm, fabsf(pv[j][e]));
            }
            if (j <= wave)
                *reinterpret_cast<float4 *>(A + (16 * wave + r) * AS + 16 * j + 4 * q4) = make_float4(av[0], av[1], av[2], av[3]);
        }
        {  // P's operand
            pm = max_quarters(pm);
            const int e = exp_of(pm) - 14;
            const float m = pow2(-e);
            if (q4 == 0) gd[G_P + 16 * wave + r] = pow2(e) * RSQRT_D;
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (2 * s <= wave) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = pv[2 * s + j / 4][j % 4] * m;
                    v4u hi, lo;
                    split8(v, hi, lo);
                    uint8_t *d = hd + PF + ((wave * 2 + s) * 2) * FRAG + lane * 16;
                    *reinterpret_cast<v4u *>(d) = hi;
                    *reinterpret_cast<v4u *>(d + FRAG) = lo;
                }
        }
        __syncthreads();
        {  // the inverse of the wave's diagonal block, lane = column l%16, by substitution
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s = i == r ? 1.0f : 0.0f;
                const float *ar = A + (16 * wave + i) * AS + 16 * wave;
#pragma unroll
                for (int j = 0; j < i; ++j) s = fmaf(-ar[j], x[j], s);
                x[i] = s;
            }
            if (q4 == 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) Md[(16 * wave + i) * MS + r] = x[i];
            }
        }
        __syncthreads();
        // the wave's block row of M, from the diagonal leftwards: M_wj = -(sum_(k > j) M_wk A_kj) M_jj, as transposes, whose
        // products leave a lane with row l%16 and columns 4 (l / 16) + e: the layout they are needed in next
        v4f mt[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) mt[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        {
            const float4 f = lds4(Md + (16 * wave + r) * MS + 4 * q4);
            const v4f dg = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j == wave) mt[j] = dg;
        }
#pragma unroll
        for (int j = 2; j >= 0; --j) {
            if (j >= wave) continue;
            v4f t = {0.0f, 0.0f, 0.0f, 0.0f}, o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = j + 1; k < 4; ++k)
                if (k <= wave) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(A[(16 * k + 4 * q4 + e) * AS + 16 * j + r], mt[k][e], t, 0, 0, 0);
                }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o = __builtin_amdgcn_mfma_f32_16x16x4f32(Md[(16 * j + 4 * q4 + e) * MS + r], t[e], o, 0, 0, 0);
            mt[j] = -o;
        }
        {  // M's operand
            float am = 0.0f, sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    am = fmaxf(am, fabsf(mt[j][e]));
                    sum += fabsf(mt[j][e]);
                }
            am = max_quarters(am);
            sum = row_max(sum_quarters(sum));
            const int e = exp_of(am) - 14;
            const float m = pow2(-e);
            if (q4 == 0) gd[G_M + 16 * wave + r] = pow2(e);
            if (lane == 0) gd[G_SC + 4 + wave] = sum;
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (2 * s <= wave) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = mt[2 * s + j / 4][j % 4] * m;
                    v4u hi, lo;
                    split8(v, hi, lo);
                    uint8_t *d = hd + MF + ((wave * 2 + s) * 2) * FRAG + lane * 16;
                    *reinterpret_cast<v4u *>(d) = hi;
                    *reinterpret_cast<v4u *>(d + FRAG) = lo;
                }
        }
    }
}

// grid (nvh, D / (16 NC), B), four waves.  Wave w owns tokens 16 w .. + 15 of X, U and o, and rows 32 w .. + 31 of S; lane = column
// l%16 of each of NC column tiles, rows 4 (l / 16) + e.  That is also the layout of an operand's slots, so what a wave
// computes it splits and writes to the LDS as it stands, and the others read whole operands: S, X and U meet there once
// a chunk each, with one barrier.
template <bool BLOCK, int NC>
__global__ void __launch_bounds__(256, 1) k_chunk_scan(const ChunkArgs a) {
    __shared__ v4u Sop[4][NC][2][64];                   // [32 rows][column tile][hi, lo][lane]
    __shared__ v4u Xop[2][NC][2][64], Uop[2][NC][2][64], Wop[2][NC][2][64];  // [32 tokens]...: X, U, e^(G63 - G) U
    __shared__ float smax[4][NC][16], sinv[4][NC][16], vmax[4][NC][16];
    const GdnChunk &p = a.p;
    const int h = blockIdx.x, col0 = blockIdx.y * 16 * NC, b = blockIdx.z;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q4 = lane >> 4;
    const int c0 = p.cu[b], len = min(p.cu[b + 1], p.T) - c0;
    if (c0 < 0 || len <= 0) return;
    const int per = p.nvh / p.nkh, kh = p.head_map == 0 ? h % p.nkh : h / per;
    const int item0 = first_item(p.cu, b, 1, C), chunks = (len + C - 1) / C;
    const int Cc = 2 * p.nkh * D + p.nvh * D;
    float s[NC][2][4];
    float *Sg = p.S + ((size_t) b * p.nvh + h) * D * D + col0 + r;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][c][e] = Sg[(32 * wave + 16 * c + 4 * q4 + e) * D + 16 * n];
    float4 cw[NC];
    if (BLOCK) {
#pragma unroll
        for (int n = 0; n < NC; ++n)
            cw[n] = *reinterpret_cast<const float4 *>(p.conv_w + 4 * (2 * p.nkh * D + h * D + col0 + 16 * n + r));
    }
    v4u kf[4][2], qf[4][2], mf[2][2], pf[2][2], kt[2][2][2];
    float v[NC][7];
    auto key = [&](int i) { return a.keys + ((size_t) (item0 + i) * p.nkh + kh) * KEY_BYTES + lane * 16; };
    auto head = [&](int i) { return a.heads + ((size_t) (item0 + i) * p.nvh + h) * HEAD_BYTES; };
    auto ld = [&](const uint8_t *x) { return *reinterpret_cast<const v4u *>(x); };
    auto load_rows = [&](int i, int at, v4u(&f)[4][2]) {
        const uint8_t *x = key(i) + at + wave * 8 * FRAG;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j / 2][j % 2] = ld(x + j * FRAG);
    };
    auto load_tri = [&](int i, int at, v4u(&f)[2][2]) {
        const uint8_t *x = head(i) + at + wave * 4 * FRAG + lane * 16;
        f[0][0] = ld(x);
        f[0][1] = ld(x + FRAG);
        if (wave >= 2) {
            f[1][0] = ld(x + 2 * FRAG);
            f[1][1] = ld(x + 3 * FRAG);
        }
    };
    auto load_kt = [&](int i) {
        const uint8_t *x = key(i) + KT + wave * 8 * FRAG;
#pragma unroll
        for (int j = 0; j < 8; ++j) kt[j / 4][j / 2 % 2][j % 2] = ld(x + j * FRAG);
    };
    // the chunk's values of the lane's tokens 16 wave + 4 q4 + e; BLOCK: raw inputs from three tokens before
    auto load_v = [&](int i) {
        const int t = i * C + 16 * wave + 4 * q4;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int e = 0; e < (BLOCK ? 7 : 4); ++e) {
                const int u = BLOCK ? t + e - 3 : t + e;
                const int col = (BLOCK ? 2 * p.nkh * D : 0) + h * D + col0 + 16 * n + r;
                v[n][e] = 0.0f;
                if (u < len) {
                    if (!BLOCK) v[n][e] = p.v[(size_t) (c0 + u) * p.nvh * D + col];
                    else if (u >= 0) v[n][e] = p.qkv[(size_t) (c0 + u) * Cc + col];
                    else v[n][e] = p.conv_ring[((size_t) b * p.ring + ((p.pos[b] + u) & (p.ring - 1))) * Cc + col];
                }
            }
    };
    float val[NC][4];
    auto take_v = [&](int i) {  // values, and their largest in the column
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float am = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (BLOCK) {
                    float y = cw[n].x * v[n][e];
                    y = fmaf(cw[n].y, v[n][e + 1], y);
                    y = fmaf(cw[n].z, v[n][e + 2], y);
                    y = fmaf(cw[n].w, v[n][e + 3], y);
                    val[n][e] = i * C + 16 * wave + 4 * q4 + e < len ? silu_(y) : 0.0f;
                } else {
                    val[n][e] = v[n][e];
                }
                am = fmaxf(am, fabsf(val[n][e]));
            }
            am = max_quarters(am);
            if (q4 == 0) vmax[wave][n][r] = am;
        }
    };
    auto put_s = [&]() {
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float am = 0.0f, x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) am = fmaxf(am, fabsf(s[n][j / 4][j % 4]));
            am = max_quarters(am);
            const int e = exp_of(am) - 14;
            const float m = pow2(-e);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[n][j / 4][j % 4] * m;
            split8(x, Sop[wave][n][0][lane], Sop[wave][n][1][lane]);
            if (q4 == 0) {
                smax[wave][n][r] = am;
                sinv[wave][n][r] = pow2(e);
            }
        }
    };
    auto put4 = [&](v4u(&op)[2][NC][2][64], int n, const float (&x)[4], float m) {  // the wave's 16 tokens of an operand
        uint32_t hi[2], lo[2];
        split2(x[0] * m, x[1] * m, hi[0], lo[0]);
        split2(x[2] * m, x[3] * m, hi[1], lo[1]);
        reinterpret_cast<v2u *>(&op[wave / 2][n][0][lane])[wave & 1] = v2u{hi[0], hi[1]};
        reinterpret_cast<v2u *>(&op[wave / 2][n][1][lane])[wave & 1] = v2u{lo[0], lo[1]};
    };
    load_v(0);
    load_rows(0, KF, kf);
    load_rows(0, QF, qf);
    load_tri(0, MF, mf);
    load_kt(0);
    load_tri(0, PF, pf);
    take_v(0);
    put_s();
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < chunks; ++i) {
        const int nx = min(i + 1, chunks - 1);
        const float *gd = reinterpret_cast<const float *>(head(i) + GATES);
        const int tok = 16 * wave + 4 * q4;
        const float4 beta4 = *reinterpret_cast<const float4 *>(gd + G_BETA + tok), ks4 = *reinterpret_cast<const float4 *>(gd + G_KS + tok);
        const float4 qs4 = *reinterpret_cast<const float4 *>(gd + G_QS + tok), up4 = *reinterpret_cast<const float4 *>(gd + G_UP + tok);
        const float4 p4 = *reinterpret_cast<const float4 *>(gd + G_P + tok), m4 = *reinterpret_cast<const float4 *>(gd + G_M + tok);
        const float4 sc = *reinterpret_cast<const float4 *>(gd + G_SC), mn4 = *reinterpret_cast<const float4 *>(gd + G_SC + 4);
        const float bt[4] = {beta4.x, beta4.y, beta4.z, beta4.w}, ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
        const float qs[4] = {qs4.x, qs4.y, qs4.z, qs4.w}, up[4] = {up4.x, up4.y, up4.z, up4.w};
        const float pp[4] = {p4.x, p4.y, p4.z, p4.w}, mm[4] = {m4.x, m4.y, m4.z, m4.w};
        const float mnorm = fmaxf(fmaxf(mn4.x, mn4.y), fmaxf(mn4.z, mn4.w));
        lds_barrier();  // S (and the largest values of the columns) is there
        float si[4][NC], xb[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float sm = 0.0f, vm = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                sm = fmaxf(sm, smax[w][n][r]);
                vm = fmaxf(vm, vmax[w][n][r]);
                si[w][n] = sinv[w][n][r];
            }
            xb[n] = fmaf(sc.x, vm, sc.y * sm);
        }
        v4f ka[NC], qa[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) ka[n] = qa[n] = zero;
        v4u sh[4][NC], sl[4][NC];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                sh[w][n] = Sop[w][n][0][lane];
                sl[w][n] = Sop[w][n][1][lane];
                v4f t = mma(kf[w][0], sl[w][n], zero);
                t = mma(kf[w][1], sh[w][n], t);
                t = mma(kf[w][0], sh[w][n], t);
                ka[n] += t * si[w][n];
            }
        load_rows(nx, KF, kf);
        int ex[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float x[4];
            ex[n] = exp_of(xb[n]) - 14;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = bt[e] * val[n][e] - ks[e] * ka[n][e];
            put4(Xop, n, x, pow2(-ex[n]));
        }
        load_v(nx);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                v4f t = mma(qf[w][0], sl[w][n], zero);
                t = mma(qf[w][1], sh[w][n], t);
                t = mma(qf[w][0], sh[w][n], t);
                qa[n] += t * si[w][n];
            }
        load_rows(nx, QF, qf);
        lds_barrier();  // X is there
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            v4f u = zero;
#pragma unroll
            for (int w = 0; w < 2; ++w)
                if (2 * w <= wave) {
                    const v4u xh = Xop[w][n][0][lane], xl = Xop[w][n][1][lane];
                    u = mma(mf[w][0], xl, u);
                    u = mma(mf[w][1], xh, u);
                    u = mma(mf[w][0], xh, u);
                }
            const float f = pow2(ex[n]), ub = xb[n] * mnorm;
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = u[e] * (mm[e] * f);
                y[e] = x[e] * up[e];
            }
            put4(Uop, n, x, pow2(14 - exp_of(ub)));
            put4(Wop, n, y, pow2(14 - exp_of(ub * sc.z)));
        }
        load_tri(nx, MF, mf);
        lds_barrier();  // U is there
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float f = pow2(exp_of(xb[n] * mnorm * sc.z) - 14);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                v4f t = zero;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const v4u uh = Wop[w][n][0][lane], ul = Wop[w][n][1][lane];
                    t = mma(kt[c][w][0], ul, t);
                    t = mma(kt[c][w][1], uh, t);
                    t = mma(kt[c][w][0], uh, t);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][c][e] = fmaf(t[e], f, sc.w * s[n][c][e]);
            }
        }
        load_kt(nx);
        take_v(nx);
        put_s();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float f = pow2(exp_of(xb[n] * mnorm) - 14);
            v4f t = zero;
#pragma unroll
            for (int w = 0; w < 2; ++w)
                if (2 * w <= wave) {
                    const v4u uh = Uop[w][n][0][lane], ul = Uop[w][n][1][lane];
                    t = mma(pf[w][0], ul, t);
                    t = mma(pf[w][1], uh, t);
                    t = mma(pf[w][0], uh, t);
                }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int u = i * C + tok + e;
                if (u < len) p.o[((size_t) (c0 + u) * p.nvh + h) * D + col0 + 16 * n + r] = fmaf(qs[e], qa[n][e], pp[e] * f * t[e]);
            }
        }
        load_tri(nx, PF, pf);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) Sg[(32 * wave + 16 * c + 4 * q4 + e) * D + 16 * n] = s[n][c][e];
}

// The fused block's end: gated RMSNorm of every (token, value head) in place, 32 lanes a row; and, in the blocks behind
// those, the last three raw inputs of each request into its conv ring.
__global__ void __launch_bounds__(256) k_chunk_finish(const ChunkArgs a, unsigned norm_blocks) {
    const GdnChunk &p = a.p;
    if (blockIdx.x >= norm_blocks) {
        const int Cc = 2 * p.nkh * D + p.nvh * D, per = (Cc + 255) / 256;
        const unsigned i = blockIdx.x - norm_blocks;
        const int b = i / per, c = i % per * 256 + threadIdx.x;
        const int c0 = p.cu[b], len = min(p.cu[b + 1], p.T) - c0;
        if (c0 < 0 || c >= Cc) return;
        for (int d = 1; d <= min(3, len); ++d)
            p.conv_ring[((size_t) b * p.ring + ((p.pos[b] + len - d) & (p.ring - 1))) * Cc + c] = p.qkv[(size_t) (c0 + len - d) * Cc + c];
        return;
    }
    const size_t row = (size_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    const int l = threadIdx.x & 31;
    const bool on = row < (size_t) min(p.cu[p.B], p.T) * p.nvh;
    const size_t at = on ? row * (D / 4) + l : 0;
    const float4 o = reinterpret_cast<const float4 *>(p.o)[at], z = reinterpret_cast<const float4 *>(p.z)[at];
    const float4 w = reinterpret_cast<const float4 *>(p.norm_w)[l];
    const float rn = rsqrtf(half_sum(sumsq4(o)) / D + p.eps);
    if (!on) return;
    float4 g;
    if (p.gate_act == 0) g = make_float4(sigmoidf_(z.x), sigmoidf_(z.y), sigmoidf_(z.z), sigmoidf_(z.w));
    else g = make_float4(silu_(z.x), silu_(z.y), silu_(z.z), silu_(z.w));
    reinterpret_cast<float4 *>(p.o)[at] = make_float4(o.x * rn * w.x * g.x, o.y * rn * w.y * g.y, o.z * rn * w.z * g.z, o.w * rn * w.w * g.w);
}

}  // namespace

size_t gdn_chunk_work_bytes(int B, int T, int nkh, int nvh) {
    return item_count(B, T, 1, C) * ((size_t) nkh * KEY_BYTES + (size_t) nvh * HEAD_BYTES);
}

int gdn_chunk_launch(const GdnChunk &p, hipStream_t st) {
    const bool block = p.block;
    if (p.B < 1 || p.T < 1 || p.nkh < 1 || p.nvh < 1) FN_FAIL("gdn_chunk: B, T, nkh and nvh must be >= 1");
    if (p.dk != D || p.dv != D) FN_FAIL("gdn_chunk: only dk = dv = 128 is built");
    if (p.nvh % p.nkh) FN_FAIL("gdn_chunk: nvh must be a multiple of nkh");
    if (p.head_map != 0 && p.head_map != 1) FN_FAIL("gdn_chunk: head_map must be 0 (tiled h % nkh) or 1 (grouped)");
    if (p.B > 65535 || p.nkh > 65535) FN_FAIL("gdn_chunk: B and nkh must be <= 65535");
    if (!p.cu || !p.S || !p.o || !p.work) FN_FAIL("gdn_chunk: null pointer");
    if (block) {
        if (p.gate_act != 0 && p.gate_act != 1) FN_FAIL("gdn_chunk: gate_act must be 0 (sigmoid) or 1 (silu)");
        if (p.ring < 4 || (p.ring & (p.ring - 1))) FN_FAIL("gdn_chunk: ring must be a power of two >= 4");
        if (!p.pos || !p.qkv || !p.conv_w || !p.conv_ring || !p.ab || !p.dt_bias || !p.ssm_a || !p.z || !p.norm_w)
            FN_FAIL("gdn_chunk: null pointer");
        if (((uintptr_t) p.conv_w | (uintptr_t) p.z | (uintptr_t) p.norm_w) & 15)
            FN_FAIL("gdn_chunk: conv_w, z, norm_w, out and work must be 16-byte aligned");
    } else {
        if (!p.q || !p.k || !p.v || !p.beta || !p.g) FN_FAIL("gdn_chunk: null pointer");
        if (((uintptr_t) p.q | (uintptr_t) p.k) & 15) FN_FAIL("gdn_chunk: q, k, o and work must be 16-byte aligned");
    }
    if (((uintptr_t) p.o | (uintptr_t) p.work) & 15)
        FN_FAIL(block ? "gdn_chunk: conv_w, z, norm_w, out and work must be 16-byte aligned"
                      : "gdn_chunk: q, k, o and work must be 16-byte aligned");
    if (p.work_bytes < gdn_chunk_work_bytes(p.B, p.T, p.nkh, p.nvh)) FN_FAIL("gdn_chunk: workspace too small");
    ChunkArgs a{p, nullptr, nullptr, 0};
    const size_t items = item_count(p.B, p.T, 1, C);
    a.items = (int) items;
    a.keys = static_cast<uint8_t *>(p.work);
    a.heads = a.keys + items * p.nkh * KEY_BYTES;
    const dim3 gi((unsigned) items, p.nkh), gs(p.nvh, D / 32, p.B);
    const size_t norm = ((size_t) p.T * p.nvh + 7) / 8;                                   // blocks of k_chunk_finish
    const size_t ring = p.B * ((((size_t) 2 * p.nkh + p.nvh) * D + 255) / 256);
    if (norm + ring > 0x7fffffffu) FN_FAIL("gdn_chunk: too many rows");
    if (block) {
        hipLaunchKernelGGL(k_chunk_intra<true>, gi, dim3(256), 0, st, a);
        hipLaunchKernelGGL((k_chunk_scan<true, 2>), gs, dim3(256), 0, st, a);
        hipLaunchKernelGGL(k_chunk_finish, dim3((unsigned) (norm + ring)), dim3(256), 0, st, a, (unsigned) norm);
    } else {
        hipLaunchKernelGGL(k_chunk_intra<false>, gi, dim3(256), 0, st, a);
        hipLaunchKernelGGL((k_chunk_scan<false, 2>), gs, dim3(256), 0, st, a);
    }
    FN_CK(hipGetLastError());
    return 0;
}

}  // namespace fn
