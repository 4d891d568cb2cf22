// The gated delta rule over whole prompts of a packed batch, chunk by chunk.
//
// A token does S <- g S, d = beta (v - S^T k), S <- S + k d^T, o = S^T q / sqrt(dk).  Within a chunk of 64 tokens, with
// G_i the sum of the log decays up to token i and S the state before the chunk, the updates d (rows of U) solve a
// unit lower triangular system:
//   U = U0 - W S,  U0 = M diag(beta) V,  W = M diag(beta e^G) K,  M = (I + A)^-1,  A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i)
//   o_i = (e^G_i S^T q_i + sum_(j <= i) e^(G_i - G_j) q_i.k_j u_j) / sqrt(dk)
//   S' = e^G_63 S + sum_j e^(G_63 - G_j) k_j u_j^T
// so that only S -> S' is sequential, in steps of 64 tokens.  Two kinds of workgroups:
//   k_chunk_intra, one a (chunk, key head), everything that does not need S: W, U0 and P_ij = e^(G_i - G_j) q_i.k_j of
//     each value head that reads the key head, and q, k as matrix operands;
//   k_chunk_scan, one a (request, value head, columns of S), which walks the request's chunks with its columns of S in
//     registers: three small products one after the other a chunk, and two exchanges through the LDS.
// W and U0 are formed before the scan, not M inside it: the scan is the sequential part, and M there is one more product
// and exchange a chunk (15k tokens, 32 value heads: scan 596 us with M, 392 us with W; the other kernel 252 and 272 us).
// Products: an fp32 operand is two f16 values (hi and lo, 11 bits each) under a power-of-two scale, and a product is hi
// hi + hi lo + lo hi on v_mfma_f32_16x16x32_f16: what is left out is 2^-22 of a product at the worst and 2^-24 in the
// mean, in half the instructions of six bf16 products and a fifth of the time of fp32 ones.  f16's range is met by
// scales: one a row of q, k, M, W and P (they are factors of output rows, folded into the gates' factors), one a column
// of V, one a column and 32 rows of S (from its largest value there), and a bound for U: |U| <= max|U0| + max|W_i|
// sqrt(128) max|S| in its column.  A bound too large by a factor of up to 2^15 costs no bit of a value as large as the
// column's largest: f16 reaches 2^-24 and lo goes down to there.
// What is far below its column's largest among the 64 tokens keeps fewer bits: values that fall by 10^4 within a chunk leave
// outputs and state at 3e-7, by 10^6 at 5e-6 and 2e-5, by 10^8 at 5e-4 and 2e-3 of themselves.
// Decays: G is summed in 64 bits, because differences of far sums are taken; all exponents are then <= 0 for decays < 1.
#include "serve.cuh"

namespace fn {

namespace {

constexpr int D = 128;                        // dk = dv
constexpr int C = 64;                         // tokens a chunk
constexpr int RS = D + 4;                     // floats a row of q, k in the LDS
constexpr int AS = C + 4, MS = 20;            // floats a row of A, of the diagonal blocks of M
constexpr int FRAG = 1024;                    // an operand of one 16 x 16 x 32 product: 16 bytes a lane
constexpr int QF = 0, KT = 32 * FRAG, KEY_BYTES = 64 * FRAG;                         // a (chunk, key head)
constexpr int WF = 0, U0 = 32 * FRAG, PF = 64 * FRAG, GATES = 80 * FRAG, HEAD_BYTES = 82 * FRAG;  // a (chunk, value head)
// GATES: floats: [64] scale of W's row, e^G 2^eq / sqrt(dk), e^(G63 - G) 2^ek, 2^ep / sqrt(dk); [128] largest |U0| of a
// column; sqrt(128) max|W_i|, largest e^(G63 - G) 2^ek, e^G63
constexpr int G_W = 0, G_QS = 64, G_UP = 128, G_P = 192, G_UM = 256, G_SC = 384;
constexpr float RSQRT_D = 0.08838834764831845f;

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

struct ChunkArgs {
    GdnChunk p;
    uint8_t *keys, *heads;  // the two parts of the workspace
};

__device__ __forceinline__ v4f mma(const v4u &a, const v4u &b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// Two values as f16 hi and lo pairs.  (The values are taken as they are in fp32: a product folded into the conversion
// is rounded once for the hi that is kept and twice for the one that is subtracted, and where the two differ lo is
// wrong by a unit of hi: one element in some thousands, by 2^-11.)
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    asm("" : "+v"(a), "+v"(b));
    const h2 h = __builtin_convertvector((v2f{a, b}), h2);
    const h2 l = __builtin_convertvector((v2f{fmaf((float) h.x, -1.0f, a), fmaf((float) h.y, -1.0f, b)}), h2);
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

__device__ __forceinline__ float silu_(float x) { return x * gate_of(x); }

__device__ __forceinline__ float4 lds4(const float *p) { return *reinterpret_cast<const float4 *>(p); }

// grid (chunks, nkh), four waves.  What bounds it: memory.  15k tokens, 16 key and 32 value heads: 0.49 GB of q, k, v in,
// 0.86 GB of operands out in 272 us, 5.0 TB/s (all rows are requested before the first is waited for, and V and the gates
// a part ahead: 332 us without).  In the block form, 4k tokens, 16 and 48 heads: 0.49 GB in 139 us, 3.5 TB/s: half of its
// time goes to vector instructions (conv and SiLU of every channel), and a chunk's three value heads one after the other
// leave two rounds of workgroups.  M = (I + A)^-1 by blocks of 16: a wave inverts its diagonal block by
// substitution, one column a lane, and forms its block row from the diagonal leftwards on fp32 matrix instructions.
template <bool BLOCK>
__global__ void __launch_bounds__(256, 2) k_chunk_intra(const ChunkArgs a) {
    __shared__ __align__(16) float rows[2][C * RS];            // q, k; later operands | A, diagonal blocks of M
    __shared__ __align__(16) float mul[2][C], back[2][C];      // row factors to f16's range and back
    __shared__ __align__(16) float bet[C], bks[C], mback[2][C];  // beta, beta e^G 2^ek; back of M's two forms
    __shared__ float wam[4][C], wsq[4][C];                     // largest value and squares of W's rows, by wave
    __shared__ double G[C];
    const GdnChunk &p = a.p;
    const int item = blockIdx.x, kh = blockIdx.y;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    int r = lane & 15, q4 = lane >> 4;
    const int b = request_of(p.cu, p.B, item, 1, C);
    const int c0 = p.cu[b], t0 = (item - first_item(p.cu, b, 1, C)) * C, n = min(C, min(p.cu[b + 1], p.T) - c0 - t0);
    if (c0 < 0 || t0 < 0 || n <= 0) return;
    const size_t row0 = (size_t) c0 + t0;
    // 16-row tiles that hold a token: of the others no row operand is written (the descriptor is empty), or read
    const int tiles = __builtin_amdgcn_readfirstlane((n + 15) / 16);
    // (the place is in the descriptor and not in a scalar offset: behind a store of 16 bytes with one this compiler may
    // write the store's registers in the next instruction, and the store was seen to take the new values)
    auto put = [&](uint8_t *to, bool on, const v4u &x) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_buffer_store_b128(x, buf(to, on ? FRAG : 0), lane * 16, 0, 0);
    };
    uint8_t *kd = a.keys + ((size_t) item * p.nkh + kh) * KEY_BYTES;

    const int per = p.nvh / p.nkh, Cc = 2 * p.nkh * D + p.nvh * D;
    auto head_of = [&](int i) { return p.head_map == 0 ? kh + i * p.nkh : kh * per + i; };
    float gate[2];  // beta, g of a head (of the block: what they are made from), a head ahead
    auto request_gates = [&](int i) __attribute__((always_inline)) {
        const size_t t = row0 + min(lane, n - 1), h = head_of(i);
        gate[0] = BLOCK ? p.ab[t * 2 * p.nvh + p.nvh + h] : p.beta[t * p.nvh + h];
        gate[1] = BLOCK ? p.ab[t * 2 * p.nvh + h] : p.g[t * p.nvh + h];
    };
    request_gates(0);
    // 1. q, k rows
    if (BLOCK) {
        const int ch = tid & (D - 1), part = tid >> 7, col = (part * p.nkh + kh) * D + ch;
        const float4 w = *reinterpret_cast<const float4 *>(p.conv_w + 4 * col);
        const float *x = p.qkv + row0 * Cc + col;
        const brsrc rd = buf(p.qkv + row0 * Cc, (uint32_t) n * Cc * 4);  // rows behind: 0
        float h[3], v[C];
#pragma unroll
        for (int t = 0; t < C; ++t) v[t] = bld(rd, (uint32_t) (t * Cc + col) * 4, 0);
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int t = t0 - 3 + j;
            h[j] = t >= 0 ? x[(ptrdiff_t) (j - 3) * Cc]
                          : p.conv_ring[((size_t) b * p.ring + ((p.pos[b] + t) & (p.ring - 1))) * Cc + col];
        }
#pragma unroll
        for (int t = 0; t < C; ++t) {
            float y = w.x * h[0];
            y = fmaf(w.y, h[1], y);
            y = fmaf(w.z, h[2], y);
            y = fmaf(w.w, v[t], y);
            rows[part][t * RS + ch] = t < n ? silu_(y) : 0.0f;
            h[0] = h[1];
            h[1] = h[2];
            h[2] = v[t];
        }
    } else {
        float4 x[16];  // all requested before the first is waited for
        const uint32_t pitch = p.nkh * D * 4, at = (tid >> 5) * pitch + (tid & 31) * 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const brsrc rd = buf((i < 8 ? p.q : p.k) + (row0 * p.nkh + kh) * D, (uint32_t) (n - 1) * pitch + D * 4);  // rows behind: 0
            x[i] = bld4(rd, at + i % 8 * 8 * pitch, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            *reinterpret_cast<float4 *>(&rows[i / 8][((tid >> 5) + i % 8 * 8) * RS + (tid & 31) * 4]) = x[i];
    }
    lds_barrier();
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
        }
    }
    lds_barrier();
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
                if (part) {
                    split8(v, kh_[s], kl[s]);
                } else {
                    split8(v, qh[s], ql[s]);
                    put(kd + QF + ((wave * 4 + s) * 2) * FRAG, wave < tiles, qh[s]);
                    put(kd + QF + ((wave * 4 + s) * 2 + 1) * FRAG, wave < tiles, ql[s]);
                }
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
    lds_barrier();
    v4u *op = reinterpret_cast<v4u *>(rows[0]);  // [tile][step][hi, lo][lane]: K's row operands, later two forms of M
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        op[((wave * 4 + s) * 2) * 64 + lane] = kh_[s];
        op[((wave * 4 + s) * 2 + 1) * 64 + lane] = kl[s];
    }
    lds_barrier();
    // 3. k_j.k_i and k_j.q_i of the wave's 16 rows i (lane: i = 16 wave + l%16, j = 16 tile + 4 (l / 16) + e)
    v4f kk[4], qk[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk[j] = qk[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (j <= wave) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const v4u h = op[((j * 4 + s) * 2) * 64 + lane], l = op[((j * 4 + s) * 2 + 1) * 64 + lane];
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
    for (int hi_ = 0; hi_ < per; ++hi_) {
        asm volatile("" : "+v"(r), "+v"(q4));  // addresses are made again for each head, not kept in some 60 registers
        const int h = head_of(hi_);
        uint8_t *hd = a.heads + ((size_t) item * p.nvh + h) * HEAD_BYTES;
        float *gd = reinterpret_cast<float *>(hd + GATES);
        float be = 0.0f, g = 0.0f;
        if (lane < n) {
            be = gate[0];
            g = gate[1];
            if (BLOCK) {
                const float ga = g + p.dt_bias[h];
                be = sigmoidf_(be);
                g = (ga > 20.0f ? ga : log1pf(expf(ga))) * p.ssm_a[h];
            }
        }
        if (hi_ + 1 < per) request_gates(hi_ + 1);
        double gs = fmax((double) g, -200.0);  // a decay below e^-200 is 0 in fp32 (and -infinity would cancel to NaN)
        if (g != g) gs = g;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double y = __shfl_up(gs, d);
            if (lane >= d) gs += y;
        }
        lds_barrier();  // what the last head left in the LDS has been read
        if (wave == 0) {
            const double g63 = __shfl(gs, 63);
            const float eg = expf((float) gs), up = expf((float) (g63 - gs)) * back[1][lane], um = wave_max(up);
            G[lane] = gs;
            bet[lane] = be;
            bks[lane] = be * eg * back[1][lane];
            gd[G_QS + lane] = eg * back[0][lane] * RSQRT_D;
            gd[G_UP + lane] = up;
            if (lane == 0) {
                gd[G_SC + 1] = um;
                gd[G_SC + 2] = expf((float) g63);
            }
        }
        lds_barrier();
        // values of the wave's columns 32 wave + 16 c + l%16, requested ahead
        float vv[2][2][8], before[2][3];
        float4 cw[2];
        {
            const int pitch = BLOCK ? Cc : p.nvh * D, col = (BLOCK ? 2 * p.nkh * D : 0) + h * D + 32 * wave + r;
            const brsrc v = buf((BLOCK ? p.qkv : p.v) + row0 * pitch, (uint32_t) n * pitch * 4);  // rows behind: 0
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (BLOCK) {
                    const int ch = col + 16 * c;
                    cw[c] = *reinterpret_cast<const float4 *>(p.conv_w + 4 * ch);
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        before[c][i] = t0 ? p.qkv[(row0 + i - 3) * Cc + ch]
                                          : p.conv_ring[((size_t) b * p.ring + ((p.pos[b] + i - 3) & (p.ring - 1))) * Cc + ch];
                }
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        vv[c][s][j] = bld(v, (uint32_t) ((32 * s + 16 * (j / 4) + 4 * q4 + j % 4) * pitch + col + 16 * c) * 4, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const double gi = G[16 * wave + r];
        const float bi = bet[16 * wave + r];
        {
            float pv[4][4], pm = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float av[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int jt = 16 * j + 4 * q4 + e, it = 16 * wave + r;
                    const float dec = j <= wave && jt <= it ? exp_((float) (gi - G[jt])) : 0.0f;
                    av[e] = j <= wave && jt < it ? bi * dec * kk[j][e] : 0.0f;
                    pv[j][e] = j <= wave && jt <= it ? dec * qk[j][e] : 0.0f;
                    pm = fmaxf(pm, fabsf(pv[j][e]));
                }
                if (j <= wave)
                    *reinterpret_cast<float4 *>(A + (16 * wave + r) * AS + 16 * j + 4 * q4) = make_float4(av[0], av[1], av[2], av[3]);
            }
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
                    put(hd + PF + ((wave * 2 + s) * 2) * FRAG, wave < tiles, hi);
                    put(hd + PF + ((wave * 2 + s) * 2 + 1) * FRAG, wave < tiles, lo);
                }
        }
        // values of the wave's columns 32 wave + 16 c + l%16 (slots as in k^T)
        if (BLOCK) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float y[3] = {before[c][0], before[c][1], before[c][2]};  // the three tokens before four of the lane's
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float *x = &vv[c][g / 2][4 * (g % 2)], nx[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {  // a quarter's last three are the next quarter's, the last quarter's the next g's
                        const float z = __shfl(x[i + 1], (lane + 48) & 63);
                        if (q4) y[i] = z;
                        nx[i] = z;
                    }
                    const float in[7] = {y[0], y[1], y[2], x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float z = cw[c].x * in[i];
                        z = fmaf(cw[c].y, in[i + 1], z);
                        z = fmaf(cw[c].z, in[i + 2], z);
                        z = fmaf(cw[c].w, in[i + 3], z);
                        x[i] = 16 * g + 4 * q4 + i < n ? silu_(z) : 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 3; ++i) y[i] = nx[i];
                }
            }
        }
        lds_barrier();
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
        lds_barrier();
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
        // K^T of the wave's dims comes back from where the lane has put it (32 registers less through the rest of the loop)
        v4u kt[2][2][2];
#pragma unroll
        for (int i = 0; i < 8; ++i) kt[i / 4][i / 2 % 2][i % 2] = *reinterpret_cast<v4u *>(kd + KT + (wave * 8 + i) * FRAG + lane * 16);
        // M diag(beta e^G 2^ek) and M diag(beta) as operands, a scale a row
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            float am = 0.0f, v[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 x = lds4((f ? bet : bks) + 16 * j + 4 * q4);
                const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[j][e] = mt[j][e] * y[e];
                    am = fmaxf(am, fabsf(v[j][e]));
                }
            }
            am = max_quarters(am);
            const int e = exp_of(am) - 14;
            const float m = pow2(-e);
            if (q4 == 0) mback[f][16 * wave + r] = pow2(e);
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (2 * s <= wave) {
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = v[2 * s + j / 4][j % 4] * m;
                    v4u *d = op + (((f * 4 + wave) * 2 + s) * 2) * 64 + lane;
                    split8(x, d[0], d[64]);
                }
        }
        lds_barrier();
        const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
        // U0 of the wave's columns: lane = column, tokens 16 i + 4 (l / 16) + e
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float am = 0.0f, um = 0.0f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) am = fmaxf(am, fabsf(vv[c][s][j]));
            am = max_quarters(am);
            const int e = exp_of(am) - 14;
            const float m = pow2(-e), f = pow2(e);
            v4u vh[2], vl[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) vv[c][s][j] *= m;
                split8(vv[c][s], vh[s], vl[s]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v4f u = zero;
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (2 * s <= i) {
                        const v4u mh = op[(((4 + i) * 2 + s) * 2) * 64 + lane], ml = op[(((4 + i) * 2 + s) * 2 + 1) * 64 + lane];
                        u = mma(mh, vl[s], u);
                        u = mma(ml, vh[s], u);
                        u = mma(mh, vh[s], u);
                    }
                const float4 bk = lds4(&mback[1][16 * i + 4 * q4]);
                const float4 o = make_float4(u[0] * bk.x * f, u[1] * bk.y * f, u[2] * bk.z * f, u[3] * bk.w * f);
                um = fmaxf(um, fmaxf(fmaxf(fabsf(o.x), fabsf(o.y)), fmaxf(fabsf(o.z), fabsf(o.w))));
                put(hd + U0 + (i * 8 + 2 * wave + c) * FRAG, i < tiles, __builtin_bit_cast(v4u, o));
            }
            um = max_quarters(um);
            if (q4 == 0) gd[G_UM + 32 * wave + 16 * c + r] = um;
        }
        __builtin_amdgcn_sched_barrier(0);
        // W^T = K^T (M diag)^T of the wave's dims, all tokens: lane = token 16 i + l%16, dims 32 wave + 16 c + 4 (l / 16) + e
        v4f w[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[0][i] = w[1][i] = zero;
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (2 * s <= i) {
                    const v4u mh = op[((i * 2 + s) * 2) * 64 + lane], ml = op[((i * 2 + s) * 2 + 1) * 64 + lane];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        w[c][i] = mma(kt[c][s][0], ml, w[c][i]);
                        w[c][i] = mma(kt[c][s][1], mh, w[c][i]);
                        w[c][i] = mma(kt[c][s][0], mh, w[c][i]);
                    }
                }
            const float f = mback[0][16 * i + r];
            w[0][i] *= f;
            w[1][i] *= f;
            float am = 0.0f, sq = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    am = fmaxf(am, fabsf(w[c][i][e]));
                    sq = fmaf(w[c][i][e], w[c][i][e], sq);
                }
            am = max_quarters(am);
            sq = sum_quarters(sq);
            if (q4 == 0) {
                wam[wave][16 * i + r] = am;
                wsq[wave][16 * i + r] = sq;
            }
        }
        lds_barrier();
        // W as the scan's row operand: step `wave` of every row tile
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 16 * i + r;
            const float am = fmaxf(fmaxf(wam[0][t], wam[1][t]), fmaxf(wam[2][t], wam[3][t]));
            const int e = exp_of(am) - 14;
            const float m = pow2(-e);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = w[j / 4][i][j % 4] * m;
            v4u hi, lo;
            split8(x, hi, lo);
            put(hd + WF + ((i * 4 + wave) * 2) * FRAG, i < tiles, hi);
            put(hd + WF + ((i * 4 + wave) * 2 + 1) * FRAG, i < tiles, lo);
            if (wave == 0 && q4 == 0) gd[G_W + t] = pow2(e);
        }
        if (wave == 1) {
            const float n2 = wave_max((wsq[0][lane] + wsq[1][lane]) + (wsq[2][lane] + wsq[3][lane]));
            if (lane == 0) gd[G_SC] = sqrtf(n2) * 11.3138f;  // sqrt(128), rounded up
        }
    }
}

// grid (nvh, D / (16 NC), B), nine waves.  Waves 0..3 carry the state: wave w owns tokens 16 w .. + 15 of U and rows 32 w
// .. + 31 of S.  Waves 4..7 compute the outputs of tokens 16 (w - 4) .. + 15.  Lane = column l%16 of each of NC column
// tiles, rows 4 (l / 16) + e.  That is also the layout of an operand's slots, so what a wave computes it splits and writes
// to the LDS as it stands, and the others read whole operands: S and U meet there once a chunk each, with one barrier.
//   state waves:   | U = U0 - W S, written | S' = e^G63 S + K^T U, written |
//   output waves:  | S^T q                 | + P U, stored                 |
// Operands are requested a chunk ahead, each as soon as its registers are free, and between other work, because a wave
// stops at a load that the address unit cannot take yet.  That reaches over the L2's latency, not the memory's, and the
// workgroups of a head read the same operands at the same time.  So wave 8 touches the operands two chunks ahead, each of
// the head's workgroups (which share an XCD where nvh is a multiple of 8) its part of the lines: 538 us without it, 392 us
// with it at 15k tokens and 32 heads.  (Loads to the LDS hold no registers, but a barrier waits for them: 402 us.)
// What bounds it then: the way round the state waves, 1.3 us a chunk of 1.7: two barriers, two trips through the LDS and
// the products between them; the rest is the operands' 113 KiB a chunk, whatever the columns, at 64 bytes a cycle and CU.
// That is why two column tiles (2.7 us a chunk) are taken as soon as one would leave more workgroups than CUs.
template <int NC>
__global__ void __launch_bounds__(576, 3) k_chunk_scan(const ChunkArgs a) {
    __shared__ v4u Sop[4][NC][2][64];                   // [32 rows][column tile][hi, lo][lane]
    __shared__ v4u Uop[2][NC][2][64], Wop[2][NC][2][64];  // [32 tokens]...: U, e^(G63 - G) U
    __shared__ float smax[4][NC][16], sinv[4][NC][16];
    constexpr int NG = (G_SC + 4) / 4;                  // the chunk's factors pass through the LDS, a chunk ahead
    __shared__ __align__(16) float gates[2][NG * 4];
    const GdnChunk &p = a.p;
    const int h = blockIdx.x, col0 = blockIdx.y * 16 * NC, b = blockIdx.z;
    const int role = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int lane = threadIdx.x & 63, r = lane & 15, q4 = lane >> 4;
    const int c0 = p.cu[b], len = min(p.cu[b + 1], p.T) - c0;
    if (c0 < 0 || len <= 0) return;
    const int per = p.nvh / p.nkh, kh = p.head_map == 0 ? h % p.nkh : h / per;
    const int item0 = first_item(p.cu, b, 1, C), chunks = (len + C - 1) / C;
    const int tok = 16 * wave + 4 * q4;  // the lane's first token
    const uint32_t lane16 = lane * 16;
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    // the chunk's operands.  Of a 16-row tile that holds no token the row operands were not written: the descriptor is
    // empty then, and loads give zeros.
    auto holds = [&](int i) { return 16 * wave < len - i * C; };
    auto key = [&](int i, bool on = true) __attribute__((always_inline)) {
        return buf(a.keys + ((size_t) (item0 + i) * p.nkh + kh) * KEY_BYTES, on ? KEY_BYTES : 0);
    };
    auto head = [&](int i, bool on = true) __attribute__((always_inline)) {
        return buf(a.heads + ((size_t) (item0 + i) * p.nvh + h) * HEAD_BYTES, on ? HEAD_BYTES : 0);
    };
    auto ld = [&](brsrc d, int at) __attribute__((always_inline)) {
        return __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(d, (int) lane16, at, 0));
    };
    auto load_rows = [&](brsrc d, int at, v4u(&f)[4][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j / 2][j % 2] = ld(d, at + (wave * 8 + j) * FRAG);
    };
    // largest |U| of the columns (a bound) from the largest |S|, and the scales of S's 32-row steps
    auto bounds = [&](const float *gd, float sc, float(&si)[4][NC], float(&ub)[NC]) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float sm = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                sm = fmaxf(sm, smax[w][n][r]);
                si[w][n] = sinv[w][n][r];
            }
            ub[n] = fmaf(sc, sm, gd[G_UM + col0 + 16 * n + r]);
        }
    };
    // S^T f of the wave's rows: the 32-row steps have scales of their own, so each is summed apart (which also keeps
    // products that wait for each other apart)
    auto times_s = [&](const v4u(&f)[4][2], const float(&si)[4][NC], v4f(&acc)[NC]) __attribute__((always_inline)) {
        v4f t[4][NC];
        v4u sh[4][NC];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                sh[w][n] = Sop[w][n][0][lane];
                t[w][n] = mma(f[w][1], sh[w][n], zero);
            }
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < NC; ++n) t[w][n] = mma(f[w][0], Sop[w][n][1][lane], t[w][n]);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < NC; ++n) t[w][n] = mma(f[w][0], sh[w][n], t[w][n]);
#pragma unroll
        for (int n = 0; n < NC; ++n) acc[n] = (t[0][n] * si[0][n] + t[1][n] * si[1][n]) + (t[2][n] * si[2][n] + t[3][n] * si[3][n]);
    };
    if (role == 2) {
        constexpr int LINES = D / 16 / NC * 64, NH = (HEAD_BYTES / 128 + LINES - 1) / LINES, NK = (KEY_BYTES / 128 + LINES - 1) / LINES;
        uint32_t x[NH + NK];
        auto touch = [&](int i) __attribute__((always_inline)) {
            const brsrc hd = head(i), kd = key(i);
            const int n = len - i * C, l0 = blockIdx.y * 64 + lane;
            // lines behind the operands, or of a tile without a token: not loaded
            auto at = [&](int l, int tile) { return 16 * tile < n ? l * 128 : HEAD_BYTES; };
#pragma unroll
            for (int k = 0; k < NH; ++k) {
                const int l = l0 + k * LINES, by = l * 128;
                x[k] = __builtin_amdgcn_raw_buffer_load_b32(
                    hd, at(l, by < PF ? by % U0 / (8 * FRAG) : by < GATES ? (by - PF) / (4 * FRAG) : 0), 0, 0);
            }
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const int l = l0 + k * LINES, by = l * 128;
                x[NH + k] = __builtin_amdgcn_raw_buffer_load_b32(kd, at(l, by < KT ? by / (8 * FRAG) : 0), 0, 0);
            }
        };
        touch(min(1, chunks - 1));
        for (int i = 0; i < chunks; ++i) {
            lds_barrier();
#pragma unroll
            for (int k = 0; k < NH + NK; ++k) asm volatile("" ::"v"(x[k]));  // the last chunk's, which have come by now
            touch(min(i + 2, chunks - 1));
            lds_barrier();
        }
#pragma unroll
        for (int k = 0; k < NH + NK; ++k) asm volatile("" ::"v"(x[k]));
    } else if (role == 0) {
        float s[NC][2][4];
        float *Sg = p.S + ((size_t) b * p.nvh + h) * D * D + col0 + r;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][c][e] = Sg[(32 * wave + 16 * c + 4 * q4 + e) * D + 16 * n];
        v4u wf[4][2], kt[2][2][2];
        float4 u0[NC];
        auto load_kt = [&](brsrc d) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) kt[j / 4][j / 2 % 2][j % 2] = ld(d, KT + (wave * 8 + j) * FRAG);
        };
        auto load_u0 = [&](brsrc d) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < NC; ++n) u0[n] = bld4(d, lane16, U0 + (wave * 8 + blockIdx.y * NC + n) * FRAG);
        };
        auto put_s = [&]() __attribute__((always_inline)) {
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
        auto put4 = [&](v4u(&op)[2][NC][2][64], int n, const float(&x)[4], float m) __attribute__((always_inline)) {
            uint32_t hi[2], lo[2];  // the wave's 16 tokens of an operand
            split2(x[0] * m, x[1] * m, hi[0], lo[0]);
            split2(x[2] * m, x[3] * m, hi[1], lo[1]);
            reinterpret_cast<v2u *>(&op[wave / 2][n][0][lane])[wave & 1] = v2u{hi[0], hi[1]};
            reinterpret_cast<v2u *>(&op[wave / 2][n][1][lane])[wave & 1] = v2u{lo[0], lo[1]};
        };
        // in the order of the loop's requests: its waits count them as both ways into it have them
        load_u0(head(0, holds(0)));
        __builtin_amdgcn_sched_barrier(0);
        load_rows(head(0, holds(0)), WF, wf);
        __builtin_amdgcn_sched_barrier(0);
        load_kt(key(0));
        __builtin_amdgcn_sched_barrier(0);
        put_s();
        for (int i = 0; i < chunks; ++i) {
            const int nx = min(i + 1, chunks - 1);
            const float *gd = gates[i & 1];
            const brsrc hn = head(nx, holds(nx)), kn = key(nx);
            lds_barrier();  // S (and the largest values of the columns) is there
            const float4 sc = lds4(gd + G_SC);
            float si[4][NC], ub[NC];
            bounds(gd, sc.x, si, ub);
            v4f wa[NC];
            times_s(wf, si, wa);
            __builtin_amdgcn_sched_barrier(0);
            float fs[NC];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const float4 fw = lds4(gd + G_W + tok), up = lds4(gd + G_UP + tok);
                const float x[4] = {u0[n].x - fw.x * wa[n][0], u0[n].y - fw.y * wa[n][1], u0[n].z - fw.z * wa[n][2],
                                    u0[n].w - fw.w * wa[n][3]};
                const float y[4] = {x[0] * up.x, x[1] * up.y, x[2] * up.z, x[3] * up.w};
                const int ew = exp_of(ub[n] * sc.y) - 14;
                fs[n] = pow2(ew);
                put4(Uop, n, x, pow2(14 - exp_of(ub[n])));
                put4(Wop, n, y, pow2(-ew));
            }
            load_u0(hn);
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();  // U is there
            load_rows(hn, WF, wf);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                v4f t[2][2];  // [16 rows][32 tokens]
#pragma unroll
                for (int q = 0; q < 3; ++q)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int w = 0; w < 2; ++w) t[c][w] = mma(kt[c][w][q == 1], Wop[w][n][q == 0][lane], q == 0 ? zero : t[c][w]);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][c][e] = fmaf(t[c][0][e] + t[c][1][e], fs[n], sc.z * s[n][c][e]);
            }
            __builtin_amdgcn_sched_barrier(0);
            load_kt(kn);
            put_s();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 8 * NC, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) Sg[(32 * wave + 16 * c + 4 * q4 + e) * D + 16 * n] = s[n][c][e];
    } else {
        v4u qf[4][2], pf[2][2];
        float4 gate;
        const int gt = threadIdx.x & 255;
        auto load_p = [&](brsrc d) __attribute__((always_inline)) {
            pf[0][0] = ld(d, PF + wave * 4 * FRAG);
            pf[0][1] = ld(d, PF + wave * 4 * FRAG + FRAG);
            if (wave >= 2) {
                pf[1][0] = ld(d, PF + wave * 4 * FRAG + 2 * FRAG);
                pf[1][1] = ld(d, PF + wave * 4 * FRAG + 3 * FRAG);
            }
        };
        auto load_gates = [&](brsrc d) __attribute__((always_inline)) {
            if (gt < NG) gate = bld4(d, gt * 16, GATES);
        };
        auto put_gates = [&](int i) __attribute__((always_inline)) {
            if (gt < NG) reinterpret_cast<float4 *>(gates[i & 1])[gt] = gate;
        };
        load_gates(head(0));
        put_gates(0);
        load_rows(key(0, holds(0)), QF, qf);
        __builtin_amdgcn_sched_barrier(0);
        load_p(head(0, holds(0)));
        __builtin_amdgcn_sched_barrier(0);
        for (int i = 0; i < chunks; ++i) {
            const int nx = min(i + 1, chunks - 1);
            const float *gd = gates[i & 1];
            const brsrc hn = head(nx, holds(nx)), kn = key(nx, holds(nx));
            load_gates(head(nx));
            lds_barrier();  // S (and the largest values of the columns) is there
            float si[4][NC], ub[NC];
            bounds(gd, gd[G_SC], si, ub);
            v4f qa[NC];
            times_s(qf, si, qa);
            __builtin_amdgcn_sched_barrier(0);
            load_rows(kn, QF, qf);
            put_gates(nx);
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();  // U is there
            const brsrc od = buf(p.o + ((size_t) (c0 + i * C) * p.nvh + h) * D + col0,
                                 (uint32_t) (min(len - i * C, C) - 1) * p.nvh * D * 4 + 16 * NC * 4);  // rows behind the last: dropped
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                // the wave's rows of P times U (tokens 32 .. only for the rows behind them)
                const v4u uh = Uop[0][n][0][lane], ul = Uop[0][n][1][lane];
                v4f t = mma(pf[0][0], ul, zero), t2 = mma(pf[0][1], uh, zero);
                if (wave >= 2) {
                    const v4u uh1 = Uop[1][n][0][lane], ul1 = Uop[1][n][1][lane];
                    t = mma(pf[1][0], ul1, t);
                    t2 = mma(pf[1][1], uh1, t2);
                    t2 = mma(pf[1][0], uh1, t2);
                }
                t = mma(pf[0][0], uh, t);
                t += t2;
                const float4 qs4 = lds4(gd + G_QS + tok), pp4 = lds4(gd + G_P + tok);
                const float qs[4] = {qs4.x, qs4.y, qs4.z, qs4.w}, pp[4] = {pp4.x, pp4.y, pp4.z, pp4.w};
                const float f = pow2(exp_of(ub[n]) - 14);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    bst(od, (uint32_t) (tok + e) * p.nvh * D * 4 + 64 * n + 4 * r, 0, fmaf(qs[e], qa[n][e], pp[e] * f * t[e]));
            }
            load_p(hn);
        }
    }
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
    // rows before the first request are no request's, as those behind the last
    const bool on = row >= (size_t) max(p.cu[0], 0) * p.nvh && row < (size_t) max(min(p.cu[p.B], p.T), 0) * p.nvh;
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
    if (p.nvh > 32768) FN_FAIL("gdn_chunk: nvh must be <= 32768 (the offsets in a chunk are 32-bit)");
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
    ChunkArgs a{p, nullptr, nullptr};
    const size_t items = item_count(p.B, p.T, 1, C);
    a.keys = static_cast<uint8_t *>(p.work);
    a.heads = a.keys + items * p.nkh * KEY_BYTES;
    // columns a scan workgroup (above): one tile while every workgroup has a CU of its own.  48 value heads of one request:
    // 277 us with one tile, 174 us with two; 32 value heads: 392 us with one (256 workgroups, 1.7 us a chunk), 2.7 us a
    // chunk with two
    const int nc = (long long) p.B * p.nvh * (D / 16) > device_cus() ? 2 : 1;
    const dim3 gi((unsigned) items, p.nkh), gs(p.nvh, D / 16 / nc, p.B);
    auto *scan = nc == 1 ? k_chunk_scan<1> : k_chunk_scan<2>;
    const size_t norm = ((size_t) p.T * p.nvh + 7) / 8;                                   // blocks of k_chunk_finish
    const size_t ring = p.B * ((((size_t) 2 * p.nkh + p.nvh) * D + 255) / 256);
    // a launch has below 2^32 threads, 256 a workgroup
    if (items > 0xffffffu || (block && norm + ring > 0xffffffu)) FN_FAIL("gdn_chunk: too many rows");
    if (block) {
        hipLaunchKernelGGL(k_chunk_intra<true>, gi, dim3(256), 0, st, a);
        hipLaunchKernelGGL(scan, gs, dim3(576), 0, st, a);
        hipLaunchKernelGGL(k_chunk_finish, dim3((unsigned) (norm + ring)), dim3(256), 0, st, a, (unsigned) norm);
    } else {
        hipLaunchKernelGGL(k_chunk_intra<false>, gi, dim3(256), 0, st, a);
        hipLaunchKernelGGL(scan, gs, dim3(576), 0, st, a);
    }
    FN_CK(hipGetLastError());
    return 0;
}

}  // namespace fn
