// The gated delta rule (formulas in delta_rule.cu) for prompts: chunks of 16 tokens on the tensor cores, 32-bit results.
//
// Inside a chunk that starts from state S0, with G_i = sum of log_decay over the chunk's tokens up to i and k, q divided by
// their lengths,
//
//   R_i = v_i - e^(G_i) S0^T k_i                      what the chunk's start leaves to be stored
//   U   = T R,  T = (I + A)^-1 diag(beta)             A_ij = beta_i (k_i.k_j) e^(G_i - G_j) for j < i, else 0
//   o_i = scale (e^(G_i) S0^T q_i + sum_(j <= i) (q_i.k_j) e^(G_i - G_j) u_j)
//   S   = e^(G_15) S0 + sum_j e^(G_15 - G_j) k_j u_j^T
//
// 16 tokens are what one matrix instruction takes along its inner dimension: a longer chunk only adds to the two products
// whose size grows with the chunk (T R and the sum over u_j).
//
// Precision.  States and outputs are 32-bit results, so no operand may be rounded to 11 bits.  q and k (bfloat16, 8 bits)
// scaled by a power of two to a length of about one are exact in half precision; what is 32-bit - the state, R, U, T and the
// weights of u_j - goes into the instructions as the sum of two half-precision numbers (22 bits), products of two low parts left
// out.  Half precision has little range: every column of the state (a row of the transposed tiles below) has a power of
// two, `sigma`, that keeps a bound on the column, its R and its U below 2^13; the bound follows the recurrence (a token
// adds at most beta |v|) and is taken anew from the state itself every 32 chunks.  The state itself stays in 32-bit registers
// and the instructions only ever sum up one chunk (their running sums are truncated, not rounded).  float32 storage: q and k
// are two parts as well.
//
// Layout.  A warp owns 16 value columns x 64 rows of S, transposed: S^T is the 16-row operand of S0^T k and S0^T q, the
// accumulator of S0^T k is (after R) the operand of the next product in the registers where it lies, and the new sums end up
// where S lies.  Heads of more than 64 rows take two warps per 16 columns, which swap their halves' sums through shared memory
// once per chunk.  Four more warps ("makers") prepare the chunks that the others walk: warp m makes chunks m, m + 4, ... in its
// own stage of a ring of four - q and k in half precision, T by substitution, the weights, the chunk's v.  Named barriers
// hand stages over; nothing spins.
//
// Values that are not finite: they spoil their column from their token on and nothing else, as in the recurrence - a product
// with a zero of T would spoil the tokens before.  Such chunks are noticed after U and redone with those values left out, and
// what they reach is set to NaN.
#include "common.cuh"
#include "delta_rule.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace fsie {

constexpr int DC_TOKENS = 16;              // tokens of a chunk
constexpr int DC_STAGES = 4;               // stages of the ring = makers
constexpr int DC_SLICE = 64;               // rows of S (columns of k) per warp
constexpr int DC_MAX_DIM = 128;
constexpr int DC_REFRESH = 32;             // chunks between two looks at the state's size
constexpr int DC_TLD = DC_TOKENS + 8;      // padded rows: ldmatrix without bank conflicts
constexpr float DC_MOST = 8192.f;          // sigma times a column's bound stays below this

__device__ __forceinline__ unsigned dc_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void dc_ldmatrix(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(dc_smem(p)) : "memory");
}
__device__ __forceinline__ void dc_ldmatrix_trans(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(dc_smem(p)) : "memory");
}
// d += a(16x16, row) * b(16x8, col), half-precision operands, float accumulators
__device__ __forceinline__ void dc_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dc_sync(int barrier, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}
__device__ __forceinline__ void dc_arrive(int barrier, int threads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}
__device__ __forceinline__ unsigned dc_bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
// x, y as half-precision numbers, and what that rounding lost
__device__ __forceinline__ void dc_split(float x, float y, unsigned& high, unsigned& low) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    high = dc_bits(h);
    low = dc_bits(__floats2half2_rn(x - f.x, y - f.y));
}
// the 16 x 16 operand of two neighbouring accumulator tiles, in two parts
__device__ __forceinline__ void dc_split_tiles(const float (&x)[4], const float (&y)[4], unsigned (&high)[4], unsigned (&low)[4]) {
    dc_split(x[0], x[1], high[0], low[0]);
    dc_split(x[2], x[3], high[1], low[1]);
    dc_split(y[0], y[1], high[2], low[2]);
    dc_split(y[2], y[3], high[3], low[3]);
}
__device__ __forceinline__ float dc_power(int e) { return __int_as_float((e + 127) << 23); }     // 2^e, e in -126..127

// eight neighbouring stored values
template <typename T> struct Raw8;
template <> struct Raw8<bf16> { uint4 x; };
template <> struct Raw8<float> { float4 x, y; };
__device__ __forceinline__ void dc_widen(const Raw8<bf16>& r, float (&v)[8]) {
    const unsigned w[4] = {r.x.x, r.x.y, r.x.z, r.x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void dc_widen(const Raw8<float>& r, float (&v)[8]) {
    v[0] = r.x.x; v[1] = r.x.y; v[2] = r.x.z; v[3] = r.x.w; v[4] = r.y.x; v[5] = r.y.y; v[6] = r.y.z; v[7] = r.y.w;
}
// WIDE: p starts on 16 bytes and all eight values are there or none; else `count` of them are
template <bool WIDE> __device__ __forceinline__ Raw8<bf16> dc_load8(const bf16* p, int count) {
    Raw8<bf16> r;
    r.x = make_uint4(0, 0, 0, 0);
    if constexpr (WIDE) {
        if (count > 0) r.x = *reinterpret_cast<const uint4*>(p);
    } else {
        unsigned w[4] = {0, 0, 0, 0};
        const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < count) w[i / 2] |= (unsigned)s[i] << (16 * (i & 1));
        r.x = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}
template <bool WIDE> __device__ __forceinline__ Raw8<float> dc_load8(const float* p, int count) {
    Raw8<float> r;
    r.x = r.y = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (WIDE) {
        if (count > 0) { r.x = *reinterpret_cast<const float4*>(p); r.y = *reinterpret_cast<const float4*>(p + 4); }
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < count ? p[i] : 0.f;
        r.x = make_float4(v[0], v[1], v[2], v[3]);
        r.y = make_float4(v[4], v[5], v[6], v[7]);
    }
    return r;
}
__device__ __forceinline__ void dc_store8(bf16* p, const Raw8<bf16>& r) { *reinterpret_cast<uint4*>(p) = r.x; }
__device__ __forceinline__ void dc_store8(float* p, const Raw8<float>& r) {
    *reinterpret_cast<float4*>(p) = r.x; *reinterpret_cast<float4*>(p + 4) = r.y;
}

template <typename T, int DK, int WALKERS>
struct DcShape {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;       // half-precision numbers that hold a stored one
    static constexpr int SLICES = DK / DC_SLICE;               // warps that share 16 value columns
    static constexpr int GROUPS = WALKERS / SLICES;            // groups of 16 value columns
    static constexpr int COLS = 16 * GROUPS;                   // value columns of a block
    static constexpr int KLD = DK + 8;                         // padded row of q and k
    static constexpr int VLD = COLS + (sizeof(T) == 4 ? 4 : 8);
    static constexpr int THREADS = 32 * (WALKERS + DC_STAGES);
    struct Stage {
        __half k[PARTS][DC_TOKENS][KLD], q[PARTS][DC_TOKENS][KLD];
        __half t[2][DC_TOKENS][DC_TLD], p[2][DC_TOKENS][DC_TLD];     // T and the weights of u_j, two parts each
        T v[DC_TOKENS][VLD];
        float before[DC_TOKENS];          // on S0^T k: e^(G_i), the key's length, the power of two
        float after[DC_TOKENS];           // on u_j in the new state: e^(G_15 - G_j), ...
        float query[DC_TOKENS];           // on an output: scale, the query's length, the power of two
        float fade[DC_TOKENS];            // e^(G_i)
        float v_most[COLS];               // largest |v| per column
    };
    struct Scratch { float a[DC_TOKENS][DC_TOKENS + 4]; double g[DC_TOKENS]; float f[DC_TOKENS], beta[DC_TOKENS]; };
    struct Shared {
        Stage stage[DC_STAGES];
        Scratch scratch[DC_STAGES];
        float4 swap[2][WALKERS][3][32];
        float norm[WALKERS][16];
    };
};

enum { DC_FULL = 1, DC_EMPTY = DC_FULL + DC_STAGES, DC_PAIR = DC_EMPTY + DC_STAGES };       // named barriers

template <typename T, int DK, int WALKERS, bool WIDE>
__device__ __forceinline__ void dc_make(const DeltaParams& p, typename DcShape<T, DK, WALKERS>::Shared& sm, int maker, int lane,
                                        int head, int col0, int t0, int count, int chunks) {
    using Sh = DcShape<T, DK, WALKERS>;
    constexpr int PARTS = Sh::PARTS, FOURS = DK / 32;          // 32 columns are a quad's eight each
    auto& st = sm.stage[maker];
    auto& own = sm.scratch[maker];
    const int g = lane >> 2, t = lane & 3;
    const T* qkv = (const T*)p.qkv;
    const int narrow = head / p.share * p.dim;
    for (int c = maker; c < chunks; c += DC_STAGES) {
        const int first = t0 + c * DC_TOKENS, n = min(DC_TOKENS, count - c * DC_TOKENS);
        // ---- q, k, v and gates on their way
        Raw8<T> kr[2][FOURS], qr[2][FOURS];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h;
            const T* row = qkv + (size_t)(first + (r < n ? r : 0)) * p.ld + narrow;
#pragma unroll
            for (int f = 0; f < FOURS; ++f) {
                const int d = f * 32 + t * 8, have = r < n ? p.dim - d : 0;
                kr[h][f] = dc_load8<WIDE>(row + p.k_off + d, have);
                qr[h][f] = dc_load8<WIDE>(row + p.q_off + d, have);
            }
        }
        constexpr int EIGHTS = Sh::COLS / 8, VLOADS = (DC_TOKENS * EIGHTS + 31) / 32;
        Raw8<T> vr[VLOADS];
#pragma unroll
        for (int i = 0; i < VLOADS; ++i) {
            const int e = lane + 32 * i, r = e / EIGHTS, d = col0 + (e % EIGHTS) * 8;
            vr[i] = dc_load8<WIDE>(qkv + (size_t)(first + (r < n ? r : 0)) * p.ld + p.v_off + head * p.vdim + d,
                                   r < n ? p.vdim - d : 0);
        }
        float decay = 0.f, beta = 0.f;
        if ((lane & 15) < n) {
            decay = p.log_decay[(size_t)(first + (lane & 15)) * p.heads + head];
            beta = p.beta[(size_t)(first + (lane & 15)) * p.heads + head];
        }
        // ---- lengths of q and k, a power of two that brings each below one, both in half precision
        float kk[2], qq[2];
        unsigned kh[PARTS][2][FOURS][4], qh[PARTS][2][FOURS][4];
        float kf[2], qf[2];                                    // length and power of two as one factor
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            kk[h] = qq[h] = 0.f;
            float x[8];
#pragma unroll
            for (int f = 0; f < FOURS; ++f) {
                dc_widen(kr[h][f], x);
#pragma unroll
                for (int i = 0; i < 8; ++i) kk[h] = fmaf(x[i], x[i], kk[h]);
                dc_widen(qr[h][f], x);
#pragma unroll
                for (int i = 0; i < 8; ++i) qq[h] = fmaf(x[i], x[i], qq[h]);
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                kk[h] += __shfl_xor_sync(0xffffffffu, kk[h], o);
                qq[h] += __shfl_xor_sync(0xffffffffu, qq[h], o);
            }
            const int ke = (((__float_as_int(kk[h]) >> 23) & 255) - 125) >> 1, qe = (((__float_as_int(qq[h]) >> 23) & 255) - 125) >> 1;
            const float ks = dc_power(-ke), qs = dc_power(-qe);
            kf[h] = dc_power(ke) / sqrtf(kk[h] + p.eps);
            qf[h] = p.scale * (dc_power(qe) / sqrtf(qq[h] + p.eps));
#pragma unroll
            for (int f = 0; f < FOURS; ++f) {
                dc_widen(kr[h][f], x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (PARTS == 2) dc_split(x[2 * i] * ks, x[2 * i + 1] * ks, kh[0][h][f][i], kh[PARTS - 1][h][f][i]);
                    else kh[0][h][f][i] = dc_bits(__floats2half2_rn(x[2 * i] * ks, x[2 * i + 1] * ks));
                }
                dc_widen(qr[h][f], x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (PARTS == 2) dc_split(x[2 * i] * qs, x[2 * i + 1] * qs, qh[0][h][f][i], qh[PARTS - 1][h][f][i]);
                    else qh[0][h][f][i] = dc_bits(__floats2half2_rn(x[2 * i] * qs, x[2 * i + 1] * qs));
                }
            }
        }
        // ---- K K^T and Q K^T: a lane's eight neighbouring values are operand registers as they are, because both operands
        // take their inner index in the same order
        float kkt[2][2][4], qkt[2][2][4];                      // [two chains][columns 0-7, 8-15]
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) kkt[i][j][e] = qkt[i][j][e] = 0.f;
#pragma unroll
        for (int f = 0; f < FOURS; ++f) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {                      // inner 16 of the 32 columns
#pragma unroll
                for (int pa = 0; pa < PARTS; ++pa) {
#pragma unroll
                    for (int pb = 0; pb + pa < PARTS; ++pb) {
                        const unsigned ka[4] = {kh[pa][0][f][2 * i], kh[pa][1][f][2 * i], kh[pa][0][f][2 * i + 1], kh[pa][1][f][2 * i + 1]};
                        const unsigned qa[4] = {qh[pa][0][f][2 * i], qh[pa][1][f][2 * i], qh[pa][0][f][2 * i + 1], qh[pa][1][f][2 * i + 1]};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            dc_mma(kkt[i][j], ka, kh[pb][j][f][2 * i], kh[pb][j][f][2 * i + 1]);
                            dc_mma(qkt[i][j], qa, kh[pb][j][f][2 * i], kh[pb][j][f][2 * i + 1]);
                        }
                    }
                }
            }
        }
        // ---- gates: sums of log_decay in 64 bits, so that a difference of two of them is as exact as its own terms
        double sum = decay < -1e4f ? -1e4 : (double)decay;     // (e^-10000 is zero)
#pragma unroll
        for (int o = 1; o < DC_TOKENS; o <<= 1) {
            const double left = __shfl_up_sync(0xffffffffu, sum, o, DC_TOKENS);
            if ((lane & 15) >= o) sum += left;
        }
        const double all = __shfl_sync(0xffffffffu, sum, DC_TOKENS - 1, DC_TOKENS);
        const int from = (lane & 7) * 4;                       // a lane of the quad that holds row lane & 7
        const float kf0 = __shfl_sync(0xffffffffu, kf[0], from), kf1 = __shfl_sync(0xffffffffu, kf[1], from);
        const float qf0 = __shfl_sync(0xffffffffu, qf[0], from), qf1 = __shfl_sync(0xffffffffu, qf[1], from);
        const float kfi = (lane & 8) ? kf1 : kf0, qfi = (lane & 8) ? qf1 : qf0;        // of token lane & 15
        const float fade = expf((float)sum), after = expf((float)(all - sum)) * kfi;
        __syncwarp();                                          // the last chunk's scratch has been read
        if (lane < DC_TOKENS) { own.g[lane] = sum; own.f[lane] = kfi; own.beta[lane] = beta; }
        __syncwarp();
        float weight[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = 8 * j + 2 * t;
            const double g0 = own.g[col], g1 = own.g[col + 1];
            const float f0 = own.f[col], f1 = own.f[col + 1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = g + 8 * h;
                const double gr = own.g[row];
                const float mine = own.beta[row] * own.f[row];
                const float e0 = expf((float)(gr - g0)), e1 = expf((float)(gr - g1));
                weight[j][2 * h] = row >= col ? (qkt[0][j][2 * h] + qkt[1][j][2 * h]) * f0 * e0 : 0.f;
                weight[j][2 * h + 1] = row > col ? (qkt[0][j][2 * h + 1] + qkt[1][j][2 * h + 1]) * f1 * e1 : 0.f;
                own.a[row][col] = row > col ? mine * f0 * (kkt[0][j][2 * h] + kkt[1][j][2 * h]) * e0 : 0.f;
                own.a[row][col + 1] = row > col + 1 ? mine * f1 * (kkt[0][j][2 * h + 1] + kkt[1][j][2 * h + 1]) * e1 : 0.f;
            }
        }
        __syncwarp();
        // ---- row i of (I + A)^-1 in lane i (and again in lane i + 16): from x (I + A) = e_i, last column first
        const int i = lane & 15;
        float x[DC_TOKENS];
#pragma unroll
        for (int j = 0; j < DC_TOKENS; ++j) x[j] = i == j ? 1.f : 0.f;
#pragma unroll
        for (int l = DC_TOKENS - 1; l >= 1; --l) {
            if (l <= i) {
#pragma unroll
                for (int j = 0; j < l; ++j) x[j] = fmaf(-x[l], own.a[l][j], x[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < DC_TOKENS; ++j) x[j] = j <= i ? x[j] * own.beta[j] : 0.f;
        // ---- into the stage, once its last chunk has been walked
        if (c >= DC_STAGES) dc_sync(DC_EMPTY + maker, 32 * (WALKERS + 1));
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int f = 0; f < FOURS; ++f) {
                    const unsigned(&a)[4] = kh[part][h][f];
                    const unsigned(&b)[4] = qh[part][h][f];
                    *reinterpret_cast<uint4*>(&st.k[part][g + 8 * h][f * 32 + t * 8]) = make_uint4(a[0], a[1], a[2], a[3]);
                    *reinterpret_cast<uint4*>(&st.q[part][g + 8 * h][f * 32 + t * 8]) = make_uint4(b[0], b[1], b[2], b[3]);
                }
        {
            unsigned high[DC_TOKENS / 2], low[DC_TOKENS / 2];
#pragma unroll
            for (int j = 0; j < DC_TOKENS / 2; ++j) dc_split(x[2 * j], x[2 * j + 1], high[j], low[j]);
            // the two lanes that hold a row write one part each
            uint4* to = reinterpret_cast<uint4*>(&st.t[lane >> 4][i][0]);
            const bool second = lane >= 16;
            to[0] = second ? make_uint4(low[0], low[1], low[2], low[3]) : make_uint4(high[0], high[1], high[2], high[3]);
            to[1] = second ? make_uint4(low[4], low[5], low[6], low[7]) : make_uint4(high[4], high[5], high[6], high[7]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                unsigned high, low;
                dc_split(weight[j][2 * h], weight[j][2 * h + 1], high, low);
                *reinterpret_cast<unsigned*>(&st.p[0][g + 8 * h][8 * j + 2 * t]) = high;
                *reinterpret_cast<unsigned*>(&st.p[1][g + 8 * h][8 * j + 2 * t]) = low;
            }
        float most[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) most[k] = 0.f;
#pragma unroll
        for (int k = 0; k < VLOADS; ++k) {
            const int e = lane + 32 * k;
            if (e < DC_TOKENS * EIGHTS) dc_store8(&st.v[e / EIGHTS][(e % EIGHTS) * 8], vr[k]);
            float y[8];
            dc_widen(vr[k], y);
#pragma unroll
            for (int z = 0; z < 8; ++z)                        // (one that is not finite must not move its column's power)
                most[z] = fmaxf(most[z], fabsf(y[z]) < INFINITY ? fabsf(y[z]) : 0.f);
        }
#pragma unroll
        for (int o = EIGHTS; o < 32; o <<= 1)
#pragma unroll
            for (int z = 0; z < 8; ++z) most[z] = fmaxf(most[z], __shfl_xor_sync(0xffffffffu, most[z], o));
        if (lane < EIGHTS) {
#pragma unroll
            for (int z = 0; z < 8; ++z) st.v_most[lane * 8 + z] = most[z];
        }
        if (lane < DC_TOKENS) {
            st.before[lane] = fade * kfi; st.after[lane] = after; st.query[lane] = qfi; st.fade[lane] = fade;
        }
        dc_arrive(DC_FULL + maker, 32 * (WALKERS + 1));
    }
}

// U = T R (both in two parts): operands R (high, low), T's parts as they lie in the stage
__device__ __forceinline__ void dc_solve(float (&u)[2][4], const unsigned (&rh)[4], const unsigned (&rl)[4], const unsigned (&th)[4],
                                         const unsigned (&tl)[4]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
        dc_mma(b, rl, th[2 * j], th[2 * j + 1]);
        dc_mma(a, rh, th[2 * j], th[2 * j + 1]);
        dc_mma(b, rh, tl[2 * j], tl[2 * j + 1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) u[j][e] = a[e] + b[e];
    }
}

// the first token of each of the thread's two rows whose value is not finite (DC_TOKENS: none), over the row's four lanes
__device__ __forceinline__ void dc_first_bad(const float (&x)[2][4], int t, int (&first)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int at = DC_TOKENS;
#pragma unroll
        for (int j = 1; j >= 0; --j)
#pragma unroll
            for (int e = 1; e >= 0; --e)
                if (!(fabsf(x[j][2 * h + e]) < INFINITY)) at = 8 * j + 2 * t + e;
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
        first[h] = min(first[h], at);
    }
}
__device__ __forceinline__ void dc_leave_out(float (&x)[2][4], int t, const int (&first)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (8 * j + 2 * t + (e & 1) >= first[e >> 1]) x[j][e] = 0.f;
}

template <typename T, int DK, int WALKERS, bool WIDE>
__global__ void __launch_bounds__(32 * (WALKERS + DC_STAGES), 1)
delta_chunk_kernel(const DeltaParams p) {
    using Sh = DcShape<T, DK, WALKERS>;
    constexpr int PARTS = Sh::PARTS, SLICES = Sh::SLICES, TILES = DC_SLICE / 8, STEPS = DC_SLICE / 16;
    extern __shared__ __align__(16) unsigned char dc_raw[];
    auto& sm = *reinterpret_cast<typename Sh::Shared*>(dc_raw);
    const int head = blockIdx.y, item = blockIdx.z, col0 = blockIdx.x * Sh::COLS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = p.item_slots[item], count = p.item_qlen[item], t0 = p.item_qstart[item];
    if (slot < 0 || count <= 0) return;                        // a padding entry of a fixed-size batch
    const int chunks = (count + DC_TOKENS - 1) / DC_TOKENS;
    if (warp >= WALKERS) {
        grid_dependency_wait();
        grid_dependents_go();
        dc_make<T, DK, WALKERS, WIDE>(p, sm, warp - WALKERS, lane, head, col0, t0, count, chunks);
        return;
    }
    const int g = lane >> 2, t = lane & 3;
    const int group = warp / SLICES, slice = warp % SLICES;
    const int row0 = slice * DC_SLICE;                         // the warp's rows of S
    const int col = col0 + group * 16 + g;                     // the thread's value columns: col and col + 8
    float* state = p.state + (size_t)slot * p.state_stride + (size_t)head * p.dim * p.vdim;
    // S^T, tile n: rows (value columns) g and g + 8, columns (rows of S) 8 n + 2 t and the next; times sigma
    float s[TILES][4];
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = row0 + 8 * n + 2 * t + (e & 1), v = col + 8 * (e >> 1);
            s[n][e] = d < p.dim && v < p.vdim ? state[(size_t)d * p.vdim + v] : 0.f;
        }
    grid_dependency_wait();
    grid_dependents_go();
    float sigma[2] = {1.f, 1.f}, bound[2] = {0.f, 0.f};        // of columns col and col + 8
    unsigned sh[STEPS][4], sl[STEPS][4];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
    const int b_row = (lane & 7) + 8 * (lane >> 4), b_col = 8 * ((lane >> 3) & 1);      // ldmatrix, operand stored [n][k]
    const int bt_row = (lane & 7) + 8 * ((lane >> 3) & 1), bt_col = 8 * (lane >> 4);    // ... and [k][n]
    float* out = p.out + (size_t)t0 * p.heads * p.vdim + (size_t)head * p.vdim + col;

    for (int c = 0; c < chunks; ++c) {
        auto& st = sm.stage[c % DC_STAGES];
        dc_sync(DC_FULL + c % DC_STAGES, 32 * (WALKERS + 1));
        // ---- the columns' powers of two
        if (c % DC_REFRESH == 0) {                             // the bounds from the columns themselves
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float sum = 0.f;
                const float back = 1.f / sigma[h];             // (a power of two)
#pragma unroll
                for (int n = 0; n < TILES; ++n) sum = fmaxf(sum, fmaxf(fabsf(s[n][2 * h]), fabsf(s[n][2 * h + 1])));
                sum *= back;
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) sum = fmaxf(sum, __shfl_xor_sync(0xffffffffu, sum, o));
                if (SLICES > 1) {
                    if (t == 0) sm.norm[warp][g + 8 * h] = sum;
                } else {
                    bound[h] = sum * 8.f;                      // 2-norm of 64 numbers, at most 8 times the largest
                }
            }
            if (SLICES > 1) {
                dc_sync(DC_PAIR + group, 64);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    bound[h] = fmaxf(sm.norm[group * SLICES][g + 8 * h], sm.norm[group * SLICES + SLICES - 1][g + 8 * h]) * 12.f;
            }
        }
        const float add[2] = {32.f * st.v_most[group * 16 + g], 32.f * st.v_most[group * 16 + g + 8]};
        float factor[2];
        bool moved = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float most = (bound[h] + add[h]) * sigma[h];
            factor[h] = 1.f;
            if (most > DC_MOST || (most < DC_MOST / 256.f && most > 0.f)) {
                // 2^12 <= most * factor < 2^13; sigma itself stays within 2^-100 .. 2^100
                int e = 12 - (((__float_as_int(most) >> 23) & 255) - 127);
                const int have = ((__float_as_int(sigma[h]) >> 23) & 255) - 127;
                e = min(max(e, -100 - have), 100 - have);
                factor[h] = dc_power(min(max(e, -126), 127));
                moved = moved || factor[h] != 1.f;
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sigma[h] *= factor[h];
#pragma unroll
                for (int n = 0; n < TILES; ++n) { s[n][2 * h] *= factor[h]; s[n][2 * h + 1] *= factor[h]; }
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
        }
        // ---- S0^T k and S0^T q of the warp's rows: 16 columns x 16 tokens
        float wk[2][4], wq[2][4];
        {
            float low_k[2][4], low_q[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) wk[j][e] = wq[j][e] = low_k[j][e] = low_q[j][e] = 0.f;
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                unsigned b[4];
                dc_ldmatrix(b, &st.k[0][b_row][row0 + 16 * k + b_col]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    dc_mma(wk[j], sh[k], b[2 * j], b[2 * j + 1]);
                    dc_mma(low_k[j], sl[k], b[2 * j], b[2 * j + 1]);
                }
                if (PARTS == 2) {
                    dc_ldmatrix(b, &st.k[PARTS - 1][b_row][row0 + 16 * k + b_col]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) dc_mma(low_k[j], sh[k], b[2 * j], b[2 * j + 1]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) wk[j][e] += low_k[j][e];
            if (SLICES > 1) {
                sm.swap[c & 1][warp][0][lane] = make_float4(wk[0][0], wk[0][1], wk[0][2], wk[0][3]);
                sm.swap[c & 1][warp][1][lane] = make_float4(wk[1][0], wk[1][1], wk[1][2], wk[1][3]);
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                unsigned b[4];
                dc_ldmatrix(b, &st.q[0][b_row][row0 + 16 * k + b_col]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    dc_mma(wq[j], sh[k], b[2 * j], b[2 * j + 1]);
                    dc_mma(low_q[j], sl[k], b[2 * j], b[2 * j + 1]);
                }
                if (PARTS == 2) {
                    dc_ldmatrix(b, &st.q[PARTS - 1][b_row][row0 + 16 * k + b_col]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) dc_mma(low_q[j], sh[k], b[2 * j], b[2 * j + 1]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) wq[j][e] += low_q[j][e];
        }
        // ---- with two warps per 16 columns: all of S0^T k for both, of S0^T q the half of the tokens that a warp finishes
        if (SLICES > 1) {
            const int other = slice ^ 1;
            sm.swap[c & 1][warp][2][lane] = other ? make_float4(wq[1][0], wq[1][1], wq[1][2], wq[1][3])
                                                  : make_float4(wq[0][0], wq[0][1], wq[0][2], wq[0][3]);
            dc_sync(DC_PAIR + group, 64);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float4 x = sm.swap[c & 1][warp ^ 1][j][lane];
                wk[j][0] += x.x; wk[j][1] += x.y; wk[j][2] += x.z; wk[j][3] += x.w;
            }
            const float4 x = sm.swap[c & 1][warp ^ 1][2][lane];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (slice == j) { wq[j][0] += x.x; wq[j][1] += x.y; wq[j][2] += x.z; wq[j][3] += x.w; }
        }
        // ---- R, U
        float r[2][4], u[2][4];
        if constexpr (sizeof(T) == 2) {
            unsigned v[4];                                     // tokens 0-7 of col, col + 8; tokens 8-15 of both
            dc_ldmatrix_trans(v, &st.v[(lane & 7) + 8 * (lane >> 4)][group * 16 + 8 * ((lane >> 3) & 1)]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    r[j][2 * h] = __uint_as_float(v[2 * j + h] << 16);
                    r[j][2 * h + 1] = __uint_as_float(v[2 * j + h] & 0xffff0000u);
                }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) r[j][e] = to_float(st.v[8 * j + 2 * t + (e & 1)][group * 16 + g + 8 * (e >> 1)]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 before = *reinterpret_cast<const float2*>(&st.before[8 * j + 2 * t]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                r[j][2 * h] = fmaf(-before.x, wk[j][2 * h], r[j][2 * h] * sigma[h]);
                r[j][2 * h + 1] = fmaf(-before.y, wk[j][2 * h + 1], r[j][2 * h + 1] * sigma[h]);
            }
        }
        unsigned rh[4], rl[4], th[4], tl[4];
        dc_ldmatrix(th, &st.t[0][b_row][b_col]);
        dc_ldmatrix(tl, &st.t[1][b_row][b_col]);
        dc_split_tiles(r[0], r[1], rh, rl);
        dc_solve(u, rh, rl, th, tl);
        int bad[2] = {DC_TOKENS, DC_TOKENS};
        {
            float probe = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) probe = fmaf(u[j][e], 0.f, probe);
            if (__any_sync(0xffffffffu, probe != 0.f)) {       // (NaN: something is not finite)
                dc_first_bad(r, t, bad);
                dc_leave_out(r, t, bad);
                dc_split_tiles(r[0], r[1], rh, rl);
                dc_solve(u, rh, rl, th, tl);
                dc_first_bad(u, t, bad);
                dc_leave_out(u, t, bad);
            }
        }
        // ---- outputs: the chunk's start and its own tokens
        unsigned uh[4], ul[4], ph[4], pl[4];
        dc_ldmatrix(ph, &st.p[0][b_row][b_col]);
        dc_ldmatrix(pl, &st.p[1][b_row][b_col]);
        dc_split_tiles(u[0], u[1], uh, ul);
        const float back[2] = {1.f / sigma[0], 1.f / sigma[1]};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (SLICES > 1 && slice != j) continue;
            float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
            dc_mma(b, ul, ph[2 * j], ph[2 * j + 1]);
            dc_mma(a, uh, ph[2 * j], ph[2 * j + 1]);
            dc_mma(b, uh, pl[2 * j], pl[2 * j + 1]);
            const float2 fade = *reinterpret_cast<const float2*>(&st.fade[8 * j + 2 * t]);
            const float2 query = *reinterpret_cast<const float2*>(&st.query[8 * j + 2 * t]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int token = 8 * j + 2 * t + (e & 1);
                float o = fmaf((e & 1) ? fade.y : fade.x, wq[j][e], a[e] + b[e]) * ((e & 1) ? query.y : query.x) * back[e >> 1];
                if (token >= bad[e >> 1]) o = __int_as_float(0x7fffffff);
                if (c * DC_TOKENS + token < count && col + 8 * (e >> 1) < p.vdim)
                    out[(size_t)(c * DC_TOKENS + token) * p.heads * p.vdim + 8 * (e >> 1)] = o;
            }
        }
        // ---- the new state
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 after = *reinterpret_cast<const float2*>(&st.after[8 * j + 2 * t]);
#pragma unroll
            for (int e = 0; e < 4; ++e) u[j][e] *= (e & 1) ? after.y : after.x;
        }
        dc_split_tiles(u[0], u[1], uh, ul);
        const float decay = st.fade[DC_TOKENS - 1];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            unsigned b[4], b2[4];
            dc_ldmatrix_trans(b, &st.k[0][bt_row][row0 + 16 * k + bt_col]);
            if (PARTS == 2) dc_ldmatrix_trans(b2, &st.k[PARTS - 1][bt_row][row0 + 16 * k + bt_col]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float a[4] = {0.f, 0.f, 0.f, 0.f};
                dc_mma(a, ul, b[2 * j], b[2 * j + 1]);
                if (PARTS == 2) dc_mma(a, uh, b2[2 * j], b2[2 * j + 1]);
                dc_mma(a, uh, b[2 * j], b[2 * j + 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[2 * k + j][e] = fmaf(s[2 * k + j][e], decay, a[e]);
            }
        }
        if (c + DC_STAGES < chunks) dc_arrive(DC_EMPTY + c % DC_STAGES, 32 * (WALKERS + 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bound[h] = fmaf(bound[h], decay, add[h]);
            if (bad[h] < DC_TOKENS) {
#pragma unroll
                for (int n = 0; n < TILES; ++n) s[n][2 * h] = s[n][2 * h + 1] = __int_as_float(0x7fffffff);
            }
        }
#pragma unroll
        for (int k = 0; k < STEPS; ++k) dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = row0 + 8 * n + 2 * t + (e & 1), v = col + 8 * (e >> 1);
            if (d < p.dim && v < p.vdim) state[(size_t)d * p.vdim + v] = s[n][e] * (1.f / sigma[e >> 1]);
        }
}

template <typename T, int DK, int WALKERS, bool WIDE>
static int launch_chunk(const DeltaParams& p, int items, int early, cudaStream_t stream) {
    using Sh = DcShape<T, DK, WALKERS>;
    auto kernel = delta_chunk_kernel<T, DK, WALKERS, WIDE>;
    static bool configured = false;            // per process and kernel; harmless if repeated
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(typename Sh::Shared));
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    const dim3 grid((p.vdim + Sh::COLS - 1) / Sh::COLS, p.heads, items);
    if (grid.y > 65535 || grid.z > 65535) return ERR_UNSUPPORTED;
    return launch_dependent_if(early, kernel, grid, dim3(Sh::THREADS), sizeof(typename Sh::Shared), stream, p);
}

template <typename T, int DK>
static int launch_chunk_any(const DeltaParams& p, int items, int early, cudaStream_t stream) {
    const bool wide = p.ld % 8 == 0 && p.q_off % 8 == 0 && p.k_off % 8 == 0 && p.v_off % 8 == 0 && p.dim % 8 == 0 &&
                      p.vdim % 8 == 0 && (uintptr_t)p.qkv % 16 == 0;
    if (wide) return launch_chunk<T, DK, 4, true>(p, items, early, stream);
    return launch_chunk<T, DK, 4, false>(p, items, early, stream);
}

// The chunked form; ERR_UNSUPPORTED where a head has more rows than it holds.
int delta_chunk(const DeltaParams& p, int items, int dtype, int early, cudaStream_t stream) {
    if (p.dim > DC_MAX_DIM) return ERR_UNSUPPORTED;
    if (dtype == DTYPE_F32)
        return p.dim <= 64 ? launch_chunk_any<float, 64>(p, items, early, stream) : launch_chunk_any<float, 128>(p, items, early, stream);
    return p.dim <= 64 ? launch_chunk_any<bf16, 64>(p, items, early, stream) : launch_chunk_any<bf16, 128>(p, items, early, stream);
}

}  // namespace fsie

extern "C" int fsie_delta_chunk_max_dim() { return fsie::DC_MAX_DIM; }
