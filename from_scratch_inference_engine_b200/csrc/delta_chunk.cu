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
// two, `sigma`, chosen from the column's and the chunk's own largest numbers every 32 chunks, and anew, with the chunk's
// sums taken again, whenever a number of R leaves the range in between.  The state itself stays in 32-bit registers
// and the instructions only ever sum up one chunk (their running sums are truncated, not rounded).  float32 storage: q and k
// are two parts as well.
//
// Two kernels.  The first prepares all chunks side by side, a warp per chunk and q/k head: q and k in half precision, T by
// substitution, the weights of u_j, the gates' factors, as records in the workspace that lie as the second kernel's shared
// memory holds them.  The second walks a head's chunks, a block for every 16 GROUPS value columns, four more warps
// keeping the records and v of the next chunks on their way into a ring of stages; all meet once per chunk and nothing spins.  (One kernel in which
// four more warps per block prepared the chunks took 951 us for 8,192 tokens of 32 heads: every block of value columns
// prepared them again, and the two roles' code did not fit the instruction cache together.)
//
// Layout.  A warp of the second kernel owns 16 value columns x 64 rows of S, transposed: S^T is the 16-row operand of S0^T k
// and S0^T q, the accumulator of S0^T k is (after R) the operand of the next product in the registers where it lies, and the
// new sums end up where S lies.  Heads of more than 64 rows take two warps per 16 columns, which swap their halves' sums
// through shared memory once per chunk.
//
// Values that are not finite: they spoil their column from their token on and nothing else, as in the recurrence - a product
// with a zero of T would spoil the tokens before.  Such chunks are noticed by R and by a mark in their record, redone with those
// values left out, and what they reach is set to NaN.
#include "common.cuh"
#include "delta_rule.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace fsie {

constexpr int DC_TOKENS = 16;              // tokens of a chunk
constexpr int DC_STAGES = 4;               // stages of the ring: the chunk's, the next one's and two on their way
constexpr int DC_WALKERS = 4;              // warps that walk a block's chunks
constexpr int DC_SLICE = 64;               // rows of S (columns of k) per warp
constexpr int DC_MAX_DIM = 128;
constexpr int DC_REFRESH = 32;             // chunks between two looks at the state's size
constexpr int DC_SIZE = 4;                 // ... which brings the largest number of a column to 2^4 .. 2^5
constexpr int DC_TLD = DC_TOKENS + 8;      // padded rows: ldmatrix without bank conflicts
// A number of R, times sigma, is below this: a row of T has at most 16 numbers of at most beta^2 <= 4 (what a token's value
// still does to a later token's u passes through contractions), so that u, and u with a factor of at most 2, fit half precision.
constexpr float DC_MOST = 500.f;

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
__device__ __forceinline__ unsigned dc_bits(__half2 h) { return *reinterpret_cast<unsigned*>(&h); }
// two floats in one register pair: the packed instructions of sm_100 work on both at once
__device__ __forceinline__ unsigned long long dc_pair(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void dc_unpair(unsigned long long p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}
__device__ __forceinline__ void dc_fma2(float& x, float& y, float ax, float ay, float bx, float by, float cx, float cy) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(dc_pair(ax, ay)), "l"(dc_pair(bx, by)), "l"(dc_pair(cx, cy)));
    dc_unpair(r, x, y);
}
__device__ __forceinline__ void dc_mul2(float& x, float& y, float ax, float ay, float bx, float by) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(dc_pair(ax, ay)), "l"(dc_pair(bx, by)));
    dc_unpair(r, x, y);
}
__device__ __forceinline__ void dc_add2(float& x, float& y, float ax, float ay, float bx, float by) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(dc_pair(ax, ay)), "l"(dc_pair(bx, by)));
    dc_unpair(r, x, y);
}
// x, y as half-precision numbers, and what that rounding lost (cutting x and y off instead would save an instruction, but
// products of two lows, which are left out, would then all have the same sign)
__device__ __forceinline__ void dc_split(float x, float y, unsigned& high, unsigned& low) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    high = dc_bits(h);
    float lx, ly;
    dc_add2(lx, ly, x, y, -f.x, -f.y);
    low = dc_bits(__floats2half2_rn(lx, ly));
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

template <typename T, int DK>
struct DcShape {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;       // half-precision numbers that hold a stored one
    static constexpr int SLICES = DK / DC_SLICE;               // warps that share 16 value columns
    static constexpr int GROUPS = DC_WALKERS / SLICES;         // groups of 16 value columns
    static constexpr int COLS = 16 * GROUPS;                   // value columns of a block
    static constexpr int KLD = DK + 8;                         // padded row of q and k
    static constexpr int VLD = COLS + (sizeof(T) == 4 ? 4 : 8);
    static constexpr int THREADS = 2 * 32 * DC_WALKERS;        // the walkers' and the fetchers'
    struct alignas(16) Keys { __half k[PARTS][DC_TOKENS][KLD], q[PARTS][DC_TOKENS][KLD]; };
    struct alignas(16) Gates {
        __half t[2][DC_TOKENS][DC_TLD], p[2][DC_TOKENS][DC_TLD];     // T and the weights of u_j, two parts each
        float before[DC_TOKENS];          // on S0^T k: e^(G_i), the key's length, the power of two
        float after[DC_TOKENS];           // on u_j in the new state: e^(G_15 - G_j), ...
        float query[DC_TOKENS];           // on an output: scale, the query's length, the power of two
        float fade[DC_TOKENS];            // e^(G_i)
        float odd[4];                     // NaN where T has a number that is not finite, else 0
    };
    struct alignas(16) Stage { Keys keys; Gates gates; T v[DC_TOKENS][VLD]; };
    struct Shared {
        Stage stage[DC_STAGES];
        float4 swap[2][DC_WALKERS][3][32];
        float most[DC_WALKERS][16];
    };
};

// What the two kernels share beside the rule's arguments: the records, [chunk][q/k head] and [chunk][head].  Chunks are
// numbered request after request, those of a request from its first token on; `chunks` is what the workspace has room for.
struct DcRecords { unsigned char* keys; unsigned char* gates; int items, chunks; };

// The number of chunks in front of request `item`, by all lanes of a warp.
__device__ __forceinline__ int dc_chunks_before(const int* __restrict__ item_qlen, int item, int lane) {
    int sum = 0;
    for (int i = lane; i < item; i += 32) sum += (max(item_qlen[i], 0) + DC_TOKENS - 1) / DC_TOKENS;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

constexpr int DC_MAKERS = 4;               // warps of a preparing block

// a warp per chunk and q/k head
template <typename T, int DK, bool WIDE>
__global__ void __launch_bounds__(32 * DC_MAKERS)
delta_records_kernel(const DeltaParams p, const DcRecords records) {
    using Sh = DcShape<T, DK>;
    constexpr int PARTS = Sh::PARTS, FOURS = DK / 32;          // 32 columns are a quad's eight each
    struct Scratch { float a[DC_TOKENS][DC_TOKENS + 4]; double g[DC_TOKENS]; float f[DC_TOKENS], beta[DC_TOKENS]; };
    __shared__ Scratch scratch[DC_MAKERS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    auto& own = scratch[warp];
    const int narrow_heads = p.heads / p.share;
    const long long unit = (long long)blockIdx.x * DC_MAKERS + warp;
    const int chunk = (int)(unit / narrow_heads), narrow = (int)(unit - (long long)chunk * narrow_heads);
    // the chunk's request and first token: 32 requests at a time
    int item = -1, place = 0;
    for (int i0 = 0, before = 0; i0 < records.items && item < 0; i0 += 32) {
        const int i = i0 + lane, have = i < records.items ? (max(p.item_qlen[i], 0) + DC_TOKENS - 1) / DC_TOKENS : 0;
        int upto = have;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += left;
        }
        const unsigned here = __ballot_sync(0xffffffffu, before + upto > chunk && before + upto - have <= chunk);
        if (here) {
            const int at = __ffs(here) - 1;
            item = i0 + at;
            place = chunk - __shfl_sync(0xffffffffu, before + upto - have, at);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const int slot = item >= 0 ? p.item_slots[item] : -1, count = item >= 0 ? p.item_qlen[item] : 0;
    const int first = item >= 0 ? p.item_qstart[item] + place * DC_TOKENS : 0, n = min(DC_TOKENS, count - place * DC_TOKENS);
    grid_dependency_wait();
    grid_dependents_go();
    if (slot < 0 || chunk >= records.chunks) return;           // beyond the step's chunks, or a padding entry
    const T* qkv = (const T*)p.qkv;
    // ---- q, k and the first head's gates on their way
    Raw8<T> kr[2][FOURS], qr[2][FOURS];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        const T* row = qkv + (size_t)(first + (r < n ? r : 0)) * p.ld + narrow * p.dim;
#pragma unroll
        for (int f = 0; f < FOURS; ++f) {
            const int d = f * 32 + t * 8, have = r < n ? p.dim - d : 0;
            kr[h][f] = dc_load8<WIDE>(row + p.k_off + d, have);
            qr[h][f] = dc_load8<WIDE>(row + p.q_off + d, have);
        }
    }
    const int i = lane & 15;                                   // the lane's token (twice per warp)
    float decay = 0.f, beta = 0.f;
    if (i < n) {
        decay = p.log_decay[(size_t)(first + i) * p.heads + narrow * p.share];
        beta = p.beta[(size_t)(first + i) * p.heads + narrow * p.share];
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
    auto* keys = reinterpret_cast<typename Sh::Keys*>(records.keys) + ((size_t)chunk * narrow_heads + narrow);
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int f = 0; f < FOURS; ++f) {
                const unsigned(&a)[4] = kh[part][h][f];
                const unsigned(&b)[4] = qh[part][h][f];
                *reinterpret_cast<uint4*>(&keys->k[part][g + 8 * h][f * 32 + t * 8]) = make_uint4(a[0], a[1], a[2], a[3]);
                *reinterpret_cast<uint4*>(&keys->q[part][g + 8 * h][f * 32 + t * 8]) = make_uint4(b[0], b[1], b[2], b[3]);
            }
    const int from = (lane & 7) * 4;                           // a lane of the quad that holds row lane & 7
    const float kf0 = __shfl_sync(0xffffffffu, kf[0], from), kf1 = __shfl_sync(0xffffffffu, kf[1], from);
    const float qf0 = __shfl_sync(0xffffffffu, qf[0], from), qf1 = __shfl_sync(0xffffffffu, qf[1], from);
    const float kfi = (lane & 8) ? kf1 : kf0, qfi = (lane & 8) ? qf1 : qf0;        // of token i
    if (lane < DC_TOKENS) own.f[lane] = kfi;
    // ---- the gates of every head that reads these q and k
#pragma unroll 1
    for (int z = 0; z < p.share; ++z) {
        const int head = narrow * p.share + z;
        auto* to = reinterpret_cast<typename Sh::Gates*>(records.gates) + ((size_t)chunk * p.heads + head);
        // sums of log_decay in 64 bits, so that a difference of two of them is as exact as its own terms
        double sum = decay < -1e4f ? -1e4 : (double)decay;     // (e^-10000 is zero)
#pragma unroll
        for (int o = 1; o < DC_TOKENS; o <<= 1) {
            const double left = __shfl_up_sync(0xffffffffu, sum, o, DC_TOKENS);
            if (i >= o) sum += left;
        }
        const double all = __shfl_sync(0xffffffffu, sum, DC_TOKENS - 1, DC_TOKENS);
        if (lane < DC_TOKENS) { own.g[lane] = sum; own.beta[lane] = beta; }
        const float fade = expf((float)sum);
        if (lane < DC_TOKENS) {
            to->before[lane] = fade * kfi; to->after[lane] = expf((float)(all - sum)) * kfi; to->query[lane] = qfi; to->fade[lane] = fade;
        }
        if (z + 1 < p.share && i < n) {                        // the next head's
            decay = p.log_decay[(size_t)(first + i) * p.heads + head + 1];
            beta = p.beta[(size_t)(first + i) * p.heads + head + 1];
        }
        __syncwarp();
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
                const float e0 = expf((float)(gr - g0)) * f0, e1 = expf((float)(gr - g1)) * f1;
                const float w0 = row >= col ? (qkt[0][j][2 * h] + qkt[1][j][2 * h]) * e0 : 0.f;
                const float w1 = row > col ? (qkt[0][j][2 * h + 1] + qkt[1][j][2 * h + 1]) * e1 : 0.f;
                unsigned high, low;
                dc_split(w0, w1, high, low);
                *reinterpret_cast<unsigned*>(&to->p[0][row][col]) = high;
                *reinterpret_cast<unsigned*>(&to->p[1][row][col]) = low;
                own.a[row][col] = row > col ? mine * (kkt[0][j][2 * h] + kkt[1][j][2 * h]) * e0 : 0.f;
                own.a[row][col + 1] = row > col + 1 ? mine * (kkt[0][j][2 * h + 1] + kkt[1][j][2 * h + 1]) * e1 : 0.f;
            }
        }
        __syncwarp();
        // row i of (I + A)^-1 in lane i (and again in lane i + 16): from x (I + A) = e_i, last column first
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
        bool finite = true;
#pragma unroll
        for (int j = 0; j < DC_TOKENS; ++j) {
            x[j] = j <= i ? x[j] * own.beta[j] : 0.f;
            finite = finite && fabsf(x[j]) < INFINITY;
        }
        const bool odd = !__all_sync(0xffffffffu, finite);
        if (lane == 0) to->odd[0] = odd ? __int_as_float(0x7fffffff) : 0.f;
        unsigned high[DC_TOKENS / 2], low[DC_TOKENS / 2];
#pragma unroll
        for (int j = 0; j < DC_TOKENS / 2; ++j) dc_split(x[2 * j], x[2 * j + 1], high[j], low[j]);
        // the two lanes that hold a row write one part each
        uint4* row = reinterpret_cast<uint4*>(&to->t[lane >> 4][i][0]);
        const bool second = lane >= 16;
        row[0] = second ? make_uint4(low[0], low[1], low[2], low[3]) : make_uint4(high[0], high[1], high[2], high[3]);
        row[1] = second ? make_uint4(low[4], low[5], low[6], low[7]) : make_uint4(high[4], high[5], high[6], high[7]);
        __syncwarp();
    }
}

__device__ __forceinline__ void dc_copy16(void* dst, const void* src, bool there) {
    const int bytes = there ? 16 : 0;                          // 0 source bytes: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dc_smem(dst)), "l"(src), "r"(bytes) : "memory");
}

enum { DC_MEET = 1, DC_PAIR = 2 };         // named barriers: all warps, and from DC_PAIR on the pairs'

// A fetching thread's share of the copies into the ring, chunk after chunk: the addresses move on by a chunk with every call.
// (Copied by the walkers themselves a chunk takes them 800 cycles more: their own reads of shared memory queue behind.)
template <typename T, int DK, bool WIDE>
struct DcFetch {
    using Sh = DcShape<T, DK>;
    using Stage = typename Sh::Stage;
    static constexpr int FETCHERS = 32 * DC_WALKERS;
    static constexpr int PER = 16 / sizeof(T), ACROSS = Sh::COLS / PER;          // 16-byte pieces of a row of v
    static constexpr int KEYS = sizeof(typename Sh::Keys) / 16, GATES = sizeof(typename Sh::Gates) / 16;
    const unsigned char* keys;
    const unsigned char* gates;
    const T* v;
    size_t keys_step, gates_step, v_step;
    int left, row, have;                                       // tokens from the next chunk on; the thread's row of v, its columns there

    __device__ __forceinline__ DcFetch(const DeltaParams& p, const DcRecords& records, int head, int col0, int t0, int count, int chunk0) {
        const int narrow_heads = p.heads / p.share, tid = threadIdx.x - FETCHERS;
        keys_step = (size_t)narrow_heads * sizeof(typename Sh::Keys);
        gates_step = (size_t)p.heads * sizeof(typename Sh::Gates);
        v_step = (size_t)DC_TOKENS * p.ld;
        keys = records.keys + chunk0 * keys_step + (size_t)(head / p.share) * sizeof(typename Sh::Keys) + tid * 16;
        gates = records.gates + chunk0 * gates_step + (size_t)head * sizeof(typename Sh::Gates) + tid * 16;
        row = WIDE ? tid / ACROSS : 0;
        const int d = WIDE ? (tid % ACROSS) * PER : 0;
        have = p.vdim - col0 - d;
        v = (const T*)p.qkv + (size_t)t0 * p.ld + p.v_off + (size_t)head * p.vdim + col0 + (WIDE && have > 0 ? d : 0);
        left = count;
    }
    __device__ __forceinline__ void next(const DeltaParams& p, Stage& st) {
        const int tid = threadIdx.x - FETCHERS;
        if (left > 0) {
#pragma unroll
            for (int i = 0; i < (KEYS + FETCHERS - 1) / FETCHERS; ++i)
                if ((i + 1) * FETCHERS <= KEYS || tid + i * FETCHERS < KEYS)
                    dc_copy16(reinterpret_cast<uint4*>(&st.keys) + tid + i * FETCHERS, keys + i * FETCHERS * 16, true);
#pragma unroll
            for (int i = 0; i < (GATES + FETCHERS - 1) / FETCHERS; ++i)
                if ((i + 1) * FETCHERS <= GATES || tid + i * FETCHERS < GATES)
                    dc_copy16(reinterpret_cast<uint4*>(&st.gates) + tid + i * FETCHERS, gates + i * FETCHERS * 16, true);
            if constexpr (WIDE) {
                constexpr int ROWS = FETCHERS / ACROSS;     // rows of v that the block's threads copy at once
#pragma unroll
                for (int r = 0; r < DC_TOKENS; r += ROWS) {
                    const bool there = r + row < left && have > 0;
                    if (r + row < DC_TOKENS)
                        dc_copy16(&st.v[r + row][(tid % ACROSS) * PER], v + (there ? (size_t)(r + row) * p.ld : 0), there);
                }
            } else {
                for (int e = tid; e < DC_TOKENS * Sh::COLS; e += FETCHERS) {
                    const int r = e / Sh::COLS, d = e % Sh::COLS;
                    st.v[r][d] = r < left && d < have ? v[(size_t)r * p.ld + d] : from_float<T>(0.f);
                }
            }
            keys += keys_step;
            gates += gates_step;
            left -= DC_TOKENS;
            if (left > 0) v += v_step;
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    }
};

// S0^T times a chunk's keys or queries, the state in two parts (in sums of their own: low parts are lost beside high ones)
template <int STEPS>
__device__ __forceinline__ void dc_state_product(float (&sum)[2][4], const unsigned (&high)[STEPS][4], const unsigned (&low)[STEPS][4],
                                                 const unsigned (&b)[STEPS][4]) {
    float lows[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[j][e] = lows[j][e] = 0.f;
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            dc_mma(sum[j], high[k], b[k][2 * j], b[k][2 * j + 1]);
            dc_mma(lows[j], low[k], b[k][2 * j], b[k][2 * j + 1]);
        }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; e += 2) dc_add2(sum[j][e], sum[j][e + 1], sum[j][e], sum[j][e + 1], lows[j][e], lows[j][e + 1]);
}

// a thread's v of one chunk as it is stored
template <typename T> struct DcValues;
template <> struct DcValues<bf16> {
    unsigned x[4];
    __device__ __forceinline__ void widen(float (&r)[2][4]) const {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                r[j][2 * h] = __uint_as_float(x[2 * j + h] << 16);
                r[j][2 * h + 1] = __uint_as_float(x[2 * j + h] & 0xffff0000u);
            }
    }
};
template <> struct DcValues<float> {
    float x[8];
    __device__ __forceinline__ void widen(float (&r)[2][4]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e >> 2][e & 3] = x[e];
    }
};

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
        for (int e = 0; e < 4; e += 2) dc_add2(u[j][e], u[j][e + 1], a[e], a[e + 1], b[e], b[e + 1]);
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

template <typename T, int DK, bool WIDE>
__global__ void __launch_bounds__(2 * 32 * DC_WALKERS, 2)
delta_walk_kernel(const DeltaParams p, const DcRecords records) {
    using Sh = DcShape<T, DK>;
    constexpr int PARTS = Sh::PARTS, SLICES = Sh::SLICES, TILES = DC_SLICE / 8, STEPS = DC_SLICE / 16;
    extern __shared__ __align__(16) unsigned char dc_raw[];
    auto& sm = *reinterpret_cast<typename Sh::Shared*>(dc_raw);
    const int head = blockIdx.y, item = blockIdx.z, col0 = blockIdx.x * Sh::COLS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = p.item_slots[item], count = p.item_qlen[item], t0 = p.item_qstart[item];
    if (slot < 0 || count <= 0) return;                        // a padding entry of a fixed-size batch
    const int chunks = (count + DC_TOKENS - 1) / DC_TOKENS;
    const int chunk0 = dc_chunks_before(p.item_qlen, item, lane);
    if (chunk0 + chunks > records.chunks) return;              // lists that name more tokens than there are
    // registers: two blocks of 256 threads have 128 each; the walkers' four warps take over most of the fetchers' (216 + 40)
    if (warp >= DC_WALKERS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");
        grid_dependency_wait();
        grid_dependents_go();
        DcFetch<T, DK, WIDE> fetch(p, records, head, col0, t0, count, chunk0);
        fetch.next(p, sm.stage[0]);
        fetch.next(p, sm.stage[1]);
        for (int c = 0; c <= chunks; ++c) {                    // (the last meeting is for a chunk that is not there)
            asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            dc_sync(DC_MEET, Sh::THREADS);                     // chunk c is there, and everybody is through with chunk c - 2:
            fetch.next(p, sm.stage[(c + 2) % DC_STAGES]);      // its stage takes chunk c + 2
        }
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
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
    float sigma[2] = {1.f, 1.f}, back[2] = {1.f, 1.f};         // of columns col and col + 8, and one over it
    unsigned sh[STEPS][4], sl[STEPS][4];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
    const int b_row = (lane & 7) + 8 * (lane >> 4), b_col = 8 * ((lane >> 3) & 1);      // ldmatrix, operand stored [n][k]
    const int bt_row = (lane & 7) + 8 * ((lane >> 3) & 1), bt_col = 8 * (lane >> 4);    // ... and [k][n]
    // two warps per 16 columns: each finishes the outputs of eight of the chunk's tokens
    constexpr int FINISH = SLICES > 1 ? 1 : 2;                 // tiles of eight tokens that a warp finishes
    const int tile0 = SLICES > 1 ? slice : 0;
    float* out = p.out + (size_t)t0 * p.heads * p.vdim + (size_t)head * p.vdim + col;
    const size_t width = (size_t)p.heads * p.vdim;
    const int left = p.vdim - col;                             // columns col and col + 8 are there
    // Operands of the next products are read well ahead of them, and sums that do not depend on one another are asked for
    // together: a warp has its scheduler nearly to itself, so what one instruction waits for, all wait for.
    unsigned bk[STEPS][4];                                     // K of the chunk (the first part), operand of S0^T k
    DcValues<T> v;                                             // its v, laid out as a tile of U
    auto ask = [&](const typename Sh::Stage& st) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) dc_ldmatrix(bk[k], &st.keys.k[0][b_row][row0 + 16 * k + b_col]);
        if constexpr (sizeof(T) == 2) {                        // tokens 0-7 of col, col + 8; tokens 8-15 of both
            dc_ldmatrix_trans(v.x, &st.v[(lane & 7) + 8 * (lane >> 4)][group * 16 + 8 * ((lane >> 3) & 1)]);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) v.x[4 * j + e] = st.v[8 * j + 2 * t + (e & 1)][group * 16 + g + 8 * (e >> 1)];
        }
    };
    dc_sync(DC_MEET, Sh::THREADS);                             // stage 0 is there
    ask(sm.stage[0]);

    for (int c = 0; c < chunks; ++c) {
        const auto& st = sm.stage[c % DC_STAGES];
        const int here = count - c * DC_TOKENS;                // tokens from the chunk's first on
        bool look = c % DC_REFRESH == 0, spoiled = false;
        int bad[2] = {DC_TOKENS, DC_TOKENS};
        float u[2][4], wq[FINISH][4];
        unsigned kt[STEPS][4];                                 // K again, operand of the new state
        for (int tries = 0;; ++tries) {
            if (look) {                                        // the columns' powers of two from the columns themselves
                float most[2], raw[2][4];
                v.widen(raw);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    most[h] = 0.f;
#pragma unroll
                    for (int n = 0; n < TILES; ++n) most[h] = fmaxf(most[h], fmaxf(fabsf(s[n][2 * h]), fabsf(s[n][2 * h + 1])));
                    most[h] *= back[h];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 2 * h; e < 2 * h + 2; ++e)        // (an infinite value must not move its column's power)
                            if (fabsf(raw[j][e]) < INFINITY) most[h] = fmaxf(most[h], fabsf(raw[j][e]));
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], o));
                }
                if (SLICES > 1) {
                    if (t == 0) { sm.most[warp][g] = most[0]; sm.most[warp][g + 8] = most[1]; }
                    dc_sync(DC_PAIR + group, 64);
                    most[0] = fmaxf(most[0], sm.most[warp ^ 1][g]);
                    most[1] = fmaxf(most[1], sm.most[warp ^ 1][g + 8]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int e = DC_SIZE - (((__float_as_int(most[h]) >> 23) & 255) - 127);
                    const float next = most[h] > 0.f ? dc_power(min(max(e, -100), 100)) : sigma[h];
                    const float factor = next * back[h];
                    sigma[h] = next;
                    back[h] = 1.f / next;
#pragma unroll
                    for (int n = 0; n < TILES; ++n) { s[n][2 * h] *= factor; s[n][2 * h + 1] *= factor; }
                }
#pragma unroll
                for (int k = 0; k < STEPS; ++k) dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
            }
            // ---- S0^T k and S0^T q of the warp's rows: 16 columns x 16 tokens
            unsigned bq[STEPS][4], th[4], tl[4];
            float wk[2][4], both[2][4];
#pragma unroll
            for (int k = 0; k < STEPS; ++k) dc_ldmatrix(bq[k], &st.keys.q[0][b_row][row0 + 16 * k + b_col]);
            dc_state_product<STEPS>(wk, sh, sl, bk);
            if (PARTS == 2) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    dc_ldmatrix(kt[k], &st.keys.k[PARTS - 1][b_row][row0 + 16 * k + b_col]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) dc_mma(wk[j], sh[k], kt[k][2 * j], kt[k][2 * j + 1]);
                }
            }
            if (SLICES > 1) {
                sm.swap[c & 1][warp][0][lane] = make_float4(wk[0][0], wk[0][1], wk[0][2], wk[0][3]);
                sm.swap[c & 1][warp][1][lane] = make_float4(wk[1][0], wk[1][1], wk[1][2], wk[1][3]);
            }
            dc_ldmatrix(th, &st.gates.t[0][b_row][b_col]);
            dc_ldmatrix(tl, &st.gates.t[1][b_row][b_col]);
            const float2 before0 = *reinterpret_cast<const float2*>(&st.gates.before[2 * t]);
            const float2 before1 = *reinterpret_cast<const float2*>(&st.gates.before[8 + 2 * t]);
            float size = st.gates.odd[0];                      // NaN where T is not finite
            dc_state_product<STEPS>(both, sh, sl, bq);
            if (PARTS == 2) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    dc_ldmatrix(kt[k], &st.keys.q[PARTS - 1][b_row][row0 + 16 * k + b_col]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) dc_mma(both[j], sh[k], kt[k][2 * j], kt[k][2 * j + 1]);
                }
            }
            if constexpr (SLICES > 1) {
                sm.swap[c & 1][warp][2][lane] = make_float4(slice ? both[0][0] : both[1][0], slice ? both[0][1] : both[1][1],
                                                            slice ? both[0][2] : both[1][2], slice ? both[0][3] : both[1][3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) wq[0][e] = slice ? both[1][e] : both[0][e];
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) wq[j % FINISH][e] = both[j][e];
            }
            // ---- one meeting per chunk: the halves' sums are there, and so is the next stage
            if (tries == 0) dc_sync(DC_MEET, Sh::THREADS);
            else if (SLICES > 1) dc_sync(DC_PAIR + group, 64);
            if (SLICES > 1) {
                float4 x[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) x[j] = sm.swap[c & 1][warp ^ 1][j][lane];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    dc_add2(wk[j][0], wk[j][1], wk[j][0], wk[j][1], x[j].x, x[j].y);
                    dc_add2(wk[j][2], wk[j][3], wk[j][2], wk[j][3], x[j].z, x[j].w);
                }
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) dc_ldmatrix_trans(kt[k], &st.keys.k[0][bt_row][row0 + 16 * k + bt_col]);
            // ---- R, U
            float r[2][4];
            v.widen(r);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 before = j ? before1 : before0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x, y;
                    dc_mul2(x, y, r[j][2 * h], r[j][2 * h + 1], sigma[h], sigma[h]);
                    dc_fma2(r[j][2 * h], r[j][2 * h + 1], -before.x, -before.y, wk[j][2 * h], wk[j][2 * h + 1], x, y);
                    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(size) : "f"(fabsf(r[j][2 * h])), "f"(fabsf(r[j][2 * h + 1])));
                }
            }
            unsigned rh[4], rl[4];
            dc_split_tiles(r[0], r[1], rh, rl);
            dc_solve(u, rh, rl, th, tl);
            if (!__any_sync(0xffffffffu, !(size < DC_MOST))) break;
            if (tries == 0) {                                  // (both warps of a pair have the same R and T)
                look = true;
                ask(st);
                continue;
            }
            // not a matter of size: something is not finite
            spoiled = true;
            dc_first_bad(r, t, bad);
            dc_leave_out(r, t, bad);
            dc_split_tiles(r[0], r[1], rh, rl);
            dc_solve(u, rh, rl, th, tl);
            dc_first_bad(u, t, bad);
            dc_leave_out(u, t, bad);
            break;
        }
        // ---- the new state
        unsigned uh[4], ul[4], zh[4], zl[4];
        const float2 after0 = *reinterpret_cast<const float2*>(&st.gates.after[2 * t]);
        const float2 after1 = *reinterpret_cast<const float2*>(&st.gates.after[8 + 2 * t]);
        const float decay = st.gates.fade[DC_TOKENS - 1];
        float faded[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 after = j ? after1 : after0;
#pragma unroll
            for (int e = 0; e < 4; e += 2) dc_mul2(faded[j][e], faded[j][e + 1], u[j][e], u[j][e + 1], after.x, after.y);
        }
        dc_split_tiles(faded[0], faded[1], uh, ul);
        float add[TILES][4];
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) add[n][e] = 0.f;
            dc_mma(add[n], ul, kt[n >> 1][2 * (n & 1)], kt[n >> 1][2 * (n & 1) + 1]);
        }
        if (PARTS == 2) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                unsigned b[4];
                dc_ldmatrix_trans(b, &st.keys.k[PARTS - 1][bt_row][row0 + 16 * k + bt_col]);
                dc_mma(add[2 * k], uh, b[0], b[1]);
                dc_mma(add[2 * k + 1], uh, b[2], b[3]);
            }
        }
#pragma unroll
        for (int n = 0; n < TILES; ++n) dc_mma(add[n], uh, kt[n >> 1][2 * (n & 1)], kt[n >> 1][2 * (n & 1) + 1]);
        dc_split_tiles(u[0], u[1], zh, zl);
        unsigned ph[4], pl[4];
        if constexpr (SLICES > 1) {                            // the eight tokens' rows: both inner halves, both parts
            dc_ldmatrix(ph, &st.gates.p[lane >> 4][8 * slice + (lane & 7)][b_col]);
            pl[0] = ph[2]; pl[1] = ph[3];
        } else {
            dc_ldmatrix(ph, &st.gates.p[0][b_row][b_col]);
            dc_ldmatrix(pl, &st.gates.p[1][b_row][b_col]);
        }
        if (SLICES > 1) {
            const float4 x = sm.swap[c & 1][warp ^ 1][2][lane];
            dc_add2(wq[0][0], wq[0][1], wq[0][0], wq[0][1], x.x, x.y);
            dc_add2(wq[0][2], wq[0][3], wq[0][2], wq[0][3], x.z, x.w);
        }
        float oa[FINISH][4], ob[FINISH][4];
#pragma unroll
        for (int j = 0; j < FINISH; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) oa[j][e] = ob[j][e] = 0.f;
            dc_mma(ob[j], zl, ph[2 * j], ph[2 * j + 1]);
            dc_mma(oa[j], zh, ph[2 * j], ph[2 * j + 1]);
            dc_mma(ob[j], zh, pl[2 * j], pl[2 * j + 1]);
        }
        if (c + 1 < chunks) ask(sm.stage[(c + 1) % DC_STAGES]);
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
#pragma unroll
            for (int n = 2 * k; n < 2 * k + 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    dc_fma2(s[n][e], s[n][e + 1], s[n][e], s[n][e + 1], decay, decay, add[n][e], add[n][e + 1]);
            dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
        }
        // ---- outputs: the chunk's start and its own tokens
#pragma unroll
        for (int j = 0; j < FINISH; ++j) {
            const int first = 8 * (tile0 + j) + 2 * t;
            const float2 fade = *reinterpret_cast<const float2*>(&st.gates.fade[first]);
            const float2 query = *reinterpret_cast<const float2*>(&st.gates.query[first]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x, y, fx, fy;
                dc_add2(x, y, oa[j][2 * h], oa[j][2 * h + 1], ob[j][2 * h], ob[j][2 * h + 1]);
                dc_fma2(x, y, fade.x, fade.y, wq[j][2 * h], wq[j][2 * h + 1], x, y);
                dc_mul2(fx, fy, query.x, query.y, back[h], back[h]);
                dc_mul2(x, y, x, y, fx, fy);
                if (spoiled) {
                    if (first >= bad[h]) x = __int_as_float(0x7fffffff);
                    if (first + 1 >= bad[h]) y = __int_as_float(0x7fffffff);
                }
                if (first < here && 8 * h < left) out[(size_t)first * width + 8 * h] = x;
                if (first + 1 < here && 8 * h < left) out[(size_t)(first + 1) * width + 8 * h] = y;
            }
        }
        out += (size_t)DC_TOKENS * width;
        if (spoiled) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (bad[h] < DC_TOKENS) {
#pragma unroll
                    for (int n = 0; n < TILES; ++n) s[n][2 * h] = s[n][2 * h + 1] = __int_as_float(0x7fffffff);
                }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) dc_split_tiles(s[2 * k], s[2 * k + 1], sh[k], sl[k]);
        }
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = row0 + 8 * n + 2 * t + (e & 1), v = col + 8 * (e >> 1);
            if (d < p.dim && v < p.vdim) state[(size_t)d * p.vdim + v] = s[n][e] * back[e >> 1];
        }
}

constexpr int DC_ALONE_BYTES = 120 * 1024;     // more than half of an SM's shared memory
static_assert(sizeof(DcShape<float, 128>::Shared) <= DC_ALONE_BYTES, "the largest shape");

template <typename T, int DK, bool WIDE>
static int launch_chunk(const DeltaParams& p, const DcRecords& records, int early, cudaStream_t stream) {
    using Sh = DcShape<T, DK>;
    auto kernel = delta_walk_kernel<T, DK, WIDE>;
    static int sms = 0;                        // per process and kernel; harmless if repeated
    if (sms == 0) {
        int device = 0, count = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DC_ALONE_BYTES);
        if (e != cudaSuccess) return (int)e;
        sms = count;
    }
    const long long units = (long long)records.chunks * (p.heads / p.share);
    const dim3 grid((p.vdim + Sh::COLS - 1) / Sh::COLS, p.heads, records.items);
    if (grid.y > 65535 || grid.z > 65535 || units > 0x7fffffffLL) return ERR_UNSUPPORTED;
    const int rc = launch_dependent_if(early, delta_records_kernel<T, DK, WIDE>, dim3((unsigned)((units + DC_MAKERS - 1) / DC_MAKERS)),
                                       dim3(32 * DC_MAKERS), 0, stream, p, records);
    if (rc != 0) return rc;
    // Two blocks on an SM take 2,200 cycles for a chunk of each, one alone 1,530: as many blocks as SMs had better not share any,
    // which they do if they start while the records' blocks still hold some (ask for more than half of the shared memory).
    const size_t smem = (long long)grid.x * grid.y * grid.z <= sms ? DC_ALONE_BYTES : sizeof(typename Sh::Shared);
    // the state is older than the records' kernel, which waits for whatever may have written it
    return launch_dependent(kernel, grid, dim3(Sh::THREADS), smem, stream, p, records);
}

template <typename T, int DK>
static int launch_chunk_any(const DeltaParams& p, int items, long long chunks, unsigned char* room, int early, cudaStream_t stream) {
    using Sh = DcShape<T, DK>;
    DcRecords records;
    records.keys = room;
    records.gates = room + (size_t)chunks * (p.heads / p.share) * sizeof(typename Sh::Keys);
    records.items = items;
    records.chunks = (int)chunks;
    const bool wide = p.ld % 8 == 0 && p.q_off % 8 == 0 && p.k_off % 8 == 0 && p.v_off % 8 == 0 && p.dim % 8 == 0 &&
                      p.vdim % 8 == 0 && (uintptr_t)p.qkv % 16 == 0;
    return wide ? launch_chunk<T, DK, true>(p, records, early, stream) : launch_chunk<T, DK, false>(p, records, early, stream);
}

static long long chunk_bytes(int heads, int share, int dim, int dtype) {
    const long long gates = (long long)heads * sizeof(DcShape<bf16, 64>::Gates), narrow = heads / share;
    if (dtype == DTYPE_F32) return gates + narrow * (dim <= 64 ? sizeof(DcShape<float, 64>::Keys) : sizeof(DcShape<float, 128>::Keys));
    return gates + narrow * (dim <= 64 ? sizeof(DcShape<bf16, 64>::Keys) : sizeof(DcShape<bf16, 128>::Keys));
}

// The chunked form; ERR_UNSUPPORTED where a head has more rows than it holds.  `room`: 16-byte aligned memory.
int delta_chunk(const DeltaParams& p, int items, int dtype, void* room, long long room_bytes, int early, cudaStream_t stream) {
    if (p.dim > DC_MAX_DIM) return ERR_UNSUPPORTED;
    const long long chunks = room_bytes / chunk_bytes(p.heads, p.share, p.dim, dtype);
    if (!room || (uintptr_t)room % 16 != 0 || chunks <= 0 || chunks > 0x7fffffffLL) return ERR_BAD_ARGUMENT;
    unsigned char* at = (unsigned char*)room;
    if (dtype == DTYPE_F32)
        return p.dim <= 64 ? launch_chunk_any<float, 64>(p, items, chunks, at, early, stream)
                           : launch_chunk_any<float, 128>(p, items, chunks, at, early, stream);
    return p.dim <= 64 ? launch_chunk_any<bf16, 64>(p, items, chunks, at, early, stream)
                       : launch_chunk_any<bf16, 128>(p, items, chunks, at, early, stream);
}

}  // namespace fsie

extern "C" {

int fsie_delta_chunk_max_dim() { return fsie::DC_MAX_DIM; }

int fsie_delta_chunk_tokens() { return fsie::DC_TOKENS; }

// bytes of the workspace per chunk
int fsie_delta_chunk_bytes(int heads, int share, int dim, int dtype) { return (int)fsie::chunk_bytes(heads, share, dim, dtype); }

}  // extern "C"
