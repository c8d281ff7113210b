// The gated delta rule (formulas in delta_rule.cu) for prompts: chunks of 32 tokens on the tensor cores, 32-bit results.
//
// Inside a chunk that starts from state S0, with G_i = sum of log_decay over the chunk's tokens up to i and k, q divided by
// their lengths,
//
//   R_i = b (v_i - e^(G_i) S0^T k_i)                  what the chunk's start leaves to be stored; b: a power of two, above every beta
//   U   = T R,  T = (I + A)^-1 diag(beta) / b         A_ij = beta_i (k_i.k_j) e^(G_i - G_j) for j < i, else 0
//   o_i = scale (e^(G_i) S0^T q_i + sum_(j <= i) (q_i.k_j) e^(G_i - G_j) u_j)
//   S   = e^(G_31) S0 + sum_j e^(G_31 - G_j) k_j u_j^T
//
// A chunk is a chain - S0^T k, R, U, S - whose steps wait for one another, and a request's heads give a warp of its own to every
// 16 columns and 64 rows of S only, so what bounds a prompt is the chain's latency.  A longer chunk puts more independent
// instructions into every step; it adds to the two products that grow with the chunk (T R and the sum over u_j), by halves only
// where the blocks of T above the diagonal are left out.
//
// Measured (bfloat16, heads of 128 x 128): 8,192 tokens of 16 q/k and 32 heads 358 us - records 61, walk 313, a part of it beside
// the records -, against 42 for their bytes; 0.7 TB/s.  A chunk of a block that has its SM alone takes 2,400 cycles for 984 of tensor
// instructions (123 of 8 cycles per warp), and no step of the chain stands out; with two blocks on an SM 3,500 for both, so that
// four prompts of 2,048 tokens of 32 heads (512 blocks in 296 places) take 335 us: records 83, walk 273.  Chunks of 16 tokens took
// 530 us for the 8,192 when those of 32, in their first form, took 443.
//
// Precision.  States and outputs are 32-bit results, so no operand may be rounded to 11 bits.  q and k (bfloat16, 8 bits)
// scaled by a power of two to a length of about one are exact in half precision (down to 2^-17 of the length; what is smaller is cut
// at 2^-24 of it); what is 32-bit - the state, R, U, T and the
// weights of u_j - goes into the instructions as the sum of two half-precision numbers (22 bits), products of two low parts left
// out.  The state itself stays in 32-bit registers and the instructions only ever sum up one chunk (their running sums are
// truncated, not rounded).  float32 storage: q and k are two parts as well.
//
// Range.  Half precision has little of it: a pair ends at 2^-25, 22 bits below a number of 2^-3.  Where a sum of its own takes the low
// parts' products they go in 2^11 times as large (DC_LOW), so that the pairs of R, U, T and the weights end at 2^-36; T and the weights
// are stored 2^11 and 2^14 times as large besides.  Every column of the state (a row of the transposed tiles below) has a power of two,
// `sigma`, chosen in a look at the largest numbers of the column and of the first chunk's b v, and anew, the chunk's sums taken again,
// when a chunk is out of range: when a number of U is too large, when next to nothing of a column's is taken into the state, or when next
// to nothing is stored at some token and the column holds no more (DC_LEAST...).  Where that is so even right behind a look - a large
// value that is forgotten within its chunk, small ones in front of a large one -, where a state is small beside the values, or where
// something is not finite, the warps of the 16 columns walk the chunk token by token in 32 bits, as the recurrence is written.  Such a
// chunk takes some nine times as long (8,192 tokens of 16 q/k and 32 heads, all so, 3.0 ms; values with e^(2 N(0, 1)) for a token's size 460
// us, half of them zeros 460, a column of zeros, decays of e^-4 or steps of 0.001 take nothing more).
//
// Two kernels.  The first prepares all chunks side by side, a block per chunk and q/k head: q and k in half precision, T by
// substitution, the weights of u_j, the gates' factors, as records in the workspace that lie as the second kernel's shared
// memory holds them.  The second walks a head's chunks, a block for every 16 to 64 value columns, four more warps keeping
// the records and v of the next chunks on their way into a ring of stages; all meet once per chunk.  (One kernel in which four
// more warps per block prepared the chunks took 951 us for 8,192 tokens of 32 heads, the first form of the two 691: every block
// of value columns prepared them again, and the two roles' code did not fit the instruction cache together.)
//
// Layout.  A warp of the second kernel owns 16 value columns x 64 or 32 rows of S, transposed: S^T is the 16-row operand of S0^T k
// and S0^T q, the accumulator of S0^T k is (after R) the operand of the next product in the registers where it lies, and the
// new sums end up where S lies.  Heads of more rows take two or four warps per 16 columns, which swap their rows' sums
// of S0^T k through shared memory, in the chunk's one meeting; those of S0^T q the fetching warps add up.
//
// Values that are not finite spoil their column from their token on and nothing else, as in the recurrence: a product with a zero
// of T would spoil the tokens before, so such chunks, noticed by U, are walked token by token.
#include "common.cuh"
#include "delta_rule.cuh"
#include "tma.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace fsie {

constexpr int DC_TOKENS = 32;              // tokens of a chunk
constexpr int DC_TILES = DC_TOKENS / 8;    // ... in tiles of eight
constexpr int DC_STAGES = 3;               // stages of the ring: the chunk's, the next one's and one on its way
constexpr int DC_WALKERS = 4;              // warps that walk a block's chunks
constexpr int DC_FETCHERS = 128;           // threads that copy
constexpr int DC_MAX_DIM = 128;
constexpr int DC_SIZE = 12;                // a look brings the largest number of a column to 2^12 .. 2^13
constexpr int DC_FIRST = -100, DC_LAST = 115;        // ... with powers of two from the one to the other
constexpr int DC_DOWN = 3;                 // ... or, where R or U are then too large, to 2^-DC_DOWN of that
constexpr float DC_LOW = 2048.f;           // on a low part whose products have a sum of their own
constexpr float DC_T_SCALE = DC_LOW;       // on T, whose numbers are below beta <= 2, as its record has it
constexpr float DC_P_SCALE = 16384.f;      // ... and on the weights of u_j, which are below 1
constexpr int DC_TLD = 16 + 8;             // padded rows of a 16 x 16 block in scratch
constexpr int DC_ALD = 16 + 4;             // ... of floats
// Numbers of U, times sigma, are below this: u with a factor of at most 2 then fits half precision.  (Those of R do if U is finite.)
// Right behind a look R is at most 2^13 (1 + sqrt(128)), 12,300 with DC_DOWN.
constexpr float DC_MOST = 32000.f;
// What a column holds at a token, times sigma, is no less than this: R and U, as pairs, end at 2^-36, and what the weights' pairs leave
// of a number of DC_MOST at 2^-32.
constexpr float DC_LEAST = 1.f / 8192;
// ... and the state in front of a chunk no less than this: its pairs end at 2^-25, a rounding there (2^-25.8, the mean square) is nine
// units of 2^-24.  What the chunk leaves: this times the root of the number of tokens that have not faded by then, whose pairs
// end at 2^-25 as well; six for 32, and DC_ENOUGH is enough in any case.
constexpr float DC_LEAST_STATE = 1.f / 32, DC_ENOUGH = 1.f / 4;
static_assert(DC_ENOUGH == DC_LEAST * DC_T_SCALE, "one register for both");

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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a * b: the first of a sum
__device__ __forceinline__ void dc_mma0(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void dc_mma_if(bool first, float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if (first) dc_mma0(d, a, b0, b1);
    else dc_mma(d, a, b0, b1);
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
// the same from x and y times DC_LOW, the low part times DC_LOW
__device__ __forceinline__ void dc_split_far(float x, float y, unsigned& high, unsigned& low) {
    float hx, hy;
    dc_mul2(hx, hy, x, y, 1.f / DC_LOW, 1.f / DC_LOW);
    const __half2 h = __floats2half2_rn(hx, hy);
    const float2 f = __half22float2(h);
    high = dc_bits(h);
    dc_fma2(hx, hy, f.x, f.y, -DC_LOW, -DC_LOW, x, y);
    low = dc_bits(__floats2half2_rn(hx, hy));
}
// the 16 x 16 operand of two neighbouring accumulator tiles, in two parts
__device__ __forceinline__ void dc_split_tiles(const float (&x)[4], const float (&y)[4], unsigned (&high)[4], unsigned (&low)[4]) {
    dc_split(x[0], x[1], high[0], low[0]);
    dc_split(x[2], x[3], high[1], low[1]);
    dc_split(y[0], y[1], high[2], low[2]);
    dc_split(y[2], y[3], high[3], low[3]);
}
__device__ __forceinline__ void dc_split_tiles_far(const float (&x)[4], const float (&y)[4], unsigned (&high)[4], unsigned (&low)[4]) {
    dc_split_far(x[0], x[1], high[0], low[0]);
    dc_split_far(x[2], x[3], high[1], low[1]);
    dc_split_far(y[0], y[1], high[2], low[2]);
    dc_split_far(y[2], y[3], high[3], low[3]);
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

// A row of a 16 x 16 block is two pieces of 16 bytes, in the other order in every second four rows: ldmatrix without bank conflicts.
__device__ __forceinline__ int dc_piece(int row, int piece) { return 8 * (piece ^ ((row >> 2) & 1)); }

// T and the weights of u_j are lower triangular: of their four 16 x 16 blocks those at (0, 0), (1, 0) and (1, 1) are kept.
template <typename T, int DK>
struct DcRecord {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;       // half-precision numbers that hold a stored one
    static constexpr int KLD = DK + 8;                         // padded row of q and k
    struct alignas(16) Keys { __half k[PARTS][DC_TOKENS][KLD], q[PARTS][DC_TOKENS][KLD]; };
    struct alignas(16) Gates {
        __half t[2][3][16][16], p[2][3][16][16];               // T and the weights of u_j, two parts each; dc_piece()
        float before[DC_TOKENS];          // on S0^T k: b, e^(G_i), the key's length, the power of two, DC_LOW
        float after[DC_TOKENS];           // on u_j in the new state: e^(G_31 - G_j), ..., one over DC_T_SCALE
        float query[DC_TOKENS];           // on an output: scale, the query's length, the power of two, one over DC_P_SCALE
        float fade[DC_TOKENS];            // e^(G_i), times DC_P_SCALE, as the weights of u_j are
        float key[DC_TOKENS], decay[DC_TOKENS], beta[DC_TOKENS];        // the key's length, the power of two; e^log_decay; beta
        float above[4];                   // b
    };
};

// SLICE: rows of S (columns of k) per warp
template <typename T, int DK, int SLICE>
struct DcShape : DcRecord<T, DK> {
    static constexpr int SLICES = DK / SLICE;                  // warps that share 16 value columns
    static constexpr int GROUPS = DC_WALKERS / SLICES;         // groups of 16 value columns
    static constexpr int COLS = 16 * GROUPS;                   // value columns of a block
    static constexpr int VLD = COLS + (sizeof(T) == 4 ? 4 : 0);         // row of v; bfloat16: v_piece()
    static constexpr int OLD = COLS + 4;                       // padded row of outputs
    static constexpr int THREADS = 32 * DC_WALKERS + DC_FETCHERS;
    static constexpr int WRITES = DC_TOKENS * COLS / 4 / DC_FETCHERS;       // rows of four outputs that a fetching thread writes
    static constexpr int FINISH = DC_TILES / SLICES;           // tiles of eight tokens whose outputs a warp finishes
    // Place of a row's 16-byte piece of bfloat16 v: in another order in every row, ldmatrix without bank conflicts.
    static __device__ __forceinline__ int v_piece(int row, int piece) { return piece ^ (COLS == 16 ? (row >> 2) & 1 : COLS == 32 ? (row >> 1) & 3 : row & 7); }
    struct alignas(16) Stage { typename DcRecord<T, DK>::Keys keys; typename DcRecord<T, DK>::Gates gates; T v[DC_TOKENS][VLD]; };
    struct Shared {
        Stage stage[DC_STAGES];
        float4 swap[2][SLICES > 1 ? DC_WALKERS : 1][DC_TILES][32];      // S0^T k of a warp's rows
        float out[2][SLICES][DC_TOKENS][OLD];      // a chunk's outputs without the factors, a summand per warp of the 16 columns
        float back[2][COLS];                       // what its columns are still to be multiplied by
        float most[2][DC_WALKERS][16];             // of looks; of the search for what is too small
        uint64_t full[DC_STAGES];                  // a stage's records are there
        int lost;                                  // ... or were waited for in vain
    };
};

// What the two kernels share beside the rule's arguments: the records, [chunk][q/k head] and [chunk][head].  Chunks are
// numbered request after request, those of a request from its first token on; `chunks` is what the workspace has room for.
struct DcRecords { unsigned char* keys; unsigned char* gates; int items, longer, chunks; };    // longer: a bound of the requests that have chunks

// A request's chunks; none for those of less than `least` tokens.
__device__ __forceinline__ int dc_chunks(int tokens, int least) { return tokens < least ? 0 : (tokens + DC_TOKENS - 1) / DC_TOKENS; }

// The request that is the `rank`-th with chunks, -1 if there are not so many, and the chunks in front of it; by all lanes of a warp.
__device__ __forceinline__ int dc_find(const int* __restrict__ item_qlen, int items, int rank, int least, int lane, int& before) {
    before = 0;
    for (int i0 = 0; i0 < items; i0 += 32) {
        const int have = i0 + lane < items ? dc_chunks(item_qlen[i0 + lane], least) : 0;
        const unsigned with = __ballot_sync(0xffffffffu, have > 0);
        const unsigned here = __ballot_sync(0xffffffffu, have > 0 && __popc(with & ((1u << lane) - 1)) == rank);
        const int at = here ? __ffs(here) - 1 : 32;
        before += __reduce_add_sync(0xffffffffu, lane < at ? have : 0);
        if (here) return i0 + at;
        rank -= __popc(with);
    }
    return -1;
}

// A product of two 16 x 16 matrices in two parts each, low ones times DC_LOW: sum += a b, b's operand registers as ldmatrix gives them.
__device__ __forceinline__ void dc_product(float (&sum)[2][4], const unsigned (&ah)[4], const unsigned (&al)[4], const unsigned (&bh)[4],
                                           const unsigned (&bl)[4]) {
    float low[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) low[j][e] = 0.f;
        dc_mma(low[j], al, bh[2 * j], bh[2 * j + 1]);
        dc_mma(sum[j], ah, bh[2 * j], bh[2 * j + 1]);
        dc_mma(low[j], ah, bl[2 * j], bl[2 * j + 1]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[j][e] = fmaf(low[j][e], 1.f / DC_LOW, sum[j][e]);
}

template <typename T, int DK>
struct DcMaker {                           // a preparing block's shared memory: the records as they go out, and scratch
    typename DcRecord<T, DK>::Keys keys;
    typename DcRecord<T, DK>::Gates gates;
    float a[2][16 * DC_ALD + 16];          // A's blocks on the diagonal; the two are read at once, from other banks
    __half w[2][16][DC_TLD];
    double g[DC_TOKENS];
    float kf[DC_TOKENS], qf[DC_TOKENS], beta[DC_TOKENS], share[DC_TOKENS], above;     // share: beta / b
};

__device__ __forceinline__ void dc_copy_out(void* to, const void* from, int bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(to), "r"(dc_smem(from)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}

// A block of four warps per chunk and q/k head: they take eight tokens' q and k each, then three of them one block of the
// products and weights each, the fourth the gates' sums.  (One warp for all of it held as much shared memory and left seven warps
// on an SM.)  8,192 tokens of 32 heads of 128 columns: 83 us, 336 MB read and written, 4.0 TB/s; 8,192 tokens of 16 q/k and 32 heads
// 61 us.  A block is a chain of nine steps behind barriers (7,300 cycles alone, 20,000 among others), shared memory is busy 63 % of
// the time, and five blocks to an SM beat six and seven (77 us against 80 and 96, before the low parts had a range of their own).
constexpr int DC_MAKERS = 4;

template <typename T, int DK, bool WIDE>
__global__ void __launch_bounds__(32 * DC_MAKERS, sizeof(T) == 2 ? 5 : 4)
delta_records_kernel(const DeltaParams p, const DcRecords records) {
    using Sh = DcRecord<T, DK>;
    constexpr int PARTS = Sh::PARTS, FOURS = DK / 32;          // 32 columns are a quad's eight each
    extern __shared__ __align__(16) unsigned char dc_raw[];
    auto& own = *reinterpret_cast<DcMaker<T, DK>*>(dc_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int narrow_heads = p.heads / p.share;
    const int chunk = blockIdx.x / narrow_heads, narrow = blockIdx.x - chunk * narrow_heads;
    // the chunk's request and first token: 32 requests at a time
    int slot = -1, count = 0, first = 0, place = 0;
    for (int i0 = 0, before = 0; i0 < records.items; i0 += 32) {
        const int i = i0 + lane, last = records.items - 1;     // (read all at once: they come from far)
        const int tokens = p.item_qlen[min(i, last)], its_slot = p.item_slots[min(i, last)], its_first = p.item_qstart[min(i, last)];
        const int have = i <= last ? dc_chunks(tokens, p.least) : 0;
        int upto = have;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += left;
        }
        const unsigned here = __ballot_sync(0xffffffffu, before + upto > chunk && before + upto - have <= chunk);
        if (here) {
            const int at = __ffs(here) - 1;
            place = chunk - __shfl_sync(0xffffffffu, before + upto - have, at);
            slot = __shfl_sync(0xffffffffu, its_slot, at);
            count = __shfl_sync(0xffffffffu, tokens, at);
            first = __shfl_sync(0xffffffffu, its_first, at) + place * DC_TOKENS;
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const int n = min(DC_TOKENS, count - place * DC_TOKENS);
    grid_dependency_wait();
    if (p.go && first_block() && threadIdx.x == 0) delta_release(p.go, 0);
    grid_dependents_go();
    if (slot < 0 || chunk >= records.chunks) return;           // beyond the step's chunks, or a padding entry
    float decay = 0.f, beta = 0.f;                             // of the lane's token, the first head's
    if (warp == 3 && lane < n) {
        decay = p.log_decay[(size_t)(first + lane) * p.heads + narrow * p.share];
        beta = p.beta[(size_t)(first + lane) * p.heads + narrow * p.share];
    }
    // ---- q and k, a quad per token: their lengths, a power of two that brings each below one, both in half precision
    {
        const int r = 8 * warp + g;
        const T* row = (const T*)p.qkv + (size_t)(first + (r < n ? r : 0)) * p.ld + narrow * p.dim;
        Raw8<T> raw[2][FOURS];
#pragma unroll
        for (int f = 0; f < FOURS; ++f) {
            const int d = f * 32 + t * 8, have = r < n ? p.dim - d : 0;
            raw[0][f] = dc_load8<WIDE>(row + p.k_off + d, have);
            raw[1][f] = dc_load8<WIDE>(row + p.q_off + d, have);
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __half* to = which ? own.keys.q[0][r] : own.keys.k[0][r];          // the second part's row comes DC_TOKENS later
            float sum = 0.f, x[8];
#pragma unroll
            for (int f = 0; f < FOURS; ++f) {
                dc_widen(raw[which][f], x);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int e = (((__float_as_int(sum) >> 23) & 255) - 125) >> 1;
            const float scale = dc_power(-e);
#pragma unroll
            for (int f = 0; f < FOURS; ++f) {
                dc_widen(raw[which][f], x);
                unsigned high[4], low[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (PARTS == 2) dc_split(x[2 * i] * scale, x[2 * i + 1] * scale, high[i], low[i]);
                    else high[i] = dc_bits(__floats2half2_rn(x[2 * i] * scale, x[2 * i + 1] * scale));
                }
                *reinterpret_cast<uint4*>(to + f * 32 + t * 8) = make_uint4(high[0], high[1], high[2], high[3]);
                if (PARTS == 2)
                    *reinterpret_cast<uint4*>(to + DC_TOKENS * Sh::KLD + f * 32 + t * 8) = make_uint4(low[0], low[1], low[2], low[3]);
            }
            if (t == 0) (which ? own.qf : own.kf)[r] = (which ? p.scale : 1.f) * (dc_power(e) / sqrtf(sum + p.eps));
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // generic writes before async-proxy reads
    __syncthreads();
    if (threadIdx.x == 96)
        dc_copy_out(records.keys + ((size_t)chunk * narrow_heads + narrow) * sizeof(typename Sh::Keys), &own.keys, sizeof(typename Sh::Keys));
    // ---- K K^T and Q K^T: warp 0 block (0, 0), warp 1 block (1, 0), warp 2 block (1, 1)
    const int rows = warp == 0 ? 0 : 16, cols = warp == 2 ? 16 : 0;
    float kkt[2][4], qkt[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) kkt[j][e] = qkt[j][e] = 0.f;
    const int a_row = lane & 15, a_col = 8 * (lane >> 4);      // ldmatrix, 16-row operand; its registers 0, 2 and 1, 3 are an 8-column one's
    const int bt_row = (lane & 7) + 8 * ((lane >> 3) & 1), bt_col = 8 * (lane >> 4);   // ldmatrix.trans, operand stored [k][n]
    if (warp < 3) {
#pragma unroll 4
        for (int d = 0; d < DK; d += 16) {
#pragma unroll
            for (int pb = 0; pb < PARTS; ++pb) {
                unsigned kb[4];
                dc_ldmatrix(kb, &own.keys.k[pb][cols + a_row][d + a_col]);
#pragma unroll
                for (int pa = 0; pa + pb < PARTS; ++pa) {
                    unsigned ka[4], qa[4];
                    dc_ldmatrix(ka, &own.keys.k[pa][rows + a_row][d + a_col]);
                    dc_ldmatrix(qa, &own.keys.q[pa][rows + a_row][d + a_col]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        dc_mma(kkt[j], ka, kb[j], kb[2 + j]);
                        dc_mma(qkt[j], qa, kb[j], kb[2 + j]);
                    }
                }
            }
        }
    }
    // ---- the gates of every head that reads these q and k
#pragma unroll 1
    for (int z = 0; z < p.share; ++z) {
        const int head = narrow * p.share + z;
        if (warp == 3) {
            // sums of log_decay in 64 bits, so that a difference of two of them is as exact as its own terms
            double sum = decay < -1e4f ? -1e4 : (double)decay;       // (e^-10000 is zero)
#pragma unroll
            for (int o = 1; o < DC_TOKENS; o <<= 1) {
                const double left = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += left;
            }
            const double all = __shfl_sync(0xffffffffu, sum, DC_TOKENS - 1);
            const float kf = own.kf[lane], fade = expf((float)sum);
            // b: 2^(n + 1) for a largest beta from 2^n on; 1 where that is nothing or not finite
            const unsigned largest = __reduce_max_sync(0xffffffffu, __float_as_uint(beta) & 0x7fffffffu) >> 23;
            const float above = largest > 0 && largest < 253 ? dc_power((int)largest - 126) : 1.f;
            if (lane == 0) own.above = above;
            own.g[lane] = sum;
            own.share[lane] = beta / above;
            own.beta[lane] = beta;
            if (z > 0) {                                       // the last head's record has left
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
                __syncwarp();
            }
            own.gates.before[lane] = fade * kf * (above * DC_LOW);
            own.gates.after[lane] = expf((float)(all - sum)) * kf * (1.f / DC_T_SCALE);
            own.gates.query[lane] = own.qf[lane] * (1.f / DC_P_SCALE);
            own.gates.fade[lane] = fade * DC_P_SCALE;
            own.gates.key[lane] = kf;
            own.gates.decay[lane] = expf(decay);
            own.gates.beta[lane] = beta;
            if (lane < 4) own.gates.above[lane] = above;
            if (z + 1 < p.share && lane < n) {                 // the next head's
                decay = p.log_decay[(size_t)(first + lane) * p.heads + head + 1];
                beta = p.beta[(size_t)(first + lane) * p.heads + head + 1];
            }
        }
        __syncthreads();
        float below[2][4];                                     // warp 1: block (1, 0) of A without beta
        if (warp < 3) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int bc = 8 * j + 2 * t, col = cols + bc;
                const double g0 = own.g[col], g1 = own.g[col + 1];
                const float f0 = own.kf[col], f1 = own.kf[col + 1];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int br = g + 8 * h, row = rows + br;
                    const double gr = own.g[row];
                    const float e0 = expf((float)(gr - g0)) * f0, e1 = expf((float)(gr - g1)) * f1;
                    unsigned high, low;
                    dc_split_far(row >= col ? qkt[j][2 * h] * e0 * (DC_P_SCALE * DC_LOW) : 0.f, row > col ? qkt[j][2 * h + 1] * e1 * (DC_P_SCALE * DC_LOW) : 0.f, high, low);
                    *reinterpret_cast<unsigned*>(&own.gates.p[0][warp][br][dc_piece(br, j) + 2 * t]) = high;
                    *reinterpret_cast<unsigned*>(&own.gates.p[1][warp][br][dc_piece(br, j) + 2 * t]) = low;
                    const float x = own.kf[row] * kkt[j][2 * h] * e0, y = own.kf[row] * kkt[j][2 * h + 1] * e1;
                    below[j][2 * h] = x; below[j][2 * h + 1] = y;
                    if (warp != 1) {
                        // (one that is not finite is left out: its token's R or beta is not finite either, and T has that)
                        const float bx = own.beta[row] * x, by = own.beta[row] * y;
                        own.a[warp / 2][br * DC_ALD + bc] = row > col && fabsf(bx) < INFINITY ? bx : 0.f;
                        own.a[warp / 2][br * DC_ALD + bc + 1] = row > col + 1 && fabsf(by) < INFINITY ? by : 0.f;
                    }
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            // blocks (0, 0) and (1, 1) of T: row i of (I + A)^-1 in a lane, from x (I + A) = e_i, last column first
            const int i = lane & 15, m = lane >> 4;
            float x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = i == j ? 1.f : 0.f;
#pragma unroll
            for (int l = 15; l >= 1; --l) {
                const float xl = l <= i ? -x[l] : 0.f;
#pragma unroll
                for (int j = 0; j < l; j += 4) {               // (A is zero on the diagonal and beyond)
                    const float4 a = *reinterpret_cast<const float4*>(&own.a[m][l * DC_ALD + j]);
                    x[j] = fmaf(xl, a.x, x[j]); x[j + 1] = fmaf(xl, a.y, x[j + 1]);
                    x[j + 2] = fmaf(xl, a.z, x[j + 2]); x[j + 3] = fmaf(xl, a.w, x[j + 3]);
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = j <= i ? x[j] * own.share[16 * m + j] : 0.f;
            unsigned high[8], low[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) dc_split_far(x[2 * j] * (DC_T_SCALE * DC_LOW), x[2 * j + 1] * (DC_T_SCALE * DC_LOW), high[j], low[j]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                *reinterpret_cast<uint4*>(&own.gates.t[0][2 * m][i][dc_piece(i, j)]) = make_uint4(high[4 * j], high[4 * j + 1], high[4 * j + 2], high[4 * j + 3]);
                *reinterpret_cast<uint4*>(&own.gates.t[1][2 * m][i][dc_piece(i, j)]) = make_uint4(low[4 * j], low[4 * j + 1], low[4 * j + 2], low[4 * j + 3]);
            }
        }
        __syncthreads();
        if (warp == 1) {
            // block (1, 0): -T_11 b (A_10 / beta) T_00, beta / b being in T_11; A / beta is below 1 and the second product's numbers, 16
            // summands, below 64: both go in DC_INNER times as large
            constexpr float DC_INNER = 512.f;
            unsigned ah[4], al[4], bh[4], bl[4];
            float w[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[j][e] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) below[j][e] *= DC_INNER * DC_LOW;
            dc_split_tiles_far(below[0], below[1], ah, al);
            dc_ldmatrix_trans(bh, &own.gates.t[0][0][bt_row][dc_piece(bt_row, lane >> 4)]);
            dc_ldmatrix_trans(bl, &own.gates.t[1][0][bt_row][dc_piece(bt_row, lane >> 4)]);
            dc_product(w, ah, al, bh, bl);
            // (one that is not finite must not reach rows above its own)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float x = w[j][2 * h], y = w[j][2 * h + 1];      // (T has DC_T_SCALE, which is DC_LOW)
                    unsigned high, low;
                    dc_split_far(fabsf(x) < INFINITY ? -x : 0.f, fabsf(y) < INFINITY ? -y : 0.f, high, low);
                    *reinterpret_cast<unsigned*>(&own.w[0][g + 8 * h][8 * j + 2 * t]) = high;
                    *reinterpret_cast<unsigned*>(&own.w[1][g + 8 * h][8 * j + 2 * t]) = low;
                }
            __syncwarp();
            dc_ldmatrix(ah, &own.gates.t[0][2][a_row][dc_piece(a_row, lane >> 4)]);
            dc_ldmatrix(al, &own.gates.t[1][2][a_row][dc_piece(a_row, lane >> 4)]);
            dc_ldmatrix_trans(bh, &own.w[0][bt_row][bt_col]);
            dc_ldmatrix_trans(bl, &own.w[1][bt_row][bt_col]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[j][e] = 0.f;
            dc_product(w, ah, al, bh, bl);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned high, low;
                    dc_split_far(w[j][2 * h] * (own.above * (DC_LOW / DC_INNER)), w[j][2 * h + 1] * (own.above * (DC_LOW / DC_INNER)), high, low);
                    *reinterpret_cast<unsigned*>(&own.gates.t[0][1][g + 8 * h][dc_piece(g, j) + 2 * t]) = high;
                    *reinterpret_cast<unsigned*>(&own.gates.t[1][1][g + 8 * h][dc_piece(g, j) + 2 * t]) = low;
                }
        }
        if (n < DC_TOKENS) {
            // Tokens that are not there have the last one's row of T, so that U repeats its value: nothing is out of range for their sake.
            // (Their keys are zero and no output reads them.)
            __syncthreads();
            const int last = n - 1;
            for (int x = threadIdx.x; x < 8 * (DC_TOKENS - n); x += 32 * DC_MAKERS) {
                const int row = n + (x >> 3), part = (x >> 2) & 1, right = (x >> 1) & 1, piece = x & 1;       // columns 0 to 15, 16 to 31
                if (row < 16 && right) continue;
                uint4 from = make_uint4(0, 0, 0, 0);
                if (last >= 16 || !right)
                    from = *reinterpret_cast<const uint4*>(&own.gates.t[part][last < 16 ? 0 : 1 + right][last & 15][dc_piece(last & 15, piece)]);
                *reinterpret_cast<uint4*>(&own.gates.t[part][row < 16 ? 0 : 1 + right][row & 15][dc_piece(row & 15, piece)]) = from;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 96)
            dc_copy_out(records.gates + ((size_t)chunk * p.heads + head) * sizeof(typename Sh::Gates), &own.gates, sizeof(typename Sh::Gates));
    }
    if (threadIdx.x == 96) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
}

__device__ __forceinline__ void dc_copy16(void* dst, const void* src, bool there) {
    const int bytes = there ? 16 : 0;                          // 0 source bytes: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dc_smem(dst)), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void dc_copy_in(void* to, const void* from, unsigned bytes, uint64_t* full) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dc_smem(to)), "l"(from), "r"(bytes), "r"(dc_smem(full)) : "memory");
}

enum { DC_MEET = 1, DC_PAIR = 2 };                   // named barriers; from DC_PAIR on the pairs'

// A fetching thread's share of the copies into the ring, chunk after chunk: the addresses move on by a chunk with every call.
// (Copied by the walkers themselves a chunk took them 800 cycles more, their own reads of shared memory queueing behind.  The
// records come as two bulk copies: 16-byte copies of all the threads queued before the walkers' reads as well, 8,192 tokens of
// 16 heads took 366 us against 343.)
template <typename T, int DK, int SLICE, bool WIDE>
struct DcFetch {
    using Sh = DcShape<T, DK, SLICE>;
    using Stage = typename Sh::Stage;
    static constexpr int PER = 16 / sizeof(T), ACROSS = Sh::COLS / PER;          // 16-byte pieces of a row of v
    const unsigned char* keys;
    const unsigned char* gates;
    const T* v;
    size_t keys_step, gates_step, v_step;
    int left, row, have;                                       // tokens from the next chunk on; the thread's row of v, its columns there

    __device__ __forceinline__ DcFetch(const DeltaParams& p, const DcRecords& records, int head, int col0, int t0, int count, int chunk0) {
        const int narrow_heads = p.heads / p.share, tid = threadIdx.x - 32 * DC_WALKERS;
        keys_step = (size_t)narrow_heads * sizeof(typename Sh::Keys);
        gates_step = (size_t)p.heads * sizeof(typename Sh::Gates);
        v_step = (size_t)DC_TOKENS * p.ld;
        keys = records.keys + chunk0 * keys_step + (size_t)(head / p.share) * sizeof(typename Sh::Keys);
        gates = records.gates + chunk0 * gates_step + (size_t)head * sizeof(typename Sh::Gates);
        row = WIDE ? tid / ACROSS : 0;
        const int d = WIDE ? (tid % ACROSS) * PER : 0;
        have = p.vdim - col0 - d;
        v = (const T*)p.qkv + (size_t)t0 * p.ld + p.v_off + (size_t)head * p.vdim + col0 + (WIDE && have > 0 ? d : 0);
        left = count;
    }
    __device__ __forceinline__ void next(const DeltaParams& p, Stage& st, uint64_t* full) {
        const int tid = threadIdx.x - 32 * DC_WALKERS;
        if (left > 0) {
            if (tid == 0) {
                mbar_expect_tx(full, sizeof(st.keys) + sizeof(st.gates));
                dc_copy_in(&st.keys, keys, sizeof(st.keys), full);
                dc_copy_in(&st.gates, gates, sizeof(st.gates), full);
            }
            if constexpr (WIDE) {
                constexpr int ROWS = DC_FETCHERS / ACROSS;     // rows of v that the block's threads copy at once
#pragma unroll
                for (int r = 0; r < DC_TOKENS; r += ROWS) {
                    const bool there = r + row < left && have > 0;
                    if (r + row < DC_TOKENS)
                        dc_copy16(&st.v[r + row][(sizeof(T) == 2 ? Sh::v_piece(r + row, tid % ACROSS) : tid % ACROSS) * PER], v + (there ? (size_t)(r + row) * p.ld : 0), there);
                }
            } else {
                for (int e = tid; e < DC_TOKENS * Sh::COLS; e += DC_FETCHERS) {
                    const int r = e / Sh::COLS, d = e % Sh::COLS;
                    st.v[r][sizeof(T) == 2 ? Sh::v_piece(r, d / 8) * 8 + d % 8 : d] = r < left && d < have ? v[(size_t)r * p.ld + d] : from_float<T>(0.f);
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

// The fetching threads also write outputs, whole lines side by side: `tokens` rows of a chunk's, from `to` on, the walkers' summands
// times the column's and the token's factor (`queries`, from the chunk's record).
template <typename Sh>
__device__ __forceinline__ void dc_write(const float (&from)[Sh::SLICES][DC_TOKENS][Sh::OLD], const float* back,
                                         const float (&queries)[Sh::WRITES], float* to, size_t width, int tokens, int columns, bool wide) {
    constexpr int FOURS = Sh::COLS / 4, AT_ONCE = DC_FETCHERS / FOURS;
    const int tid = threadIdx.x - 32 * DC_WALKERS, d = (tid % FOURS) * 4;
    if (d >= columns) return;
    const float4 b = *reinterpret_cast<const float4*>(back + d);
#pragma unroll
    for (int i = 0; i < DC_TOKENS / AT_ONCE; ++i) {
        const int r = tid / FOURS + i * AT_ONCE;
        if (r >= tokens) continue;
        const float query = queries[i];
        float4 o = *reinterpret_cast<const float4*>(&from[0][r][d]);
#pragma unroll
        for (int s = 1; s < Sh::SLICES; ++s) {
            const float4 x = *reinterpret_cast<const float4*>(&from[s][r][d]);
            o = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
        }
        o = make_float4(o.x * b.x * query, o.y * b.y * query, o.z * b.z * query, o.w * b.w * query);
        float* at = to + (size_t)r * width + d;
        if (wide && d + 4 <= columns) {
            *reinterpret_cast<float4*>(at) = o;
        } else {
            at[0] = o.x;
            if (d + 1 < columns) at[1] = o.y;
            if (d + 2 < columns) at[2] = o.z;
            if (d + 3 < columns) at[3] = o.w;
        }
    }
}

// a thread's v of one chunk as it is stored
template <typename T> struct DcValues;
template <> struct DcValues<bf16> {
    unsigned x[2 * DC_TILES];
    __device__ __forceinline__ void widen(float (&r)[DC_TILES][4]) const {
#pragma unroll
        for (int j = 0; j < DC_TILES; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                r[j][2 * h] = __uint_as_float(x[2 * j + h] << 16);
                r[j][2 * h + 1] = __uint_as_float(x[2 * j + h] & 0xffff0000u);
            }
    }
};
template <> struct DcValues<float> {
    float x[4 * DC_TILES];
    __device__ __forceinline__ void widen(float (&r)[DC_TILES][4]) const {
#pragma unroll
        for (int e = 0; e < 4 * DC_TILES; ++e) r[e >> 2][e & 3] = x[e];
    }
};

// U = T R, times DC_T_SCALE, all in two parts; th, tl: T's blocks (0, 0), (1, 0), (1, 1)
__device__ __forceinline__ void dc_solve(float (&u)[DC_TILES][4], const unsigned (&rh)[2][4], const unsigned (&rl)[2][4],
                                         const unsigned (&th)[3][4], const unsigned (&tl)[3][4]) {
    float low[DC_TILES][4];
    // (tile after tile, so that no sum waits for its own last instruction)
#pragma unroll
    for (int b = 0; b < 3; ++b) {
        const int block = b == 0 ? 1 : b == 1 ? 0 : 2, in = block == 2, to = 2 * (block > 0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            dc_mma_if(block < 2, low[to + j], rl[in], th[block][2 * j], th[block][2 * j + 1]);
            dc_mma_if(block < 2, u[to + j], rh[in], th[block][2 * j], th[block][2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) dc_mma(low[to + j], rh[in], tl[block][2 * j], tl[block][2 * j + 1]);
    }
#pragma unroll
    for (int j = 0; j < DC_TILES; ++j)
#pragma unroll
        for (int e = 0; e < 4; e += 2) dc_fma2(u[j][e], u[j][e + 1], low[j][e], low[j][e + 1], 1.f / DC_LOW, 1.f / DC_LOW, u[j][e], u[j][e + 1]);
}

template <typename T, int DK, int SLICE, bool WIDE>
__global__ void __launch_bounds__(32 * DC_WALKERS + DC_FETCHERS, sizeof(T) == 2 ? 2 : 1)
delta_walk_kernel(const DeltaParams p, const DcRecords records) {
    using Sh = DcShape<T, DK, SLICE>;
    constexpr int PARTS = Sh::PARTS, SLICES = Sh::SLICES, TILES = SLICE / 8, STEPS = SLICE / 16, FINISH = Sh::FINISH;
    extern __shared__ __align__(16) unsigned char dc_raw[];
    auto& sm = *reinterpret_cast<typename Sh::Shared*>(dc_raw);
    const int head = blockIdx.y, col0 = blockIdx.x * Sh::COLS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int chunk0;                                                // the request's first
    const int item = dc_find(p.item_qlen, records.items, blockIdx.z, p.least, lane, chunk0);
    const int slot = item < 0 ? -1 : p.item_slots[item], count = item < 0 ? 0 : p.item_qlen[item], t0 = item < 0 ? 0 : p.item_qstart[item];
    const int chunks = dc_chunks(count, p.least);
    // fewer requests than blocks, a padding entry of a fixed-size batch, or lists that name more tokens than there are
    const bool tells = p.go && first_block() && threadIdx.x == 32 * DC_WALKERS;
    if (slot < 0 || chunk0 > records.chunks - chunks) {
        grid_dependency_wait();
        if (tells) delta_release(p.go, DELTA_GO);
        return;
    }
    // registers (bfloat16): two blocks of 256 threads have 128 each; the walking warps take over some of the fetching ones' (216 + 40)
    if (warp >= DC_WALKERS) {
        if (sizeof(T) == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");
        grid_dependency_wait();
        if (tells) delta_release(p.go, DELTA_GO);
        grid_dependents_go();
        DcFetch<T, DK, SLICE, WIDE> fetch(p, records, head, col0, t0, count, chunk0);
        const size_t width = (size_t)p.heads * p.vdim;
        float* out = p.out + (size_t)t0 * width + (size_t)head * p.vdim + col0;
        const bool wide = p.vdim % 4 == 0 && (uintptr_t)p.out % 16 == 0;
        const float* queries = (reinterpret_cast<const typename Sh::Gates*>(records.gates) + (size_t)chunk0 * p.heads + head)->query;
        const bool first = threadIdx.x == 32 * DC_WALKERS;
        if (first) {
            for (int i = 0; i < DC_STAGES; ++i) mbar_init(&sm.full[i], 1);
            sm.lost = 0;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        fetch.next(p, sm.stage[0], &sm.full[0]);
        fetch.next(p, sm.stage[1], &sm.full[1]);
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");
        // (A copy between checked addresses ends; should one be waited for in vain, no more are asked for, the outputs and the state
        // become NaN, and the copies on their way are waited for once more at the end.)
        int lost = -1;                                         // the chunk that did not come
        auto await_chunk = [&](int c) {
            if (first && lost < 0 && !mbar_wait(&sm.full[c % DC_STAGES], (c / DC_STAGES) & 1)) {
                sm.lost = 1;
                lost = c;
                fetch.left = 0;
            }
            __syncwarp();
        };
        await_chunk(0);
        dc_sync(DC_MEET, Sh::THREADS);                         // chunk 0 is there
        for (int c = 1; c <= chunks + 1; ++c) {                // (the last meetings are for chunks that are not there)
            float query[Sh::WRITES];                           // of the chunk that is written next
            if (c >= 2) {
#pragma unroll
                for (int i = 0; i < Sh::WRITES; ++i) query[i] = queries[(threadIdx.x - 32 * DC_WALKERS) / (Sh::COLS / 4) + i * (DC_TOKENS / Sh::WRITES)];
                queries += (size_t)p.heads * (sizeof(typename Sh::Gates) / sizeof(float));
            }
            asm volatile("cp.async.wait_group 0;\n" ::: "memory");
            if (c < chunks) await_chunk(c);
            dc_sync(DC_MEET, Sh::THREADS);                     // chunk c is there, and everybody is through with chunk c - 2:
            fetch.next(p, sm.stage[(c + 1) % DC_STAGES], &sm.full[(c + 1) % DC_STAGES]);       // its stage takes chunk c + 1
            if (c >= 2) {
                if (__builtin_expect(sm.lost, 0)) {
#pragma unroll
                    for (int i = 0; i < Sh::WRITES; ++i) query[i] = __int_as_float(0x7fffffff);
                }
                dc_write<Sh>(sm.out[c & 1], sm.back[c & 1], query, out, width, count - (c - 2) * DC_TOKENS, p.vdim - col0, wide);
                out += DC_TOKENS * width;
            }
        }
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        if (lost >= 0)
            for (int c = lost; c < min(chunks, max(lost + 1, 2)); ++c) mbar_wait(&sm.full[c % DC_STAGES], (c / DC_STAGES) & 1);
        return;
    }
    if (sizeof(T) == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
    const int g = lane >> 2, t = lane & 3;
    const int group = warp / SLICES, slice = warp % SLICES;
    const int row0 = slice * SLICE;                            // the warp's rows of S
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
    const int b_row = (lane & 7) + 8 * (lane >> 4), b_col = 8 * ((lane >> 3) & 1);      // ldmatrix, operand stored [n][k]
    const int bt_row = (lane & 7) + 8 * ((lane >> 3) & 1), bt_col = 8 * (lane >> 4);    // ... and [k][n]
    const int b_piece = dc_piece(lane & 7, (lane >> 3) & 1);   // ... of a 16 x 16 block
    // Each of the warps of 16 columns finishes the outputs of some of the four token tiles: of two the first 0 and 3, the second 1 and 2
    // (tiles 2 and 3 have two blocks of weights), of four each one.  S0^T q has tile `place ^ slice` at a place, so that a warp's own
    // tiles are at the same places in every warp.
    const int q_row = (lane & 7) + 8 * ((lane >> 4) ^ (slice & 1)), q_half = 16 * (slice >> 1);
    constexpr int OWN = SLICES == 2 ? 3 : 1;                   // steps between the places of a warp's own tiles
    auto tile_of = [&](int j) { return OWN * j ^ slice; };
    // Operands of the next products are read well ahead of them, and sums that do not depend on one another are asked for
    // together: a warp has its scheduler nearly to itself, so what one instruction waits for, all wait for.
    unsigned bk[2][2][4];                                      // K, operand of S0^T k, 16 rows of S and two times 16 tokens each; two in turn
    DcValues<T> v;                                             // the chunk's v, laid out as a tile of U
    auto ask_keys = [&](const typename Sh::Stage& st, int k) {
#pragma unroll
        for (int m = 0; m < 2; ++m) dc_ldmatrix(bk[k & 1][m], &st.keys.k[0][16 * m + b_row][row0 + 16 * k + b_col]);
    };
    auto ask = [&](const typename Sh::Stage& st) {
        ask_keys(st, 0);
        if constexpr (sizeof(T) == 2) {                        // tokens 0-7 of col, col + 8; tokens 8-15 of both
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                unsigned x[4];
                dc_ldmatrix_trans(x, &st.v[16 * m + b_row][Sh::v_piece(b_row, group * 2 + ((lane >> 3) & 1)) * 8]);
#pragma unroll
                for (int e = 0; e < 4; ++e) v.x[4 * m + e] = x[e];
            }
        } else {
#pragma unroll
            for (int j = 0; j < DC_TILES; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) v.x[4 * j + e] = st.v[8 * j + 2 * t + (e & 1)][group * 16 + g + 8 * (e >> 1)];
        }
    };
    // v of a token in the thread's columns
    auto value = [&](const typename Sh::Stage& st, int i, int h) {
        return to_float(st.v[i][sizeof(T) == 2 ? Sh::v_piece(i, group * 2 + h) * 8 + g : group * 16 + 8 * h + g]);
    };
    // the largest number of the thread's two columns of S, over all the warps that have rows of them, without sigma
    auto largest = [&](float (&most)[2], float (&swap)[DC_WALKERS][16]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            most[h] = 0.f;
#pragma unroll
            for (int n = 0; n < TILES; ++n) most[h] = fmaxf(most[h], fmaxf(fabsf(s[n][2 * h]), fabsf(s[n][2 * h + 1])));
            most[h] *= back[h];
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], o));
        }
        if (SLICES > 1) {
            if (t == 0) { swap[warp][g] = most[0]; swap[warp][g + 8] = most[1]; }
            dc_sync(DC_PAIR + group, 32 * SLICES);
#pragma unroll
            for (int s = 1; s < SLICES; ++s) {
                most[0] = fmaxf(most[0], swap[warp ^ s][g]);
                most[1] = fmaxf(most[1], swap[warp ^ s][g + 8]);
            }
        }
    };
    // What the two columns' numbers are held against.  A column of zeros (S and v; those beyond the last among them) is out of the check
    // and gets the largest power of two, so that the first number that is not zero is too large for it.
    float least[2];
    auto arm = [&](int h, bool there) { least[h] = there ? DC_ENOUGH : -1.f; };
    enum { FRESH, LITTLE, MUCH };                              // why a chunk is not walked just so: no sigma yet, small numbers, large ones
    int why = FRESH, down = 0, c = 0, stage = 0;
    bool looked = false, met = false;                          // sigma is this chunk's own; the chunk's meeting has been
    auto through = [&] {                                       // with chunk c
        ++c;
        stage = stage + 1 < DC_STAGES ? stage + 1 : 0;
        looked = met = false;
    };
    dc_sync(DC_MEET, Sh::THREADS);                             // stage 0 is there

    while (c < chunks) {
        bool by_token = false, passed = false;
        {
            const auto& st = sm.stage[stage];
            const int tokens = min(DC_TOKENS, count - c * DC_TOKENS);
            ask(st);
            if (why == LITTLE) {
                // Nearly nothing is stored at a token, or taken in.  What the columns hold: the state's largest number and the values, faded.
                float most[2], all[2];                         // faded; not faded, and as a look counts them
                largest(most, sm.most[1]);
                bool small = false;
#pragma unroll
                for (int h = 0; h < 2; ++h) all[h] = most[h] *= sigma[h];
#pragma unroll 2
                for (int i = 0; i < tokens; ++i) {
                    const float decay = st.gates.decay[i], beta = st.gates.beta[i];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float x = fabsf(value(st, i, h));
                        all[h] = fmaxf(all[h], x);
                        most[h] = fmaxf(most[h] * decay, x * beta * sigma[h]);
                        small = small || (most[h] > 0.f && most[h] < DC_LEAST);
                    }
                }
                float fade = 1.f, there = 0.f;                 // of the tokens behind; tokens that are still there
                for (int i = tokens - 1; i >= 0 && fade >= 1.f / (1 << 21); --i) {
                    there += 1.f;
                    fade *= st.gates.decay[i];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) small = small || (most[h] > 0.f && most[h] * most[h] < there * (DC_LEAST_STATE * DC_LEAST_STATE));
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (all[h] == 0.f) { sigma[h] = dc_power(DC_LAST); back[h] = dc_power(-DC_LAST); arm(h, false); }
                passed = !__any_sync(0xffffffffu, small);
            }
            if (!passed && looked && !(why == MUCH && down == 0)) {
                by_token = true;                               // not a matter of sigma
            } else if (!passed) {
                // the columns' powers of two from the columns themselves; token by token where a state is small beside the values
                down = looked ? DC_DOWN : 0;
                looked = true;
                float most[2], held[2], raw[DC_TILES][4];
                v.widen(raw);
                largest(most, sm.most[0]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = 0.f;
#pragma unroll
                    for (int j = 0; j < DC_TILES; ++j)
#pragma unroll
                        for (int e = 2 * h; e < 2 * h + 2; ++e)        // (an infinite value must not move its column's power)
                            if (fabsf(raw[j][e]) < INFINITY) x = fmaxf(x, fabsf(raw[j][e]));
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                    held[h] = most[h];
                    most[h] = fmaxf(most[h], x * st.gates.above[0]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int e = DC_SIZE - down - (((__float_as_int(most[h]) >> 23) & 255) - 127);
                    const float next = dc_power(most[h] > 0.f ? min(max(e, DC_FIRST), DC_LAST) : DC_LAST);
                    arm(h, most[h] > 0.f);
                    const float factor = next * back[h];
                    sigma[h] = next;
                    back[h] = 1.f / next;
                    by_token = by_token || (held[h] > 0.f && held[h] * next < DC_LEAST_STATE);
#pragma unroll
                    for (int n = 0; n < TILES; ++n) { s[n][2 * h] *= factor; s[n][2 * h + 1] *= factor; }
                }
                by_token = __any_sync(0xffffffffu, by_token);
            }
            if (by_token) {
                // ---- the recurrence, token by token
                if (!met) dc_sync(DC_MEET, Sh::THREADS);
                else if (SLICES > 1) dc_sync(DC_PAIR + group, 32 * SLICES);       // the swapped sums have been read
#pragma unroll 1
                for (int i = 0; i < tokens; ++i) {
                    float with_k[2] = {0.f, 0.f}, with_q[2] = {0.f, 0.f}, kq = 0.f;
                    auto both = [&](const __half (&rows)[PARTS][DC_TOKENS][Sh::KLD], int n) {
                        float2 x = __half22float2(*reinterpret_cast<const __half2*>(&rows[0][i][row0 + 8 * n + 2 * t]));
                        if (PARTS == 2) {
                            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&rows[PARTS - 1][i][row0 + 8 * n + 2 * t]));
                            x.x += y.x; x.y += y.y;
                        }
                        return x;
                    };
#pragma unroll
                    for (int n = 0; n < TILES; ++n) {
                        const float2 k = both(st.keys.k, n), q = both(st.keys.q, n);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            with_k[h] = fmaf(s[n][2 * h + 1], k.y, fmaf(s[n][2 * h], k.x, with_k[h]));
                            with_q[h] = fmaf(s[n][2 * h + 1], q.y, fmaf(s[n][2 * h], q.x, with_q[h]));
                        }
                        kq = fmaf(k.y, q.y, fmaf(k.x, q.x, kq));
                    }
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            with_k[h] += __shfl_xor_sync(0xffffffffu, with_k[h], o);
                            with_q[h] += __shfl_xor_sync(0xffffffffu, with_q[h], o);
                        }
                        kq += __shfl_xor_sync(0xffffffffu, kq, o);
                    }
                    if (SLICES > 1) {                          // (two places in turn: one meeting a token)
                        if (t == 0) sm.swap[c & 1][warp][i & 1][g] = make_float4(with_k[0], with_k[1], 0.f, 0.f);
                        dc_sync(DC_PAIR + group, 32 * SLICES);
                        with_k[0] = with_k[1] = 0.f;
#pragma unroll
                        for (int x = 0; x < SLICES; ++x) {     // the same sum in all the warps
                            const float4 part = sm.swap[c & 1][group * SLICES + x][i & 1][g];
                            with_k[0] += part.x; with_k[1] += part.y;
                        }
                    }
                    const float key = st.gates.key[i], decay = st.gates.decay[i], beta = st.gates.beta[i];
                    float now[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        now[h] = value(st, i, h) * beta * sigma[h] - beta * (decay * key * with_k[h]);
                        // a warp's own rows' summand of the output
                        if (t == 0) sm.out[c & 1][slice][i][group * 16 + 8 * h + g] = DC_P_SCALE * (decay * with_q[h] + kq * key * now[h]);
                    }
#pragma unroll
                    for (int n = 0; n < TILES; ++n) {
                        const float2 k = both(st.keys.k, n);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            s[n][2 * h] = fmaf(k.x * key, now[h], decay * s[n][2 * h]);
                            s[n][2 * h + 1] = fmaf(k.y * key, now[h], decay * s[n][2 * h + 1]);
                        }
                    }
                }
                if (slice == 0 && t == 0) {
                    sm.back[c & 1][group * 16 + g] = back[0];
                    sm.back[c & 1][group * 16 + g + 8] = back[1];
                }
                why = FRESH;
                through();
                continue;
            }
        }
        // ---- chunk after chunk, until one is out of range
        for (;;) {
            const auto& st = sm.stage[stage];
            float u[DC_TILES][4], wq[DC_TILES][4];             // U, times DC_T_SCALE; S0^T q
            unsigned bq[2][4];                                 // Q
            unsigned sh[STEPS][4], sl[STEPS][4];               // the state in two parts
            auto ask_query = [&](int k) {
#pragma unroll
                for (int m = 0; m < 2; ++m) dc_ldmatrix(bq[m], &st.keys.q[0][(16 * m ^ q_half) + q_row][row0 + 16 * k + b_col]);
            };
            // a quarter of the instructions of S0^T q: they stand where the chain of R, U and the new state has to wait
            auto query_step = [&](int k) {
                if (k >= STEPS) return;
#pragma unroll
                for (int j = 0; j < DC_TILES; ++j) dc_mma_if(k == 0, wq[j], sl[k], bq[j >> 1][2 * (j & 1)], bq[j >> 1][2 * (j & 1) + 1]);
                if (PARTS == 2) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        unsigned b[4];
                        dc_ldmatrix(b, &st.keys.q[PARTS - 1][(16 * m ^ q_half) + q_row][row0 + 16 * k + b_col]);
                        dc_mma(wq[2 * m], sh[k], b[0], b[1]);
                        dc_mma(wq[2 * m + 1], sh[k], b[2], b[3]);
                    }
                }
#pragma unroll
                for (int j = 0; j < DC_TILES; ++j) dc_mma(wq[j], sh[k], bq[j >> 1][2 * (j & 1)], bq[j >> 1][2 * (j & 1) + 1]);
                if (k + 1 < STEPS) ask_query(k + 1);
            };
            float add[TILES][4], oa[FINISH][4], ob[FINISH][4];     // what the new state takes in; outputs
            // ---- S0^T k of the warp's rows: 16 columns x 32 tokens; the next rows are taken apart meanwhile
            float wk[DC_TILES][4], lk[DC_TILES][4];
            dc_split_tiles(s[0], s[1], sh[0], sl[0]);
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                if (k + 1 < STEPS) ask_keys(st, k + 1);
#pragma unroll
                for (int j = 0; j < DC_TILES; ++j) {
                    dc_mma_if(k == 0, wk[j], sh[k], bk[k & 1][j >> 1][2 * (j & 1)], bk[k & 1][j >> 1][2 * (j & 1) + 1]);
                    dc_mma_if(k == 0, lk[j], sl[k], bk[k & 1][j >> 1][2 * (j & 1)], bk[k & 1][j >> 1][2 * (j & 1) + 1]);
                }
                if (k + 1 < STEPS) dc_split_tiles(s[2 * k + 2], s[2 * k + 3], sh[(k + 1) % STEPS], sl[(k + 1) % STEPS]);
                if (PARTS == 2) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        unsigned b[4];
                        dc_ldmatrix(b, &st.keys.k[PARTS - 1][16 * m + b_row][row0 + 16 * k + b_col]);
                        dc_mma(lk[2 * m], sh[k], b[0], b[1]);
                        dc_mma(lk[2 * m + 1], sh[k], b[2], b[3]);
                    }
                }
            }
            ask_query(0);
#pragma unroll
            for (int j = 0; j < DC_TILES; ++j) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) dc_add2(wk[j][e], wk[j][e + 1], wk[j][e], wk[j][e + 1], lk[j][e], lk[j][e + 1]);
                if (SLICES > 1) sm.swap[c & 1][warp][j][lane] = make_float4(wk[j][0], wk[j][1], wk[j][2], wk[j][3]);
            }
            float2 before[DC_TILES];
#pragma unroll
            for (int j = 0; j < DC_TILES; ++j) before[j] = *reinterpret_cast<const float2*>(&st.gates.before[8 * j + 2 * t]);
            // ---- one meeting per chunk: the halves' sums are there, and so is the next stage
            if (!met) dc_sync(DC_MEET, Sh::THREADS);
            else if (SLICES > 1) dc_sync(DC_PAIR + group, 32 * SLICES);
            if constexpr (SLICES > 1) {
                float4 x[DC_TILES];
#pragma unroll
                for (int j = 0; j < DC_TILES; ++j) x[j] = sm.swap[c & 1][warp ^ 1][j][lane];
                float4 y[DC_TILES], z[DC_TILES];
                if (SLICES > 2) {
#pragma unroll
                    for (int j = 0; j < DC_TILES; ++j) { y[j] = sm.swap[c & 1][warp ^ 2][j][lane]; z[j] = sm.swap[c & 1][warp ^ 3][j][lane]; }
                }
                query_step(0);
#pragma unroll
                for (int j = 0; j < DC_TILES; ++j) {
                    dc_add2(wk[j][0], wk[j][1], wk[j][0], wk[j][1], x[j].x, x[j].y);
                    dc_add2(wk[j][2], wk[j][3], wk[j][2], wk[j][3], x[j].z, x[j].w);
                    if (SLICES > 2) {                          // (pairs first: the same sum in all four warps)
                        dc_add2(y[j].x, y[j].y, y[j].x, y[j].y, z[j].x, z[j].y);
                        dc_add2(y[j].z, y[j].w, y[j].z, y[j].w, z[j].z, z[j].w);
                        dc_add2(wk[j][0], wk[j][1], wk[j][0], wk[j][1], y[j].x, y[j].y);
                        dc_add2(wk[j][2], wk[j][3], wk[j][2], wk[j][3], y[j].z, y[j].w);
                    }
                }
            } else {
                query_step(0);
            }
            // ---- R, times DC_LOW, and U
            const float above = st.gates.above[0] * DC_LOW, sigma_far[2] = {sigma[0] * above, sigma[1] * above};
            float r[DC_TILES][4];
            v.widen(r);
#pragma unroll
            for (int j = 0; j < DC_TILES; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x, y;
                    dc_mul2(x, y, r[j][2 * h], r[j][2 * h + 1], sigma_far[h], sigma_far[h]);
                    dc_fma2(r[j][2 * h], r[j][2 * h + 1], -before[j].x, -before[j].y, wk[j][2 * h], wk[j][2 * h + 1], x, y);
                }
            unsigned rh[2][4], rl[2][4], th[3][4], tl[3][4];
#pragma unroll
            for (int b = 0; b < 3; ++b) {
                dc_ldmatrix(th[b], &st.gates.t[0][b][b_row][b_piece]);
                dc_ldmatrix(tl[b], &st.gates.t[1][b][b_row][b_piece]);
            }
            dc_split_tiles_far(r[0], r[1], rh[0], rl[0]);
            query_step(1);
            dc_split_tiles_far(r[2], r[3], rh[1], rl[1]);
            dc_solve(u, rh, rl, th, tl);
            query_step(2);
            // ---- the new state
            unsigned uh[2][4], ul[2][4], kt[STEPS][4];
            float taken[2] = {0.f, 0.f};                       // the largest number that the new state takes in, of the thread's tokens
#pragma unroll
            for (int k = 0; k < STEPS; ++k) dc_ldmatrix_trans(kt[k], &st.keys.k[0][bt_row][row0 + 16 * k + bt_col]);
            query_step(3);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float faded[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 after = *reinterpret_cast<const float2*>(&st.gates.after[16 * m + 8 * j + 2 * t]);
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
                        dc_mul2(faded[j][e], faded[j][e + 1], u[2 * m + j][e], u[2 * m + j][e + 1], after.x, after.y);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        asm("max.f32 %0, %0, %1, %2;" : "+f"(taken[h]) : "f"(fabsf(faded[j][2 * h])), "f"(fabsf(faded[j][2 * h + 1])));
                }
                dc_split_tiles(faded[0], faded[1], uh[m], ul[m]);
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) {                      // tokens 16 m on
#pragma unroll
                for (int n = 0; n < TILES; ++n) dc_mma_if(m == 0, add[n], ul[m], kt[n >> 1][2 * (n & 1)], kt[n >> 1][2 * (n & 1) + 1]);
                if (PARTS == 2) {
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) {
                        unsigned b[4];
                        dc_ldmatrix_trans(b, &st.keys.k[PARTS - 1][16 * m + bt_row][row0 + 16 * k + bt_col]);
                        dc_mma(add[2 * k], uh[m], b[0], b[1]);
                        dc_mma(add[2 * k + 1], uh[m], b[2], b[3]);
                    }
                }
#pragma unroll
                for (int n = 0; n < TILES; ++n) dc_mma(add[n], uh[m], kt[n >> 1][2 * (n & 1)], kt[n >> 1][2 * (n & 1) + 1]);
                if (m == 0) {
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) dc_ldmatrix_trans(kt[k], &st.keys.k[0][16 + bt_row][row0 + 16 * k + bt_col]);
                }
            }
            // ---- is everything in range?  (all warps of 16 columns have the same U)
            float size, low[2], most[DC_TILES], little[2][2];  // (short chains: three at a time)
#pragma unroll
            for (int j = 0; j < DC_TILES; ++j) {
                asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(most[j]) : "f"(fabsf(u[j][0])), "f"(fabsf(u[j][1])), "f"(fabsf(u[j][2])));
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(most[j]) : "f"(fabsf(u[j][3])));
            }
            asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(size) : "f"(most[0]), "f"(most[1]), "f"(most[2]));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(size) : "f"(most[3]));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    asm("min.f32 %0, %1, %2, %3;" : "=f"(little[h][m])
                        : "f"(fabsf(u[2 * m][2 * h])), "f"(fabsf(u[2 * m][2 * h + 1])), "f"(fabsf(u[2 * m + 1][2 * h])));
                    little[h][m] = fminf(little[h][m], fabsf(u[2 * m + 1][2 * h + 1]));
                }
                low[h] = fminf(little[h][0], little[h][1]);
            }
            const bool high = !(size < DC_MOST * DC_T_SCALE);
            // of a column's four lanes one at least has taken in enough, of both columns
            unsigned enough = __ballot_sync(0xffffffffu, taken[0] >= least[0] && taken[1] >= least[1]);
            enough |= enough >> 2;
            enough |= enough >> 1;
            if (__builtin_expect(!passed && ((enough & 0x11111111u) != 0x11111111u ||
                                             __any_sync(0xffffffffu, high || low[0] < least[0] || low[1] < least[1])), 0)) {
                why = __any_sync(0xffffffffu, high) ? MUCH : LITTLE;
                met = true;
                break;
            }
            // ---- outputs: the chunk's start and its own tokens; the fetching warps add up what two warps have of S0^T q and write them
            unsigned zh[2][4], zl[2][4], w[FINISH][2][4];      // U again, weights: high and low part, two inner halves each
            float2 fade[FINISH];
            auto second = [&](int j) { return SLICES == 4 ? slice >= 2 : OWN * j >= 2; };      // the tile's tokens are in the chunk's second half
#pragma unroll
            for (int j = 0; j < FINISH; ++j) {
                fade[j] = *reinterpret_cast<const float2*>(&st.gates.fade[8 * tile_of(j) + 2 * t]);
#pragma unroll
                for (int m = 0; m < 2; ++m)
                    if (m == 0 || second(j)) dc_ldmatrix(w[j][m], &st.gates.p[lane >> 4][second(j) ? 1 + m : 0][8 * (tile_of(j) & 1) + (lane & 7)][b_piece]);
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) dc_split_tiles_far(u[2 * m], u[2 * m + 1], zh[m], zl[m]);
#pragma unroll
            for (int j = 0; j < FINISH; ++j) {
                const float(&own)[4] = wq[OWN * j];
#pragma unroll
                for (int h = 0; h < 2; ++h) dc_mul2(oa[j][2 * h], oa[j][2 * h + 1], own[2 * h], own[2 * h + 1], fade[j].x, fade[j].y);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    if (m > 0 && !second(j)) continue;
                    dc_mma_if(m == 0, ob[j], zl[m], w[j][m][0], w[j][m][1]);
                    dc_mma(oa[j], zh[m], w[j][m][0], w[j][m][1]);
                    dc_mma(ob[j], zh[m], w[j][m][2], w[j][m][3]);
                }
            }
            const float decay = st.gates.fade[DC_TOKENS - 1] * (1.f / DC_P_SCALE);
            if (c + 1 < chunks) ask(sm.stage[stage + 1 < DC_STAGES ? stage + 1 : 0]);
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    dc_fma2(s[n][e], s[n][e + 1], s[n][e], s[n][e + 1], decay, decay, add[n][e], add[n][e + 1]);
            auto leave = [&](int which, int tile, const float (&o)[4]) {
                float* to = &sm.out[c & 1][which][8 * tile + 2 * t][group * 16 + g];
                to[0] = o[0]; to[8] = o[2]; to[Sh::OLD] = o[1]; to[Sh::OLD + 8] = o[3];
            };
            if constexpr (SLICES > 1) {
#pragma unroll
                for (int j = 1; j < (SLICES > 2 ? 4 : 3); ++j) {   // the other warps' tiles
                    const int tile = j ^ slice;
                    const float2 f = *reinterpret_cast<const float2*>(&st.gates.fade[8 * tile + 2 * t]);
                    float o[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) dc_mul2(o[2 * h], o[2 * h + 1], wq[j][2 * h], wq[j][2 * h + 1], f.x, f.y);
                    leave(SLICES > 2 ? j : 1, tile, o);
                }
            }
#pragma unroll
            for (int j = 0; j < FINISH; ++j) {
                const int tile = tile_of(j);
                float o[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) dc_fma2(o[2 * h], o[2 * h + 1], ob[j][2 * h], ob[j][2 * h + 1], 1.f / DC_LOW, 1.f / DC_LOW, oa[j][2 * h], oa[j][2 * h + 1]);
                leave(0, tile, o);
            }
            if (slice == 0 && t == 0) {                        // (one over sigma as this chunk had it)
                sm.back[c & 1][group * 16 + g] = back[0];
                sm.back[c & 1][group * 16 + g + 8] = back[1];
            }
            passed = false;
            through();
            if (c >= chunks) break;
        }
    }
    dc_sync(DC_MEET, Sh::THREADS);
    if (__builtin_expect(sm.lost, 0)) back[0] = back[1] = __int_as_float(0x7fffffff);
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = row0 + 8 * n + 2 * t + (e & 1), v = col + 8 * (e >> 1);
            if (d < p.dim && v < p.vdim) state[(size_t)d * p.vdim + v] = s[n][e] * back[e >> 1];
        }
}

// An SM for each block: asks for more than half of the SM's shared memory.
constexpr int DC_ALONE_BYTES = 180 * 1024;
static_assert(sizeof(DcShape<float, 128, 64>::Shared) <= DC_ALONE_BYTES && sizeof(DcShape<float, 128, 32>::Shared) <= DC_ALONE_BYTES, "the largest shapes");

template <typename T, int DK, int SLICE, bool WIDE>
static int launch_walk(const DeltaParams& p, const DcRecords& records, dim3 grid, int sms, cudaStream_t stream) {
    using Sh = DcShape<T, DK, SLICE>;
    auto walker = delta_walk_kernel<T, DK, SLICE, WIDE>;
    static bool ready = false;                 // per process and kernel; harmless if repeated
    if (!ready) {
        const cudaError_t e = cudaFuncSetAttribute(walker, cudaFuncAttributeMaxDynamicSharedMemorySize, DC_ALONE_BYTES);
        if (e != cudaSuccess) return (int)e;
        ready = true;
    }
    // As many blocks as SMs had better not share any, which they do if they start while the records' blocks still hold some:
    // 8,192 tokens of 16 heads of 128 x 128 (64 blocks) take 366 us alone, 546 two to an SM.  More blocks, some of which may have
    // nothing to do (p.least: requests of many lengths), start behind the records' end and spread: 13 requests of 1 to 700 tokens,
    // 16 heads of 64 x 64 (208 blocks) 54 against 64 us; three of 256 to 1,024 of 16 heads of 128 x 128 (192) 89 against 85.
    // The state is older than the records' kernel, which waits for whatever may have written it.
    const long long blocks = (long long)grid.x * grid.y * grid.z;
    const bool alone = blocks <= sms, spread = !alone && blocks <= 2 * sms && p.least > 1;
    return launch_dependent_if(!spread, walker, grid, dim3(Sh::THREADS), alone ? (size_t)DC_ALONE_BYTES : sizeof(typename Sh::Shared),
                               stream, p, records);
}

template <typename T, int DK, bool WIDE>
static int launch_chunk(const DeltaParams& p, const DcRecords& records, int early, cudaStream_t stream) {
    auto maker = delta_records_kernel<T, DK, WIDE>;
    static int sms = 0;                        // per process and kernel; harmless if repeated
    if (sms == 0) {
        int device = 0, count = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(maker, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(DcMaker<T, DK>));
        if (e != cudaSuccess) return (int)e;
        sms = count;
    }
    const long long units = (long long)records.chunks * (p.heads / p.share);
    if (units > 0x7fffffffLL || p.heads > 65535 || records.longer > 65535) return ERR_UNSUPPORTED;
    const int rc = launch_dependent_if(early, maker, dim3((unsigned)units), dim3(32 * DC_MAKERS), sizeof(DcMaker<T, DK>), stream, p, records);
    if (rc != 0) return rc;
    // Half the rows per warp shorten a chunk's chain, twice the blocks solve for U twice as often: where they have an SM each it pays.
    // 8,192 tokens of 16 heads of 128 x 128 (128 blocks) 312 us against 349, 1,024 in float32 56 against 65; 2,048 tokens of 20
    // heads (160 blocks) 124 against 101.
    constexpr int NARROW = DcShape<T, DK, 32>::COLS, COLS = DcShape<T, DK, 64>::COLS;
    const dim3 narrow((p.vdim + NARROW - 1) / NARROW, p.heads, records.longer), wide((p.vdim + COLS - 1) / COLS, p.heads, records.longer);
    return (long long)narrow.x * narrow.y * narrow.z <= sms ? launch_walk<T, DK, 32, WIDE>(p, records, narrow, sms, stream)
                                                            : launch_walk<T, DK, 64, WIDE>(p, records, wide, sms, stream);
}

template <typename T, int DK>
static int launch_chunk_any(const DeltaParams& p, int items, int longer, long long chunks, unsigned char* room, int early, cudaStream_t stream) {
    DcRecords records;
    records.keys = room;
    records.gates = room + (size_t)chunks * (p.heads / p.share) * sizeof(typename DcRecord<T, DK>::Keys);
    records.items = items;
    records.longer = longer;
    records.chunks = (int)chunks;
    const bool wide = p.ld % 8 == 0 && p.q_off % 8 == 0 && p.k_off % 8 == 0 && p.v_off % 8 == 0 && p.dim % 8 == 0 &&
                      p.vdim % 8 == 0 && (uintptr_t)p.qkv % 16 == 0;
    return wide ? launch_chunk<T, DK, true>(p, records, early, stream) : launch_chunk<T, DK, false>(p, records, early, stream);
}

static long long chunk_bytes(int heads, int share, int dim, int dtype) {
    const long long gates = (long long)heads * sizeof(DcRecord<bf16, 64>::Gates), narrow = heads / share;
    if (dtype == DTYPE_F32) return gates + narrow * (dim <= 64 ? sizeof(DcRecord<float, 64>::Keys) : sizeof(DcRecord<float, 128>::Keys));
    return gates + narrow * (dim <= 64 ? sizeof(DcRecord<bf16, 64>::Keys) : sizeof(DcRecord<bf16, 128>::Keys));
}

// The chunked form; ERR_UNSUPPORTED where a head has more rows than it holds.  `longer`: at most so many requests are of p.least tokens
// or more; `room`: 16-byte aligned memory, 16 bytes and the records.
int delta_chunk(const DeltaParams& p, int items, int longer, int dtype, void* room, long long room_bytes, int early, cudaStream_t stream) {
    if (p.dim > DC_MAX_DIM) return ERR_UNSUPPORTED;
    const long long chunks = (room_bytes - 16) / chunk_bytes(p.heads, p.share, p.dim, dtype);        // (behind p.go's word)
    if (!room || (uintptr_t)room % 16 != 0 || chunks <= 0 || chunks > 0x7fffffffLL) return ERR_BAD_ARGUMENT;
    unsigned char* at = (unsigned char*)room + 16;
    if (dtype == DTYPE_F32)
        return p.dim <= 64 ? launch_chunk_any<float, 64>(p, items, longer, chunks, at, early, stream)
                           : launch_chunk_any<float, 128>(p, items, longer, chunks, at, early, stream);
    return p.dim <= 64 ? launch_chunk_any<bf16, 64>(p, items, longer, chunks, at, early, stream)
                       : launch_chunk_any<bf16, 128>(p, items, longer, chunks, at, early, stream);
}

}  // namespace fsie

extern "C" {

int fsie_delta_chunk_max_dim() { return fsie::DC_MAX_DIM; }

int fsie_delta_chunk_tokens() { return fsie::DC_TOKENS; }

// bytes of the workspace per chunk
int fsie_delta_chunk_bytes(int heads, int share, int dim, int dtype) { return (int)fsie::chunk_bytes(heads, share, dim, dtype); }

}  // extern "C"
