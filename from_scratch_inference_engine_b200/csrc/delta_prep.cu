// What stands in front of the gated delta rule (delta_rule.cu), per token of the stored projection:
//
//   c_t         = silu(sum_j w[j] u_(t - taps + 1 + j))       per channel (the q, k and v columns), taps inputs
//   log_decay_t = -exp(a_log) softplus(a_t + dt_bias)          per head
//   beta_t      = sigmoid(b_t)                                 per head
//
// The inputs u of the taps - 1 tokens before a step's first live in the request's state slot (32-bit, oldest first), and the
// same launch moves them on: only the thread that has read a channel's old inputs - in the tile with the request's first
// token - writes its new ones.  Sums, activation and gates are 32-bit; c is rounded once, to the storage type, as all
// activations between kernels are.
//
// Bound by memory: the projection's columns are read and c is written once.  A thread owns four neighbouring channels
// (8-byte accesses in bfloat16) of up to PREP_AHEAD tokens and asks for all their inputs, and the taps - 1 in front of
// them, before it does anything else; what stands in front of another thread's tokens comes from L2 a second time.
// 4,096 tokens of 8,192 channels and 32 heads: 29 us for 135 MB (4.7 TB/s; the bytes at the copy rate: 21); the instructions of the
// sums and of silu stand beside the loads (the first form, one channel per thread, took 102 us).  24 decoded tokens of 6,144
// channels: 4.7 us, a chain of list, state and inputs.
#include "common.cuh"
#include <math.h>

namespace fsie {

constexpr int PREP_THREADS = 128;
constexpr int PREP_AHEAD = 8;
constexpr int PREP_MAX_TAPS = 16;

__device__ __forceinline__ float prep_silu(float z) { return z / (1.0f + expf(-z)); }
// two floats in one register pair: the packed instructions of sm_100 work on both at once
__device__ __forceinline__ unsigned long long prep_pair(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void prep_unpair(unsigned long long p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}
__device__ __forceinline__ unsigned long long prep_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long prep_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float prep_exp2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float prep_rcp(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
// silu of four numbers.  Stored in 8 bits it needs no more than the approximate exponential and reciprocal (2^-22): the kernel is
// bound by its instructions with the exact ones.
template <typename T> __device__ __forceinline__ void prep_silu4(const unsigned long long (&z)[2], float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float x, y;
        prep_unpair(z[i], x, y);
        if (sizeof(T) == 2) {
            constexpr float L = -1.4426950408889634f;
            float ex, ey;
            prep_unpair(prep_mul2(z[i], prep_pair(L, L)), ex, ey);
            prep_unpair(prep_mul2(z[i], prep_pair(prep_rcp(1.0f + prep_exp2(ex)), prep_rcp(1.0f + prep_exp2(ey)))), v[2 * i], v[2 * i + 1]);
        } else {
            v[2 * i] = prep_silu(x);
            v[2 * i + 1] = prep_silu(y);
        }
    }
}
__device__ __forceinline__ float prep_softplus(float z) { return z > 20.f ? z : log1pf(expf(z)); }
// four neighbouring values
template <typename T> struct Stored4;
template <> struct Stored4<bf16> {
    uint2 x;
    __device__ __forceinline__ void load(const bf16* p) { x = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void widen(float (&v)[4]) const {
        v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
        v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
    }
};
template <> struct Stored4<float> {
    float4 x;
    __device__ __forceinline__ void load(const float* p) { x = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void widen(float (&v)[4]) const { v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
};
__device__ __forceinline__ void prep_load(const float* p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void prep_store(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void prep_store(bf16* p, const float (&v)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

struct PrepParams {
    int ld, conv_off, a_off, b_off;
    const int* item_qstart; const int* item_qlen; const int* item_slots;
    const int* seg_item; const int* seg_row0; int seg_tokens;
    float* state; long long state_stride, tail_off;
    const float* conv; int taps, channels;         // conv [taps, channels], the last row the current token's
    const float* a_log; const float* dt_bias; int heads;
    float* log_decay; float* beta;
};

// the gates of a tile's tokens
template <typename T>
__device__ __forceinline__ void prep_gates(const PrepParams& p, const T* __restrict__ proj, int t0, int count) {
    for (int e = threadIdx.x; e < count * p.heads; e += blockDim.x) {
        const int t = t0 + e / p.heads, h = e % p.heads;
        const T* row = proj + (size_t)t * p.ld;
        const float step = prep_softplus(to_float(row[p.a_off + h]) + p.dt_bias[h]);
        p.log_decay[(size_t)t * p.heads + h] = -expf(p.a_log[h]) * step;
        p.beta[(size_t)t * p.heads + h] = 1.0f / (1.0f + expf(-to_float(row[p.b_off + h])));
    }
}

// grid (tiles, slices of channels and one more for the gates, parts of PREP_AHEAD tokens of a tile)
template <typename T, int TAPS>
__global__ void __launch_bounds__(PREP_THREADS, 8)
delta_prep_kernel(const T* __restrict__ proj, T* __restrict__ act, const PrepParams p) {
    const int tile = blockIdx.x;
    const int item = p.seg_item[tile], row0 = p.seg_row0[tile] + blockIdx.z * PREP_AHEAD;
    const int qlen = p.item_qlen[item], slot = p.item_slots[item];
    const int count = min(min(PREP_AHEAD, p.seg_tokens - (int)blockIdx.z * PREP_AHEAD), qlen - row0), t0 = p.item_qstart[item] + row0;
    const int c = (blockIdx.y * PREP_THREADS + threadIdx.x) * 4;
    const bool gates = blockIdx.y == gridDim.y - 1, mine = !gates && c < p.channels;
    unsigned long long w[TAPS][2];
    if (mine) {
#pragma unroll
        for (int j = 0; j < TAPS; ++j) {
            const float4 x = *reinterpret_cast<const float4*>(p.conv + (size_t)j * p.channels + c);
            w[j][0] = prep_pair(x.x, x.y);
            w[j][1] = prep_pair(x.z, x.w);
        }
    }
    grid_dependency_wait();
    grid_dependents_go();
    if (slot < 0 || count <= 0) return;                    // a padding entry of a fixed-size batch
    if (gates) { prep_gates(p, proj, t0, count); return; }
    if (!mine) return;
    const T* from = proj + (size_t)t0 * p.ld + p.conv_off + c;
    T* to = act + (size_t)t0 * p.channels + c;
    float* tail = p.state + (size_t)slot * p.state_stride + p.tail_off + c;
    Stored4<T> u[PREP_AHEAD];
#pragma unroll
    for (int r = 0; r < PREP_AHEAD; ++r)
        if (r < count) u[r].load(from + (size_t)r * p.ld);
    // The inputs in front of the thread's first token, oldest first: in front of the request's first token the slot's.  Only the
    // part with that token looks at the slot, and the same thread writes there behind it.
    float last[TAPS - 1][4];
    Stored4<T> ahead[TAPS - 1];
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) {
        const int back = TAPS - 1 - j;
        if (row0 == 0) prep_load(tail + (size_t)j * p.channels, last[j]);
        else ahead[j].load(from - (ptrdiff_t)back * p.ld);                    // row0 >= taps - 1
    }
    if (row0 != 0) {
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) ahead[j].widen(last[j]);
    }
#pragma unroll
    for (int r = 0; r < PREP_AHEAD; ++r) {
        if (r < count) {
            float sum[4], x[4];
            unsigned long long z[2];
            u[r].widen(x);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                z[i] = prep_mul2(w[0][i], prep_pair(last[0][2 * i], last[0][2 * i + 1]));
#pragma unroll
                for (int j = 1; j < TAPS - 1; ++j) z[i] = prep_fma2(w[j][i], prep_pair(last[j][2 * i], last[j][2 * i + 1]), z[i]);
                z[i] = prep_fma2(w[TAPS - 1][i], prep_pair(x[2 * i], x[2 * i + 1]), z[i]);
            }
            prep_silu4<T>(z, sum);
            prep_store(to, sum);
            to += p.channels;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j + 1 < TAPS - 1; ++j) last[j][i] = last[j + 1][i];
                last[TAPS - 2][i] = x[i];
            }
        }
    }
    if (row0 == 0) {
        if (count < qlen) {                                // the request's last tokens are another thread's
            const T* end = from + (size_t)qlen * p.ld;
#pragma unroll
            for (int j = 0; j < TAPS - 1; ++j) {
                const int back = TAPS - 1 - j;
                if (back <= qlen) { ahead[j].load(end - (ptrdiff_t)back * p.ld); ahead[j].widen(last[j]); }
            }
        }
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) prep_store(tail + (size_t)j * p.channels, last[j]);
    }
}

// Any number of taps and any alignment: a thread per channel.
template <typename T>
__global__ void __launch_bounds__(PREP_THREADS)
delta_prep_any_kernel(const T* __restrict__ proj, T* __restrict__ act, const PrepParams p) {
    grid_dependency_wait();
    grid_dependents_go();
    const int tile = blockIdx.x;
    const int item = p.seg_item[tile], row0 = p.seg_row0[tile];
    const int qlen = p.item_qlen[item], slot = p.item_slots[item];
    const int count = min(p.seg_tokens, qlen - row0), t0 = p.item_qstart[item] + row0;
    if (slot < 0 || count <= 0) return;
    if (blockIdx.y == gridDim.y - 1) { prep_gates(p, proj, t0, count); return; }
    const int c = blockIdx.y * PREP_THREADS + threadIdx.x;
    if (c >= p.channels) return;
    const int back = p.taps - 1;
    const T* from = proj + (size_t)(t0 - row0) * p.ld + p.conv_off + c;      // the request's first new token
    float* tail = back ? p.state + (size_t)slot * p.state_stride + p.tail_off + c : nullptr;
    // input number r of the request's new tokens, those before the first from the slot
    auto input = [&](int r) { return r >= 0 ? to_float(from[(size_t)r * p.ld]) : tail[(size_t)(back + r) * p.channels]; };
    for (int r = row0; r < row0 + count; ++r) {
        float sum = 0.f;
        for (int j = 0; j < p.taps; ++j) sum = fmaf(p.conv[(size_t)j * p.channels + c], input(r - back + j), sum);
        act[(size_t)(t0 - row0 + r) * p.channels + c] = from_float<T>(prep_silu(sum));
    }
    if (row0 == 0) {
        float moved[PREP_MAX_TAPS - 1];
        for (int j = 0; j < back; ++j) moved[j] = input(qlen - back + j);
        for (int j = 0; j < back; ++j) tail[(size_t)j * p.channels] = moved[j];
    }
}

template <typename T>
static int launch_prep(const void* proj, void* act, const PrepParams& p, int tokens, int tiles, int early, cudaStream_t stream) {
    const bool wide = p.channels % 4 == 0 && p.ld % 4 == 0 && p.conv_off % 4 == 0 && (uintptr_t)proj % 16 == 0 &&
                      (uintptr_t)act % 16 == 0 && (uintptr_t)p.conv % 16 == 0 && (uintptr_t)p.state % 16 == 0 &&
                      p.state_stride % 4 == 0 && p.tail_off % 4 == 0;
    if (wide && p.taps >= 2 && p.taps <= 4) {
        // (no tile holds more tokens than there are)
        const dim3 grid(tiles, (p.channels / 4 + PREP_THREADS - 1) / PREP_THREADS + 1,
                        (min(p.seg_tokens, tokens) + PREP_AHEAD - 1) / PREP_AHEAD);
        if (grid.z > 65535) return ERR_UNSUPPORTED;
        auto kernel = p.taps == 2 ? delta_prep_kernel<T, 2> : p.taps == 3 ? delta_prep_kernel<T, 3> : delta_prep_kernel<T, 4>;
        return launch_dependent_if(early, kernel, grid, dim3(PREP_THREADS), 0, stream, (const T*)proj, (T*)act, p);
    }
    const dim3 grid(tiles, (p.channels + PREP_THREADS - 1) / PREP_THREADS + 1);
    return launch_dependent_if(early, delta_prep_any_kernel<T>, grid, dim3(PREP_THREADS), 0, stream, (const T*)proj, (T*)act, p);
}

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_delta_prep_max_taps() { return PREP_MAX_TAPS; }

int fsie_delta_prep(const void* proj, int tokens, int ld, int conv_off, int a_off, int b_off, const int* item_qstart, const int* item_qlen,
                    const int* item_slots, const int* seg_item, const int* seg_row0, int tiles, int seg_tokens, float* state,
                    long long state_stride, long long tail_off, const float* conv, int taps, int channels, const float* a_log,
                    const float* dt_bias, int heads, void* act, float* log_decay, float* beta, int dtype, int early,
                    cudaStream_t stream) {
    if (tiles <= 0 || tokens <= 0) return 0;
    if (taps < 1 || taps > PREP_MAX_TAPS || (channels + PREP_THREADS - 1) / PREP_THREADS > 65534) return ERR_UNSUPPORTED;
    // only the tile with a request's first token may look at the slot, which that tile also writes
    if (channels <= 0 || heads <= 0 || seg_tokens < 1 || seg_tokens < taps - 1 || (taps > 1 && !state)) return ERR_BAD_ARGUMENT;
    PrepParams p;
    p.ld = ld; p.conv_off = conv_off; p.a_off = a_off; p.b_off = b_off;
    p.item_qstart = item_qstart; p.item_qlen = item_qlen; p.item_slots = item_slots;
    p.seg_item = seg_item; p.seg_row0 = seg_row0; p.seg_tokens = seg_tokens;
    p.state = state; p.state_stride = state_stride; p.tail_off = tail_off;
    p.conv = conv; p.taps = taps; p.channels = channels;
    p.a_log = a_log; p.dt_bias = dt_bias; p.heads = heads; p.log_decay = log_decay; p.beta = beta;
    if (dtype == DTYPE_F32) return launch_prep<float>(proj, act, p, tokens, tiles, early, stream);
    if (dtype == DTYPE_BF16) return launch_prep<bf16>(proj, act, p, tokens, tiles, early, stream);
    return ERR_BAD_ARGUMENT;
}

}  // extern "C"
