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
// Bound by memory: the projection's columns are read and c is written once.  A thread owns eight neighbouring channels
// (16-byte accesses in bfloat16) and walks the tile's tokens with the last taps - 1 inputs in registers, so that no input
// is read for every tap again; the loads of PREP_AHEAD tokens go out together.
#include "common.cuh"
#include <math.h>

namespace fsie {

constexpr int PREP_THREADS = 128;
constexpr int PREP_AHEAD = 8;
constexpr int PREP_MAX_TAPS = 16;

__device__ __forceinline__ float prep_silu(float z) { return z / (1.0f + expf(-z)); }
__device__ __forceinline__ float prep_softplus(float z) { return z > 20.f ? z : log1pf(expf(z)); }

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

// grid (tiles, slices of channels and one more for the gates)
template <typename T, int TAPS>
__global__ void __launch_bounds__(PREP_THREADS)
delta_prep_kernel(const T* __restrict__ proj, T* __restrict__ act, const PrepParams p) {
    const int tile = blockIdx.x;
    const int item = p.seg_item[tile], row0 = p.seg_row0[tile];
    const int qlen = p.item_qlen[item], slot = p.item_slots[item];
    const int count = min(p.seg_tokens, qlen - row0), t0 = p.item_qstart[item] + row0;
    const int c = (blockIdx.y * PREP_THREADS + threadIdx.x) * 8;
    const bool gates = blockIdx.y == gridDim.y - 1, mine = !gates && c < p.channels;
    float w[TAPS][8];
    if (mine) {
#pragma unroll
        for (int j = 0; j < TAPS; ++j) load8(p.conv + (size_t)j * p.channels + c, w[j]);
    }
    grid_dependency_wait();
    grid_dependents_go();
    if (slot < 0 || count <= 0) return;                    // a padding entry of a fixed-size batch
    if (gates) { prep_gates(p, proj, t0, count); return; }
    if (!mine) return;
    const T* from = proj + (size_t)t0 * p.ld + p.conv_off + c;
    T* to = act + (size_t)t0 * p.channels + c;
    float* tail = p.state + (size_t)slot * p.state_stride + p.tail_off + c;
    float last[TAPS - 1][8];                               // the inputs before the next token, oldest first
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) {
        if (row0 == 0) load8(tail + (size_t)j * p.channels, last[j]);
        else load8(from - (ptrdiff_t)(TAPS - 1 - j) * p.ld, last[j]);     // row0 >= taps - 1
    }
    for (int r0 = 0; r0 < count; r0 += PREP_AHEAD) {
        float u[PREP_AHEAD][8];
#pragma unroll
        for (int r = 0; r < PREP_AHEAD; ++r)
            if (r0 + r < count) load8(from + (size_t)(r0 + r) * p.ld, u[r]);
#pragma unroll
        for (int r = 0; r < PREP_AHEAD; ++r) {
            if (r0 + r < count) {
                float sum[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum[i] = w[0][i] * last[0][i];
#pragma unroll
                    for (int j = 1; j < TAPS - 1; ++j) sum[i] = fmaf(w[j][i], last[j][i], sum[i]);
                    sum[i] = prep_silu(fmaf(w[TAPS - 1][i], u[r][i], sum[i]));
                }
                store8(to + (size_t)(r0 + r) * p.channels, sum);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
#pragma unroll
                    for (int j = 0; j + 1 < TAPS - 1; ++j) last[j][i] = last[j + 1][i];
                    last[TAPS - 2][i] = u[r][i];
                }
            }
        }
    }
    if (row0 == 0) {
        if (count < qlen) {                                // the request's last tokens are another tile's
            const T* end = from + (size_t)qlen * p.ld;
#pragma unroll
            for (int j = 0; j < TAPS - 1; ++j) load8(end - (ptrdiff_t)(TAPS - 1 - j) * p.ld, last[j]);
        }
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) store8(tail + (size_t)j * p.channels, last[j]);
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
static int launch_prep(const void* proj, void* act, const PrepParams& p, int tiles, int early, cudaStream_t stream) {
    const bool wide = p.channels % 8 == 0 && p.ld % 8 == 0 && p.conv_off % 8 == 0 && (uintptr_t)proj % 16 == 0 &&
                      (uintptr_t)act % 16 == 0 && (uintptr_t)p.conv % 16 == 0 && (uintptr_t)p.state % 16 == 0 &&
                      p.state_stride % 4 == 0 && p.tail_off % 4 == 0;
    if (wide && p.taps >= 2 && p.taps <= 4) {
        const dim3 grid(tiles, (p.channels / 8 + PREP_THREADS - 1) / PREP_THREADS + 1);
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

int fsie_delta_prep(const void* proj, int ld, int conv_off, int a_off, int b_off, const int* item_qstart, const int* item_qlen,
                    const int* item_slots, const int* seg_item, const int* seg_row0, int tiles, int seg_tokens, float* state,
                    long long state_stride, long long tail_off, const float* conv, int taps, int channels, const float* a_log,
                    const float* dt_bias, int heads, void* act, float* log_decay, float* beta, int dtype, int early,
                    cudaStream_t stream) {
    if (tiles <= 0) return 0;
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
    if (dtype == DTYPE_F32) return launch_prep<float>(proj, act, p, tiles, early, stream);
    if (dtype == DTYPE_BF16) return launch_prep<bf16>(proj, act, p, tiles, early, stream);
    return ERR_BAD_ARGUMENT;
}

}  // extern "C"
