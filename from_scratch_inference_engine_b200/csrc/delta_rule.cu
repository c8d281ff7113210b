// The gated delta rule over per-request state.  Per request and head, token by token:
//
//   k' = k / sqrt(|k|^2 + eps)      q' = q / sqrt(|q|^2 + eps)      a_t = exp(log_decay_t)
//   u_t = beta_t (v_t - a_t S_(t-1)^T k'_t)       S_t = a_t S_(t-1) + k'_t u_t^T       o_t = scale S_t^T q'_t
//
// S [heads, dim, vdim] is 32-bit and lives in the request's state slot; a step carries it on from where the step before
// left it.  `share` heads in a row read the same q and k columns.  What a key already holds is taken out before its new
// value goes in, so - other than in the scans of lightning.cu - a chunk's tokens depend on one another through a
// triangular system and not only through sums.
//
// This file: the recurrent form, for steps of few tokens per request and for any sizes.  delta_chunk.cu: the chunked form.
#include "common.cuh"
#include "delta_rule.cuh"
#include <math.h>

namespace fsie {

// ---------------------------------------------------------------------------------------------- recurrent form
// grid (slices of 32 value columns, heads, requests), 256 threads.  A thread keeps rows r, r + GROUPS, ... of its columns
// of S in registers; the two sums over the rows that a token needs, S^T k and S^T q (of the S before the token: the new
// S's sum with q is a S^T q + (k.q) u), are taken in one pass, so a token costs one meeting of the block's warps.
//
// Bound by memory for one token per request: S is read and written once, nothing else is of that size.  The slices are
// narrow (32 columns, a 128-byte line a row) so that one request's heads already give work to many SMs, and all of a
// thread's loads of S are asked for before the kernel in front has finished (`early`).
constexpr int STEP_COLS = 32;
constexpr int STEP_THREADS = 256;
constexpr int STEP_WARPS = STEP_THREADS / 32;
constexpr int STEP_MAX_DIM = 256;

template <int V> struct Cols { float v[V]; };
__device__ __forceinline__ Cols<4> load_cols(const float* p, Cols<4>) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    return {{x.x, x.y, x.z, x.w}};
}
__device__ __forceinline__ Cols<1> load_cols(const float* p, Cols<1>) { return {{*p}}; }
__device__ __forceinline__ void store_cols(float* p, const Cols<4>& c) {
    *reinterpret_cast<float4*>(p) = make_float4(c.v[0], c.v[1], c.v[2], c.v[3]);
}
__device__ __forceinline__ void store_cols(float* p, const Cols<1>& c) { *p = c.v[0]; }

// V columns a thread (4: vdim, the slots and out in whole 16 bytes; else 1), ROWS rows a thread
template <typename T, int V, int ROWS>
__global__ void __launch_bounds__(STEP_THREADS)
delta_step_kernel(const DeltaParams p) {
    constexpr int ACROSS = STEP_COLS / V;                  // threads side by side in a slice's row
    constexpr int GROUPS = STEP_THREADS / ACROSS;          // row groups of the block
    constexpr int IN_WARP = 32 / ACROSS;                   // ... of a warp
    __shared__ float ks[2][STEP_MAX_DIM], qs[2][STEP_MAX_DIM];
    __shared__ float sums[2][STEP_WARPS][2][STEP_COLS];
    const int head = blockIdx.y, item = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = p.item_slots[item], count = p.item_qlen[item], t0 = p.item_qstart[item];
    if (slot < 0 || count <= 0) return;                    // a padding entry of a fixed-size batch
    const int group = tid / ACROSS, at = (tid % ACROSS) * V, col = blockIdx.x * STEP_COLS + at;
    const bool in = col < p.vdim;
    float* state = p.state + (size_t)slot * p.state_stride + (size_t)head * p.dim * p.vdim + col;
    Cols<V> s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = group + i * GROUPS;
#pragma unroll
        for (int x = 0; x < V; ++x) s[i].v[x] = 0.f;
        if (in && r < p.dim) s[i] = load_cols(state + (size_t)r * p.vdim, Cols<V>());
    }
    grid_dependency_wait();
    grid_dependents_go();
    const T* row = (const T*)p.qkv + (size_t)t0 * p.ld;
    const int narrow = head / p.share * p.dim;
    // a thread's part of the next token's q and k (dim is 256 at most, one number of each per thread)
    auto ask = [&](const T* from, float& k, float& q) {
        k = tid < p.dim ? to_float(from[p.k_off + narrow + tid]) : 0.f;
        q = tid < p.dim ? to_float(from[p.q_off + narrow + tid]) : 0.f;
    };
    float k_next, q_next;
    ask(row, k_next, q_next);
    for (int r = 0; r < count; ++r) {
        const int b = r & 1, t = t0 + r;
        if (tid < p.dim) { ks[b][tid] = k_next; qs[b][tid] = q_next; }
        Cols<V> v;
#pragma unroll
        for (int x = 0; x < V; ++x) v.v[x] = in ? to_float(row[p.v_off + head * p.vdim + col + x]) : 0.f;
        const float decay = expf(p.log_decay[(size_t)t * p.heads + head]), beta = p.beta[(size_t)t * p.heads + head];
        row += p.ld;
        __syncthreads();
        if (r + 1 < count) ask(row, k_next, q_next);
        // lengths and product of q and k: every warp by itself, all in the same order
        float kk = 0.f, qq = 0.f, kq = 0.f;
        for (int d = lane; d < p.dim; d += 32) {
            const float k = ks[b][d], q = qs[b][d];
            kk = fmaf(k, k, kk); qq = fmaf(q, q, qq); kq = fmaf(k, q, kq);
        }
        kk = warp_sum(kk); qq = warp_sum(qq); kq = warp_sum(kq);
        const float k_norm = 1.0f / sqrtf(kk + p.eps), q_norm = p.scale / sqrtf(qq + p.eps);
        Cols<V> with_k, with_q;
#pragma unroll
        for (int x = 0; x < V; ++x) with_k.v[x] = with_q.v[x] = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int d = group + i * GROUPS;
            const float k = d < p.dim ? ks[b][d] : 0.f, q = d < p.dim ? qs[b][d] : 0.f;
#pragma unroll
            for (int x = 0; x < V; ++x) {
                with_k.v[x] = fmaf(s[i].v[x], k, with_k.v[x]);
                with_q.v[x] = fmaf(s[i].v[x], q, with_q.v[x]);
            }
        }
#pragma unroll
        for (int o = ACROSS; o < 32; o <<= 1) {
#pragma unroll
            for (int x = 0; x < V; ++x) {
                with_k.v[x] += __shfl_xor_sync(0xffffffffu, with_k.v[x], o);
                with_q.v[x] += __shfl_xor_sync(0xffffffffu, with_q.v[x], o);
            }
        }
        if (IN_WARP == 1 || lane < ACROSS) {
            store_cols(&sums[b][warp][0][at], with_k);
            store_cols(&sums[b][warp][1][at], with_q);
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < V; ++x) with_k.v[x] = with_q.v[x] = 0.f;
#pragma unroll
        for (int w = 0; w < STEP_WARPS; ++w) {
            const Cols<V> a = load_cols(&sums[b][w][0][at], Cols<V>()), c = load_cols(&sums[b][w][1][at], Cols<V>());
#pragma unroll
            for (int x = 0; x < V; ++x) { with_k.v[x] += a.v[x]; with_q.v[x] += c.v[x]; }
        }
        Cols<V> u, o;
#pragma unroll
        for (int x = 0; x < V; ++x) {
            u.v[x] = beta * (v.v[x] - decay * k_norm * with_k.v[x]);
            o.v[x] = q_norm * (decay * with_q.v[x] + kq * k_norm * u.v[x]);
        }
        if (in && group == 0) store_cols(p.out + (size_t)t * p.heads * p.vdim + head * p.vdim + col, o);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int d = group + i * GROUPS;
            const float k = d < p.dim ? ks[b][d] * k_norm : 0.f;
#pragma unroll
            for (int x = 0; x < V; ++x) s[i].v[x] = fmaf(k, u.v[x], decay * s[i].v[x]);
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = group + i * GROUPS;
        if (in && r < p.dim) store_cols(state + (size_t)r * p.vdim, s[i]);
    }
}

template <typename T>
static int launch_step(const DeltaParams& p, int items, int early, cudaStream_t stream) {
    if (p.dim > STEP_MAX_DIM) return ERR_UNSUPPORTED;
    const bool wide = p.vdim % 4 == 0 && p.state_stride % 4 == 0 && (uintptr_t)p.state % 16 == 0 && (uintptr_t)p.out % 16 == 0;
    const dim3 grid((p.vdim + STEP_COLS - 1) / STEP_COLS, p.heads, items);
    if (grid.y > 65535 || grid.z > 65535) return ERR_UNSUPPORTED;
    void (*kernel)(const DeltaParams);
    if (wide) kernel = p.dim <= 64 ? delta_step_kernel<T, 4, 2> : p.dim <= 128 ? delta_step_kernel<T, 4, 4> : delta_step_kernel<T, 4, 8>;
    else kernel = p.dim <= 64 ? delta_step_kernel<T, 1, 8> : p.dim <= 128 ? delta_step_kernel<T, 1, 16> : delta_step_kernel<T, 1, 32>;
    return launch_dependent_if(early, kernel, grid, dim3(STEP_THREADS), 0, stream, p);
}

// delta_chunk.cu
int delta_chunk(const DeltaParams& p, int items, int dtype, void* room, long long room_bytes, int early, cudaStream_t stream);

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_delta_max_dim() { return STEP_MAX_DIM; }

// `form`: 0 the recurrent form, 1 the chunked one, with a workspace `room` of fsie_delta_chunk_bytes() for every chunk
// (of fsie_delta_chunk_tokens() tokens of a request, its last one begun)
int fsie_delta_rule(int form, const void* qkv, int ld, int q_off, int k_off, int v_off, const float* log_decay, const float* beta,
                    const int* item_qstart, const int* item_qlen, const int* item_slots, int items, float* state,
                    long long state_stride, float* out, int heads, int dim, int vdim, int share, float scale, float eps,
                    int dtype, void* room, long long room_bytes, int early, cudaStream_t stream) {
    if (items <= 0) return 0;
    if (heads <= 0 || dim <= 0 || vdim <= 0 || share <= 0 || heads % share != 0 || form < 0 || form > 1) return ERR_BAD_ARGUMENT;
    DeltaParams p;
    p.qkv = qkv; p.ld = ld; p.q_off = q_off; p.k_off = k_off; p.v_off = v_off; p.log_decay = log_decay; p.beta = beta;
    p.item_qstart = item_qstart; p.item_qlen = item_qlen; p.item_slots = item_slots;
    p.state = state; p.state_stride = state_stride; p.out = out;
    p.heads = heads; p.dim = dim; p.vdim = vdim; p.share = share; p.scale = scale; p.eps = eps;
    if (dtype != DTYPE_F32 && dtype != DTYPE_BF16) return ERR_BAD_ARGUMENT;
    if (form == 1) return delta_chunk(p, items, dtype, room, room_bytes, early, stream);
    return dtype == DTYPE_F32 ? launch_step<float>(p, items, early, stream) : launch_step<bf16>(p, items, early, stream);
}

}  // extern "C"
