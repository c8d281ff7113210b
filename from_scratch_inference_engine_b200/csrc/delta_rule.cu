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
#include <limits.h>
#include <math.h>

namespace fsie {

// ---------------------------------------------------------------------------------------------- recurrent form
// grid (slices of 32 value columns, heads, requests), 256 threads.  A thread keeps rows r, r + GROUPS, ... of its columns
// of S in registers; the two sums over the rows that a token needs, S^T k and S^T q (of the S before the token: the new
// S's sum with q is a S^T q + (k.q) u), are taken in one pass, so a token costs one meeting of the block's warps.
//
// Bound by memory for one token per request: S is read and written once, nothing else is of that size.  The slices are
// narrow (32 columns, a 128-byte line a row) so that one request's heads already give work to many SMs, and all of a
// thread's loads of S are asked for before the kernel in front has finished (`early`).  One request of 16 heads of 128 x 128
// takes 5.0 us: a chain of list, S and two meetings, 2 MB being nothing.
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
    __shared__ __align__(16) float sums[2][STEP_WARPS][2][STEP_COLS];
    const int head = blockIdx.y, item = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = p.item_slots[item], count = p.item_qlen[item], t0 = p.item_qstart[item];
    if (slot < 0 || count < p.least || count > p.most) {   // a padding entry of a fixed-size batch, or the other form's
        if (!p.beside || first_block()) grid_dependency_wait();
        return;
    }
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
    if (p.beside) {
        delta_await(p.go);
    } else {
        grid_dependency_wait();
        grid_dependents_go();
    }
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
    if (p.beside && first_block()) grid_dependency_wait();
}

// ---------------------------------------------------------------------------------------------- many requests
// The same for steps whose states are more than what the SMs work on at once.  What bounds the kernel above then is its
// instructions: a thread has 16 numbers of S, and reading k and q, the sums over the warps and the lengths take it several times
// what the S takes.  Here it has 64 or 32: a block of 2 DIM threads owns DIM rows (64, 96 or 128) x 4 ACROSS columns, ACROSS
// threads side by side in a row and groups of ACROSS / 2 rows.
// 64 requests of 32 heads of 128 x 128 take 49 us (268 MB, 5.4 TB/s; the kernel above 61; a kernel that only reads and
// writes such a state in place 43), 100 of 16 heads of 128 x 160 52 us (57 with a block less per SM), 33 of 6 heads of 96 x 160
// 7.6 us (9.4 with 128 rows to a block), 200 of 12 heads of 64 x 64 15 us.  What is left is the block's own chain: lists, S,
// three meetings, S.  (One block per SM with the next two S on their way into its shared memory took 70 us: its meetings hold up
// everything.)
constexpr int HEAD_MAX_DIM = 128;
constexpr int HEAD_FROM = 64;              // blocks

template <typename T, int ACROSS, int DIM>
__global__ void __launch_bounds__(2 * DIM, ACROSS == 16 ? (DIM == 128 ? 4 : DIM == 96 ? 5 : 8) : DIM == 128 ? 2 : DIM == 96 ? 3 : 4)
delta_head_kernel(const DeltaParams p) {
    constexpr int COLS = 4 * ACROSS, ROWS = ACROSS / 2, WARPS = 2 * DIM / 32;
    __shared__ __align__(16) float ks[2][DIM], qs[2][DIM], sums[2][WARPS][COLS], us[2][COLS];
    const int head = blockIdx.y, item = blockIdx.z, col0 = blockIdx.x * COLS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slot = p.item_slots[item], count = p.item_qlen[item], t0 = p.item_qstart[item];
    if (slot < 0 || count < p.least || count > p.most) {   // a padding entry of a fixed-size batch, or the other form's
        if (!p.beside || first_block()) grid_dependency_wait();
        return;
    }
    const int row0 = tid / ACROSS * ROWS, at = (tid % ACROSS) * 4;     // the thread's rows and columns
    const bool in = col0 + at < p.vdim;
    float* state = p.state + (size_t)slot * p.state_stride + ((size_t)head * p.dim + row0) * p.vdim + col0 + at;
    float4 s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        s[i] = in && row0 + i < p.dim ? *reinterpret_cast<const float4*>(state + (size_t)i * p.vdim) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.beside) {
        delta_await(p.go);
    } else {
        grid_dependency_wait();
        grid_dependents_go();
    }
    // k by the first half of the threads, q by the other; v by the threads that sum up S^T k, later
    const int d = tid < DIM ? tid : tid - DIM, narrow = head / p.share * p.dim;
    const T* row = (const T*)p.qkv + (size_t)t0 * p.ld;
    auto part = [&](const T* from) { return d < p.dim ? to_float(from[(tid < DIM ? p.k_off : p.q_off) + narrow + d]) : 0.f; };
    float mine = part(row);
    for (int r = 0; r < count; ++r) {
        const int turn = r & 1, t = t0 + r;
        (tid < DIM ? ks : qs)[turn][d] = mine;
        const float v = tid < COLS && col0 + tid < p.vdim ? to_float(row[p.v_off + head * p.vdim + col0 + tid]) : 0.f;
        const float decay = expf(p.log_decay[(size_t)t * p.heads + head]), beta = p.beta[(size_t)t * p.heads + head];
        row += p.ld;
        __syncthreads();
        if (r + 1 < count) mine = part(row);
        float4 with_k = make_float4(0.f, 0.f, 0.f, 0.f), with_q = with_k;
#pragma unroll
        for (int i = 0; i < ROWS; i += 4) {
            const float4 k = *reinterpret_cast<const float4*>(&ks[turn][row0 + i]), q = *reinterpret_cast<const float4*>(&qs[turn][row0 + i]);
            const float kx[4] = {k.x, k.y, k.z, k.w}, qx[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 x = s[i + j];
                with_k.x = fmaf(x.x, kx[j], with_k.x); with_k.y = fmaf(x.y, kx[j], with_k.y);
                with_k.z = fmaf(x.z, kx[j], with_k.z); with_k.w = fmaf(x.w, kx[j], with_k.w);
                with_q.x = fmaf(x.x, qx[j], with_q.x); with_q.y = fmaf(x.y, qx[j], with_q.y);
                with_q.z = fmaf(x.z, qx[j], with_q.z); with_q.w = fmaf(x.w, qx[j], with_q.w);
            }
        }
        if (ACROSS == 16) {
            with_k.x += __shfl_xor_sync(0xffffffffu, with_k.x, 16); with_k.y += __shfl_xor_sync(0xffffffffu, with_k.y, 16);
            with_k.z += __shfl_xor_sync(0xffffffffu, with_k.z, 16); with_k.w += __shfl_xor_sync(0xffffffffu, with_k.w, 16);
            with_q.x += __shfl_xor_sync(0xffffffffu, with_q.x, 16); with_q.y += __shfl_xor_sync(0xffffffffu, with_q.y, 16);
            with_q.z += __shfl_xor_sync(0xffffffffu, with_q.z, 16); with_q.w += __shfl_xor_sync(0xffffffffu, with_q.w, 16);
        }
        if (lane < ACROSS) {
            *reinterpret_cast<float4*>(&sums[0][warp][at]) = with_k;
            *reinterpret_cast<float4*>(&sums[1][warp][at]) = with_q;
        }
        // lengths and product of q and k: every warp by itself, all in the same order (zeros beyond dim)
        float kk = 0.f, qq = 0.f, kq = 0.f;
        {
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i) {
                const float k = ks[turn][lane + 32 * i], q = qs[turn][lane + 32 * i];
                kk = fmaf(k, k, kk); qq = fmaf(q, q, qq); kq = fmaf(k, q, kq);
            }
            kk = warp_sum(kk); qq = warp_sum(qq); kq = warp_sum(kq);
        }
        const float k_norm = 1.0f / sqrtf(kk + p.eps);
        __syncthreads();
        // S^T k in COLS threads, S^T q in as many others where there are that many
        constexpr bool HALVES = 2 * DIM >= 2 * COLS;
        float sum_k = 0.f, sum_q = 0.f;
        const int c = tid & (COLS - 1);
        if (tid < COLS) {
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum_k += sums[0][w][c];
            us[turn][c] = beta * (v - decay * k_norm * sum_k) * k_norm;          // u times one over the key's length
        }
        const bool writes = HALVES ? tid >= COLS && tid < 2 * COLS : tid < COLS;
        if (writes) {
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum_q += sums[1][w][c];
        }
        __syncthreads();
        if (writes && col0 + c < p.vdim)
            p.out[(size_t)t * p.heads * p.vdim + head * p.vdim + col0 + c] =
                p.scale / sqrtf(qq + p.eps) * (decay * sum_q + kq * us[turn][c]);
        const float4 u = *reinterpret_cast<const float4*>(&us[turn][at]);
#pragma unroll
        for (int i = 0; i < ROWS; i += 4) {
            const float4 k = *reinterpret_cast<const float4*>(&ks[turn][row0 + i]);
            const float kx[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float4& x = s[i + j];
                x.x = fmaf(kx[j], u.x, decay * x.x); x.y = fmaf(kx[j], u.y, decay * x.y);
                x.z = fmaf(kx[j], u.z, decay * x.z); x.w = fmaf(kx[j], u.w, decay * x.w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (in && row0 + i < p.dim) *reinterpret_cast<float4*>(state + (size_t)i * p.vdim) = s[i];
    if (p.beside && first_block()) grid_dependency_wait();
}

template <typename T>
static int launch_step(const DeltaParams& p, int items, int early, cudaStream_t stream) {
    if (p.dim > STEP_MAX_DIM) return ERR_UNSUPPORTED;
    const bool wide = p.vdim % 4 == 0 && p.state_stride % 4 == 0 && (uintptr_t)p.state % 16 == 0 && (uintptr_t)p.out % 16 == 0;
    // Four requests of 16 heads (64 blocks) take both kernels 6.6 us; fewer blocks leave SMs idle (one request: 6.6 against 5.0).
    // Several tokens: 64 requests of 32 heads and 4 tokens 90 us against 170, 16 of 12 heads of 64 x 64 12 against 16.
    if (wide && p.dim <= HEAD_MAX_DIM) {
        const int across = p.vdim % 128 == 0 || p.vdim % 128 > 64 ? 32 : 16;
        const dim3 grid((p.vdim + 4 * across - 1) / (4 * across), p.heads, items);
        if ((long long)grid.x * grid.y * grid.z >= HEAD_FROM && grid.y <= 65535 && grid.z <= 65535)
            return p.dim <= 64   ? launch_dependent_if(early, across == 32 ? delta_head_kernel<T, 32, 64> : delta_head_kernel<T, 16, 64>,
                                                       grid, dim3(128), 0, stream, p)
                   : p.dim <= 96 ? launch_dependent_if(early, across == 32 ? delta_head_kernel<T, 32, 96> : delta_head_kernel<T, 16, 96>,
                                                       grid, dim3(192), 0, stream, p)
                                 : launch_dependent_if(early, across == 32 ? delta_head_kernel<T, 32, 128> : delta_head_kernel<T, 16, 128>,
                                                       grid, dim3(256), 0, stream, p);
    }
    const dim3 grid((p.vdim + STEP_COLS - 1) / STEP_COLS, p.heads, items);
    if (grid.y > 65535 || grid.z > 65535) return ERR_UNSUPPORTED;
    void (*kernel)(const DeltaParams);
    if (wide) kernel = p.dim <= 64 ? delta_step_kernel<T, 4, 2> : p.dim <= 128 ? delta_step_kernel<T, 4, 4> : delta_step_kernel<T, 4, 8>;
    else kernel = p.dim <= 64 ? delta_step_kernel<T, 1, 8> : p.dim <= 128 ? delta_step_kernel<T, 1, 16> : delta_step_kernel<T, 1, 32>;
    return launch_dependent_if(early, kernel, grid, dim3(STEP_THREADS), 0, stream, p);
}

// delta_chunk.cu
int delta_chunk(const DeltaParams& p, int items, int longer, int dtype, void* room, long long room_bytes, int early, cudaStream_t stream);

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_delta_max_dim() { return STEP_MAX_DIM; }

// `form`: 0 the recurrent form, 1 the chunked one, with a workspace `room` of 16 bytes and
// fsie_delta_chunk_bytes() for every chunk (of fsie_delta_chunk_tokens() tokens of a request, its last one begun).  Form 1 with
// `few` > 0: requests of up to `few` tokens, `ones` at least, in the recurrent form, beside the others.
int fsie_delta_rule(int form, int few, int ones, const void* qkv, int ld, int q_off, int k_off, int v_off, const float* log_decay, const float* beta,
                    const int* item_qstart, const int* item_qlen, const int* item_slots, int items, float* state,
                    long long state_stride, float* out, int heads, int dim, int vdim, int share, float scale, float eps,
                    int dtype, void* room, long long room_bytes, int early, cudaStream_t stream) {
    if (items <= 0) return 0;
    if (heads <= 0 || dim <= 0 || vdim <= 0 || share <= 0 || heads % share != 0 || form < 0 || form > 1) return ERR_BAD_ARGUMENT;
    if (ones < 0 || (form == 1 && ones >= items)) return ERR_BAD_ARGUMENT;
    DeltaParams p;
    p.qkv = qkv; p.ld = ld; p.q_off = q_off; p.k_off = k_off; p.v_off = v_off; p.log_decay = log_decay; p.beta = beta;
    p.item_qstart = item_qstart; p.item_qlen = item_qlen; p.item_slots = item_slots;
    p.state = state; p.state_stride = state_stride; p.out = out;
    p.heads = heads; p.dim = dim; p.vdim = vdim; p.share = share; p.scale = scale; p.eps = eps;
    if (dtype != DTYPE_F32 && dtype != DTYPE_BF16) return ERR_BAD_ARGUMENT;
    p.least = 1; p.most = INT_MAX; p.beside = false; p.go = nullptr;
    if (form == 1) {
        p.least = few > 0 ? few + 1 : 1;
        if (few > 0) p.go = (unsigned*)room;
        const int rc = delta_chunk(p, items, few > 0 ? items - ones : items, dtype, room, room_bytes, early, stream);
        if (rc != 0 || few <= 0) return rc;
        // Behind the walk in the stream, beside it on the GPU: its blocks start when the walk's have, and the first waits for the
        // walk's end at its own, so that whoever waits for them all waits for both.
        p.least = 1; p.most = few; p.beside = true; early = 1;
    }
    return dtype == DTYPE_F32 ? launch_step<float>(p, items, early, stream) : launch_step<bf16>(p, items, early, stream);
}

}  // extern "C"
