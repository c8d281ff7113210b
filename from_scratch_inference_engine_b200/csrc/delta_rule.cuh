// Arguments shared by the two forms of the gated delta rule (delta_rule.cu has the formulas).
#pragma once

namespace fsie {

__device__ __forceinline__ bool first_block() { return (blockIdx.x | blockIdx.y | blockIdx.z) == 0; }

struct DeltaParams {
    const void* qkv; int ld, q_off, k_off, v_off;          // [tokens, ld]; heads / share q and k columns of dim, heads of vdim
    const float* log_decay; const float* beta;             // [tokens, heads]
    const int* item_qstart; const int* item_qlen; const int* item_slots;   // [items]
    float* state; long long state_stride;                  // [slots], S [heads, dim, vdim] in front of each
    float* out;                                            // [tokens, heads * vdim]
    int heads, dim, vdim, share;
    int least, most;                                       // tokens of a request that the launch takes; it leaves others alone
    bool beside;                                           // the recurrent form runs beside the chunked one's launches
    unsigned* go;                                          // ... and its inputs are there when this is 1 (delta_await)
    float scale, eps;
};

// The recurrent launch beside the walk starts when every block of the walk has, whose wait for the records' kernel is over, whose own
// wait made visible to it what stands in front of the rule.  No wait of the launch's own is among these: it would be one for the walk's end.
// So the order is handed on: the records' kernel clears the word behind its wait, the walk's first block, behind its own, releases it
// as 1, and a block here acquires that before it reads what the kernels in front may have written.  The poll's first answer is
// 1 but for a few hundred cycles; a block that is not answered waits for the walk's end.
constexpr unsigned DELTA_GO = 1;
__device__ __forceinline__ void delta_release(unsigned* word, unsigned value) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(word), "r"(value) : "memory");
}
__device__ __forceinline__ void delta_await(const unsigned* word) {
    if (threadIdx.x == 0) {
        unsigned seen = 0;
        for (int i = 0; i < 1000 && seen != DELTA_GO; ++i)
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(word) : "memory");
        if (seen != DELTA_GO) grid_dependency_wait();
    }
    __syncthreads();
}

}  // namespace fsie
