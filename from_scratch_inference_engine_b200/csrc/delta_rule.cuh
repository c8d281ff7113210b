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
    float scale, eps;
};

}  // namespace fsie
