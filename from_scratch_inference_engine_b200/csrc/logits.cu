// Logits changed before a token is chosen: penalties for tokens that a request's history holds, biases, masks of the
// allowed tokens - and the histories themselves.
//
// A history is a row of counts[slots, vocab] (how often the token was generated) and a row of bits seen[slots, words] (bit
// v % 32 of word v / 32: the token occurs, in the prompt or among the generated).  For row r of the logits with history s,
// penalties (theta, presence, frequency), biases b and a mask:
//
//   z' = (z > 0 ? z / theta : z * theta) - presence * [counts[s, v] > 0] - frequency * counts[s, v]      where seen[s, v]
//   z'' = z' + b[v]      and -inf, whatever z'' is (NaN too), where the mask's bit is clear
//
// in place and in 32 bits.
//
// Bound by memory, and by little of it: the bits tell which logits and counts have to be read at all (a row of 151,936
// tokens: 19 KB of bits per history and mask, against 608 KB of logits and as much of counts).  A thread owns four tokens
// in a row, half a byte of the bits: 16 bytes of logits and counts, read only where a bit of the history is set, written
// without a read where the mask forbids all four.  All of a thread's words are asked for before the first is used.
#include "common.cuh"
#include <math.h>

namespace fsie {

constexpr int ADJUST_THREADS = 256;
constexpr int ADJUST_STEPS = 4;                                        // groups of four tokens per thread
constexpr int ADJUST_SPAN = ADJUST_THREADS * 4 * ADJUST_STEPS;         // tokens of a row that a block owns
enum { ERR_TOKEN_ID = 1, ERR_BIAS_ORDER = 5, ERR_HISTORY_RANGE = 6 };

struct AdjustArgs {
    float* logits; int rows, vocab, words;
    const int* slots; const float* penalties; const int* counts; const unsigned* seen; int slot_count;      // slots: null, or [rows], -1 none
    const int* bias_start; const int* bias_token; const float* bias_value; int bias_count;                  // null, or a list per row
    const int* mask_of; const unsigned* masks; int mask_count;                                              // null, or [rows], -1 none
    int* error;
};

// VEC: rows of logits and counts start on 16 bytes
template <bool VEC>
__global__ void __launch_bounds__(ADJUST_THREADS)
adjust_logits_kernel(const AdjustArgs a) {
    grid_dependency_wait();
    grid_dependents_go();
    const int row = blockIdx.y, first = blockIdx.x * ADJUST_SPAN;
    int slot = a.slots ? a.slots[row] : -1, mask_row = a.mask_of ? a.mask_of[row] : -1;
    if (slot >= a.slot_count || mask_row >= a.mask_count) {
        if (threadIdx.x == 0) atomicExch(a.error, ERR_HISTORY_RANGE);
        if (slot >= a.slot_count) slot = -1;
        if (mask_row >= a.mask_count) mask_row = -1;
    }
    float theta = 1.f, presence = 0.f, frequency = 0.f;
    if (slot >= 0) {
        theta = a.penalties[3 * row]; presence = a.penalties[3 * row + 1]; frequency = a.penalties[3 * row + 2];
        if (theta == 1.f && presence == 0.f && frequency == 0.f) slot = -1;          // a history that changes nothing
    }
    float* logits = a.logits + (size_t)row * a.vocab;
    const unsigned* mask = mask_row >= 0 ? a.masks + (size_t)mask_row * a.words : nullptr;
    if (slot >= 0 || mask) {
        const unsigned* seen = a.seen + (size_t)max(slot, 0) * a.words;
        const int* counts = a.counts + (size_t)max(slot, 0) * a.vocab;
        unsigned held[ADJUST_STEPS], allowed[ADJUST_STEPS];
#pragma unroll
        for (int j = 0; j < ADJUST_STEPS; ++j) {
            const int v = first + (j * ADJUST_THREADS + threadIdx.x) * 4;
            held[j] = slot >= 0 && v < a.vocab ? seen[v >> 5] : 0u;
            allowed[j] = mask && v < a.vocab ? mask[v >> 5] : 0xffffffffu;
        }
#pragma unroll
        for (int j = 0; j < ADJUST_STEPS; ++j) {
            const int v = first + (j * ADJUST_THREADS + threadIdx.x) * 4;
            if (v >= a.vocab) break;
            const unsigned there = a.vocab - v >= 4 ? 15u : (1u << (a.vocab - v)) - 1u;
            const unsigned open = (allowed[j] >> (v & 31)) & there;
            const unsigned hold = (held[j] >> (v & 31)) & open;           // what is forbidden need not be computed
            if (open == there && hold == 0) continue;
            float z[4];
            int n[4];
            if (VEC) {                                                    // (there is 15: the vocabulary is a multiple of 4)
                if (open != 0) {
                    const float4 x = *reinterpret_cast<const float4*>(logits + v);
                    z[0] = x.x; z[1] = x.y; z[2] = x.z; z[3] = x.w;
                }
                if (hold) {
                    const int4 x = *reinterpret_cast<const int4*>(counts + v);
                    n[0] = x.x; n[1] = x.y; n[2] = x.z; n[3] = x.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (hold >> e & 1) { z[e] = logits[v + e]; n[e] = counts[v + e]; }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (hold >> e & 1) {
                    const float repeated = z[e] > 0.f ? z[e] / theta : z[e] * theta;
                    z[e] = repeated - (n[e] > 0 ? presence : 0.f) - frequency * (float)n[e];
                }
                if (!(open >> e & 1)) z[e] = -INFINITY;
            }
            if (VEC) {
                *reinterpret_cast<float4*>(logits + v) = make_float4(z[0], z[1], z[2], z[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((there & (hold | ~open)) >> e & 1) logits[v + e] = z[e];
            }
        }
    }
    if (!a.bias_start) return;
    // biases come behind the penalties: this block's tokens have them now
    __syncthreads();
    const int begin = max(a.bias_start[row], 0), end = min(a.bias_start[row + 1], a.bias_count);
    for (int i = begin + (int)threadIdx.x; i < end; i += ADJUST_THREADS) {
        const int v = a.bias_token[i];
        if ((unsigned)v >= (unsigned)a.vocab) {
            atomicExch(a.error, ERR_TOKEN_ID);
            continue;
        }
        if (v < first || v - first >= ADJUST_SPAN) continue;
        if (i > begin && a.bias_token[i - 1] >= v) {             // a token twice: which of the two would come first is open
            atomicExch(a.error, ERR_BIAS_ORDER);
            continue;
        }
        if (!mask || (mask[v >> 5] >> (v & 31) & 1)) logits[v] += a.bias_value[i];
    }
}

// tokens[i] into history slots[i] (-1: into none).  Sums of whole numbers and bits: the order of the atomics changes nothing.
__global__ void __launch_bounds__(256)
count_tokens_kernel(const int* __restrict__ tokens, const int* __restrict__ slots, int n, int vocab, int words, int slot_count,
                    int* __restrict__ counts, unsigned* __restrict__ seen, int generated, int* __restrict__ error) {
    grid_dependency_wait();
    grid_dependents_go();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int v = tokens[i], slot = slots[i];
    if (slot < 0) return;
    if ((unsigned)v >= (unsigned)vocab) { atomicExch(error, ERR_TOKEN_ID); return; }
    if (slot >= slot_count) { atomicExch(error, ERR_HISTORY_RANGE); return; }
    if (generated) atomicAdd(counts + (size_t)slot * vocab + v, 1);
    unsigned* word = seen + (size_t)slot * words + (v >> 5);
    const unsigned bit = 1u << (v & 31);
    if (!(*(volatile unsigned*)word & bit)) atomicOr(word, bit);
}

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_adjust_logits(float* logits, int rows, int vocab, const int* slots, const float* penalties, const int* counts,
                       const int* seen, int slot_count, const int* bias_start, const int* bias_token, const float* bias_value,
                       int bias_count, const int* mask_of, const int* masks, int mask_count, int* error, cudaStream_t stream) {
    if (rows < 0 || vocab <= 0 || slot_count < 0 || bias_count < 0 || mask_count < 0 || !error) return ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    if (!logits || (slots && (!penalties || (slot_count && (!counts || !seen)))) ||
        (bias_start && bias_count && (!bias_token || !bias_value)) || (mask_of && mask_count && !masks))
        return ERR_BAD_ARGUMENT;
    if (rows > 65535 || vocab > 1 << 30) return ERR_UNSUPPORTED;          // rows are the grid's y dimension
    if (!slots && !bias_start && !mask_of) return 0;
    AdjustArgs a;
    a.logits = logits; a.rows = rows; a.vocab = vocab; a.words = (vocab - 1) / 32 + 1;
    a.slots = slots; a.penalties = penalties; a.counts = counts; a.seen = (const unsigned*)seen; a.slot_count = slot_count;
    a.bias_start = bias_start; a.bias_token = bias_token; a.bias_value = bias_value; a.bias_count = bias_count;
    a.mask_of = mask_of; a.masks = (const unsigned*)masks; a.mask_count = mask_count;
    a.error = error;
    const bool vec = vocab % 4 == 0 && (((uintptr_t)logits | (uintptr_t)counts) & 15) == 0;
    const dim3 grid((vocab - 1) / ADJUST_SPAN + 1, rows);
    return launch_dependent(vec ? adjust_logits_kernel<true> : adjust_logits_kernel<false>, grid, dim3(ADJUST_THREADS), 0,
                            stream, a);
}

int fsie_count_tokens(const int* tokens, const int* slots, int n, int vocab, int slot_count, int* counts, int* seen,
                      int generated, int* error, cudaStream_t stream) {
    if (n < 0 || vocab <= 0 || slot_count < 0 || !error) return ERR_BAD_ARGUMENT;
    if (n == 0) return 0;
    if (!tokens || !slots || !seen || (generated && !counts)) return ERR_BAD_ARGUMENT;
    return launch_dependent(count_tokens_kernel, dim3((n - 1) / 256 + 1), dim3(256), 0, stream, tokens, slots, n, vocab,
                            (vocab - 1) / 32 + 1, slot_count, counts, (unsigned*)seen, generated, error);
}

}  // extern "C"
