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
// Bound by latency and by little memory: the bits tell which logits and counts have to be read at all (a row of 151,936 tokens:
// 19 KB of bits per history and mask, against 608 KB of logits and as much of counts).  A warp owns 1,024 tokens, a word of 32
// bits to a lane.  The tokens that the history holds and the mask allows go into a list, so that a lane has one of them and all
// of a warp's logits and counts are asked for at once; what the mask forbids is written without a read, a word's 32 tokens side
// by side.  64 rows of 152,064 tokens with 1,500 in every history, 22 of them masked, 40 biases: 6.6 us, where 16 bytes were written at a
// time and single tokens where a word is mixed 9.2, and threads that walked four groups of four tokens each, with a wait at each,
// took 12.0; 200 rows with 800 in every history 8.7, those threads 21.7.  Blocks of 2, 4, 8 warps (of the form before): 8.3, 9.2,
// 10.2 us for those 64 rows, 16.1, 9.1, 8.0 for those 200.
#include "common.cuh"
#include <math.h>

namespace fsie {

constexpr int ADJUST_WARPS = 4, ADJUST_THREADS = 32 * ADJUST_WARPS;
constexpr int WARP_TOKENS = 32 * 32, ADJUST_SPAN = ADJUST_WARPS * WARP_TOKENS;           // tokens of a row that a warp, a block owns
enum { ERR_TOKEN_ID = 1, ERR_BIAS_ORDER = 5, ERR_HISTORY_RANGE = 6 };

struct AdjustArgs {
    float* logits; int rows, vocab, words;
    const int* slots; const float* penalties; const int* counts; const unsigned* seen; int slot_count;      // slots: null, or [rows], -1 none
    const int* bias_start; const int* bias_token; const float* bias_value; int bias_count;                  // null, or a list per row
    const int* mask_of; const unsigned* masks; int mask_count;                                              // null, or [rows], -1 none
    int* error;
};

__global__ void __launch_bounds__(ADJUST_THREADS)
adjust_logits_kernel(const AdjustArgs a) {
    __shared__ unsigned short lists[ADJUST_WARPS][WARP_TOKENS];
    grid_dependency_wait();
    grid_dependents_go();
    const int row = blockIdx.y, first = blockIdx.x * ADJUST_SPAN, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int slot = a.slots ? a.slots[row] : -1, mask_row = a.mask_of ? a.mask_of[row] : -1;
    if (slot >= a.slot_count || mask_row >= a.mask_count) {
        if (threadIdx.x == 0) atomicExch(a.error, ERR_HISTORY_RANGE);
        if (slot >= a.slot_count) slot = -1;
        if (mask_row >= a.mask_count) mask_row = -1;
    }
    float theta = 1.f, presence = 0.f, frequency = 0.f;
    if (slot >= 0) { theta = a.penalties[3 * row]; presence = a.penalties[3 * row + 1]; frequency = a.penalties[3 * row + 2]; }
    float* logits = a.logits + (size_t)row * a.vocab;
    const unsigned* mask = mask_row >= 0 ? a.masks + (size_t)mask_row * a.words : nullptr;
    const int base = first + warp * WARP_TOKENS, word = (base >> 5) + lane;                   // the warp's first token, the lane's word
    if ((slot >= 0 || mask) && base < a.vocab) {
        const unsigned held = slot >= 0 && word < a.words ? a.seen[(size_t)slot * a.words + word] : 0u;
        unsigned allowed = mask && word < a.words ? mask[word] : 0xffffffffu;
        if (word == a.words - 1 && a.vocab % 32) allowed &= (1u << a.vocab % 32) - 1u;        // (bits behind the vocabulary)
        // ---- held and allowed: a history that changes nothing is passed over
        unsigned mine = theta == 1.f && presence == 0.f && frequency == 0.f ? 0u : held & allowed;
        int upto = __popc(mine), count = upto;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        const int total = __shfl_sync(0xffffffffu, upto, 31);
        for (int at = upto - count; mine; mine &= mine - 1) lists[warp][at++] = (unsigned short)(32 * lane + __ffs(mine) - 1);
        __syncwarp();
        const int* counts = a.counts + (size_t)max(slot, 0) * a.vocab;
        for (int i = lane; i < total; i += 32) {
            const int v = base + lists[warp][i];
            const float z = logits[v];
            const int n = counts[v];
            const float repeated = z > 0.f ? z / theta : z * theta;
            logits[v] = repeated - (n > 0 ? presence : 0.f) - frequency * (float)n;
        }
        // ---- forbidden: a word's tokens side by side
        if (mask) {
#pragma unroll
            for (int w = 0; w < 32; ++w) {
                const unsigned bits = __shfl_sync(0xffffffffu, allowed, w);
                const int v = base + 32 * w + lane;
                if (!(bits >> lane & 1) && v < a.vocab) logits[v] = -INFINITY;
            }
        }
    }
    if (!a.bias_start) return;
    const int begin = max(a.bias_start[row], 0), end = min(a.bias_start[row + 1], a.bias_count);
    auto add = [&](int i, int v) {
        if ((unsigned)v >= (unsigned)a.vocab) atomicExch(a.error, ERR_TOKEN_ID);
        else if (i > begin && a.bias_token[i - 1] >= v) atomicExch(a.error, ERR_BIAS_ORDER);
        else if (!mask || (mask[v >> 5] >> (v & 31) & 1)) logits[v] += a.bias_value[i];
    };
    // what this block has to do with (whatever is outside the vocabulary is the first block's)
    auto is_mine = [&](int v) { return (unsigned)v < (unsigned)a.vocab ? v >= first && v - first < ADJUST_SPAN : first == 0; };
    int mine = 0, at = 0, token = 0;                             // of the thread's share of the list; the last of them
    bool disordered = false;                                     // somewhere in the row's list
    for (int i = begin + (int)threadIdx.x; i < end; i += ADJUST_THREADS) {
        const int v = a.bias_token[i];
        disordered |= i > begin && a.bias_token[i - 1] >= v;
        if (is_mine(v)) { ++mine; at = i; token = v; }
    }
    // biases come behind the penalties: this block's tokens have them now
    if (__syncthreads_or(disordered)) {                          // a token may be there twice: one after the other
        if (threadIdx.x == 0)
            for (int i = begin; i < end; ++i) { const int v = a.bias_token[i]; if (is_mine(v)) add(i, v); }
    } else if (mine == 1) {
        add(at, token);
    } else if (mine) {
        for (int i = begin + (int)threadIdx.x; i < end; i += ADJUST_THREADS) { const int v = a.bias_token[i]; if (is_mine(v)) add(i, v); }
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
    const dim3 grid((vocab - 1) / ADJUST_SPAN + 1, rows);
    return launch_dependent(adjust_logits_kernel, grid, dim3(ADJUST_THREADS), 0, stream, a);
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
