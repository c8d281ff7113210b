// Attention of a step's new tokens over a paged cache in which several requests hold the same leading pages: the keys and
// values that they share are read once for all of them.  Compiled per head size (-DHEAD_DIM=N, a multiple of 16 up to 256),
// for bfloat16 and float32 storage; 32-bit scores, softmax statistics and sums.
//
// Mathematics.  The keys that token t sees are cut into runs: ranges of keys, each with all tokens that see it there.  For
// row x (a token's query head) and a set K of keys
//
//   m = max_K s_j     l = sum_K e^(s_j - m)     o = sum_K e^(s_j - m) v_j         s_j = (q_x . k_j) * scale
//
// and two such triples over disjoint sets join to one over their union; the result is o / l over all of the row's runs.
// `order` lists the tokens so that every run's are neighbours in it; a run is (first place in order, count, first key, end
// of keys, row of the block tables that names the keys' pages, the run around it or -1), and comes behind the run around
// it.  own_run[place] is the innermost run of the token at that place: one request's own keys, of which each of its tokens
// sees those up to its position, so it is worked on token by token.  The runs around it hold keys that all of their
// tokens see, so their rows - a row is a (token, head of the group) pair - fill tiles whatever request they are of, and no
// row of any tile sees other keys than the tile's other rows.
//
// Two launches.  What the runs are is known on the device only (a captured graph replays with others), so every block works
// the plan out by itself: all (tile, kv head) lines of the runs laid end to end, in steps of keys, cut into equal pieces, one
// per worker; runs of few rows (a token's own keys) and of many (shared ones) are two such rows of lines.  The first launch
// walks through both, a worker from line to line with the next steps' keys on their way, and leaves the triple of every
// stretch of a line that it has worked on in `room`:
//
//   many rows   tcgen05 (head sizes 64 and 128), mma.sync or FFMA: a worker is a block
//   few rows    a worker is a warp (bfloat16; fed by the copy engine beside tcgen05, by copies of 16 bytes beside mma.sync) or a
//               block (float32)
//
// The second joins the triples of a row, in a fixed order; it makes its plan while the first still runs.
//
// What a small call waits for is a chain of reads of what other multiprocessors hold, 750 cycles each, and instructions that
// run for the first time.  8 requests of a 4,096-token prompt, 28 heads over 4 of 128: 23.9 us with a launch for the plan in
// front, one each for many and few rows and one for the merge; 31.5 in one cooperative launch whose blocks meet twice
// (6 of them between two such launches); 20.7 in two, and 15.2 since their code is shorter and more of their warps join.
#include "common.cuh"
#include "tma.cuh"
#include "attention_tc.cuh"
#include <math.h>
#include <atomic>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head size: 16..256 in steps of 16");

namespace fsie {

constexpr int HD = HEAD_DIM;
constexpr int FEW = 16;                  // rows that count as few: those of a tile
constexpr int MMA_FEW_KEYS = 16, MMA_MANY_KEYS = HD <= 128 ? 64 : 32, F32_KEYS = 32;       // keys of a step
constexpr int MAX_RUNS = 768;
constexpr int MAX_LEVELS = 32;           // runs that lie around each other, the innermost among them
constexpr int RUN_INTS = 6;
// A line is cut into no more pieces than this: what joins them reads them all.  Two requests with 32,768 keys in common: 32 pieces
// 97 us, 128 35, 256 29, 512 28; with 8,192 in common 128 19, 256 21.
constexpr int LINE_PIECES = 256;
constexpr int FEW_LEAST = 2, MANY_LEAST = 1;                              // steps of a piece, at least
enum { ERR_PAGE = 3, ERR_RUNS = 7, ERR_ROOM = 8 };

// Division by a number that the host knows, for dividends below 2^31: a product's upper half, a sum and a shift (Granlund and
// Montgomery, Division by invariant integers using multiplication, 1994).  A division by any number is some forty instructions,
// and a call of few steps waits for every one of them, which runs for the first time.
struct Div {
    unsigned factor; int shift;
    __device__ __forceinline__ int of(int n) const { return (int)((__umulhi(factor, (unsigned)n) + (unsigned)n) >> shift); }
};
static int log2_of(int n) { int shift = 0; while (1 << shift < n) ++shift; return shift; }
static Div div_by(long long d) {
    int shift = 0;
    while ((1LL << shift) < d) ++shift;
    return {(unsigned)(((1ULL << 32) * ((1ULL << shift) - (unsigned long long)d)) / (unsigned long long)d + 1), shift};
}

// One side of the plan: the runs of few rows or of many.
struct Side {
    int workers, line_room, tile, keys, align, least;         // (align: where steps begin; it, tile and keys are powers of two)
    int tile_shift, key_shift;
    int tokens, parts;                   // tokens of a shared run's tile; tiles of a token, where there are several
    Div by_tokens, by_parts, by_workers;
    int of_block;                        // (few) workers of a block
    int fixed, of_step;                  // (few) tenths of steps in whose time a worker's block does a piece of many rows: to begin, per step
    long long row0;                      // the triples of stretch s are rows row0 + s * tile ..
};

struct SharedArgs {
    const void* q; int q_ld;                                  // [tokens, q_ld]; head h of token t at t * q_ld + h * HD
    const void* k_pages; const void* v_pages; long long page_stride; int page_size, num_pages;
    const int* block_tables; int table_rows, table_width;
    const int* positions; int tokens;                         // [tokens]
    const int* order; int places;                             // [places]
    const int* runs; int run_count;                           // [run_count, RUN_INTS]
    const int* own_run;                                       // [places]
    void* out; int out_ld;
    int heads, kv_heads, group; float scale;
    Side few, many;
    float* part_ml; float* part_o;                            // the triples: [rows, 2], [rows, HD]
    int early;                                                // the lists are older than the stream's last kernel
    int most_steps;                                           // of a run, so that no sum of all passes 2^31
    Div by_kv_heads, by_group, by_chunks, by_place;           // (the last two: see the join)
    int* error;
};

// ---------------------------------------------------------------------------------------------------- plan
struct Run { int first, count, begin, end, table, parent; };
enum { RUN_INNERMOST = 1, RUN_FEW = 2 };

// Tiles of up to `most` rows.  One holds whole tokens (in an innermost run a single one), or, of a group that is larger, a
// part of one token: so all rows of a token and kv head that lie in one tile lie side by side, here and in what is left for
// the merge.
__device__ __forceinline__ int line_steps(const Run& run, const Side& side) { return ((run.end - (run.begin & ~(side.align - 1)) - 1) >> side.key_shift) + 1; }
__device__ __forceinline__ int tile_tokens(const Side& side, int kind) { return kind & RUN_INNERMOST ? 1 : side.tokens; }

// What every block keeps in shared memory.
struct Plan {
    Run* runs;                           // [run_count]; count 0 where a run has no keys or places, or points outside of what there is
    int *sums, stride;                   // see line0 and step0
    unsigned char* kind;
    int few_piece, many_piece, few_total, many_total, few_lines, many_lines;      // steps of a piece, steps and lines in all
    int free_workers, free_piece;        // few: the first workers, whose blocks have no piece of many, and the steps of their pieces
    // [run_count + 1] lines and steps in front of each run, few (0) and many (1)
    __device__ __forceinline__ int* line0(int many) const { return sums + many * stride; }
    __device__ __forceinline__ int* step0(int many) const { return sums + (2 + many) * stride; }
};
__host__ __device__ __forceinline__ size_t plan_bytes(int runs) { return ((size_t)runs * (sizeof(Run) + 1) + 4 * ((size_t)runs + 1) * 4 + 15) / 16 * 16; }
constexpr int MAX_WARPS = 10;            // of a block
struct PlanSums { int sums[4][MAX_WARPS], longest[2][MAX_WARPS]; };

__device__ __forceinline__ int run_kind(const SharedArgs& a, const Run& run, int r) {
    const int innermost = a.own_run[run.first] == r ? RUN_INNERMOST : 0;
    return innermost | ((innermost ? a.group : run.count * a.group) <= FEW ? RUN_FEW : 0);
}

// All PLAN_THREADS threads of a block; false (and *error): it does not fit the room.
template <int PLAN_THREADS>
__device__ __forceinline__ bool make_plan(const SharedArgs& a, unsigned char* smem, PlanSums& s, Plan& plan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    plan.runs = reinterpret_cast<Run*>(smem);
    plan.sums = reinterpret_cast<int*>(plan.runs + a.run_count);
    plan.stride = a.run_count + 1;
    plan.kind = reinterpret_cast<unsigned char*>(plan.sums + 4 * plan.stride);
    for (int e = tid; e < a.run_count * RUN_INTS; e += PLAN_THREADS) reinterpret_cast<int*>(plan.runs)[e] = a.runs[e];
    __syncthreads();
    // ---- runs: checked, sorted into few and many, summed up
    int before[4] = {0, 0, 0, 0}, longest[2] = {0, 0};                    // lines of few and many, steps of few and many
    bool overflow = false;
    for (int base = 0; base < a.run_count; base += PLAN_THREADS) {
        const int r = base + tid;
        int mine[4] = {0, 0, 0, 0};
        if (r < a.run_count) {
            Run run = plan.runs[r];
            int kind = 0;
            if (run.count <= 0 || run.end <= run.begin) {
                run.count = 0;
            } else if (run.first < 0 || run.count > a.places || run.first > a.places - run.count || run.begin < 0 ||
                       run.end > (long long)a.table_width * a.page_size || (unsigned)run.table >= (unsigned)a.table_rows ||
                       run.parent < -1 || run.parent >= r) {
                atomicExch(a.error, ERR_RUNS);
                run.count = 0;
            } else {
                kind = run_kind(a, run, r);
                const int many = kind & RUN_FEW ? 0 : 1;
                const Side& side = many ? a.many : a.few;
                const int of_line = line_steps(run, side);
                const int lines = (tile_tokens(side, kind) == 1 ? run.count * side.parts : side.by_tokens.of(run.count - 1) + 1) * a.kv_heads;
                const long long steps = (long long)lines * of_line;
                overflow = overflow || max(steps, (long long)lines) > a.most_steps;
                mine[many] = lines; mine[2 + many] = (int)steps;
                longest[many] = max(longest[many], of_line);
            }
            plan.runs[r].count = run.count;
            plan.kind[r] = (unsigned char)kind;
        }
        int upto[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            upto[i] = mine[i];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int u = __shfl_up_sync(0xffffffffu, upto[i], o);
                if (lane >= o) upto[i] += u;
            }
            if (lane == 31) s.sums[i][warp] = upto[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int of_warp = lane < PLAN_THREADS / 32 ? s.sums[i][lane] : 0;
            upto[i] += before[i] + (int)__reduce_add_sync(0xffffffffu, lane < warp ? (unsigned)of_warp : 0u);
            before[i] += (int)__reduce_add_sync(0xffffffffu, (unsigned)of_warp);
        }
        if (r < a.run_count) {
#pragma unroll
            for (int i = 0; i < 4; ++i) plan.sums[i * plan.stride + r] = upto[i] - mine[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        longest[i] = __reduce_max_sync(0xffffffffu, longest[i]);
        if (lane == 0) s.longest[i][warp] = longest[i];
        if (tid == 0) { plan.line0(i)[a.run_count] = before[i]; plan.step0(i)[a.run_count] = before[2 + i]; }
    }
    overflow = __syncthreads_or(overflow);
    bool fits = !overflow;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Side& side = i ? a.many : a.few;
        const int l = __reduce_max_sync(0xffffffffu, lane < PLAN_THREADS / 32 ? s.longest[i][lane] : 0);
        (i ? plan.many_lines : plan.few_lines) = before[i];
        (i ? plan.many_total : plan.few_total) = before[2 + i];
        const int least = max(side.least, (l + LINE_PIECES - 1) / LINE_PIECES);
        (i ? plan.many_piece : plan.few_piece) = max(side.by_workers.of(max(before[2 + i] - 1, 0)) + 1, least);
        if (i == 0) plan.free_piece = least;
        // pieces that end where long lines do: a piece in two lines loads two sets of queries and leaves two sets of triples
        // (100 requests with 16,384 keys in common 67.8 -> 55.1 us)
        if (i == 1 && plan.many_piece > 4 && plan.many_piece < l) {
            const int pieces = l / plan.many_piece, even = (l - 1) / pieces + 1;
            if (4 * even <= 5 * plan.many_piece) plan.many_piece = even;
        }
        fits = fits && before[i] <= side.line_room;
    }
    if (!fits && tid == 0) atomicExch(a.error, ERR_ROOM);
    // ---- blocks without a piece of many rows take more of the few, so that all are done at about the same time.  (Whole numbers:
    // every block of both launches comes to the same.)
    plan.free_workers = 0;
    const int least = plan.free_piece, blocks = a.many.workers, of_block = a.few.of_block;
    if (plan.many_total == 0 || plan.many_piece > 4096 || plan.few_total > 1 << 30) return fits;
    // (the few go to the last blocks first: where the least pieces of them find room on blocks without many, all is well)
    if (plan.many_piece == 1 && plan.few_total <= (blocks - plan.many_total) * of_block * least) return fits;
    if (plan.many_piece <= 2) {                           // pieces of 2 or 4 steps on fewer blocks: what it takes to begin weighs less
        long long best = 0x7fffffffffffffffLL;
        int piece = 0;
#pragma unroll
        for (int shift = 0; shift < 3; ++shift) {
            const int later = a.few.fixed + (a.few.of_step << shift), busy = ((plan.many_total - 1) >> shift) + 1;
            const long long until = max((long long)later * a.few.workers, 10LL * plan.few_total + (long long)busy * of_block * later);
            if (1 << shift >= plan.many_piece && until < best) { best = until; piece = 1 << shift; }
        }
        plan.many_piece = piece;
    }
    const int busy = (plan.many_total - 1) / plan.many_piece + 1, free_workers = (blocks - busy) * of_block;
    if (free_workers > 0) {
        const int later = (a.few.fixed + a.few.of_step * plan.many_piece + 9) / 10;
        const int alone = max((plan.few_total + free_workers - 1) / free_workers, least);
        const int all = a.few.by_workers.of(plan.few_total + busy * of_block * later - 1) + 1;
        plan.free_workers = free_workers;
        plan.few_piece = alone <= later + least ? 0 : max(all - later, least);           // (0: the others have none)
        plan.free_piece = plan.few_piece == 0 ? alone : plan.few_piece + later;
    }
    return fits;
}

// ---- a worker's piece, as stretches: the part of a line that lies in it.  The lines of a side are numbered through, so the
// k-th stretch of a worker belongs to the k-th line behind its first, and any thread can work out any stretch by itself.
struct __align__(16) Stretch {
    int steps, k0, kend, slot;           // 0: there is none; first step's first key, end of the keys; where the triple goes, in tiles
    int table, kvh, place, row0;         // row of the block tables; the tile's rows are rows row0 .. of the tokens from `place` on
    int rows, begin, token, spare;       // (begin: the run's first key: steps may begin in front of it; token: that of a tile of one)
};
struct Piece { int from, end, first_line, worker; };          // steps, and the line in which the piece starts; from = end: no piece

// largest r with at[r] <= value, for at[0] <= value < at[count]
__device__ __forceinline__ int find_run(const int* at, int count, int value) {
    int low = 0, high = count;
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (at[middle] <= value) low = middle; else high = middle;
    }
    return low;
}

template <int MANY>
__device__ __forceinline__ Piece piece_of(const SharedArgs& a, const Plan& plan, int worker) {
    const Side& side = MANY ? a.many : a.few;
    const int step_piece = MANY ? plan.many_piece : plan.few_piece, total = MANY ? plan.many_total : plan.few_total;
    Piece piece = {0, 0, 0, worker};
    long long from = (long long)worker * step_piece;
    int size = step_piece;
    if (!MANY && plan.free_workers > 0) {
        const int further = max(worker - plan.free_workers, 0);
        from = (long long)(worker - further) * plan.free_piece + (long long)further * step_piece;
        if (worker < plan.free_workers) size = plan.free_piece;
    }
    if (from >= total || size == 0) return piece;
    piece.from = (int)from;
    piece.end = piece.from + min(size, total - piece.from);
    const int r = find_run(plan.step0(MANY), a.run_count, piece.from);
    piece.first_line = plan.line0(MANY)[r] + (piece.from - plan.step0(MANY)[r]) / line_steps(plan.runs[r], side);
    return piece;
}
// the worker whose piece a step lies in
__device__ __forceinline__ int piece_at(const Plan& plan, int many, int step) {
    if (many) return step / plan.many_piece;
    const long long free_steps = (long long)plan.free_workers * plan.free_piece;
    if (step < free_steps) return step / plan.free_piece;
    return plan.free_workers + (int)(step - free_steps) / plan.few_piece;
}
template <int MANY>
__device__ __forceinline__ void stretch_of(const SharedArgs& a, const Plan& plan, const Piece& piece, int k, Stretch& n) {
    const Side& side = MANY ? a.many : a.few;
    n.steps = 0;
    const int number = piece.first_line + k;
    if (piece.from == piece.end || number >= (MANY ? plan.many_lines : plan.few_lines)) return;
    const int r = find_run(plan.line0(MANY), a.run_count, number);
    const Run run = plan.runs[r];
    const int kind = plan.kind[r], line = number - plan.line0(MANY)[r], of_line = line_steps(run, side), begin = plan.step0(MANY)[r] + line * of_line;
    const int first = max(begin, piece.from), last = min(begin + of_line, piece.end);
    if (first >= last) return;
    const int tokens = tile_tokens(side, kind), tile = a.by_kv_heads.of(line);
    n.kvh = line - tile * a.kv_heads;
    const int token = side.parts > 1 ? side.by_parts.of(tile) : tile * tokens;
    n.place = run.first + token;
    n.row0 = side.parts > 1 ? (tile - token * side.parts) * side.tile : 0;
    n.rows = min(side.tile, side.parts > 1 ? a.group - n.row0 : min(tokens, run.count - token) * a.group);
    n.k0 = (run.begin & ~(side.align - 1)) + (first - begin) * side.keys;
    n.begin = run.begin; n.kend = run.end; n.table = run.table;
    n.slot = number + piece.worker;
    n.token = tokens == 1 ? a.order[n.place] : -1;
    if (kind & RUN_INNERMOST) {
        const int position = (unsigned)n.token < (unsigned)a.tokens ? a.positions[n.token] : -1;
        if (position < run.end) n.kend = position + 1;
    }
    n.steps = last - first;
}

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {
    const int bytes = valid ? 16 : 0;                      // 0 source bytes: zeros arrive
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix_x4(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
// d += a (16 x 16, rows) b (16 x 8, columns)
__device__ __forceinline__ void mma_bf16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}

constexpr float LOG2E = 1.4426950408889634f;
// (volatile: several of them in a row go out before the first result is used)
__device__ __forceinline__ float4 load_now(const float4* p) {
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float2 load_now(const float2* p) {
    float2 v;
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
    return v;
}

// ---- blocks of 128 threads that share steps: the ring of steps, and their keys and query rows on the way
constexpr int THREADS = 128;
struct Step {
    Stretch of;
    int valid, k0, first, last;          // whether there is one; its first key; first or last of its stretch
    int stretch;                         // how many stretches the worker has begun before
};
template <typename T, int ROWS, bool IS_FEW, int KEYS, int STAGES, int K_LD, int V_LD, int Q_LD>
struct Feed {
    static constexpr int PIECES = HD * (int)sizeof(T) / 16;               // 16-byte pieces of a head
    static constexpr int EACH = 16 / (int)sizeof(T);
    static constexpr int RECORDS = STAGES + 2, BASES = STAGES + 1;
    struct Shared {
        long long key_base[BASES][KEYS];                                  // element offset of a key's row in the pages; -1: no key
        Stretch stretch;                                                  // thread 0's: the stretch it is at
        Step steps[RECORDS];
    };
    const SharedArgs& a;
    const Plan& plan;
    Shared& sh;
    T *ks, *vs, *qs;
    Piece piece;
    int stretches, at;                                                    // thread 0's: the stretch, and the step of it

    __device__ Feed(const SharedArgs& args, const Plan& p, Shared& shared, T* k, T* v, T* q) : a(args), plan(p), sh(shared), ks(k), vs(v), qs(q) {}

    __device__ void next(Step& out) {                                     // (thread 0)
        out.valid = sh.stretch.steps != 0;
        if (!out.valid) return;
        out.of = sh.stretch;
        out.k0 = sh.stretch.k0 + at * KEYS;
        out.first = at == 0;
        out.last = at + 1 == sh.stretch.steps;
        out.stretch = stretches;
        if (++at < sh.stretch.steps) return;
        at = 0;
        stretch_of<!IS_FEW>(a, plan, piece, ++stretches, sh.stretch);
    }
    __device__ void find(int n) {                                         // where the keys of step n lie
        const Step& st = sh.steps[n % RECORDS];
        if (threadIdx.x >= KEYS || !st.valid) return;
        const int key = st.k0 + (int)threadIdx.x;
        long long base = -1;
        if (key < st.of.kend) {
            const int block = key / a.page_size;
            const int page = a.block_tables[(size_t)st.of.table * a.table_width + block];
            if ((unsigned)page < (unsigned)a.num_pages)
                base = (long long)page * a.page_stride + ((long long)st.of.kvh * a.page_size + (key - block * a.page_size)) * HD;
            else
                atomicExch(a.error, ERR_PAGE);
        }
        sh.key_base[n % BASES][threadIdx.x] = base;
    }
    __device__ void fetch(int n) {                                        // step n's keys and values, a stretch's queries
        const Step& st = sh.steps[n % RECORDS];
        if (st.valid) {
            T* kd = ks + (size_t)(n % STAGES) * KEYS * K_LD;
            T* vd = vs + (size_t)(n % STAGES) * KEYS * V_LD;
            const T* kp = (const T*)a.k_pages;
            const T* vp = (const T*)a.v_pages;
#pragma unroll 4
            for (int e = threadIdx.x; e < KEYS * PIECES; e += THREADS) {
                const int j = e / PIECES, c = (e - j * PIECES) * EACH;
                const long long base = sh.key_base[n % BASES][j];
                const long long from = (base >= 0 ? base : 0) + c;
                copy16(kd + j * K_LD + c, kp + from, base >= 0);
                copy16(vd + j * V_LD + c, vp + from, base >= 0);
            }
            if (st.first) {
                T* qd = qs + (size_t)(st.stretch % STAGES) * ROWS * Q_LD;
                const T* q = (const T*)a.q;
#pragma unroll 1
                for (int e = threadIdx.x; e < ROWS * PIECES; e += THREADS) {
                    const int r = e / PIECES, c = (e - r * PIECES) * EACH, row = st.of.row0 + r, further = a.by_group.of(row);
                    const int token = r < st.of.rows ? a.order[st.of.place + further] : -1;
                    const bool ok = (unsigned)token < (unsigned)a.tokens;
                    copy16(qd + r * Q_LD + c, q + (ok ? (long long)token * a.q_ld + (st.of.kvh * a.group + row - further * a.group) * HD + c : 0), ok);
                }
            }
        }
        copies_commit();
    }
    // first steps; false: nothing to do
    __device__ bool start() {
        // few rows from the last block on: it has the fewest pieces of many rows
        piece = piece_of<!IS_FEW>(a, plan, IS_FEW ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (piece.from == piece.end) return false;
        if (threadIdx.x == 0) {
            stretches = at = 0;
            stretch_of<!IS_FEW>(a, plan, piece, 0, sh.stretch);
#pragma unroll 1
            for (int n = 0; n <= STAGES; ++n) next(sh.steps[n]);
        }
        __syncthreads();
#pragma unroll 1
        for (int n = 0; n < STAGES; ++n) find(n);
        __syncthreads();
#pragma unroll 1
        for (int n = 0; n < STAGES - 1; ++n) fetch(n);
        return true;
    }
    __device__ void finish() {                                            // (the shared memory may serve for something else)
        copies_wait<0>();
        __syncthreads();
    }
    // step n has landed: on with the steps behind it
    __device__ void advance(int n) {
        copies_wait<STAGES - 2>();
        __syncthreads();
        fetch(n + STAGES - 1);
        find(n + STAGES);
        if (threadIdx.x == 0) next(sh.steps[(n + STAGES + 1) % RECORDS]);
    }
    __device__ const Step& step(int n) const { return sh.steps[n % RECORDS]; }
};

// ------------------------------------------------------------------------------------- bfloat16, few rows
// A tile of 16 rows in one warp, steps of 16 keys: lane 4 g + t has of rows g and g + 8 keys and columns 2 t, 2 t + 1 of every eight.
struct FewState {
    float m_lo, m_hi, l_lo, l_hi, o[HD / 8][4];
    __device__ __forceinline__ void begin() {
        m_lo = m_hi = -INFINITY; l_lo = l_hi = 0.f;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) { o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f; }
    }
    // k_at(i), v_at(c): where this lane's row of the i-th (c-th) 16 columns of keys (values) lies; q_of(i, f): the queries' fragment;
    // bit j of `keys`: key j counts
    template <typename KeysAt, typename ValuesAt, typename QueryOf>
    __device__ __forceinline__ void step(KeysAt k_at, ValuesAt v_at, QueryOf q_of, unsigned keys, int t, float sc) {
        // ---- scores: two chains of products for each eight keys
        float s[2][4], s2[2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[c][e] = s2[c][e] = 0.f;
        constexpr int TOGETHER = HD / 16 < 8 ? HD / 16 : 8;               // fragments asked for before the first is used
#pragma unroll
        for (int i0 = 0; i0 < HD / 16; i0 += TOGETHER) {
            unsigned b[TOGETHER][4], q4[4];
#pragma unroll
            for (int i = 0; i < TOGETHER; ++i)
                if (i0 + i < HD / 16) ldmatrix_x4(b[i], k_at(i0 + i));
#pragma unroll
            for (int i = 0; i < TOGETHER; ++i) {
                if (i0 + i >= HD / 16) break;
                q_of(i0 + i, q4);
                mma_bf16(i & 1 ? s2[0] : s[0], q4, b[i][0], b[i][1]);
                mma_bf16(i & 1 ? s2[1] : s[1], q4, b[i][2], b[i][3]);
            }
        }
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool there = keys >> (c * 8 + 2 * t + e) & 1;
                s[c][e] = there ? s[c][e] + s2[c][e] : -INFINITY;
                s[c][2 + e] = there ? s[c][2 + e] + s2[c][2 + e] : -INFINITY;
                mx_lo = fmaxf(mx_lo, s[c][e]);
                mx_hi = fmaxf(mx_hi, s[c][2 + e]);
            }
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1));
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
        const float mn_lo = fmaxf(m_lo, mx_lo), mn_hi = fmaxf(m_hi, mx_hi);
        const float base_lo = mn_lo == -INFINITY ? 0.f : mn_lo * sc, base_hi = mn_hi == -INFINITY ? 0.f : mn_hi * sc;
        const float corr_lo = fast_exp2(m_lo * sc - base_lo), corr_hi = fast_exp2(m_hi * sc - base_hi);
        m_lo = mn_lo; m_hi = mn_hi;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            s[c][0] = fast_exp2(fmaf(s[c][0], sc, -base_lo)); s[c][1] = fast_exp2(fmaf(s[c][1], sc, -base_lo));
            s[c][2] = fast_exp2(fmaf(s[c][2], sc, -base_hi)); s[c][3] = fast_exp2(fmaf(s[c][3], sc, -base_hi));
        }
        l_lo = l_lo * corr_lo + ((s[0][0] + s[0][1]) + (s[1][0] + s[1][1]));       // of this thread's keys
        l_hi = l_hi * corr_hi + ((s[0][2] + s[0][3]) + (s[1][2] + s[1][3]));
        if (__any_sync(0xffffffffu, corr_lo != 1.f || corr_hi != 1.f)) {
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) { o[c][0] *= corr_lo; o[c][1] *= corr_lo; o[c][2] *= corr_hi; o[c][3] *= corr_hi; }
        }
        // ---- weighted values: the weights are rounded to bfloat16, as the values are; the sums l hold them unrounded
        const unsigned p4[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]), pack_bf16(s[1][2], s[1][3])};
#pragma unroll
        for (int c0 = 0; c0 < HD / 16; c0 += TOGETHER) {
            unsigned b[TOGETHER][4];
#pragma unroll
            for (int c = 0; c < TOGETHER; ++c)
                if (c0 + c < HD / 16) ldmatrix_x4_trans(b[c], v_at(c0 + c));
#pragma unroll
            for (int c = 0; c < TOGETHER; ++c) {
                if (c0 + c >= HD / 16) break;
                mma_bf16(o[2 * (c0 + c)], p4, b[c][0], b[c][1]);
                mma_bf16(o[2 * (c0 + c) + 1], p4, b[c][2], b[c][3]);
            }
        }
    }
    __device__ __forceinline__ void leave(const SharedArgs& a, int rows, int slot, int g, int t) {
        l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
        l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = g + 8 * half;
            if (r >= rows) continue;
            const size_t row = (size_t)slot * FEW + r;
            float* dst = a.part_o + row * HD;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c)
                *reinterpret_cast<float2*>(dst + c * 8 + 2 * t) = make_float2(o[c][2 * half], o[c][2 * half + 1]);
            if (t == 0) {
                const float m = half ? m_hi : m_lo;
                *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m == -INFINITY ? m : m * a.scale, half ? l_hi : l_lo);
            }
        }
    }
};

// Every warp is a worker of its own: one tile of 16 rows, steps of 16 keys, its own ring of STAGES steps in shared memory, and
// no meeting of warps on the way.  What a step costs is its chain of dependent instructions, so what counts is how many warps
// an SM has at it and how few instructions they take: four warps that shared a step of 32 keys took 442 instructions each,
// and 62 us where these take 40 (200 requests, 40 heads over 8 of 128, 32 to 512 keys of their own each).
template <int MOST_WARPS, int ROOM>
struct FewShape {
    static constexpr int KEYS = MMA_FEW_KEYS, STAGES = 3;
    static constexpr int LD = HD + 8;                    // padded rows: ldmatrix without bank conflicts
    static constexpr bool Q_IN_REGS = HD <= 128;
    static constexpr int Q_SLOTS = Q_IN_REGS ? 2 : 3;
    static constexpr int AT_ONCE = 8;                    // stretches that a worker works out at once
    static constexpr size_t WORKER = ((size_t)STAGES * 2 * KEYS + (size_t)Q_SLOTS * FEW) * LD * sizeof(bf16) + FEW * 8 + AT_ONCE * sizeof(Stretch);
    static constexpr int FIT = (int)(ROOM / WORKER);
    static constexpr int WORKERS = FIT < MOST_WARPS ? FIT : MOST_WARPS;
    static constexpr size_t SMEM = WORKERS * WORKER;
};

template <typename S>
__device__ __forceinline__ void few_phase(const SharedArgs& a, const Plan& plan, unsigned char* smem, int workers) {
    constexpr int KEYS = S::KEYS, STAGES = S::STAGES, LD = S::LD, PIECES = HD / 8, ROUNDS = KEYS * PIECES / 32;
    static_assert(KEYS == FEW, "keys and queries are copied alike");
    if (threadIdx.x >= 32 * workers) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bf16* ring = reinterpret_cast<bf16*>(smem + warp * S::WORKER);        // [stage][K, V][KEYS][LD]
    bf16* qs = ring + STAGES * 2 * KEYS * LD;                             // [slot][FEW][LD]
    long long* row_at = reinterpret_cast<long long*>(qs + S::Q_SLOTS * FEW * LD);       // where the rows to copy begin
    Stretch* stretches = reinterpret_cast<Stretch*>(row_at + FEW);
    // the blocks that have the fewest pieces of many rows come first
    const Piece piece = piece_of<0>(a, plan, (gridDim.x - 1 - blockIdx.x) * workers + warp);
    if (piece.from == piece.end) return;
    // (held in registers: a parameter is read from where it lies, again and again, otherwise)
    const bf16 *kp = (const bf16*)a.k_pages, *vp = (const bf16*)a.v_pages, *qp = (const bf16*)a.q;
    long long page_stride = a.page_stride;
    int page_size = a.page_size, num_pages = a.num_pages, q_ld = a.q_ld, group = a.group, table_width = a.table_width, tokens = a.tokens;
    const int* block_tables = a.block_tables;
    asm volatile("" : "+l"(kp), "+l"(vp), "+l"(qp), "+l"(page_stride), "+l"(block_tables), "+r"(page_size), "+r"(num_pages), "+r"(q_ld), "+r"(group), "+r"(table_width), "+r"(tokens));
    // ---- the walk: the step that comes next, and its keys' pages, asked for a turn before its keys and values are
    int k = -1, left = 0, k0 = 0;                         // stretch, steps left of it, the step's first key
    bool first = false, more = true;
    Stretch at = {};
    int page = 0, inside = -1;                            // of key `lane % 16`: its page, and its place there (-1: no key)
    auto look_up = [&]() {
        inside = -1;
        if (!more) return;
        first = left == 0;
        if (first) {
            if (++k % S::AT_ONCE == 0) {
                __syncwarp();
                if (lane < S::AT_ONCE) stretch_of<0>(a, plan, piece, k + lane, stretches[lane]);
                __syncwarp();
            }
            at = stretches[k % S::AT_ONCE];
            left = at.steps;
            more = left > 0;
            if (!more) return;
            k0 = at.k0;
        } else {
            k0 += KEYS;
        }
        --left;
        const int key = k0 + (lane & 15);
        if (key < at.kend) {
            const int block = key / page_size;
            inside = key - block * page_size;
            page = block_tables[(size_t)at.table * table_width + block];
        }
    };
    // what a step needs when it has landed: bits 0 .. 15 its keys, 16 .. 18 first, last and valid; rows and slot
    struct Landing { unsigned bits; int rows, slot; };
    auto fetch = [&](int n) {
        Landing landing = {0u, 0, 0};
        if (more) {
            const bool there = inside >= 0 && (unsigned)page < (unsigned)num_pages;
            if (inside >= 0 && !there) atomicExch(a.error, ERR_PAGE);
            landing.bits = (__ballot_sync(0xffffffffu, there) & 0xffffu) | (first ? 1u << 16 : 0u) | (left == 0 ? 1u << 17 : 0u) | 1u << 18;
            landing.rows = at.rows; landing.slot = at.slot;
            const long long base = there ? (long long)page * page_stride + ((long long)at.kvh * page_size + inside) * HD : 0;
            bf16* kd = ring + (n % STAGES) * 2 * KEYS * LD;
            __syncwarp();
            if (lane < KEYS) row_at[lane] = base;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < ROUNDS; ++i) {
                const int e = i * 32 + lane, j = e / PIECES, c = (e - j * PIECES) * 8;
                const bool ok = landing.bits >> j & 1;
                const long long from = row_at[j] + c;
                copy16(kd + j * LD + c, kp + from, ok);
                copy16(kd + (KEYS + j) * LD + c, vp + from, ok);
            }
            if (first) {
                long long query_at = 0;                   // of row `lane`
                bool row_there = false;
                if (lane < at.rows) {
                    const int row = at.row0 + lane, further = row < group ? 0 : row / group;
                    const int token = at.token >= 0 ? at.token : a.order[at.place + further];
                    row_there = (unsigned)token < (unsigned)tokens;
                    if (row_there) query_at = (long long)token * q_ld + (at.kvh * group + row - further * group) * HD;
                }
                const unsigned rows = __ballot_sync(0xffffffffu, row_there);
                bf16* qd = qs + (k % S::Q_SLOTS) * FEW * LD;
                __syncwarp();
                if (lane < FEW) row_at[lane] = query_at;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < ROUNDS; ++i) {
                    const int e = i * 32 + lane, r = e / PIECES, c = (e - r * PIECES) * 8;
                    copy16(qd + r * LD + c, qp + row_at[r] + c, rows >> r & 1);
                }
            }
        }
        copies_commit();
        return landing;
    };

    const int g = lane >> 2, t = lane & 3;
    const float sc = a.scale * LOG2E;                     // scores in base-2 units
    FewState state;
    unsigned qf[S::Q_IN_REGS ? HD / 16 : 1][4];
    int stretch = -1;
    Landing now = {0u, 0, 0}, next = {0u, 0, 0};
    static_assert(STAGES == 3, "landings held: this step's and the next two");
    look_up();
    for (int n = 1 - STAGES;; ++n) {                      // (the first turns only fetch)
        if (n >= 0) {
            copies_wait<STAGES - 2>();
            __syncwarp();
            if (!(now.bits >> 18)) break;
        }
        const bool begins = now.bits >> 16 & 1;
        stretch += begins;
        const bf16* q_at = qs + (stretch & (S::Q_IN_REGS ? 1 : 0)) * FEW * LD + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + 8 * (lane >> 4);
        if (!S::Q_IN_REGS) q_at += (stretch % 3) * FEW * LD;
        if (begins) {
            state.begin();
            if (S::Q_IN_REGS) {
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) ldmatrix_x4(qf[i], q_at + i * 16);
                __syncwarp();                             // the slot may be filled again
            }
        }
        const Landing behind = fetch(n + STAGES - 1);
        look_up();
        if (n >= 0) {
            const bf16* kt = ring + (n % STAGES) * 2 * KEYS * LD;
            const bf16* vt = kt + KEYS * LD;
            state.step([&](int i) { return kt + ((lane & 7) + 8 * (lane >> 4)) * LD + i * 16 + 8 * ((lane >> 3) & 1); },
                       [&](int c) { return vt + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + c * 16 + 8 * (lane >> 4); },
                       [&](int i, unsigned (&q4)[4]) {
                           if constexpr (S::Q_IN_REGS) { q4[0] = qf[i][0]; q4[1] = qf[i][1]; q4[2] = qf[i][2]; q4[3] = qf[i][3]; }
                           else ldmatrix_x4(q4, q_at + i * 16);
                       }, now.bits, t, sc);
            if (now.bits >> 17 & 1) state.leave(a, now.rows, now.slot, g, t);
            __syncwarp();                                 // the step's place in the ring may be filled again
        }
        now = next; next = behind;
    }
    copies_wait<0>();
}

// ------------------------------------------------------------------------------------- bfloat16, many rows
// Head sizes and pages that the tcgen05 kernel below does not take: tiles of 64 rows, 16 to a warp.
struct ManyShape {
    static constexpr int ROWS = 64, KEYS = MMA_MANY_KEYS, STAGES = 2;
    static constexpr int LD = HD + 8;
    using F = Feed<bf16, ROWS, false, KEYS, STAGES, LD, LD, LD>;
    static constexpr size_t SMEM = (size_t)STAGES * (2 * KEYS + ROWS) * LD * sizeof(bf16) + (sizeof(F::Shared) + 15) / 16 * 16;
};

__device__ __forceinline__ void many_phase(const SharedArgs& a, const Plan& plan, unsigned char* smem) {
    using S = ManyShape;
    constexpr int KEYS = S::KEYS, NT = KEYS / 8;
    bf16* ks = reinterpret_cast<bf16*>(smem);
    bf16* vs = ks + (size_t)S::STAGES * KEYS * S::LD;
    bf16* qs = vs + (size_t)S::STAGES * KEYS * S::LD;
    S::F::Shared& sh = *reinterpret_cast<S::F::Shared*>(qs + (size_t)S::STAGES * S::ROWS * S::LD);
    S::F feed(a, plan, sh, ks, vs, qs);
    if (!feed.start()) return;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int r_lo = warp * 16 + g, r_hi = r_lo + 8;
    const float sc = a.scale * LOG2E;
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    float o[HD / 8][4];

    for (int n = 0; feed.step(n).valid; ++n) {
        feed.advance(n);
        const Step st = feed.step(n);
        const bf16* q_at = qs + (size_t)(st.stretch % S::STAGES) * S::ROWS * S::LD +
                           (warp * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * S::LD + 8 * (lane >> 4);
        if (st.first) {
            m_lo = m_hi = -INFINITY; l_lo = l_hi = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) { o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f; }
        }
        const bf16* kt = ks + (size_t)(n % S::STAGES) * KEYS * S::LD;
        const bf16* vt = vs + (size_t)(n % S::STAGES) * KEYS * S::LD;
        float s[NT][4];
#pragma unroll
        for (int c = 0; c < NT; ++c) { s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f; }
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            unsigned q4[4];
            ldmatrix_x4(q4, q_at + k * 16);
#pragma unroll
            for (int c = 0; c < NT / 2; ++c) {
                unsigned b[4];
                ldmatrix_x4(b, kt + (c * 16 + (lane & 7) + 8 * (lane >> 4)) * S::LD + k * 16 + 8 * ((lane >> 3) & 1));
                mma_bf16(s[2 * c], q4, b[0], b[1]);
                mma_bf16(s[2 * c + 1], q4, b[2], b[3]);
            }
        }
        // ---- keys that are not there (behind the end; a page that is none)
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
        const long long* base = sh.key_base[n % S::F::BASES];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (base[c * 8 + 2 * t + e] < 0) s[c][e] = s[c][2 + e] = -INFINITY;
                mx_lo = fmaxf(mx_lo, s[c][e]);
                mx_hi = fmaxf(mx_hi, s[c][2 + e]);
            }
        }
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1));
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
        const float mn_lo = fmaxf(m_lo, mx_lo), mn_hi = fmaxf(m_hi, mx_hi);
        const float base_lo = mn_lo == -INFINITY ? 0.f : mn_lo * sc, base_hi = mn_hi == -INFINITY ? 0.f : mn_hi * sc;
        const float corr_lo = exp2f(m_lo * sc - base_lo), corr_hi = exp2f(m_hi * sc - base_hi);
        m_lo = mn_lo; m_hi = mn_hi;
        float sum_lo = 0.f, sum_hi = 0.f;
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            s[c][0] = exp2f(s[c][0] * sc - base_lo); s[c][1] = exp2f(s[c][1] * sc - base_lo);
            s[c][2] = exp2f(s[c][2] * sc - base_hi); s[c][3] = exp2f(s[c][3] * sc - base_hi);
            sum_lo += s[c][0] + s[c][1];
            sum_hi += s[c][2] + s[c][3];
        }
        l_lo = l_lo * corr_lo + sum_lo;
        l_hi = l_hi * corr_hi + sum_hi;
        if (__any_sync(0xffffffffu, corr_lo != 1.f || corr_hi != 1.f)) {
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) { o[c][0] *= corr_lo; o[c][1] *= corr_lo; o[c][2] *= corr_hi; o[c][3] *= corr_hi; }
        }
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k) {             // weights rounded to bfloat16, the sums l hold them unrounded
            const unsigned p4[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]), pack_bf16(s[2 * k][2], s[2 * k][3]),
                                    pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]), pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
                unsigned b[4];
                ldmatrix_x4_trans(b, vt + (k * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * S::LD + c * 16 + 8 * (lane >> 4));
                mma_bf16(o[2 * c], p4, b[0], b[1]);
                mma_bf16(o[2 * c + 1], p4, b[2], b[3]);
            }
        }
        if (!st.last) continue;
        // ---- the stretch's triples
        l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
        l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
        const size_t row = (size_t)a.many.row0 + (size_t)st.of.slot * S::ROWS;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = half ? r_hi : r_lo;
            if (r >= st.of.rows) continue;
            float* dst = a.part_o + (row + r) * HD;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c)
                *reinterpret_cast<float2*>(dst + c * 8 + 2 * t) = make_float2(o[c][2 * half], o[c][2 * half + 1]);
            if (t == 0) {
                const float m = half ? m_hi : m_lo;
                *reinterpret_cast<float2*>(a.part_ml + (row + r) * 2) = make_float2(m == -INFINITY ? m : m * a.scale, half ? l_hi : l_lo);
            }
        }
    }
    feed.finish();
}

// ------------------------------------------------------------------------------------------------- float32
// FFMA.  A warp has 8 rows: its lanes' halves four each, 16 lanes side by side along the keys (scores) and the columns
// (values); WARPS_K warps share the keys of a step and then the columns, as above.
template <int WARPS_M, int WARPS_K, bool FEW_ROWS>
struct F32Shape {
    static constexpr int ROWS = 8 * WARPS_M, STAGES = 2, KEYS = F32_KEYS;
    static constexpr int K_LD = HD + 4, P_LD = KEYS + 4;
    static constexpr int JN = KEYS / 16 / WARPS_K;                              // keys of a lane
    static constexpr int VEC = WARPS_K == 1 ? 4 : 2;                      // columns side by side
    static constexpr int GROUPS = (HD / VEC + 16 * WARPS_K - 1) / (16 * WARPS_K);
    static constexpr bool IS_FEW = FEW_ROWS;
    using F = Feed<float, ROWS, IS_FEW, KEYS, STAGES, K_LD, HD, HD>;
    static constexpr size_t SMEM = sizeof(float) * ((size_t)STAGES * KEYS * (K_LD + HD) + (size_t)STAGES * ROWS * HD + (size_t)ROWS * P_LD +
                                                    2 * WARPS_K * ROWS) + (sizeof(typename F::Shared) + 15) / 16 * 16;
};

template <int WARPS_M, int WARPS_K, bool FEW_ROWS>
__device__ __forceinline__ void f32_phase(const SharedArgs& a, const Plan& plan, unsigned char* smem) {
    using S = F32Shape<WARPS_M, WARPS_K, FEW_ROWS>;
    constexpr int STAGES = S::STAGES, VEC = S::VEC, KEYS = S::KEYS;
    float* ks = reinterpret_cast<float*>(smem);
    float* vs = ks + STAGES * KEYS * S::K_LD;
    float* qs = vs + STAGES * KEYS * HD;
    float* ps = qs + STAGES * S::ROWS * HD;
    float* row_max = ps + S::ROWS * S::P_LD;
    float* row_sum = row_max + WARPS_K * S::ROWS;
    typename S::F::Shared& sh = *reinterpret_cast<typename S::F::Shared*>(row_sum + WARPS_K * S::ROWS);
    typename S::F feed(a, plan, sh, ks, vs, qs);
    if (!feed.start()) return;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = warp / WARPS_K, wk = warp % WARPS_K;
    const int tx = lane & 15, r0 = wm * 8 + (lane >> 4) * 4;
    float m[4], l[4], acc[S::GROUPS][4][VEC];

    for (int n = 0; feed.step(n).valid; ++n) {
        feed.advance(n);
        const Step st = feed.step(n);
        const float* q_at = qs + (size_t)(st.stretch % STAGES) * S::ROWS * HD + r0 * HD;
        if (st.first) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
#pragma unroll
            for (int c = 0; c < S::GROUPS; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) acc[c][i][e] = 0.f;
        }
        const float* kt = ks + (size_t)(n % STAGES) * KEYS * S::K_LD;
        const float* vt = vs + (size_t)(n % STAGES) * KEYS * HD;
        const long long* base = sh.key_base[n % S::F::BASES];
        float s[4][S::JN];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < S::JN; ++j) s[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < HD; d += 4) {
            float4 x[4], y[S::JN];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(q_at + i * HD + d);
#pragma unroll
            for (int j = 0; j < S::JN; ++j) y[j] = *reinterpret_cast<const float4*>(kt + (wk * 16 * S::JN + tx + 16 * j) * S::K_LD + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < S::JN; ++j)
                    s[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, s[i][j]))));
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top[i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < S::JN; ++j) {
                s[i][j] = base[wk * 16 * S::JN + tx + 16 * j] >= 0 ? s[i][j] * a.scale : -INFINITY;
                top[i] = fmaxf(top[i], s[i][j]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], w));
        }
        if constexpr (WARPS_K > 1) {
            if (tx < 4) row_max[wk * S::ROWS + r0 + tx] = tx == 0 ? top[0] : tx == 1 ? top[1] : tx == 2 ? top[2] : top[3];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < WARPS_K; ++w) top[i] = fmaxf(top[i], row_max[w * S::ROWS + r0 + i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float m_new = fmaxf(m[i], top[i]);
            const float corr = m[i] == -INFINITY ? 0.f : expf(m[i] - m_new);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < S::JN; ++j) {
                const float w = s[i][j] == -INFINITY ? 0.f : expf(s[i][j] - m_new);
                ps[(r0 + i) * S::P_LD + wk * 16 * S::JN + tx + 16 * j] = w;
                sum += w;
            }
            l[i] = l[i] * corr + sum;
            m[i] = m_new;
#pragma unroll
            for (int c = 0; c < S::GROUPS; ++c)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[c][i][e] *= corr;
        }
        if constexpr (WARPS_K > 1) __syncthreads();
        else __syncwarp();
#pragma unroll 2
        for (int j = 0; j < KEYS; j += 4) {
            float w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(ps + (r0 + i) * S::P_LD + j);
                w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int c = 0; c < S::GROUPS; ++c) {
                    const int column = (wk * 16 + tx + c * 16 * WARPS_K) * VEC;
                    if (HD / VEC % (16 * WARPS_K) == 0 || column < HD) {
                        float v[VEC];
                        if constexpr (VEC == 4) {
                            const float4 x = *reinterpret_cast<const float4*>(vt + (j + u) * HD + column);
                            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                        } else {
                            const float2 x = *reinterpret_cast<const float2*>(vt + (j + u) * HD + column);
                            v[0] = x.x; v[1] = x.y;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < VEC; ++e) acc[c][i][e] = fmaf(w[i][u], v[e], acc[c][i][e]);
                    }
                }
        }
        if (!st.last) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        if constexpr (WARPS_K > 1) {
            if (tx < 4) row_sum[wk * S::ROWS + r0 + tx] = tx == 0 ? l[0] : tx == 1 ? l[1] : tx == 2 ? l[2] : l[3];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                l[i] = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS_K; ++w) l[i] += row_sum[w * S::ROWS + r0 + i];
            }
        }
        const size_t row = (S::IS_FEW ? 0 : (size_t)a.many.row0) + (size_t)st.of.slot * S::ROWS;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r0 + i >= st.of.rows) continue;
            float* dst = a.part_o + (row + r0 + i) * HD;
#pragma unroll
            for (int c = 0; c < S::GROUPS; ++c) {
                const int column = (wk * 16 + tx + c * 16 * WARPS_K) * VEC;
                if (HD / VEC % (16 * WARPS_K) == 0 || column < HD) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) dst[column + e] = acc[c][i][e];
                }
            }
            if (wk == 0 && tx == 0) *reinterpret_cast<float2*>(a.part_ml + (row + r0 + i) * 2) = make_float2(m[i], l[i]);
        }
    }
    feed.finish();
}

// ------------------------------------------------------------------------------------ bfloat16, many rows, tcgen05
// Tiles of 256 rows as two streams of 128 (a tensor-memory lane each), keys in tiles of 128 by TMA, scores and outputs in
// tensor memory; a block walks its stretches with all of this set up once.
//
//   producer warp   K and V tiles by turns into a ring of SLOTS, page by page
//   MMA warp        S_X = Q_X K^T, O_X += P_X V for the streams in turn; in a tile that reaches beyond the keys that the run
//                   has it sets those rows of V to zero first, so that whatever lies there is multiplied with nothing
//                   (keys of a page outside the pool arrive as zeros, K and V, and are masked by the softmax warps)
//   2 x 4 warps     a stream's queries into shared memory, then a thread per row: scores, running maximum and sum, the weights as
//                   bfloat16 over the scores in tensor memory; at a stretch's end its row's triple
//
// Waits are bounded: when one runs out *error is set, all roles leave, tensor memory is freed.
#if HEAD_DIM == 64 || HEAD_DIM == 128
#define FSIE_SHARED_TC 1
namespace tc {

constexpr int BM = 128, STREAMS = 2, ROWS = STREAMS * BM, KEYS = 128;
constexpr int SLOTS = 4;
constexpr int SOFTMAX_WARPS = 4 * STREAMS, THREADS = 64 + 32 * SOFTMAX_WARPS;
constexpr int HALVES = HD / 64, ATOM = 128 * 128;        // 128-byte column halves of a row; 128 rows of one
constexpr int Q_BYTES = HALVES * ATOM, KV_BYTES = HALVES * ATOM;
constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_O = STREAMS * KEYS;
constexpr int STRETCHES = 32;                            // of a block's piece, worked out at once
constexpr int BOX = 16;                                  // keys that a copy brings, where a page has as many
constexpr int NO_ROW = 0x7fffff00;                       // behind the rows of all pages
enum { ERR_TC_PRODUCER = 31, ERR_TC_MMA = 32, ERR_TC_SOFTMAX = 33, ERR_TC_LAYOUT = 34, ERR_FEW = 39 };

struct Control {
    uint64_t ring_full[SLOTS], ring_empty[SLOTS], s_full[STREAMS], p_ready[STREAMS], o_done[STREAMS], q_ready[STREAMS];
    uint32_t tmem_slot;
    int abort_flag;
    int page_missing;                                    // a page that a step asks for is none: see missing_boxes
    Stretch stretches[STRETCHES];
};
constexpr int CONTROL_BYTES = 2048;
static_assert(sizeof(Control) <= CONTROL_BYTES, "control block");
constexpr size_t SMEM = CONTROL_BYTES + STREAMS * Q_BYTES + SLOTS * KV_BYTES;

// Two 32-bit numbers to an instruction, and the largest of three: the softmax warps wait for their turn to issue.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float x, float y) { Pair p; asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y)); return p; }
__device__ __forceinline__ float2 apart(Pair p) { float2 v; asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p)); return v; }
__device__ __forceinline__ Pair fma2(Pair x, Pair y, Pair z) { Pair p; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(x), "l"(y), "l"(z)); return p; }
__device__ __forceinline__ Pair add2(Pair x, Pair y) { Pair p; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(x), "l"(y)); return p; }
__device__ __forceinline__ float max3(float x, float y, float z) { float v; asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(x), "f"(y), "f"(z)); return v; }

__device__ __forceinline__ bool mbar_done(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return done;
}

// Which of a step's boxes, from key `from` on, lie in pages outside the pool, a bit each: lane j looks box j up.
__device__ __forceinline__ unsigned missing_boxes(const int* table, int page_size, int num_pages, int from, int kend, int lane) {
    const int box = min(page_size, BOX), key = from + lane * box;
    const int page = lane * box < KEYS && key < kend ? table[key >> (__ffs(page_size) - 1)] : 0;
    return __ballot_sync(0xffffffffu, (unsigned)page >= (unsigned)num_pages);
}

// 32 keys, in boxes of 8 or 16, of which those with a bit in `missing` do not count.
__device__ __forceinline__ unsigned there_of(unsigned missing, bool boxes_of_8) {
    if (!boxes_of_8) return ~((missing & 1 ? 0xffffu : 0u) | (missing & 2 ? 0xffff0000u : 0u));
    return ~((missing & 1 ? 0xffu : 0u) | (missing & 2 ? 0xff00u : 0u) | (missing & 4 ? 0xff0000u : 0u) | (missing & 8 ? 0xff000000u : 0u));
}

__device__ __forceinline__ void tc_phase(const CUtensorMap& k_map, const CUtensorMap& v_map, const SharedArgs& a, const Plan& plan, unsigned char* smem_all) {
    Control& ctl = *reinterpret_cast<Control*>(smem_all);
    unsigned char* q_s = smem_all + CONTROL_BYTES;       // [stream][HALVES][128 rows][128 B]
    unsigned char* ring = q_s + STREAMS * Q_BYTES;       // [slot][HALVES][128 keys][128 B]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Piece piece = piece_of<1>(a, plan, blockIdx.x);
    if ((smem_addr(smem_all) & 1023) != 0) {             // the swizzle goes by addresses
        if (tid == 0) atomicExch(a.error, ERR_TC_LAYOUT);
        return;
    }
    if (piece.from == piece.end) return;
    if (tid == 0) {
        for (int s = 0; s < SLOTS; ++s) { mbar_init(&ctl.ring_full[s], 1); mbar_init(&ctl.ring_empty[s], 1); }
        for (int st = 0; st < STREAMS; ++st) {
            mbar_init(&ctl.s_full[st], 1); mbar_init(&ctl.p_ready[st], BM); mbar_init(&ctl.o_done[st], 1);
            mbar_init(&ctl.q_ready[st], BM);
        }
        ctl.abort_flag = ctl.page_missing = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    static_assert(STRETCHES == 32, "a lane each");
    if (warp == 2) stretch_of<1>(a, plan, piece, lane, ctl.stretches[lane]);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&ctl.tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = ctl.tmem_slot;
    int done = 0;                                         // stretches of the rounds before
    auto give_up = [&](int code) { atomicExch(a.error, code); atomicExch(&ctl.abort_flag, 1); };

    // what the roles count on from stretch to stretch
    int e = 0;                                            // producer, MMA: ring entries so far (K, V, K, ...)
    int tiles_of[STREAMS] = {0, 0}, stretches_of[STREAMS] = {0, 0};       // MMA: of each stream; softmax: [0] of its own
    bool ok = true;
    const int st_own = (warp - 2) / 4;                    // softmax warps: their stream
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_base + COL_S + st_own * KEYS, o_addr = lane_base + COL_O + st_own * KEYS;
    const float sc = a.scale * LOG2E;

    for (;;) {
        for (int k = 0; k < STRETCHES && ok; ++k) {
            const Stretch sr = ctl.stretches[k];
            if (sr.steps == 0) break;
            const int tiles = sr.steps, streams = sr.rows > BM ? 2 : 1;
            if (warp == 0) {
                // -------------------------------------------------------------- producer: lane j has box j of a tile
                const int ps = a.page_size, shift = __ffs(ps) - 1, box = min(ps, BOX), boxes = KEYS / box;
                const long long rows_per_page = a.page_stride / HD;
                const int* table = a.block_tables + (size_t)sr.table * a.table_width;
                auto look_up = [&](int i) {               // beyond the keys any page will do: they count for nothing
                    const int key = sr.k0 + i * KEYS + lane * box;
                    return lane < boxes && i < tiles && key < sr.kend ? table[key >> shift] : 0;
                };
                int ahead = look_up(0);
                for (int i = 0; i < tiles && ok; ++i) {
                    const int page = ahead;
                    ahead = look_up(i + 1);
                    const bool there = (unsigned)page < (unsigned)a.num_pages;
                    if (!there) {                         // (whoever waits for these keys finds the flag set)
                        atomicExch(a.error, ERR_PAGE);
                        atomicExch(&ctl.page_missing, 1);
                    }
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv, ++e) {
                        const int s = e % SLOTS;
                        if (lane == 0 && e >= SLOTS) ok = mbar_wait(&ctl.ring_empty[s], (e / SLOTS - 1) & 1);
                        ok = __shfl_sync(0xffffffffu, ok, 0) && !*(volatile int*)&ctl.abort_flag;
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_expect_tx(&ctl.ring_full[s], (uint32_t)KV_BYTES);
                        __syncwarp();
                        if (lane < boxes) {
                            unsigned char* dst = ring + (size_t)s * KV_BYTES + lane * box * 128;
                            const int row = there ? (int)(page * rows_per_page + (long long)sr.kvh * ps) + (sr.k0 + lane * box & (ps - 1)) : NO_ROW;
#pragma unroll
                            for (int h = 0; h < HALVES; ++h) tma_load_2d(dst + h * ATOM, kv ? &v_map : &k_map, h * 64, row, &ctl.ring_full[s]);
                        }
                    }
                }
                if (!ok) {
                    if (lane == 0) give_up(ERR_TC_PRODUCER);
                    for (int j = max(0, e - SLOTS); j < e; ++j) mbar_wait(&ctl.ring_full[j % SLOTS], (j / SLOTS) & 1);    // copies on the way
                }
            } else if (warp == 1) {
                // -------------------------------------------------------------- MMA: one lane issues, all take part in the waits
                // The streams by turns, each one's product with V and its next scores together, so that one stream's products run
                // beside the other's softmax (a warp for each stream: both fall into step, 5,000 cycles a step).  Little else stands
                // between a stream's weights and its next scores: what the copy engine brings is waited for beside the softmax,
                // whether all lanes are well is asked once a tile.  3,950 cycles a step of 256 rows; with a vote and a fence at
                // every wait, and the waits where their data is used, 4,890.
                const uint32_t idesc_s = idesc_bf16(BM, KEYS, 0), idesc_o = idesc_bf16(BM, HD, 1);
                const uint64_t q_base = desc_k_major(q_s), k_base = desc_k_major(ring), v_base = desc_mn_major(ring, ATOM);
                auto wait = [&](uint64_t* bar, int parity) { if (!mbar_done(bar, parity & 1)) ok = mbar_wait(bar, parity & 1) && ok; };
                auto scores = [&](int st, int entry) {    // S_st = Q_st K^T
                    const uint64_t qd = q_base + (uint64_t)(st * (Q_BYTES >> 4)), kd = k_base + (uint64_t)((entry % SLOTS) * (KV_BYTES >> 4));
#pragma unroll
                    for (int c = 0; c < HD / 16; ++c) {
                        const uint32_t step = (c >> 2) * (ATOM >> 4) + 2 * (c & 3);
                        mma_ss(tmem + COL_S + st * KEYS, qd + step, kd + step, idesc_s, c > 0);
                    }
                    mma_commit(&ctl.s_full[st]);
                };
                wait(&ctl.ring_full[e % SLOTS], e / SLOTS);
#pragma unroll 1
                for (int st = 0; st < streams; ++st) {
                    wait(&ctl.q_ready[st], stretches_of[st]++);
                    if (lane == 0 && ok) {
                        scores(st, e);
                        if (st == streams - 1) mma_commit(&ctl.ring_empty[e % SLOTS]);
                    }
                    __syncwarp();
                }
                for (int i = 0; i < tiles; ++i, e += 2) {
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const bool on = i + 1 < tiles;
                    wait(&ctl.ring_full[(e + 1) % SLOTS], (e + 1) / SLOTS);            // V of this tile, K of the next
                    if (on) wait(&ctl.ring_full[(e + 2) % SLOTS], (e + 2) / SLOTS);
                    const int from = sr.k0 + i * KEYS;
                    if (from < sr.begin || from + KEYS > sr.kend) {        // rows of V that are none of the run's keys
                        unsigned char* v = ring + (size_t)((e + 1) % SLOTS) * KV_BYTES;
                        for (int at = lane; at < KEYS * 8 * HALVES; at += 32) {
                            const int key = from + (at >> 3) % KEYS;
                            if (key < sr.begin || key >= sr.kend) *reinterpret_cast<uint4*>(v + (size_t)at * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
#pragma unroll 1
                    for (int st = 0; st < streams; ++st) {
                        wait(&ctl.p_ready[st], tiles_of[st]++);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (lane == 0 && ok) {            // O_st += P_st V: 16 keys are 8 columns of P, 16 rows of V
                            const uint64_t vd = v_base + (uint64_t)(((e + 1) % SLOTS) * (KV_BYTES >> 4));
#pragma unroll
                            for (int c = 0; c < KEYS / 16; ++c)
                                mma_ts(tmem + COL_O + st * KEYS, tmem + COL_S + st * KEYS + c * 8, vd + (uint64_t)(c * (16 * 128 >> 4)), idesc_o,
                                       (i > 0 || c > 0) ? 1u : 0u);
                            if (on) scores(st, e + 2);
                            else mma_commit(&ctl.o_done[st]);
                            if (st == streams - 1) {
                                mma_commit(&ctl.ring_empty[(e + 1) % SLOTS]);
                                if (on) mma_commit(&ctl.ring_empty[(e + 2) % SLOTS]);
                            }
                        }
                        __syncwarp();
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok && lane == 0) give_up(ERR_TC_MMA);
            } else if (st_own < streams) {
                // -------------------------------------------------------------- softmax, a thread per row of a stream
                const int rows = sr.rows - st_own * BM;
                const bool valid = r < rows;
                // ---- the queries, K-major and swizzled (zero beyond the tile's rows); all S of the stretch before are done
                long long mine = -1;
                if (valid) {
                    const int row = sr.row0 + st_own * BM + r, further = a.by_group.of(row), token = a.order[sr.place + further];
                    if ((unsigned)token < (unsigned)a.tokens) mine = (long long)token * a.q_ld + (sr.kvh * a.group + row - further * a.group) * HD;
                }
                constexpr int CHUNKS = HD / 8, AT_ONCE = 32 / CHUNKS;     // 16-byte pieces of a row; rows that a warp copies at once
#pragma unroll 4
                for (int j = 0; j < 32; j += AT_ONCE) {   // a warp's rows by that warp
                    const int mate = j + lane / CHUNKS, c = lane % CHUNKS;
                    const long long from = __shfl_sync(0xffffffffu, mine, mate);
                    copy16(q_s + st_own * Q_BYTES + (c >> 3) * ATOM + swizzled(quarter * 32 + mate, c & 7),
                           (const bf16*)a.q + (from >= 0 ? from + c * 8 : 0), from >= 0);
                }
                copies_commit();
                copies_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&ctl.q_ready[st_own]);
                float m_run = -INFINITY, l_run = 0.f;
                for (int i = 0; i < tiles && ok; ++i) {
                    const int from = sr.k0 + i * KEYS;
                    const bool came = mbar_wait(&ctl.s_full[st_own], tiles_of[0]++ & 1);
                    unsigned missing = 0u;                // boxes, in pages that are none
                    if (!__all_sync(0xffffffffu, came && !*(volatile int*)&ctl.page_missing)) {
                        if (!__all_sync(0xffffffffu, came)) {
                            if (lane == 0) give_up(ERR_TC_SOFTMAX);
                            ok = false;
                            break;
                        }
                        missing = missing_boxes(a.block_tables + (size_t)sr.table * a.table_width, a.page_size, a.num_pages, from, sr.kend, lane);
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    // (32 keys at a time, twice: a step alone, as a short prompt has it, waits for its instructions, which all
                    // 128 in registers are four times as many of)
                    const bool part = missing || from < sr.begin || from + KEYS > sr.kend;
                    auto scores = [&](int c, uint32_t (&sv)[32]) {
                        tmem_ld32_issue(s_addr + c, sv);
                        tmem_wait_ld();
                        if (part) {                       // bit j: key j of these 32 counts (what is missing in a branch behind this one
                                                          // and a vote of its own: 89.6 us for 86.9, 200 requests that share 8,192 keys)
                            const int below = min(max(sr.begin - from - c, 0), 32), upto = min(max(sr.kend - from - c, 0), 32);
                            unsigned keys = below < upto ? (0xffffffffu >> (32 - (upto - below))) << below : 0u;
                            if (missing) keys &= there_of(missing >> (c >> (a.page_size < BOX ? 3 : 4)), a.page_size < BOX);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(keys >> j & 1)) sv[j] = 0xff800000u;        // -inf
                        }
                    };
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int c = 0; c < KEYS; c += 32) {
                        uint32_t sv[32];
                        scores(c, sv);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) mx4[j / 2 & 3] = max3(mx4[j / 2 & 3], __uint_as_float(sv[j]), __uint_as_float(sv[j + 1]));
                    }
                    const float mx = valid ? fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) : -INFINITY;
                    // the reference point of the exponentials moves only when the maximum has grown by more than 2^8 since it was
                    // set: until then a weight may exceed 1, by at most that, and O and the row sum stay as they are
                    float m_new = m_run;
                    if (mx > m_run && (m_run == -INFINITY || (mx - m_run) * sc > 8.f)) m_new = mx;
                    const float base = m_new == -INFINITY ? 0.f : m_new * sc;
                    const float corr = m_new == m_run ? 1.f : fast_exp2(m_run * sc - base);
                    if (i > 0 && __any_sync(0xffffffffu, valid && corr != 1.f)) {
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32_issue(o_addr + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                            tmem_st32_issue(o_addr + c, o);
                            tmem_wait_st();
                        }
                    }
                    Pair sum2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                    const Pair sc2 = pair(sc, sc), base2 = pair(-base, -base);
#pragma unroll 1
                    for (int c = 0; c < KEYS; c += 32) {  // (weights go over scores that are done with)
                        uint32_t sv[32];
                        scores(c, sv);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 x = apart(fma2(pair(__uint_as_float(sv[j]), __uint_as_float(sv[j + 1])), sc2, base2));
                            const float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
                            sum2[(j >> 1) & 1] = add2(sum2[(j >> 1) & 1], pair(p0, p1));
                            sv[j >> 1] = pack_bf16(p0, p1);
                        }
                        tmem_st16_issue(s_addr + c / 2, sv);
                    }
                    tmem_wait_st();
                    const float2 sum = apart(add2(sum2[0], sum2[1]));
                    l_run = l_run * corr + (valid ? sum.x + sum.y : 0.f);
                    m_run = m_new;
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    mbar_arrive(&ctl.p_ready[st_own]);
                }
                if (ok && !__all_sync(0xffffffffu, mbar_wait(&ctl.o_done[st_own], stretches_of[0]++ & 1))) {
                    if (lane == 0) give_up(ERR_TC_SOFTMAX);
                    ok = false;
                }
                if (ok) {
                    // ---- the row's triple
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const size_t row = (size_t)a.many.row0 + (size_t)sr.slot * ROWS + st_own * BM + r;
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float v[32];
                        tmem_ld32(o_addr + c, v);         // (all lanes take part)
                        if (valid) {                      // (whole sectors: a warp's rows lie 4 * HD bytes apart)
#pragma unroll
                            for (int j = 0; j < 32; j += 8)
                                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(a.part_o + row * HD + c + j), "f"(v[j]),
                                             "f"(v[j + 1]), "f"(v[j + 2]), "f"(v[j + 3]), "f"(v[j + 4]), "f"(v[j + 5]), "f"(v[j + 6]), "f"(v[j + 7]) : "memory");
                        }
                    }
                    if (valid) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m_run == -INFINITY ? m_run : m_run * a.scale, l_run);
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                }
            }
        }
        __syncthreads();                                  // all roles are done with these stretches
        const bool more = ctl.stretches[STRETCHES - 1].steps != 0 && !ctl.abort_flag;
        __syncthreads();
        if (!more) break;
        done += STRETCHES;
        if (warp == 2) stretch_of<1>(a, plan, piece, done + lane, ctl.stretches[lane]);
        __syncthreads();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Few rows: as few_phase, a warp a worker, but the copy engine brings a step's keys and values, so that a step costs neither 32
// addresses nor copies of 16 bytes, and the queries come straight into registers, which leaves room for more workers.
// 200 requests, 40 heads over 8 of 128, 32 to 512 keys of their own each: 34 us by copies of 16 bytes and as much
// here, but 63 requests of 1,024 to 2,048 keys, 28 heads over 4, 50.6 and 45.9 in all (193 MB: 5.4 TB/s behind what such a call
// takes with few keys).
struct TmaFew {
    static constexpr int KEYS = MMA_FEW_KEYS, STAGES = 3, AT_ONCE = 8;
    static constexpr int HALF = KEYS * 128, STAGE = 2 * HALVES * HALF;                  // bytes: 64 columns of a step's keys; a stage
    struct Worker { uint64_t full[STAGES]; Stretch stretches[AT_ONCE]; };
    static constexpr int CONTROL = (sizeof(Worker) + 15) / 16 * 16;
    static constexpr size_t WORKER = STAGES * STAGE + CONTROL;
    static constexpr int FIT = (int)((227 * 1024 - CONTROL_BYTES) / WORKER);
    // (a ninth leaves the second launch's blocks no room beside the first's: 8 requests of a 300-token prompt 13.0 us for 12.0 with
    // seven; 64 requests with 512 keys in common 25.1 us with nine, 20.4 with eight, 25.8 with seven)
    static constexpr int WORKERS = FIT < 8 ? FIT : 8;
};

__device__ __forceinline__ void few_phase(const CUtensorMap& k_map, const CUtensorMap& v_map, const SharedArgs& a, const Plan& plan, unsigned char* smem, int workers) {
    using S = TmaFew;
    constexpr int KEYS = S::KEYS, STAGES = S::STAGES;
    if (threadIdx.x >= 32 * workers) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* ring = smem + warp * STAGES * S::STAGE;                // [stage][K, V][HALVES][KEYS][128 B], swizzled
    S::Worker& own = *reinterpret_cast<S::Worker*>(smem + workers * STAGES * S::STAGE + warp * S::CONTROL);
    // the blocks that have the fewest pieces of many rows come first
    const Piece piece = piece_of<0>(a, plan, (gridDim.x - 1 - blockIdx.x) * workers + warp);
    if (piece.from == piece.end) return;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&own.full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    const int group = a.group, tokens = a.tokens, num_pages = a.num_pages, page_size = a.page_size, shift = __ffs(page_size) - 1;
    const int box = min(page_size, KEYS), boxes = KEYS / box, rows_per_page = (int)(a.page_stride / HD);
    // ---- the walk: the step that comes next, and its pages, asked for a turn before its keys and values are
    int k = -1, left = 0, k0 = 0;                         // stretch, steps left of it, the step's first key
    bool first = false, more = true;
    Stretch at = {};
    int page = 0;                                         // lane j < boxes: of the step's j-th box
    const int* table = a.block_tables;
    auto look_up = [&]() {
        if (!more) return;
        first = left == 0;
        if (first) {
            if (++k % S::AT_ONCE == 0) {
                __syncwarp();
                if (lane < S::AT_ONCE) stretch_of<0>(a, plan, piece, k + lane, own.stretches[lane]);
                __syncwarp();
            }
            at = own.stretches[k % S::AT_ONCE];
            left = at.steps;
            more = left > 0;
            if (!more) return;
            k0 = at.k0;
            table = a.block_tables + (size_t)at.table * a.table_width;
        } else {
            k0 += KEYS;
        }
        --left;
        const int key = k0 + lane * box;
        page = lane < boxes && key < at.kend ? table[key >> shift] : -1;
    };
    // what a step needs when it has landed: bits 0 .. 15 its keys, 16 .. 18 first, last and valid; rows and slot; lane r: where
    // row r of the queries lies
    struct Landing { unsigned bits; int rows, slot; long long query; };
    auto fetch = [&](int stage) {
        Landing landing = {0u, 0, 0, 0};
        if (!more) return landing;
        const int key = k0 + lane * box;
        const bool asked = lane < boxes && key < at.kend, there = asked && (unsigned)page < (unsigned)num_pages;
        if (asked && !there) atomicExch(a.error, ERR_PAGE);
        const unsigned missing = __ballot_sync(0xffffffffu, asked && !there);
        unsigned keys = (0xffffu >> min(max(KEYS - (at.kend - k0), 0), KEYS)) & (0xffffu << max(at.begin - k0, 0));
        if (missing) keys &= missing & 1 ? (missing & 2 ? 0u : 0xff00u) : 0x00ffu;
        if (missing && boxes == 1) keys = 0u;
        landing.bits = (keys & 0xffffu) | (first ? 1u << 16 : 0u) | (left == 0 ? 1u << 17 : 0u) | 1u << 18;
        landing.rows = at.rows; landing.slot = at.slot;
        if (lane == 0) mbar_expect_tx(&own.full[stage], (uint32_t)S::STAGE);
        __syncwarp();
        if (lane < boxes) {
            // (a box that is not there: rows behind all pages, which arrive as zeros)
            const int row = there ? page * rows_per_page + (at.kvh << shift) + (key & (page_size - 1)) : NO_ROW;
            unsigned char* dst = ring + stage * S::STAGE + lane * box * 128;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                tma_load_2d(dst + h * S::HALF, &k_map, h * 64, row, &own.full[stage]);
                tma_load_2d(dst + (HALVES + h) * S::HALF, &v_map, h * 64, row, &own.full[stage]);
            }
        }
        if (first && lane < at.rows) {
            const int row = at.row0 + lane, further = row < group ? 0 : row / group;
            const int token = at.token >= 0 ? at.token : a.order[at.place + further];
            if ((unsigned)token < (unsigned)tokens) landing.query = (long long)token * a.q_ld + (at.kvh * group + row - further * group) * HD;
        }
        return landing;
    };

    const int g = lane >> 2, t = lane & 3;
    const float sc = a.scale * LOG2E;                     // scores in base-2 units
    FewState state;
    state.begin();
    unsigned qf[HD / 16][4];
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) qf[i][0] = qf[i][1] = qf[i][2] = qf[i][3] = 0u;
    // ldmatrix: this lane's row of 16 keys, and its 16-byte piece c of a row at 16 * (c ^ row % 8)
    const int k_row = ((lane & 7) + 8 * (lane >> 4)) * 128, k_piece = ((lane >> 3) & 1) ^ (lane & 7);
    const int v_row = ((lane & 7) + 8 * ((lane >> 3) & 1)) * 128, v_piece = (lane >> 4) ^ (lane & 7);
    Landing now = {0u, 0, 0, 0}, next = {0u, 0, 0, 0};
    static_assert(STAGES == 3, "landings held: this step's and the next two");
    int stage = 1, parity = 0;                            // of the step n (in front of the first: those of step -2)
    look_up();
    for (int n = 1 - STAGES;; ++n) {                      // (the first turns only fetch)
        if (n >= 0) {
            if (!(now.bits >> 18)) break;
            if (now.bits >> 16 & 1) {                     // a stretch begins: its queries, on their way beside the wait
                state.begin();
                const long long lo = __shfl_sync(0xffffffffu, now.query, g), hi = __shfl_sync(0xffffffffu, now.query, g + 8);
                const unsigned *q_lo = reinterpret_cast<const unsigned*>((const bf16*)a.q + lo) + t, *q_hi = reinterpret_cast<const unsigned*>((const bf16*)a.q + hi) + t;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) { qf[i][0] = q_lo[8 * i]; qf[i][1] = q_hi[8 * i]; qf[i][2] = q_lo[8 * i + 4]; qf[i][3] = q_hi[8 * i + 4]; }
            }
            if (!__all_sync(0xffffffffu, mbar_wait(&own.full[stage], parity))) {
                if (lane == 0) atomicExch(a.error, ERR_FEW);
                for (int i = 1; i < STAGES; ++i) {        // copies on the way
                    if (++stage == STAGES) { stage = 0; parity ^= 1; }
                    if ((i == 1 ? next.bits : 0u) >> 18) mbar_wait(&own.full[stage], parity);
                }
                return;
            }
        }
        const int ahead = stage == 0 ? STAGES - 1 : stage - 1;            // of step n + STAGES - 1
        const Landing behind = fetch(ahead);
        look_up();
        if (n >= 0) {
            unsigned char* kt = ring + stage * S::STAGE;
            unsigned char* vt = kt + HALVES * S::HALF;
            if ((now.bits & 0xffffu) != 0xffffu) {        // whatever lies behind the keys is multiplied with nothing
                for (int e = lane; e < HALVES * KEYS * 8; e += 32)
                    if (!(now.bits >> ((e >> 3) % KEYS) & 1)) *reinterpret_cast<uint4*>(vt + e * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            state.step([&](int i) { return kt + (i >> 2) * S::HALF + k_row + ((k_piece ^ (2 * (i & 3))) << 4); },
                       [&](int c) { return vt + (c >> 2) * S::HALF + v_row + ((v_piece ^ (2 * (c & 3))) << 4); },
                       [&](int i, unsigned (&q4)[4]) { q4[0] = qf[i][0]; q4[1] = qf[i][1]; q4[2] = qf[i][2]; q4[3] = qf[i][3]; }, now.bits, t, sc);
            if (now.bits >> 17 & 1) state.leave(a, now.rows, now.slot, g, t);
            __syncwarp();                                 // the step's place in the ring may be filled again
        }
        if (++stage == STAGES) { stage = 0; if (n >= 0) parity ^= 1; }
        now = next; next = behind;
    }
}

// Pages of keys or values as a matrix of HD columns, boxes of up to 16 rows x 64 columns, 128-byte swizzle.
static int pages_map(CUtensorMap& map, const void* pages, long long rows, int page_size) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return ERR_UNSUPPORTED;
    const cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)min(page_size, BOX)};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pages), dims, strides, box, elem,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : (int)ERR_BAD_ARGUMENT;
}

}  // namespace tc
#endif

// --------------------------------------------------------------------------------------------------- merge
// A unit is up to ROWS heads of one token and kv head, whose triples lie in the same tiles, side by side.  Lane d has the d-th
// run around the token: how many triples it left and where.  Then, in turns of 32 triples, lane j puts the j-th's
// place into a list in shared memory, each lane has the maxima and sums of one of the rows and of every (32 / ROWS)-th
// triple, the weights go into shared memory, and the columns are summed four per lane, in the order of the triples.  SPLIT
// warps have a share of a unit's triples each and join through shared memory, in order.
template <int ROWS, int SPLIT>
struct MergeShared {
    static constexpr int WARPS = SPLIT > 1 ? SPLIT : 1;
    int listed[32];                                       // of each warp: a turn's triples, their first rows
    float weights[32][ROWS];
    float4 joined[SPLIT > 1 ? ROWS : 1][SPLIT > 1 ? HD / 4 : 1];
    float2 joined_ml[ROWS];
};

template <typename T, int ROWS, int SPLIT, int WARPS>
__device__ __forceinline__ void merge_units(const SharedArgs& a, const Plan& plan, unsigned char* smem) {
    constexpr int CHUNKS = (HD / 4 + 31) / 32;
    constexpr int PARTS = 32 / ROWS, AHEAD = ROWS * CHUNKS >= 16 ? 1 : 16 / (ROWS * CHUNKS) < 8 ? 16 / (ROWS * CHUNKS) : 8;
    constexpr int TEAMS = WARPS / SPLIT;                                  // units that a block works on at once
    static_assert(sizeof(MergeShared<ROWS, SPLIT>) % 16 == 0 && sizeof(PlanSums) % 16 == 0, "what follows starts on 16 bytes");
    static_assert(FEW % ROWS == 0, "a unit lies in one tile");
    MergeShared<ROWS, SPLIT>* mine = reinterpret_cast<MergeShared<ROWS, SPLIT>*>(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % SPLIT, team = warp / SPLIT;
    MergeShared<ROWS, SPLIT>& own = mine[warp];
    if (team >= TEAMS) return;
    const int chunks = (a.group + ROWS - 1) / ROWS;                       // units of a token and kv head
    const int per_place = a.kv_heads * chunks, units = a.places * per_place;
    bool waited = false;
    for (int unit = blockIdx.x * TEAMS + team; unit < units; unit += gridDim.x * TEAMS) {
    const int place = a.by_place.of(unit), in_place = unit - place * per_place, kvh = a.by_chunks.of(in_place), g0 = (in_place - kvh * chunks) * ROWS;
    const int rows = min(ROWS, a.group - g0);
    const int token = a.order[place];
    int r = a.own_run[place], levels = 0, own_level = -1;
    const bool no_such_run = r < -1 || r >= a.run_count;
    if (no_such_run) r = -1;
    // ---- lane d: the d-th run around the token; its triples of row g0 are rows first_at, first_at + tile, ..
    for (; r >= 0 && levels < MAX_LEVELS; ++levels) {
        if (lane == levels) own_level = r;
        const int parent = plan.runs[r].parent;
        r = parent < r ? parent : -1;
    }
    const bool there = (unsigned)token < (unsigned)a.tokens;
    const int position = there ? a.positions[token] : -1;
    if ((no_such_run || r >= 0 || !there) && lane == 0) atomicExch(a.error, ERR_RUNS);
    int first_at = 0, count = 0, tile_rows = FEW;
    if (own_level >= 0) {
        const Run run = plan.runs[own_level];
        if (run.count > 0 && (place < run.first || place >= run.first + run.count)) {
            atomicExch(a.error, ERR_RUNS);                // a run that the token is not in
        } else if (run.count > 0) {
            const int kind = plan.kind[own_level], many = kind & RUN_FEW ? 0 : 1;
            const Side& side = many ? a.many : a.few;
            tile_rows = side.tile;
            const int token_in = place - run.first, tokens = tile_tokens(side, kind), part = side.parts > 1 ? g0 >> side.tile_shift : 0;
            const int tile = side.parts > 1 ? token_in * side.parts + part : tokens == 1 ? token_in : side.by_tokens.of(token_in);
            const int row = side.parts > 1 ? g0 - part * tile_rows : (token_in - tile * tokens) * a.group + g0;
            const int line = tile * a.kv_heads + kvh, of_line = line_steps(run, side), from = plan.step0(many)[own_level] + line * of_line;
            const int b0 = piece_at(plan, many, from);
            count = piece_at(plan, many, from + of_line - 1) - b0 + 1;
            first_at = (int)side.row0 + (plan.line0(many)[own_level] + line + b0) * tile_rows + row;
            // (a shared run ends in front of its tokens)
            if (!(kind & RUN_INNERMOST) && run.end - 1 > position) atomicExch(a.error, ERR_RUNS);
        }
    }
    if (!waited) {                                        // (all of the above is older than the kernel in front)
        grid_dependency_wait();
        grid_dependents_go();
        waited = true;
    }
    if (!there) continue;                                 // (all warps of a unit)
    int upto = count;
#pragma unroll
    for (int o = 1; o < MAX_LEVELS; o *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
    }
    const int triples = __shfl_sync(0xffffffffu, upto, MAX_LEVELS - 1);
    const int column = HD / 4 % 32 == 0 ? lane : min(lane, HD / 4 - 1);    // (lanes beyond the head read what another does)
    float4 sum[ROWS][CHUNKS];
#pragma unroll
    for (int g = 0; g < ROWS; ++g)
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) sum[g][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, denom = 0.f;                   // of row x
    const int x = lane % ROWS, part = lane / ROWS;
    int* list = own.listed;
    const int each = (triples + SPLIT - 1) / SPLIT, last = min(triples, (share + 1) * each);
    for (int t0 = share * each; t0 < last; t0 += 32) {
        const int have = min(32, last - t0);
        int at = 0;                                       // (places beyond the triples: row 0, which counts for nothing)
        for (int d = 0; d < levels; ++d) {
            const int n = __shfl_sync(0xffffffffu, count, d), j = t0 + lane - (__shfl_sync(0xffffffffu, upto, d) - n);
            const int from = __shfl_sync(0xffffffffu, first_at, d), step = __shfl_sync(0xffffffffu, tile_rows, d);
            if (j >= 0 && j < n) at = from + j * step;
        }
        __syncwarp();
        list[lane] = at;
        __syncwarp();
        float m[ROWS], l[ROWS], top_new = top;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int j = part + PARTS * i;
            m[i] = -INFINITY; l[i] = 0.f;
            if (j < have && x < rows) {
                const float2 ml = load_now(reinterpret_cast<const float2*>(a.part_ml) + list[j] + x);
                m[i] = ml.x; l[i] = ml.y;
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) top_new = fmaxf(top_new, m[i]);
#pragma unroll
        for (int o = ROWS; o < 32; o *= 2) top_new = fmaxf(top_new, __shfl_xor_sync(0xffffffffu, top_new, o));
        const float before = top == -INFINITY ? 0.f : expf(top - top_new);
        float sum_l = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const float w = m[i] == -INFINITY ? 0.f : expf(m[i] - top_new);
            own.weights[part + PARTS * i][x] = w;
            sum_l += l[i] * w;
        }
#pragma unroll
        for (int o = ROWS; o < 32; o *= 2) sum_l += __shfl_xor_sync(0xffffffffu, sum_l, o);
        denom = denom * before + sum_l;
        top = top_new;
        __syncwarp();
        if (t0 > share * each) {
#pragma unroll
            for (int g = 0; g < ROWS; ++g) {
                const float f = __shfl_sync(0xffffffffu, before, g);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) { sum[g][c].x *= f; sum[g][c].y *= f; sum[g][c].z *= f; sum[g][c].w *= f; }
            }
        }
        for (int j0 = 0; j0 < have; j0 += AHEAD) {
            // AHEAD triples' columns are asked for before the first is used
            float4 v[AHEAD][ROWS][CHUNKS];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const float4* from = reinterpret_cast<const float4*>(a.part_o) + (size_t)list[j0 + j] * (HD / 4) + column;
#pragma unroll
                for (int g = 0; g < ROWS; ++g)
                    if (g < rows) {
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c)
                            v[j][g][c] = load_now(from + g * (HD / 4) + (HD / 4 % 32 == 0 ? 32 * c : min(32 * c, HD / 4 - 1 - column)));
                    }
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
#pragma unroll
                for (int g = 0; g < ROWS; ++g)
                    if (g < rows) {
                        const float w = own.weights[j0 + j][g];
                        const bool counts = w != 0.f;     // (a stretch without a key may hold anything)
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            sum[g][c].x = fmaf(w, counts ? v[j][g][c].x : 0.f, sum[g][c].x);
                            sum[g][c].y = fmaf(w, counts ? v[j][g][c].y : 0.f, sum[g][c].y);
                            sum[g][c].z = fmaf(w, counts ? v[j][g][c].z : 0.f, sum[g][c].z);
                            sum[g][c].w = fmaf(w, counts ? v[j][g][c].w : 0.f, sum[g][c].w);
                        }
                    }
        }
    }
    // (lane g has row g's denominator)
    if constexpr (SPLIT > 1) {
#pragma unroll
        for (int g = 0; g < ROWS; ++g)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
                if (HD / 4 % 32 == 0 || lane + 32 * c < HD / 4) own.joined[g][lane + 32 * c] = sum[g][c];
        if (lane < ROWS) own.joined_ml[lane] = make_float2(top, denom);
        // (a unit's warps meet; behind the join again, since the next unit's sums go to the same place)
        auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * SPLIT) : "memory"); };
        meet();
        const MergeShared<ROWS, SPLIT>* of = mine + team * SPLIT;
        float f[SPLIT];
        float top_all = -INFINITY;
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) top_all = fmaxf(top_all, of[w].joined_ml[x].x);
        denom = 0.f;
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) {
            const float2 ml = of[w].joined_ml[x];
            f[w] = ml.x == -INFINITY ? 0.f : expf(ml.x - top_all);
            denom += ml.y * f[w];
        }
#pragma unroll
        for (int g = 0; g < ROWS; ++g)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                float4 all = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < SPLIT; ++w) {
                    const float fw = __shfl_sync(0xffffffffu, f[w], g);
                    const float4 v = of[w].joined[g][HD / 4 % 32 == 0 ? lane + 32 * c : min(lane + 32 * c, HD / 4 - 1)];
                    if (fw != 0.f) { all.x = fmaf(fw, v.x, all.x); all.y = fmaf(fw, v.y, all.y); all.z = fmaf(fw, v.z, all.z); all.w = fmaf(fw, v.w, all.w); }
                }
                sum[g][c] = all;
            }
        meet();
        if (share > 0) continue;
    }
    const float inverse = denom > 0.f ? 1.0f / denom : denom == denom ? 0.f : denom;     // no key: zeros; NaN stays NaN
#pragma unroll
    for (int g = 0; g < ROWS; ++g) {
        const float inv = __shfl_sync(0xffffffffu, inverse, g);
        if (g >= rows) continue;
        T* out = (T*)a.out + (size_t)token * a.out_ld + (kvh * a.group + g0 + g) * HD;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int d = (lane + 32 * c) * 4;
            if (HD / 4 % 32 == 0 || d < HD) {
                out[d] = from_float<T>(sum[g][c].x * inv); out[d + 1] = from_float<T>(sum[g][c].y * inv);
                out[d + 2] = from_float<T>(sum[g][c].z * inv); out[d + 3] = from_float<T>(sum[g][c].w * inv);
            }
        }
    }
    }
}

constexpr int MERGE_WARPS = 4;
template <typename T, int ROWS, int SPLIT>
__global__ void __launch_bounds__(32 * MERGE_WARPS)
shared_merge_kernel(const __grid_constant__ SharedArgs a) {
    extern __shared__ __align__(1024) unsigned char smem[];
    MergeShared<ROWS, SPLIT>* shared = reinterpret_cast<MergeShared<ROWS, SPLIT>*>(smem);
    PlanSums& sums = *reinterpret_cast<PlanSums*>(shared + MERGE_WARPS);
    Plan plan;
    const bool fits = make_plan<32 * MERGE_WARPS>(a, reinterpret_cast<unsigned char*>(&sums + 1), sums, plan);
    if (fits) merge_units<T, ROWS, SPLIT, MERGE_WARPS>(a, plan, smem);
    grid_dependency_wait();
    grid_dependents_go();
}
template <int ROWS, int SPLIT> constexpr size_t merge_smem() { return MERGE_WARPS * sizeof(MergeShared<ROWS, SPLIT>) + sizeof(PlanSums); }

using F32Few = F32Shape<2, 2, true>;
using F32Many = F32Shape<HD <= 128 ? 4 : 2, HD <= 128 ? 1 : 2, false>;
static_assert(F32Few::ROWS == FEW, "tiles of few rows");

// ----------------------------------------------------------------------------------------- the first launch
enum { ON_F32, ON_MMA, ON_TC };
constexpr size_t most_of(size_t a, size_t b) { return a > b ? a : b; }
constexpr size_t MOST_SMEM = 227 * 1024;
// FIXED, OF_STEP: see Side.  Equal pieces for all / these, us in a graph, 28 heads over 4, requests x keys in common and of their own:
//   tcgen05   32 x 1,024 + 1,024  28.5 / 22.2   64 x 1,024 + 1,024  40.3 / 31.2   128 x 512 + 200  32.8 / 26.9   8 x 4,096 + 200  16.0 / 15.1
//   mma.sync  (pages of 24)       29.3 / 27.8                       46.6 / 45.0                    34.8 / 32.5                    18.9 / 14.9
//   FFMA                          84.4 / 78.9                      145.7 / 144.5                    104 / 102                     42.9 / 33.9
// (200 x 8,192 + 512, 40 heads over 8: FIXED, OF_STEP 40, 21 99.3, 60, 16 92.2, 60, 12 86.7; the others within 4 %.  mma.sync and FFMA
// up to 40 % slower with twice as much.)
// WORKER_SMEM: shared memory of a worker of few rows where a block has several, 0 where it is one
template <int FORM> struct Form;
template <> struct Form<ON_F32> {
    static constexpr int THREADS = 128, FEW_WORKERS = 1, FEW_KEYS = F32Few::KEYS, MANY_TILE = F32Many::ROWS, MANY_KEYS = F32Many::KEYS;
    static constexpr size_t SMEM = most_of(F32Few::SMEM, F32Many::SMEM), FEW_AT = 0, WORKER_SMEM = 0;
    static constexpr int FIXED = 10, OF_STEP = 10;
};
template <> struct Form<ON_MMA> {
    using Few = FewShape<4, 190 * 1024>;
    static constexpr int THREADS = 128, FEW_WORKERS = Few::WORKERS, FEW_KEYS = Few::KEYS, MANY_TILE = ManyShape::ROWS, MANY_KEYS = ManyShape::KEYS;
    static constexpr size_t SMEM = most_of(Few::SMEM, ManyShape::SMEM), FEW_AT = 0, WORKER_SMEM = 0;
    static constexpr int FIXED = 20, OF_STEP = 10;
};
#ifdef FSIE_SHARED_TC
template <> struct Form<ON_TC> {
    using Few = tc::TmaFew;
    static constexpr int THREADS = tc::THREADS, FEW_WORKERS = Few::WORKERS, FEW_KEYS = Few::KEYS, MANY_TILE = tc::ROWS, MANY_KEYS = tc::KEYS;
    static constexpr size_t SMEM = tc::SMEM, FEW_AT = tc::CONTROL_BYTES, WORKER_SMEM = Few::WORKER;
    static constexpr int FIXED = 60, OF_STEP = 12;
};
#endif
template <int FORM> constexpr size_t plan_at(int few_workers) {
    return (most_of(Form<FORM>::SMEM, Form<FORM>::FEW_AT + few_workers * Form<FORM>::WORKER_SMEM) + 15) / 16 * 16;
}

template <int FORM>
__global__ void __launch_bounds__(Form<FORM>::THREADS, 1)
shared_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ SharedArgs a,
                        int few_workers, int plan_offset) {
    extern __shared__ __align__(1024) unsigned char smem[];
    if (!a.early) grid_dependency_wait();
    PlanSums& sums = *reinterpret_cast<PlanSums*>(smem + plan_offset);
    Plan plan;
    const bool fits = make_plan<Form<FORM>::THREADS>(a, smem + plan_offset + sizeof(PlanSums), sums, plan);
    if (a.early) grid_dependency_wait();
    grid_dependents_go();
    if (!fits) return;
    if constexpr (FORM == ON_F32) {
        f32_phase<HD <= 128 ? 4 : 2, HD <= 128 ? 1 : 2, false>(a, plan, smem);
        f32_phase<2, 2, true>(a, plan, smem);
    } else if constexpr (FORM == ON_MMA) {
        many_phase(a, plan, smem);
        few_phase<typename Form<FORM>::Few>(a, plan, smem, few_workers);
    }
#ifdef FSIE_SHARED_TC
    else {
        tc::tc_phase(k_map, v_map, a, plan, smem);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // what was written there comes before the copies of the few
        __syncthreads();
        tc::few_phase(k_map, v_map, a, plan, smem + tc::CONTROL_BYTES, few_workers);
    }
#endif
}

struct Shape { int blocks, few_workers, few_keys, many_tile, many_keys, fixed, of_step; };       // (few_workers: of a block)
constexpr int MAX_DEVICES = 64;

static bool tcgen05_takes(int page_size, long long page_stride, long long page_rows) {
#ifdef FSIE_SHARED_TC
    return (page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128) && page_stride % HD == 0 && page_rows <= tc::NO_ROW;
#else
    return false;
#endif
}

// How a form's launch looks on the current device: as many blocks as run at once beside plans of middling size.
template <int FORM>
static int shape_of(Shape& shape) {
    // Per process.  Calls come from several threads at once: one number is all that is kept, and whoever sees it sees the
    // kernel's attribute set as well; two that find none work out the same.
    static std::atomic<int> known[MAX_DEVICES];
    using F = Form<FORM>;
    int device = 0, sms = 0, per_sm = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (device < 0 || device >= MAX_DEVICES) return ERR_UNSUPPORTED;
    int blocks = known[device].load(std::memory_order_acquire);
    if (blocks == 0) {
        e = cudaFuncSetAttribute(shared_attention_kernel<FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST_SMEM);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (e == cudaSuccess)
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, shared_attention_kernel<FORM>, F::THREADS,
                                                              most_of(F::SMEM, F::FEW_AT + F::FEW_WORKERS * F::WORKER_SMEM) + plan_bytes(100));
        if (e != cudaSuccess) return (int)e;
        blocks = sms * per_sm;
        if (blocks <= 0) return ERR_UNSUPPORTED;
        known[device].store(blocks, std::memory_order_release);
    }
    shape = {blocks, F::FEW_WORKERS, F::FEW_KEYS, F::MANY_TILE, F::MANY_KEYS, F::FIXED, F::OF_STEP};
    return 0;
}
static int shape_of(int dtype, bool on_tcgen05, Shape& shape) {
    if (dtype == DTYPE_F32) return shape_of<ON_F32>(shape);
#ifdef FSIE_SHARED_TC
    if (on_tcgen05) return shape_of<ON_TC>(shape);
#endif
    return shape_of<ON_MMA>(shape);
}

template <int FORM>
static int launch(const Shape& shape, const CUtensorMap& k_map, const CUtensorMap& v_map, SharedArgs& a, cudaStream_t stream) {
    // a large plan takes the place of workers of few rows
    const size_t plan = sizeof(PlanSums) + plan_bytes(a.run_count);
    int workers = shape.few_workers;
    while (Form<FORM>::WORKER_SMEM && workers > 1 && plan_at<FORM>(workers) + plan > MOST_SMEM) --workers;
    const size_t at = plan_at<FORM>(workers);
    if (at + plan > MOST_SMEM) return ERR_UNSUPPORTED;
    a.few.of_block = workers;
    a.few.workers = shape.blocks * workers;
    a.few.by_workers = div_by(a.few.workers);
    return launch_dependent(shared_attention_kernel<FORM>, dim3(shape.blocks), dim3(Form<FORM>::THREADS), at + plan, stream, k_map, v_map, a, workers, (int)at);
}

// Few rows in all: a row to a unit and several warps on it, since what such a call waits for is one warp's chain of loads.
// More: what counts are instructions, and a warp takes several heads of a kv head together.  The whole call in a graph in us,
// 28 heads over 4 of 128, 16 to 256 keys of their own, for <rows of a unit, warps on it>:
//   requests x keys in common    rows    <1,4>  <1,2>  <2,2>  <8,1>
//   8 x 4,096                     224     15.0   15.6   17.8   32.5
//   16 x 1,024                    448     14.0   12.6   13.1   20.3
//   32 x 1,024                    896     18.2   15.3   15.8   22.6
//   64 x 2,048                  1,792     35.4   31.1   28.7   37.0
//   128 x 128                   3,584     34.8   25.9   23.0   20.3
// Up to four blocks to a multiprocessor.
template <typename T, int ROWS, int SPLIT>
static int launch_merge_as(SharedArgs& a, int blocks, cudaStream_t stream) {
    a.by_chunks = div_by((a.group + ROWS - 1) / ROWS);
    a.by_place = div_by((long long)a.kv_heads * ((a.group + ROWS - 1) / ROWS));
    const size_t smem = merge_smem<ROWS, SPLIT>() + plan_bytes(a.run_count);
    if (smem > 48 * 1024) return ERR_UNSUPPORTED;
    const long long units = (long long)a.places * a.kv_heads * ((a.group + ROWS - 1) / ROWS), teams = MERGE_WARPS / SPLIT;
    return launch_dependent(shared_merge_kernel<T, ROWS, SPLIT>, dim3((unsigned)min((units + teams - 1) / teams, (long long)blocks)), dim3(32 * MERGE_WARPS),
                            smem, stream, a);
}
template <typename T>
static int launch_merge(SharedArgs& a, int blocks, cudaStream_t stream) {
    const long long rows = (long long)a.places * a.heads;
    if (rows <= 2 * blocks) return launch_merge_as<T, 1, 4>(a, 4 * blocks, stream);
    if (rows <= 6 * blocks) return launch_merge_as<T, 1, 2>(a, 4 * blocks, stream);
    if (rows <= 16 * blocks) return launch_merge_as<T, 2, 2>(a, 4 * blocks, stream);
    return launch_merge_as<T, 8, 1>(a, 4 * blocks, stream);
}

// Where everything lies in the room, for `lines` lines of many rows; returns the bytes.
static long long lay_out(const Shape& shape, long long places, long long runs, int kv_heads, long long lines, unsigned char* room, SharedArgs& a) {
    a.few = {shape.blocks * shape.few_workers, (int)((places + runs) * kv_heads), FEW, shape.few_keys, 1, FEW_LEAST};
    a.few.fixed = shape.fixed; a.few.of_step = shape.of_step;
    const long long few_rows = (long long)(a.few.line_room + a.few.workers) * FEW, many_rows = (lines + shape.blocks) * shape.many_tile;
    a.many = {shape.blocks, (int)lines, shape.many_tile, shape.many_keys, 1, MANY_LEAST};
    a.many.row0 = few_rows;
    a.part_o = (float*)room;                             // (stores of 32 bytes: it starts on 128)
    a.part_ml = a.part_o + (few_rows + many_rows) * HD;
    return few_rows + many_rows > 0x7fffffffLL ? -1 : (few_rows + many_rows) * (HD + 2) * 4 + 128;
}

// Lines of many rows: the tiles of the runs around a token are at most `levels` deep, a shared run has one begun tile; with a
// group of more than few rows a token's own keys are among them.
static long long many_lines(const Shape& shape, long long places, long long shared, int heads, int kv_heads, int levels) {
    const long long group = heads / kv_heads, most = shape.many_tile;
    const long long of_all = group > most ? places * ((group + most - 1) / most) : (places + most / group - 1) / (most / group);
    return (levels * of_all + shared + (group > FEW ? places * ((group + most - 1) / most) : 0)) * kv_heads;
}

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_shared_attention_head_dim() { return HD; }
int fsie_shared_attention_max_runs() { return MAX_RUNS; }

// Bytes of room for `places` tokens in `runs` runs, `shared` of which are no token's innermost and lie at most `levels` deep
// around a token; negative: an error.
long long fsie_shared_attention_room(int places, int runs, int shared, int levels, int heads, int kv_heads, int dtype) {
    if (places < 0 || runs < 0 || runs > MAX_RUNS || shared < 0 || shared > runs || levels < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads ||
        (dtype != DTYPE_F32 && dtype != DTYPE_BF16))
        return ERR_BAD_ARGUMENT;
    long long most = 0;
    for (int on_tcgen05 = 0; on_tcgen05 < 2; ++on_tcgen05) {        // (which of the two takes the call the pages decide)
        if (on_tcgen05 && (dtype != DTYPE_BF16 || !tcgen05_takes(16, HD, 0))) continue;
        Shape shape;
        const int rc = shape_of(dtype, on_tcgen05, shape);
        if (rc != 0) return rc > 0 ? -1000 - rc : rc;
        SharedArgs a;
        const long long bytes = lay_out(shape, places, runs, kv_heads, many_lines(shape, places, shared, heads, kv_heads, levels), nullptr, a);
        if (bytes < 0) return ERR_UNSUPPORTED;
        most = max(most, bytes);
    }
    return most;
}

int fsie_shared_attention(const void* q, int q_ld, const void* k_pages, const void* v_pages, long long page_stride,
                          int page_size, int num_pages, const int* block_tables, int table_rows, int table_width,
                          const int* positions, int tokens, const int* order, int places, const int* runs, int run_count,
                          const int* own_run, void* out, int out_ld, int heads, int kv_heads, int head_dim, float scale,
                          void* room, long long room_bytes, int dtype, int early, int* error, cudaStream_t stream) {
    if (places < 0 || tokens < 0 || run_count < 0 || !error) return ERR_BAD_ARGUMENT;
    if (places == 0) return 0;
    if (head_dim != HD || run_count > MAX_RUNS) return ERR_UNSUPPORTED;
    const int each = dtype == DTYPE_BF16 ? 8 : 4;
    if ((dtype != DTYPE_F32 && dtype != DTYPE_BF16) || kv_heads <= 0 || heads <= 0 || heads % kv_heads || page_size <= 0 ||
        num_pages < 0 || table_rows < 0 || table_width < 0 || !q || !out || !order || !own_run || !positions || !room ||
        (run_count && (!runs || !block_tables || !k_pages || !v_pages)))
        return ERR_BAD_ARGUMENT;
    // rows are copied 16 bytes at a time
    if (q_ld % each || page_stride % each || (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)room) & 15))
        return ERR_BAD_ARGUMENT;
    if ((long long)places * heads > 0x7fffffffLL / 2) return ERR_UNSUPPORTED;
    const long long page_rows = num_pages > 0 ? (num_pages - 1) * (page_stride / HD) + (long long)kv_heads * page_size : 0;
    const bool on_tcgen05 = dtype == DTYPE_BF16 && page_rows > 0 && run_count > 0 && tcgen05_takes(page_size, page_stride, page_rows);
    Shape shape;
    int rc = shape_of(dtype, on_tcgen05, shape);
    if (rc != 0) return rc;
    // as many lines of many rows as the room has place for (its last 128 bytes are for a start on 128)
    room = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(room) + 127) & ~uintptr_t(127));
    SharedArgs a;
    const long long needed = lay_out(shape, places, run_count, kv_heads, 0, (unsigned char*)room, a);
    if (needed < 0) return ERR_UNSUPPORTED;
    if (needed > room_bytes) return ERR_BAD_ARGUMENT;
    const long long of_line = (long long)shape.many_tile * (HD + 2) * 4;
    const long long lines = min((room_bytes - needed) / of_line, 0x7fffffffLL / shape.many_tile - shape.blocks - (a.many.row0 + shape.many_tile) / shape.many_tile);
    if (lay_out(shape, places, run_count, kv_heads, lines, (unsigned char*)room, a) < 0) return ERR_UNSUPPORTED;
    a.many.align = a.few.align = on_tcgen05 ? min(page_size, 16) : 1;     // (a box of the copy engine)
    a.q = q; a.q_ld = q_ld; a.k_pages = k_pages; a.v_pages = v_pages; a.page_stride = page_stride; a.page_size = page_size;
    a.num_pages = num_pages; a.block_tables = block_tables; a.table_rows = table_rows; a.table_width = table_width;
    a.positions = positions; a.tokens = tokens; a.order = order; a.places = places; a.runs = runs; a.run_count = run_count;
    a.own_run = own_run; a.out = out; a.out_ld = out_ld; a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads;
    a.scale = scale; a.early = early; a.error = error;
    a.most_steps = 0x7fffffff / max(run_count, 1);
    a.by_kv_heads = div_by(kv_heads); a.by_group = div_by(a.group);
    for (Side* side : {&a.few, &a.many}) {
        side->tile_shift = log2_of(side->tile); side->key_shift = log2_of(side->keys);
        side->tokens = max(side->tile / a.group, 1); side->parts = (a.group + side->tile - 1) / side->tile;
        side->by_tokens = div_by(side->tokens); side->by_parts = div_by(side->parts); side->by_workers = div_by(side->workers);
    }
    CUtensorMap k_map = {}, v_map = {};
    if (dtype == DTYPE_F32) {
        rc = launch<ON_F32>(shape, k_map, v_map, a, stream);
        return rc != 0 ? rc : launch_merge<float>(a, shape.blocks, stream);
    }
#ifdef FSIE_SHARED_TC
    if (on_tcgen05) {
        rc = tc::pages_map(k_map, k_pages, page_rows, page_size);
        if (rc == 0) rc = tc::pages_map(v_map, v_pages, page_rows, page_size);
        if (rc == 0) rc = launch<ON_TC>(shape, k_map, v_map, a, stream);
        return rc != 0 ? rc : launch_merge<bf16>(a, shape.blocks, stream);
    }
#endif
    rc = launch<ON_MMA>(shape, k_map, v_map, a, stream);
    return rc != 0 ? rc : launch_merge<bf16>(a, shape.blocks, stream);
}

}  // extern "C"
