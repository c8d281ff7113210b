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
// Schedule.  What a run holds is known on the device only (a captured graph replays with other runs), so the blocks share
// the work out themselves: all (tile, kv head) lines of the runs laid end to end, in steps of KEYS keys, are cut into equal
// pieces, one per block; a block walks from line to line, with the next steps' keys on their way, and leaves the triple of
// every stretch of a line that it has worked on in `room`.  shared_merge_kernel joins the triples of a row, in a fixed
// order.  Two launches split the runs between them by their rows: few (a token's own keys) and many (shared ones).
#include "common.cuh"
#include "tma.cuh"
#include "attention_tc.cuh"
#include <math.h>
#include <string.h>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head size: 16..256 in steps of 16");

namespace fsie {

constexpr int HD = HEAD_DIM;
constexpr int FEW = 16;                  // rows that count as few: those of a tile
constexpr int MMA_FEW_KEYS = 16, MMA_MANY_KEYS = 64, F32_KEYS = 32;       // keys of a step
constexpr int MAX_RUNS = 1024;
constexpr int MAX_LEVELS = 32;           // runs that lie around each other, the innermost among them
constexpr int RUN_INTS = 6;
constexpr int LINE_PIECES = 32;          // a line is cut into no more pieces than this: what joins them reads them all
constexpr int LEAST_KEYS = 128;          // keys of a piece, at least
constexpr int LISTS_BYTES = 12 * 1024;   // lists of up to this size are read into shared memory first
enum { ERR_PAGE = 3, ERR_RUNS = 7, ERR_ROOM = 8 };

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
    int* few_table; int* many_table;                          // the launches' schedules, for the merge: [2 + 2 * run_count]
    float* part_ml; float* part_o;                            // [rows, 2], [rows, HD]
    int few_rows, many_rows;                                  // rows for the triples of either launch, few's in front
    int many_tile, many_keys, many_align;                     // rows of a tile of many rows, keys of its steps, where those begin
    int lists_in_smem;
    int early;                                                // the lists are older than the stream's last kernel
    int* error;
};

struct Run { int first, count, begin, end, table, innermost; };

// The lists, in shared or global memory.
struct Lists {
    const int* runs; const int* own_run; const int* order;
    const int* place_position;           // null: to be looked up by the place's token

    __device__ int position(const SharedArgs& a, int place) const {
        if (place_position) return place_position[place];
        const int token = order[place];
        return (unsigned)token < (unsigned)a.tokens ? a.positions[token] : -1;
    }
};

// A run as the lists give it; count 0 where it has no keys or places, or (and *error) points outside of what there is.
__device__ __forceinline__ Run load_run(const SharedArgs& a, const int* runs, const int* own_run, int r) {
    const int* p = runs + (size_t)r * RUN_INTS;
    Run run = {p[0], p[1], p[2], p[3], p[4], 0};
    const int parent = p[5];
    if (run.count <= 0 || run.end <= run.begin) { run.count = 0; return run; }
    if (run.first < 0 || run.count > a.places || run.first > a.places - run.count || run.begin < 0 ||
        run.end > (long long)a.table_width * a.page_size || (unsigned)run.table >= (unsigned)a.table_rows || parent < -1 || parent >= r) {
        atomicExch(a.error, ERR_RUNS);
        run.count = 0;
        return run;
    }
    run.innermost = own_run[run.first] == r;
    return run;
}

// A tile's rows are those of the whole run, or, in an innermost run, of one of its tokens.
__device__ __forceinline__ int rows_to_tile(const SharedArgs& a, const Run& run) { return run.innermost ? a.group : run.count * a.group; }
// Steps of a line, from the border of `align` keys (a power of two) in front of the run's first on.
__device__ __forceinline__ int line_steps(const Run& run, int keys, int align) {
    return (int)(((unsigned)run.end - (unsigned)(run.begin & ~(align - 1)) + (unsigned)keys - 1u) / (unsigned)keys);
}
// Lines and steps of a line that a launch - of the runs of up to FEW rows, or of the others - makes of a run.
template <bool IS_FEW>
__device__ __forceinline__ void count_run(const SharedArgs& a, const Run& run, int tile_rows, int keys, int align, int& lines, int& of_line) {
    lines = of_line = 0;
    const int rows = rows_to_tile(a, run);
    if (run.count == 0 || (rows <= FEW) != IS_FEW) return;
    of_line = line_steps(run, keys, align);
    lines = (rows + tile_rows - 1) / tile_rows * (run.innermost ? run.count : 1) * a.kv_heads;
}

// ---- the schedule
// What a block keeps in shared memory behind everything else: steps and lines in front of each run (step0 and line0, both
// [run_count + 1]), and the lists where they fit.
constexpr int MAX_WARPS = 10;            // of a block
struct Schedule { int steps[MAX_WARPS], lines[MAX_WARPS], longest[MAX_WARPS], size[MAX_WARPS]; };
struct Plan {
    int *step0, *line0;
    Lists lists;
    int piece, total;                    // steps of a worker's piece, steps in all
};

__host__ __device__ __forceinline__ size_t lists_bytes(long long runs, long long places) { return (runs * RUN_INTS + 3 * places) * 4; }
__host__ __device__ __forceinline__ size_t plan_bytes(int runs, int places, int lists_in_smem) {
    return ((2 * ((size_t)runs + 1)) * 4 + (lists_in_smem ? lists_bytes(runs, places) : 0) + 15) / 16 * 16;
}

// All THREADS threads of a block; `workers` in the whole launch.  False: there is nothing to do.
template <bool IS_FEW, int ROWS, int KEYS, int THREADS>
__device__ bool make_plan(const SharedArgs& a, int align, int workers, unsigned char* smem, Schedule& s, Plan& plan) {
    constexpr int WARPS = THREADS / 32;
    static_assert(WARPS <= MAX_WARPS, "warps of a block");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    plan.step0 = reinterpret_cast<int*>(smem);
    plan.line0 = plan.step0 + a.run_count + 1;
    plan.lists = {a.runs, a.own_run, a.order, nullptr};
    int* positions = nullptr;
    int position = -1;                   // of place `tid`: asked for here, put down below
    if (a.lists_in_smem) {
        int* runs = plan.line0 + a.run_count + 1;
        int* own_run = runs + a.run_count * RUN_INTS;
        int* order = own_run + a.places;
        positions = order + a.places;
        for (int e = tid; e < a.places; e += THREADS) { order[e] = a.order[e]; own_run[e] = a.own_run[e]; }
        for (int e = tid; e < a.run_count * RUN_INTS; e += THREADS) runs[e] = a.runs[e];
        if (tid < a.places && (unsigned)order[tid] < (unsigned)a.tokens) position = a.positions[order[tid]];
        for (int e = tid + THREADS; e < a.places; e += THREADS)
            positions[e] = (unsigned)order[e] < (unsigned)a.tokens ? a.positions[order[e]] : -1;
        plan.lists = {runs, own_run, order, positions};
        __syncthreads();
    }
    int steps_before = 0, lines_before = 0, longest = 0, size = 0;
    for (int base = 0; base < a.run_count; base += THREADS) {
        const int r = base + tid;
        int lines = 0, of_line = 0;
        if (r < a.run_count)
            count_run<IS_FEW>(a, load_run(a, plan.lists.runs, plan.lists.own_run, r), ROWS, KEYS, align, lines, of_line);
        longest = max(longest, of_line);
        size += (int)min(((long long)lines * of_line >> 10) + 1, 1ll << 20);        // in 1,024 steps: says whether `steps` may overflow
        const int steps = lines * of_line;
        int steps_upto = steps, lines_upto = lines;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int su = __shfl_up_sync(0xffffffffu, steps_upto, o), lu = __shfl_up_sync(0xffffffffu, lines_upto, o);
            if (lane >= o) { steps_upto += su; lines_upto += lu; }
        }
        if (base > 0) __syncthreads();
        if (lane == 31) { s.steps[warp] = steps_upto; s.lines[warp] = lines_upto; }
        const bool last = base + THREADS >= a.run_count;
        if (last) {
            const int l = __reduce_max_sync(0xffffffffu, longest), z = (int)__reduce_add_sync(0xffffffffu, (unsigned)size);
            if (lane == 0) { s.longest[warp] = l; s.size[warp] = z; }
        }
        __syncthreads();
        // the warps' sums: lane w has warp w's
        const int ws = lane < WARPS ? s.steps[lane] : 0, wl = lane < WARPS ? s.lines[lane] : 0;
        const bool before = lane < warp;
        steps_upto += steps_before + (int)__reduce_add_sync(0xffffffffu, before ? (unsigned)ws : 0u);
        lines_upto += lines_before + (int)__reduce_add_sync(0xffffffffu, before ? (unsigned)wl : 0u);
        steps_before += (int)__reduce_add_sync(0xffffffffu, (unsigned)ws);
        lines_before += (int)__reduce_add_sync(0xffffffffu, (unsigned)wl);
        if (r < a.run_count) { plan.step0[r] = steps_upto - steps; plan.line0[r] = lines_upto - lines; }
        if (last) {
            longest = __reduce_max_sync(0xffffffffu, lane < WARPS ? s.longest[lane] : 0);
            size = (int)__reduce_add_sync(0xffffffffu, lane < WARPS ? (unsigned)s.size[lane] : 0u);
        }
    }
    if (tid == 0) { plan.step0[a.run_count] = steps_before; plan.line0[a.run_count] = lines_before; }
    if (positions && tid < a.places) positions[tid] = position;
    plan.total = steps_before;
    plan.piece = max((steps_before + workers - 1) / workers, max((LEAST_KEYS + KEYS - 1) / KEYS, (longest + LINE_PIECES - 1) / LINE_PIECES));
    const bool fits = size < (1 << 20) && ((long long)lines_before + workers) * ROWS <= (IS_FEW ? a.few_rows : a.many_rows);
    __syncthreads();
    // what the merge has to know (a piece of 0: nothing was done)
    if (blockIdx.x == gridDim.x - 1) {
        int* table = IS_FEW ? a.few_table : a.many_table;
        if (tid == 0) { table[0] = fits ? plan.piece : 0; table[1] = fits ? steps_before : 0; }
        for (int r = tid; r < a.run_count; r += THREADS) { table[2 + 2 * r] = plan.step0[r]; table[3 + 2 * r] = plan.line0[r]; }
    }
    if (!fits && tid == 0) atomicExch(a.error, ERR_ROOM);
    return fits && steps_before > 0;
}

// ---- one step of a worker's walk: KEYS keys of a line
struct Step {
    int valid, first, last;              // whether there is one; first or last of the worker's stretch of the line
    int k0, begin, kend, table, kvh;     // (begin: the run's first key, where steps begin in front of it)
    int place, row0, rows;               // the tile's rows are rows row0 .. of the tokens from `place` on
    int slot;                            // where the stretch's triple goes, in tiles
    int outer;                           // a run whose tokens must all see all of its keys
    int stretch;                         // how many stretches the worker has begun before
};

template <int ROWS, int KEYS>
struct Walker {
    int run_index, lines, line, of_line, i, i_end, at, from, end, per_token, all_rows, align, worker;
    Run run;
    Step line_step;                      // what the steps of the line have in common

    __device__ void start(const SharedArgs& a, const Plan& plan, int which, int step_align) {
        align = step_align; worker = which;
        const long long begin = (long long)worker * plan.piece;
        from = at = end = 0;
        line_step.stretch = 0;
        if (begin >= plan.total) return;
        from = at = (int)begin;
        end = min(at + min(plan.piece, plan.total - at), plan.total);
        int low = 0, high = a.run_count;                                  // step0[low] <= at < step0[high]
        while (high - low > 1) {
            const int middle = (low + high) >> 1;
            if (plan.step0[middle] <= at) low = middle; else high = middle;
        }
        run_index = low;
        enter_run(a, plan);
        const int inside = at - plan.step0[run_index];
        line = inside / of_line;
        i = inside - line * of_line;
        enter_line(a, plan);
    }
    __device__ void enter_run(const SharedArgs& a, const Plan& plan) {
        run = load_run(a, plan.lists.runs, plan.lists.own_run, run_index);
        all_rows = rows_to_tile(a, run);
        per_token = (all_rows + ROWS - 1) / ROWS;                         // tiles of the run, or of one of its tokens
        lines = per_token * (run.innermost ? run.count : 1) * a.kv_heads;
        of_line = line_steps(run, KEYS, align);
        line = i = 0;
    }
    __device__ void enter_line(const SharedArgs& a, const Plan& plan) {
        Step& n = line_step;
        const int tile = line / a.kv_heads;
        n.kvh = line - tile * a.kv_heads;
        int part = tile, token = 0;
        if (run.innermost) {
            token = per_token == 1 ? tile : tile / per_token;
            part = tile - token * per_token;
        } else if (part > 0) {
            token = part * ROWS / a.group;
        }
        n.place = run.first + token;
        n.row0 = run.innermost ? part * ROWS : part * ROWS - token * a.group;
        n.rows = min(ROWS, all_rows - part * ROWS);
        n.kend = run.end;
        if (run.innermost) {
            const int position = plan.lists.position(a, n.place);
            if (position < run.end) n.kend = position + 1;
        }
        n.begin = run.begin; n.table = run.table; n.outer = !run.innermost;
        n.slot = plan.line0[run_index] + line + worker;
        i_end = min(of_line, i + (end - at));
    }
    __device__ bool more() const { return at < end; }
    __device__ int first_key() const { return (run.begin & ~(align - 1)) + i * KEYS; }
    __device__ void go_on(const SharedArgs& a, const Plan& plan) {       // to the next line, at the end of a stretch
        ++line_step.stretch;
        if (at >= end) return;
        i = 0;
        if (++line == lines) {
            do ++run_index; while (plan.step0[run_index + 1] == plan.step0[run_index]);
            enter_run(a, plan);
        }
        enter_line(a, plan);
    }
    __device__ void next(const SharedArgs& a, const Plan& plan, Step& out) {
        if (!more()) { out.valid = 0; return; }
        out = line_step;
        out.valid = 1;
        out.first = i == 0 || at == from;
        out.last = i + 1 == i_end;
        out.k0 = first_key();
        ++at; ++i;
        if (i == i_end) go_on(a, plan);
    }
    // a whole stretch: out.k0 is its first step's first key, out.last its number of steps
    __device__ void next_stretch(const SharedArgs& a, const Plan& plan, Step& out) {
        if (!more()) { out.valid = 0; return; }
        out = line_step;
        out.valid = 1;
        out.k0 = first_key();
        out.last = i_end - i;
        at += i_end - i;
        go_on(a, plan);
    }
};

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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}

constexpr float LOG2E = 1.4426950408889634f;

// ---- blocks of 128 threads that share steps: the ring of steps, and their keys and query rows on the way
constexpr int THREADS = 128;
template <typename T, int ROWS, bool IS_FEW, int KEYS, int STAGES, int K_LD, int V_LD, int Q_LD>
struct Feed {
    static constexpr int PIECES = HD * (int)sizeof(T) / 16;               // 16-byte pieces of a head
    static constexpr int EACH = 16 / (int)sizeof(T);
    static constexpr int RECORDS = STAGES + 2, BASES = STAGES + 1;
    struct Shared {
        long long key_base[BASES][KEYS];                                  // element offset of a key's row in the pages; -1: no key
        Schedule schedule;
        Step steps[RECORDS];
    };
    const SharedArgs& a;
    Shared& sh;
    unsigned char* plan_at;
    T *ks, *vs, *qs;
    Plan plan;
    Walker<ROWS, KEYS> walker;                                            // thread 0's

    __device__ Feed(const SharedArgs& args, Shared& shared, unsigned char* behind, T* k, T* v, T* q)
        : a(args), sh(shared), plan_at(behind), ks(k), vs(v), qs(q) {}

    __device__ void find(int n) {                                         // where the keys of step n lie
        const Step& st = sh.steps[n % RECORDS];
        if (threadIdx.x >= KEYS || !st.valid) return;
        const int key = st.k0 + (int)threadIdx.x;
        long long base = -1;
        if (key < st.kend) {
            const int block = key / a.page_size;
            const int page = a.block_tables[(size_t)st.table * a.table_width + block];
            if ((unsigned)page < (unsigned)a.num_pages)
                base = (long long)page * a.page_stride + ((long long)st.kvh * a.page_size + (key - block * a.page_size)) * HD;
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
                const long long at = (base >= 0 ? base : 0) + c;
                copy16(kd + j * K_LD + c, kp + at, base >= 0);
                copy16(vd + j * V_LD + c, vp + at, base >= 0);
            }
            if (st.first) {
                T* qd = qs + (size_t)(st.stretch % STAGES) * ROWS * Q_LD;
                const T* q = (const T*)a.q;
                for (int e = threadIdx.x; e < ROWS * PIECES; e += THREADS) {
                    const int r = e / PIECES, c = (e - r * PIECES) * EACH;
                    bool ok = r < st.rows;
                    long long at = 0;
                    if (ok) {
                        const int row = st.row0 + r, place = st.place + row / a.group, token = plan.lists.order[place];
                        ok = (unsigned)token < (unsigned)a.tokens;
                        if (ok) at = (long long)token * a.q_ld + (st.kvh * a.group + row % a.group) * HD + c;
                        // (a shared run ends in front of its tokens)
                        if (!ok || (st.outer && plan.lists.position(a, place) < st.kend - 1)) atomicExch(a.error, ERR_RUNS);
                    }
                    copy16(qd + r * Q_LD + c, q + at, ok);
                }
            }
        }
        copies_commit();
    }
    // Plan and first steps; false: nothing to do.  The launch of the many rows comes first and waits for the kernel in
    // front of it.  That of the few rows reads nothing that the many's wrote, and starts when all of its blocks have waited:
    // it works beside it and waits when it is done, so that the merge behind it finds both done.
    __device__ bool start() {
        if (!IS_FEW && !a.early) grid_dependency_wait();
        const bool any = make_plan<IS_FEW, ROWS, KEYS, THREADS>(a, 1, gridDim.x, plan_at, sh.schedule, plan);
        if (any) {
            if (threadIdx.x == 0) {
                walker.start(a, plan, blockIdx.x, 1);
                for (int n = 0; n <= STAGES; ++n) walker.next(a, plan, sh.steps[n]);
            }
            __syncthreads();
            for (int n = 0; n < STAGES; ++n) find(n);
        }
        if (!IS_FEW && a.early) grid_dependency_wait();
        grid_dependents_go();
        if (!any) { finish(); return false; }
        __syncthreads();
        for (int n = 0; n < STAGES - 1; ++n) fetch(n);
        return true;
    }
    __device__ void finish() {
        copies_wait<0>();
        if (IS_FEW) grid_dependency_wait();
    }
    // step n has landed: on with the steps behind it
    __device__ void advance(int n) {
        copies_wait<STAGES - 2>();
        __syncthreads();
        fetch(n + STAGES - 1);
        find(n + STAGES);
        if (threadIdx.x == 0) walker.next(a, plan, sh.steps[(n + STAGES + 1) % RECORDS]);
    }
    __device__ const Step& step(int n) const { return sh.steps[n % RECORDS]; }
};

// ------------------------------------------------------------------------------------- bfloat16, few rows
// Every warp is a worker of its own: one tile of 16 rows, steps of 16 keys, its own ring of STAGES steps in shared memory, and
// no meeting of warps on the way.  What a step costs is its chain of dependent instructions, so what counts is how many warps
// an SM has at it and how few instructions they take: four warps that shared a step of 32 keys took 442 instructions each,
// and 62 us where these take XX (200 requests, 40 heads over 8 of 128, 32 to 512 keys of their own each).
struct FewShape {
    static constexpr int KEYS = MMA_FEW_KEYS, STAGES = 3;
    static constexpr int LD = HD + 8;                    // padded rows: ldmatrix without bank conflicts
    static constexpr bool Q_IN_REGS = HD <= 128;
    static constexpr int Q_SLOTS = Q_IN_REGS ? 2 : 3;
    static constexpr size_t WORKER = ((size_t)STAGES * 2 * KEYS + (size_t)Q_SLOTS * FEW) * LD * sizeof(bf16);
    static constexpr int FIT = (int)(205 * 1024 / WORKER);
    static constexpr int WORKERS = FIT < 8 ? FIT : 8;
    static constexpr int THREADS = 32 * WORKERS;
    static constexpr size_t SMEM = WORKERS * WORKER + (sizeof(Schedule) + 15) / 16 * 16;
};

__global__ void __launch_bounds__(FewShape::THREADS, 1)
shared_few_kernel(const SharedArgs a) {
    using S = FewShape;
    constexpr int KEYS = S::KEYS, STAGES = S::STAGES, LD = S::LD, PIECES = HD / 8;
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bf16* ring = reinterpret_cast<bf16*>(smem + warp * S::WORKER);        // [stage][K, V][KEYS][LD]
    bf16* qs = ring + STAGES * 2 * KEYS * LD;                             // [slot][FEW][LD]
    Schedule& schedule = *reinterpret_cast<Schedule*>(smem + S::WORKERS * S::WORKER);
    Plan plan;
    const int worker = blockIdx.x * S::WORKERS + warp;
    const bool any = make_plan<true, FEW, KEYS, S::THREADS>(a, 1, gridDim.x * S::WORKERS, smem + S::SMEM, schedule, plan);
    grid_dependents_go();
    if (!any) { grid_dependency_wait(); return; }
    Walker<FEW, KEYS> walker;
    walker.start(a, plan, worker, 1);

    // ---- a step on its way: first its keys' pages are asked for, a turn later its keys and values
    Step coming;                                          // the step whose pages have been asked for
    int page = 0, inside = -1;                            // of key `lane % 16` of it: its page and its place there (-1: no key)
    auto look_up = [&]() {
        walker.next(a, plan, coming);
        inside = -1;
        const int key = coming.k0 + (lane & 15);
        if (coming.valid && key < coming.kend) {
            const int block = key / a.page_size;
            inside = key - block * a.page_size;
            page = a.block_tables[(size_t)coming.table * a.table_width + block];
        }
    };
    // what the step needs when it has landed: bits 0 .. 15 its keys, 16 .. 18 first, last and valid; rows and slot
    struct Landing { unsigned bits; int rows, slot; };
    auto fetch = [&](int n) {
        Landing landing = {0u, 0, 0};
        if (coming.valid) {
            const bool there = inside >= 0 && (unsigned)page < (unsigned)a.num_pages;
            if (inside >= 0 && !there) atomicExch(a.error, ERR_PAGE);
            const long long base = there ? (long long)page * a.page_stride + ((long long)coming.kvh * a.page_size + inside) * HD : -1;
            landing.bits = (__ballot_sync(0xffffffffu, there) & 0xffffu) | (coming.first ? 1u << 16 : 0u) | (coming.last ? 1u << 17 : 0u) | 1u << 18;
            landing.rows = coming.rows; landing.slot = coming.slot;
            bf16* kd = ring + (n % STAGES) * 2 * KEYS * LD;
            const bf16* kp = (const bf16*)a.k_pages;
            const bf16* vp = (const bf16*)a.v_pages;
#pragma unroll
            for (int e0 = 0; e0 < KEYS * PIECES; e0 += 32) {
                const int e = e0 + lane, j = e / PIECES, c = (e - j * PIECES) * 8;
                const long long at = __shfl_sync(0xffffffffu, base, j);
                copy16(kd + j * LD + c, kp + (at >= 0 ? at + c : 0), at >= 0);
                copy16(kd + (KEYS + j) * LD + c, vp + (at >= 0 ? at + c : 0), at >= 0);
            }
            if (coming.first) {
                long long row_at = -1;                    // of row `lane`
                if (lane < coming.rows) {
                    const int row = coming.row0 + lane, further = row < a.group ? 0 : row / a.group, place = coming.place + further;
                    const int token = plan.lists.order[place];
                    if ((unsigned)token < (unsigned)a.tokens)
                        row_at = (long long)token * a.q_ld + (coming.kvh * a.group + row - further * a.group) * HD;
                    // (a shared run ends in front of its tokens)
                    if (row_at < 0 || (coming.outer && plan.lists.position(a, place) < coming.kend - 1)) atomicExch(a.error, ERR_RUNS);
                }
                __syncwarp();
                bf16* qd = qs + (coming.stretch % S::Q_SLOTS) * FEW * LD;
#pragma unroll
                for (int e0 = 0; e0 < FEW * PIECES; e0 += 32) {
                    const int e = e0 + lane, r = e / PIECES, c = (e - r * PIECES) * 8;
                    const long long at = __shfl_sync(0xffffffffu, row_at, r);
                    copy16(qd + r * LD + c, (const bf16*)a.q + (at >= 0 ? at + c : 0), at >= 0);
                }
            }
        }
        copies_commit();
        return landing;
    };

    static_assert(STAGES == 3, "landings held: this step's and the next two");
    look_up();
    Landing now = fetch(0);
    look_up();
    Landing next = fetch(1);
    look_up();
    const int g = lane >> 2, t = lane & 3;
    const float sc = a.scale * LOG2E;                     // scores in base-2 units
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    float o[HD / 8][4];
    unsigned qf[S::Q_IN_REGS ? HD / 16 : 1][4];
    int stretch = -1;

    for (int n = 0; now.bits >> 18; ++n) {
        copies_wait<STAGES - 2>();
        __syncwarp();
        if (now.bits >> 16 & 1) ++stretch;
        const bf16* q_at = qs + (stretch % S::Q_SLOTS) * FEW * LD + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + 8 * (lane >> 4);
        if (now.bits >> 16 & 1) {
            m_lo = m_hi = -INFINITY; l_lo = l_hi = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) { o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f; }
            if (S::Q_IN_REGS) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) ldmatrix_x4(qf[k], q_at + k * 16);
                __syncwarp();                             // the slot may be filled again
            }
        }
        const Landing behind = fetch(n + STAGES - 1);
        look_up();
        const bf16* kt = ring + (n % STAGES) * 2 * KEYS * LD;
        const bf16* vt = kt + KEYS * LD;
        // ---- scores: two chains of products for each eight keys
        float s[2][4], s2[2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[c][e] = s2[c][e] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            unsigned q4[4], b[4];
            if (S::Q_IN_REGS) { q4[0] = qf[k][0]; q4[1] = qf[k][1]; q4[2] = qf[k][2]; q4[3] = qf[k][3]; }
            else ldmatrix_x4(q4, q_at + k * 16);
            ldmatrix_x4(b, kt + ((lane & 7) + 8 * (lane >> 4)) * LD + k * 16 + 8 * ((lane >> 3) & 1));
            mma_bf16(k & 1 ? s2[0] : s[0], q4, b[0], b[1]);
            mma_bf16(k & 1 ? s2[1] : s[1], q4, b[2], b[3]);
        }
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool there = now.bits >> (c * 8 + 2 * t + e) & 1;
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
        const float corr_lo = exp2f(m_lo * sc - base_lo), corr_hi = exp2f(m_hi * sc - base_hi);
        m_lo = mn_lo; m_hi = mn_hi;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            s[c][0] = exp2f(s[c][0] * sc - base_lo); s[c][1] = exp2f(s[c][1] * sc - base_lo);
            s[c][2] = exp2f(s[c][2] * sc - base_hi); s[c][3] = exp2f(s[c][3] * sc - base_hi);
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
        for (int c = 0; c < HD / 16; ++c) {
            unsigned b[4];
            ldmatrix_x4_trans(b, vt + ((lane & 7) + 8 * ((lane >> 3) & 1)) * LD + c * 16 + 8 * (lane >> 4));
            mma_bf16(o[2 * c], p4, b[0], b[1]);
            mma_bf16(o[2 * c + 1], p4, b[2], b[3]);
        }
        if (now.bits >> 17 & 1) {
            // ---- the stretch's triples
            l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
            l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = g + 8 * half;
                if (r >= now.rows) continue;
                const size_t row = (size_t)now.slot * FEW + r;
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
        __syncwarp();                                     // the step's place in the ring may be filled again
        now = next; next = behind;
    }
    copies_wait<0>();
    grid_dependency_wait();                               // (beside the many's kernel: see Feed::start)
}

// ------------------------------------------------------------------------------------- bfloat16, many rows
// Head sizes and pages that the tcgen05 kernel below does not take: tiles of 64 rows, 16 to a warp.
struct ManyShape {
    static constexpr int ROWS = 64, KEYS = MMA_MANY_KEYS, STAGES = 2;
    static constexpr int LD = HD + 8;
    using F = Feed<bf16, ROWS, false, KEYS, STAGES, LD, LD, LD>;
    static constexpr size_t SMEM = (size_t)STAGES * (2 * KEYS + ROWS) * LD * sizeof(bf16) + (sizeof(F::Shared) + 15) / 16 * 16;
};

__global__ void __launch_bounds__(THREADS)
shared_many_kernel(const SharedArgs a) {
    using S = ManyShape;
    constexpr int KEYS = S::KEYS, NT = KEYS / 8;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* ks = reinterpret_cast<bf16*>(smem);
    bf16* vs = ks + (size_t)S::STAGES * KEYS * S::LD;
    bf16* qs = vs + (size_t)S::STAGES * KEYS * S::LD;
    S::F::Shared& sh = *reinterpret_cast<S::F::Shared*>(qs + (size_t)S::STAGES * S::ROWS * S::LD);
    S::F feed(a, sh, smem + S::SMEM, ks, vs, qs);
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
        const size_t row = (size_t)a.few_rows + (size_t)st.slot * S::ROWS;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = half ? r_hi : r_lo;
            if (r >= st.rows) continue;
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
__global__ void __launch_bounds__(THREADS)
shared_f32_kernel(const SharedArgs a) {
    using S = F32Shape<WARPS_M, WARPS_K, FEW_ROWS>;
    constexpr int STAGES = S::STAGES, VEC = S::VEC, KEYS = S::KEYS;
    extern __shared__ __align__(16) unsigned char smem[];
    float* ks = reinterpret_cast<float*>(smem);
    float* vs = ks + STAGES * KEYS * S::K_LD;
    float* qs = vs + STAGES * KEYS * HD;
    float* ps = qs + STAGES * S::ROWS * HD;
    float* row_max = ps + S::ROWS * S::P_LD;
    float* row_sum = row_max + WARPS_K * S::ROWS;
    typename S::F::Shared& sh = *reinterpret_cast<typename S::F::Shared*>(row_sum + WARPS_K * S::ROWS);
    typename S::F feed(a, sh, smem + S::SMEM, ks, vs, qs);
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
        const size_t row = (S::IS_FEW ? 0 : (size_t)a.few_rows) + (size_t)st.slot * S::ROWS;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r0 + i >= st.rows) continue;
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
static_assert(THREADS / 32 <= MAX_WARPS, "warps of a block");
constexpr int HALVES = HD / 64, ATOM = 128 * 128;        // 128-byte column halves of a row; 128 rows of one
constexpr int Q_BYTES = HALVES * ATOM, KV_BYTES = HALVES * ATOM;
constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_O = STREAMS * KEYS;
enum { ROLE_PRODUCER, ROLE_MMA, ROLE_SOFTMAX, ROLES = ROLE_SOFTMAX + STREAMS };
enum { ERR_TC_PRODUCER = 31, ERR_TC_MMA = 32, ERR_TC_SOFTMAX = 33, ERR_TC_LAYOUT = 34 };

struct Control {
    uint64_t ring_full[SLOTS], ring_empty[SLOTS], s_full[STREAMS], p_ready[STREAMS], o_done[STREAMS], q_ready[STREAMS];
    uint32_t tmem_slot;
    int abort_flag;
    Schedule schedule;
    Plan plan;
    Walker<ROWS, KEYS> walkers[ROLES];
    Step stretches[ROLES][2];            // a role's stretch, by turns
    long long query_at[STREAMS][BM];     // where a stream's rows begin in q; -1: no row
};
constexpr int CONTROL_BYTES = 4096;
static_assert(sizeof(Control) <= CONTROL_BYTES, "control block");
constexpr size_t SMEM = CONTROL_BYTES + STREAMS * Q_BYTES + SLOTS * KV_BYTES;

// a stream's 128 threads meet
__device__ __forceinline__ void stream_meet(int st) {
    if (st == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
    else asm volatile("bar.sync 2, 128;" ::: "memory");
}

__global__ void __launch_bounds__(THREADS, 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const SharedArgs a) {
    extern __shared__ __align__(1024) unsigned char smem_all[];
    Control& ctl = *reinterpret_cast<Control*>(smem_all);
    unsigned char* q_s = smem_all + CONTROL_BYTES;       // [stream][HALVES][128 rows][128 B]
    unsigned char* ring = q_s + STREAMS * Q_BYTES;       // [slot][HALVES][128 keys][128 B]
    if ((smem_addr(smem_all) & 1023) != 0) {             // the swizzle goes by addresses
        if (threadIdx.x == 0) atomicExch(a.error, ERR_TC_LAYOUT);
        grid_dependency_wait();
        if (blockIdx.x == gridDim.x - 1 && threadIdx.x < 2) a.many_table[threadIdx.x] = 0;
        return;
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (!a.early) grid_dependency_wait();
    Plan planned;
    const bool any = make_plan<false, ROWS, KEYS, THREADS>(a, a.page_size, gridDim.x, smem_all + SMEM, ctl.schedule, planned);
    if (!any) {
        if (a.early) grid_dependency_wait();
        grid_dependents_go();
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < SLOTS; ++s) { mbar_init(&ctl.ring_full[s], 1); mbar_init(&ctl.ring_empty[s], 1); }
        for (int st = 0; st < STREAMS; ++st) {
            mbar_init(&ctl.s_full[st], 1); mbar_init(&ctl.p_ready[st], BM); mbar_init(&ctl.o_done[st], 1);
            mbar_init(&ctl.q_ready[st], BM);
        }
        ctl.abort_flag = 0;
        ctl.plan = planned;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp >= 2 && warp < 2 + ROLES && lane == 0) ctl.walkers[warp - 2].start(a, planned, blockIdx.x, a.page_size);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&ctl.tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = ctl.tmem_slot;
    const Plan& plan = ctl.plan;
    if (a.early) grid_dependency_wait();
    grid_dependents_go();
    auto give_up = [&](int code) { atomicExch(a.error, code); atomicExch(&ctl.abort_flag, 1); };

    if (warp == 0) {
        // ------------------------------------------------------------------ producer: lane j has page j of a tile
        const int ps = a.page_size, pages_per_tile = KEYS / ps;
        const long long rows_per_page = a.page_stride / HD;
        int e = 0;                                        // ring entries so far: K, V, K, ...
        bool ok = true;
        for (int turn = 0; ok; turn ^= 1) {
            if (lane == 0) ctl.walkers[ROLE_PRODUCER].next_stretch(a, plan, ctl.stretches[ROLE_PRODUCER][turn]);
            __syncwarp();
            const Step& st = ctl.stretches[ROLE_PRODUCER][turn];
            if (!st.valid) break;
            const int tiles = st.last, kend = st.kend;
            const int* table = a.block_tables + (size_t)st.table * a.table_width;
            auto look_up = [&](int i) {                   // beyond the keys any page will do: they count for nothing
                const int key = st.k0 + i * KEYS + lane * ps;
                return lane < pages_per_tile && i < tiles && key < kend ? table[key / ps] : 0;
            };
            int ahead = look_up(0);
            for (int i = 0; i < tiles && ok; ++i) {
                int page = ahead;
                ahead = look_up(i + 1);
                if ((unsigned)page >= (unsigned)a.num_pages) {
                    atomicExch(a.error, ERR_PAGE);
                    page = 0;
                }
#pragma unroll
                for (int kv = 0; kv < 2 && ok; ++kv, ++e) {
                    const int s = e % SLOTS;
                    if (lane == 0 && e >= SLOTS) ok = mbar_wait(&ctl.ring_empty[s], (e / SLOTS - 1) & 1);
                    ok = __shfl_sync(0xffffffffu, ok, 0) && !*(volatile int*)&ctl.abort_flag;
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&ctl.ring_full[s], (uint32_t)KV_BYTES);
                    __syncwarp();
                    if (lane < pages_per_tile) {
                        unsigned char* dst = ring + (size_t)s * KV_BYTES + lane * ps * 128;
                        const int row = (int)(page * rows_per_page + (long long)st.kvh * ps);
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) tma_load_2d(dst + h * ATOM, kv ? &v_map : &k_map, h * 64, row, &ctl.ring_full[s]);
                    }
                }
            }
            if (!ok) {
                if (lane == 0) give_up(ERR_TC_PRODUCER);
                for (int k = max(0, e - SLOTS); k < e; ++k) mbar_wait(&ctl.ring_full[k % SLOTS], (k / SLOTS) & 1);    // copies on the way
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA: one lane issues, all take part in the waits
        const uint32_t idesc_s = idesc_bf16(BM, KEYS, 0), idesc_o = idesc_bf16(BM, HD, 1);
        const uint64_t q_base = desc_k_major(q_s), k_base = desc_k_major(ring), v_base = desc_mn_major(ring, ATOM);
        int e = 0, tiles_of[STREAMS] = {0, 0}, stretches_of[STREAMS] = {0, 0};
        bool ok = true;
        auto wait = [&](uint64_t* bar, int parity) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar, parity & 1))) {
                if (lane == 0) give_up(ERR_TC_MMA);
                ok = false;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        };
        auto ring_wait = [&](int entry) { wait(&ctl.ring_full[entry % SLOTS], entry / SLOTS); };
        for (int turn = 0; ok; turn ^= 1) {
            if (lane == 0) ctl.walkers[ROLE_MMA].next_stretch(a, plan, ctl.stretches[ROLE_MMA][turn]);
            __syncwarp();
            const Step& sr = ctl.stretches[ROLE_MMA][turn];
            if (!sr.valid) break;
            const int tiles = sr.last, k0 = sr.k0, begin = sr.begin, kend = sr.kend, streams = sr.rows > BM ? 2 : 1;
            auto scores = [&](int st, int entry) {        // S_st = Q_st K^T
                if (lane == 0) {
                    const uint64_t qd = q_base + (uint64_t)(st * (Q_BYTES >> 4));
                    const uint64_t kd = k_base + (uint64_t)((entry % SLOTS) * (KV_BYTES >> 4));
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t step = (k >> 2) * (ATOM >> 4) + 2 * (k & 3);
                        mma_ss(tmem + COL_S + st * KEYS, qd + step, kd + step, idesc_s, k > 0);
                    }
                    mma_commit(&ctl.s_full[st]);
                    if (st == streams - 1) mma_commit(&ctl.ring_empty[entry % SLOTS]);
                }
                __syncwarp();
            };
            for (int st = 0; st < streams && ok; ++st) wait(&ctl.q_ready[st], stretches_of[st]++);
            if (ok) ring_wait(e);
            for (int st = 0; st < streams && ok; ++st) scores(st, e);
            for (int i = 0; i < tiles && ok; ++i, e += 2) {
                for (int st = 0; st < streams && ok; ++st) {
                    wait(&ctl.p_ready[st], tiles_of[st]++);
                    if (!ok) break;
                    if (st == 0) {
                        ring_wait(e + 1);
                        if (!ok) break;
                        const int from = k0 + i * KEYS;
                        if (from < begin || from + KEYS > kend) {          // rows of V that are none of the run's keys
                            unsigned char* v = ring + (size_t)((e + 1) % SLOTS) * KV_BYTES;
                            for (int at = lane; at < KEYS * 8 * HALVES; at += 32) {
                                const int key = from + (at >> 3) % KEYS;
                                if (key < begin || key >= kend) *reinterpret_cast<uint4*>(v + (size_t)at * 16) = make_uint4(0, 0, 0, 0);
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                        }
                    }
                    if (lane == 0) {
                        const uint64_t vd = v_base + (uint64_t)(((e + 1) % SLOTS) * (KV_BYTES >> 4));
#pragma unroll
                        for (int k = 0; k < KEYS / 16; ++k)               // 16 keys: 8 columns of P, 16 rows of V
                            mma_ts(tmem + COL_O + st * KEYS, tmem + COL_S + st * KEYS + k * 8, vd + (uint64_t)(k * (16 * 128 >> 4)),
                                   idesc_o, (i > 0 || k > 0) ? 1u : 0u);
                        if (i + 1 == tiles) mma_commit(&ctl.o_done[st]);
                        if (st == streams - 1) mma_commit(&ctl.ring_empty[(e + 1) % SLOTS]);
                    }
                    __syncwarp();
                    if (i + 1 < tiles) {                                   // the stream's next scores, beside the other's softmax
                        if (st == 0) ring_wait(e + 2);
                        if (ok) scores(st, e + 2);
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax, a thread per row of a stream
        const int st = (warp - 2) / 4, quarter = warp & 3, r = quarter * 32 + lane, role = ROLE_SOFTMAX + st;
        const int in_group = tid - 64 - st * BM;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_addr = lane_base + COL_S + st * KEYS, o_addr = lane_base + COL_O + st * KEYS;
        const float sc = a.scale * LOG2E;
        const bf16* q = (const bf16*)a.q;
        int tiles_done = 0, stretches_done = 0;
        bool ok = true;
        for (int turn = 0; ok; turn ^= 1) {
            if (in_group == 0) ctl.walkers[role].next_stretch(a, plan, ctl.stretches[role][turn]);
            stream_meet(st);
            const Step& sr = ctl.stretches[role][turn];
            if (!sr.valid) break;
            const int tiles = sr.last, k0 = sr.k0, begin = sr.begin, kend = sr.kend, rows = sr.rows - st * BM;
            if (rows <= 0) continue;
            const bool valid = r < rows;
            // ---- the stream's queries, K-major and swizzled (zero beyond the tile's rows); all S of the stretch before are done
            long long mine = -1;
            if (valid) {
                const int row = sr.row0 + st * BM + r, further = row / a.group, place = sr.place + further, token = plan.lists.order[place];
                if ((unsigned)token < (unsigned)a.tokens) mine = (long long)token * a.q_ld + (sr.kvh * a.group + row - further * a.group) * HD;
                // (a shared run ends in front of its tokens)
                if (mine < 0 || (sr.outer && plan.lists.position(a, place) < kend - 1)) atomicExch(a.error, ERR_RUNS);
            }
            ctl.query_at[st][r] = mine;
            stream_meet(st);
            {
                constexpr int CHUNKS = HD / 8;            // 16-byte pieces of a row: all of a thread's are asked for at once
                uint4 held[CHUNKS];
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j) {
                    const int at = in_group + j * BM, rr = at / CHUNKS, c = at - rr * CHUNKS;
                    const long long from = ctl.query_at[st][rr];
                    held[j] = make_uint4(0, 0, 0, 0);
                    if (from >= 0) held[j] = *reinterpret_cast<const uint4*>(q + from + c * 8);
                }
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j) {
                    const int at = in_group + j * BM, rr = at / CHUNKS, c = at - rr * CHUNKS;
                    *reinterpret_cast<uint4*>(q_s + st * Q_BYTES + (c >> 3) * ATOM + swizzled(rr, c & 7)) = held[j];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&ctl.q_ready[st]);
            }
            float m_run = -INFINITY, l_run = 0.f;
            for (int i = 0; i < tiles && ok; ++i, ++tiles_done) {
                if (!__all_sync(0xffffffffu, mbar_wait(&ctl.s_full[st], tiles_done & 1))) {
                    if (lane == 0) give_up(ERR_TC_SOFTMAX);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int from = k0 + i * KEYS;
                uint32_t sv[KEYS];
#pragma unroll
                for (int c = 0; c < KEYS; c += 32) tmem_ld32_issue(s_addr + c, sv + c);
                tmem_wait_ld();
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (from >= begin && from + KEYS <= kend) {
#pragma unroll
                    for (int j = 0; j < KEYS; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(sv[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < KEYS; ++j) {
                        if (from + j < begin || from + j >= kend) sv[j] = 0xff800000u;        // -inf
                        mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(sv[j]));
                    }
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
                float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KEYS; j += 2) {
                    const float p0 = fast_exp2(fmaf(__uint_as_float(sv[j]), sc, -base));
                    const float p1 = fast_exp2(fmaf(__uint_as_float(sv[j + 1]), sc, -base));
                    sum4[(j >> 1) & 1] += p0;
                    sum4[2 + ((j >> 1) & 1)] += p1;
                    sv[j >> 1] = pack_bf16(p0, p1);
                }
#pragma unroll
                for (int c = 0; c < KEYS / 2; c += 32) tmem_st32_issue(s_addr + c, sv + c);
                tmem_wait_st();
                l_run = l_run * corr + (valid ? (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]) : 0.f);
                m_run = m_new;
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                mbar_arrive(&ctl.p_ready[st]);
            }
            if (!ok) break;
            // ---- the row's triple
            if (!__all_sync(0xffffffffu, mbar_wait(&ctl.o_done[st], stretches_done & 1))) {
                if (lane == 0) give_up(ERR_TC_SOFTMAX);
                ok = false;
                break;
            }
            ++stretches_done;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const size_t row = (size_t)a.few_rows + (size_t)sr.slot * ROWS + st * BM + r;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                float v[32];
                tmem_ld32(o_addr + c, v);                 // (all lanes take part)
                if (valid) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4*>(a.part_o + row * HD + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                }
            }
            if (valid) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m_run == -INFINITY ? m_run : m_run * a.scale, l_run);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Pages of keys or values as a matrix of HD columns, boxes of page_size rows x 64 columns, 128-byte swizzle.
static int pages_map(CUtensorMap& map, const void* pages, long long rows, int page_size) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return ERR_UNSUPPORTED;
    const cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)page_size};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pages), dims, strides, box, elem,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : (int)ERR_BAD_ARGUMENT;
}

}  // namespace tc
#endif

// --------------------------------------------------------------------------------------------------- merge
// A warp per (place, head).  Lane d has the d-th run around the token and finds how many triples of the row it left and where;
// then lane j has the j-th triple, in turns of 32, the weights travel by shuffles, and the columns are summed four per lane
// in the order of the triples.
constexpr int MERGE_WARPS = 4;

template <typename T, int FEW_KEYS>
__global__ void __launch_bounds__(32 * MERGE_WARPS)
shared_merge_kernel(const SharedArgs a) {
    const int unit = blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int place = unit / a.heads, h = unit - place * a.heads, kvh = h / a.group, g = h - kvh * a.group;
    // ---- the token's runs, from the innermost on (the lists are older than the kernels in front of this one)
    int token = -1, mine = -1, levels = 0;
    Run run = {};
    if (place < a.places) {
        token = a.order[place];
        int r = a.own_run[place];
        if (r >= a.run_count) r = -1;
        while (r >= 0 && levels < MAX_LEVELS) {
            if (lane == levels) mine = r;
            ++levels;
            const int parent = a.runs[(size_t)r * RUN_INTS + 5];
            r = parent < r ? parent : -1;
        }
        if (r >= 0) atomicExch(a.error, ERR_RUNS);
        if (mine >= 0) run = load_run(a, a.runs, a.own_run, mine);
    }
    grid_dependency_wait();
    grid_dependents_go();
    if (place >= a.places) return;
    if ((unsigned)token >= (unsigned)a.tokens) {
        if (lane == 0) atomicExch(a.error, ERR_RUNS);
        return;
    }
    // ---- this lane's run: its triples of the row are rows first_at, first_at + tile, ..
    long long first_at = 0;
    int count = 0, tile_rows = FEW;
    if (mine >= 0 && run.count > 0 && place >= run.first && place < run.first + run.count) {
        const bool few = rows_to_tile(a, run) <= FEW;
        const int* table = few ? a.few_table : a.many_table;
        const int2 shape = *reinterpret_cast<const int2*>(table), at = *reinterpret_cast<const int2*>(table + 2 + 2 * mine);
        tile_rows = few ? FEW : a.many_tile;
        const int of_line = few ? line_steps(run, FEW_KEYS, 1) : line_steps(run, a.many_keys, a.many_align);
        const int row_in = (run.innermost ? 0 : (place - run.first) * a.group) + g, part = row_in / tile_rows;
        const int tile = part + (run.innermost ? (place - run.first) * ((a.group + tile_rows - 1) / tile_rows) : 0);
        const int line = tile * a.kv_heads + kvh;
        const long long from = (long long)at.x + (long long)line * of_line;
        if (shape.x > 0 && from + of_line <= shape.y) {                   // (pieces of shape.x steps, shape.y steps in all)
            const int b0 = (int)from / shape.x;
            count = (int)(from + of_line - 1) / shape.x - b0 + 1;
            first_at = (few ? 0 : (long long)a.few_rows) + (long long)(at.y + line + b0) * tile_rows + (row_in - part * tile_rows);
        }
    }
    int upto = count;
#pragma unroll
    for (int o = 1; o < MAX_LEVELS; o *= 2) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
    }
    const int triples = __shfl_sync(0xffffffffu, upto, MAX_LEVELS - 1);
    constexpr int CHUNKS = (HD / 4 + 31) / 32;
    float4 sum[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) sum[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, denom = 0.f;
    for (int t0 = 0; t0 < triples; t0 += 32) {
        const int have = min(32, triples - t0);
        long long at = 0;
        for (int d = 0; d < levels; ++d) {
            const int behind = __shfl_sync(0xffffffffu, upto, d), n = __shfl_sync(0xffffffffu, count, d);
            const long long from = __shfl_sync(0xffffffffu, first_at, d);
            const int step = __shfl_sync(0xffffffffu, tile_rows, d), j = t0 + lane - (behind - n);
            if (j >= 0 && j < n) at = from + (long long)j * step;
        }
        float m = -INFINITY, l = 0.f;
        if (lane < have) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
            m = ml.x; l = ml.y;
        }
        // the columns are asked for beside the maxima and sums; eight triples' at a time
        float4 v[8][CHUNKS];
        auto ask = [&](int j0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const long long from = __shfl_sync(0xffffffffu, at, (j0 + j) & 31);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
                    if (j0 + j < have && (HD / 4 % 32 == 0 || lane + 32 * c < HD / 4))
                        v[j][c] = *reinterpret_cast<const float4*>(a.part_o + from * HD + (lane + 32 * c) * 4);
            }
        };
        ask(0);
        const float top_new = fmaxf(top, warp_max(m));
        const float before = top == -INFINITY ? 0.f : expf(top - top_new);
        const float w = m == -INFINITY ? 0.f : expf(m - top_new);
        denom = denom * before + warp_sum(l * w);
        top = top_new;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) { sum[c].x *= before; sum[c].y *= before; sum[c].z *= before; sum[c].w *= before; }
        for (int j0 = 0; j0 < have; j0 += 8) {
            if (j0 > 0) ask(j0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, (j0 + j) & 31);
                if (j0 + j < have && wj != 0.f) {         // (a stretch without a key may hold anything)
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        sum[c].x = fmaf(wj, v[j][c].x, sum[c].x); sum[c].y = fmaf(wj, v[j][c].y, sum[c].y);
                        sum[c].z = fmaf(wj, v[j][c].z, sum[c].z); sum[c].w = fmaf(wj, v[j][c].w, sum[c].w);
                    }
                }
            }
        }
    }
    const float inv = denom > 0.f ? 1.0f / denom : denom == denom ? 0.f : denom;     // no key: zeros; NaN stays NaN
    T* out = (T*)a.out + (size_t)token * a.out_ld + h * HD;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int d = (lane + 32 * c) * 4;
        if (HD / 4 % 32 == 0 || d < HD) {
            out[d] = from_float<T>(sum[c].x * inv); out[d + 1] = from_float<T>(sum[c].y * inv);
            out[d + 2] = from_float<T>(sum[c].z * inv); out[d + 3] = from_float<T>(sum[c].w * inv);
        }
    }
}

using F32Few = F32Shape<2, 2, true>;
using F32Many = F32Shape<4, 1, false>;
static_assert(F32Few::ROWS == FEW, "tiles of few rows");

// blocks of `kernel` that the current device runs at once, with its own shared memory and a plan of middling size
constexpr size_t MIDDLING_PLAN = 4096;
constexpr size_t MOST_PLAN = 2 * (MAX_RUNS + 1) * 4 + LISTS_BYTES + 16;
template <typename K>
static int blocks_at_once(K kernel, int threads, size_t smem, int& blocks) {
    int device = 0, sms = 0, per_sm = 0, most = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
    if (e == cudaSuccess && smem + MOST_PLAN > (size_t)most) return ERR_UNSUPPORTED;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(smem + MOST_PLAN));
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem + MIDDLING_PLAN);
    blocks = sms * per_sm;
    return e != cudaSuccess ? (int)e : blocks > 0 ? 0 : (int)ERR_UNSUPPORTED;
}

struct Shape { int few_blocks, few_workers, many_blocks, many_tile, many_keys, on_tcgen05; };       // (a worker: a block, or a warp of one)
constexpr int MAX_DEVICES = 64;

static bool tcgen05_takes(int page_size, long long page_stride) {
#ifdef FSIE_SHARED_TC
    return (page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128) && page_stride % HD == 0;
#else
    return false;
#endif
}

// How the two launches of a storage type look on the current device.
static int shape_of(int dtype, bool on_tcgen05, Shape& shape) {
    static Shape known[3][MAX_DEVICES] = {};             // per process; the same whoever writes it
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (device < 0 || device >= MAX_DEVICES) return ERR_UNSUPPORTED;
    Shape& have = known[dtype == DTYPE_F32 ? 0 : on_tcgen05 ? 2 : 1][device];
    if (have.many_blocks == 0) {
        Shape found = {};
        int rc;
        if (dtype == DTYPE_F32) {
            rc = blocks_at_once(shared_f32_kernel<2, 2, true>, THREADS, F32Few::SMEM, found.few_blocks);
            if (rc == 0) rc = blocks_at_once(shared_f32_kernel<4, 1, false>, THREADS, F32Many::SMEM, found.many_blocks);
            found.few_workers = found.few_blocks;
            found.many_tile = F32Many::ROWS; found.many_keys = F32Many::KEYS;
        } else {
            rc = blocks_at_once(shared_few_kernel, FewShape::THREADS, FewShape::SMEM, found.few_blocks);
            found.few_workers = found.few_blocks * FewShape::WORKERS;
#ifdef FSIE_SHARED_TC
            if (rc == 0 && on_tcgen05) {
                rc = blocks_at_once(tc::shared_tc_kernel, tc::THREADS, tc::SMEM, found.many_blocks);
                found.many_tile = tc::ROWS; found.many_keys = tc::KEYS; found.on_tcgen05 = 1;
            }
#endif
            if (rc == 0 && !found.on_tcgen05) {
                rc = blocks_at_once(shared_many_kernel, THREADS, ManyShape::SMEM, found.many_blocks);
                found.many_tile = ManyShape::ROWS; found.many_keys = ManyShape::KEYS;
            }
        }
        if (rc != 0) return rc;
        have = found;
    }
    shape = have;
    return 0;
}

// Rows of triples that the two launches may need.  Innermost runs are tiled token by token, other runs of few rows have a
// tile each; the many-row tiles of the runs around a token are at most `levels` deep.
static void rows_needed(const Shape& shape, long long places, long long runs, int heads, int kv_heads, int levels, long long& few, long long& many) {
    const long long group = heads / kv_heads;
    few = ((places + runs) * kv_heads + shape.few_workers) * FEW;
    long long tiles = levels * ((places * group + shape.many_tile - 1) / shape.many_tile) + runs;
    if (group > FEW) tiles += places * ((group + shape.many_tile - 1) / shape.many_tile);
    many = (tiles * kv_heads + shape.many_blocks) * shape.many_tile;
}
constexpr long long TABLE_BYTES = 2 * (2 + 2 * MAX_RUNS) * 4;       // both schedules, in front of the triples
static_assert(TABLE_BYTES % 16 == 0, "the triples start on 16 bytes");

}  // namespace fsie

using namespace fsie;

extern "C" {

int fsie_shared_attention_head_dim() { return HD; }
int fsie_shared_attention_max_runs() { return MAX_RUNS; }

// Bytes of room for `places` tokens in `runs` runs that are at most `levels` deep around a token; negative: an error.
long long fsie_shared_attention_room(int places, int runs, int levels, int heads, int kv_heads, int dtype) {
    if (places < 0 || runs < 0 || runs > MAX_RUNS || levels < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads ||
        (dtype != DTYPE_F32 && dtype != DTYPE_BF16))
        return ERR_BAD_ARGUMENT;
    long long most = 0;
    for (int on_tcgen05 = 0; on_tcgen05 < 2; ++on_tcgen05) {        // (which of the two takes the call the pages decide)
        if (on_tcgen05 && (dtype != DTYPE_BF16 || !tcgen05_takes(16, HD))) continue;
        Shape shape;
        const int rc = shape_of(dtype, on_tcgen05, shape);
        if (rc != 0) return rc > 0 ? -1000 - rc : rc;
        long long few, many;
        rows_needed(shape, places, runs, heads, kv_heads, levels, few, many);
        most = max(most, few + many);
    }
    return most * (HD + 2) * 4 + TABLE_BYTES;
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
    if ((long long)places * heads > 0x7fffffffLL - MERGE_WARPS) return ERR_UNSUPPORTED;
    const long long page_rows = num_pages > 0 ? (num_pages - 1) * (page_stride / HD) + (long long)kv_heads * page_size : 0;
    const bool on_tcgen05 = dtype == DTYPE_BF16 && page_rows > 0 && page_rows < (1ll << 31) && run_count > 0 && tcgen05_takes(page_size, page_stride);
    Shape shape;
    int rc = shape_of(dtype, on_tcgen05, shape);
    if (rc != 0) return rc;
    long long few, many;
    rows_needed(shape, places, run_count, heads, kv_heads, 0, few, many);
    const long long rows = (room_bytes - TABLE_BYTES) / ((HD + 2) * 4);
    if (rows - few < many || few > 0x7fffffffLL) return ERR_BAD_ARGUMENT;
    SharedArgs a;
    a.q = q; a.q_ld = q_ld; a.k_pages = k_pages; a.v_pages = v_pages; a.page_stride = page_stride; a.page_size = page_size;
    a.num_pages = num_pages; a.block_tables = block_tables; a.table_rows = table_rows; a.table_width = table_width;
    a.positions = positions; a.tokens = tokens; a.order = order; a.places = places; a.runs = runs; a.run_count = run_count;
    a.own_run = own_run; a.out = out; a.out_ld = out_ld; a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.scale = scale;
    a.few_table = (int*)room; a.many_table = a.few_table + 2 + 2 * MAX_RUNS;
    a.few_rows = (int)few; a.many_rows = (int)min(rows - few, 0x7fffffffLL);
    a.many_tile = shape.many_tile; a.many_keys = shape.many_keys; a.many_align = on_tcgen05 ? page_size : 1;
    a.part_o = reinterpret_cast<float*>((unsigned char*)room + TABLE_BYTES);
    a.part_ml = a.part_o + (few + a.many_rows) * HD;
    a.lists_in_smem = lists_bytes(run_count, places) <= LISTS_BYTES;
    a.early = early; a.error = error;
    const size_t plan = plan_bytes(run_count, places, a.lists_in_smem);
    const dim3 few_grid(shape.few_blocks), many_grid(shape.many_blocks);
    if (dtype == DTYPE_F32) {
        rc = launch_dependent(shared_f32_kernel<4, 1, false>, many_grid, dim3(THREADS), F32Many::SMEM + plan, stream, a);
        if (rc == 0) rc = launch_dependent(shared_f32_kernel<2, 2, true>, few_grid, dim3(THREADS), F32Few::SMEM + plan, stream, a);
    } else {
#ifdef FSIE_SHARED_TC
        if (on_tcgen05) {
            CUtensorMap k_map, v_map;
            rc = tc::pages_map(k_map, k_pages, page_rows, page_size);
            if (rc == 0) rc = tc::pages_map(v_map, v_pages, page_rows, page_size);
            if (rc == 0) rc = launch_dependent(tc::shared_tc_kernel, many_grid, dim3(tc::THREADS), tc::SMEM + plan, stream, k_map, v_map, a);
        } else
#endif
            rc = launch_dependent(shared_many_kernel, many_grid, dim3(THREADS), ManyShape::SMEM + plan, stream, a);
        if (rc == 0) rc = launch_dependent(shared_few_kernel, few_grid, dim3(FewShape::THREADS), FewShape::SMEM + plan, stream, a);
    }
    if (rc != 0) return rc;
    const dim3 grid((unsigned)(((long long)places * heads + MERGE_WARPS - 1) / MERGE_WARPS));
    return dtype == DTYPE_F32 ? launch_dependent(shared_merge_kernel<float, F32_KEYS>, grid, dim3(32 * MERGE_WARPS), 0, stream, a)
                              : launch_dependent(shared_merge_kernel<bf16, MMA_FEW_KEYS>, grid, dim3(32 * MERGE_WARPS), 0, stream, a);
}

}  // extern "C"
