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
#include <math.h>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head size: 16..256 in steps of 16");

namespace fsie {

constexpr int HD = HEAD_DIM;
constexpr int MMA_KEYS = 64;             // keys of a step
constexpr int F32_KEYS = HD <= 128 ? 64 : 32;                         // (two steps' keys and values fit in shared memory)
constexpr int F32_FEW = HD <= 128 ? 8 : 16;                           // rows that count as few; at 32 keys two warps share a step's
constexpr int THREADS = 128;
constexpr int MAX_RUNS = 1024;
constexpr int RUN_INTS = 6;
constexpr int LINE_PIECES = 48;          // a line is cut into no more pieces than this: what joins them reads them all
constexpr int LEAST_STEPS = 2;           // steps of a piece, at least
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
    int heads, kv_heads; float scale;
    int* few_table; int* many_table;                          // the launches' schedules, for the merge: [2 + 2 * run_count]
    float* part_ml; float* part_o;                            // [rows, 2], [rows, HD]
    int few_rows, many_rows;                                  // rows for the triples of either launch, few's in front
    int early;                                                // the lists are older than the stream's last kernel
    int* error;
};

struct Run { int first, count, begin, end, table, innermost; };

// Rows and tiles of a run under a split into FEW (tiles of up to few rows) and MANY.
struct RunTiles { int per_token; int rows; int tiles; };      // rows of a token's or of the run's tiles; tiles in all

template <int FEW, int ROWS, bool IS_FEW>
__device__ __forceinline__ bool run_tiles(const Run& run, int group, RunTiles& t) {
    t.per_token = run.innermost;
    t.rows = run.innermost ? group : run.count * group;
    if ((t.rows <= FEW) != IS_FEW) return false;
    t.tiles = (t.rows + ROWS - 1) / ROWS * (run.innermost ? run.count : 1);
    return true;
}

// A run as the lists give it, with innermost set; false (and *error) where it points outside of what there is.
__device__ __forceinline__ bool load_run(const SharedArgs& a, int r, Run& run) {
    const int* p = a.runs + (size_t)r * RUN_INTS;
    run.first = p[0]; run.count = p[1]; run.begin = p[2]; run.end = p[3]; run.table = p[4];
    if (run.count <= 0 || run.end <= run.begin) { run.count = 0; return true; }
    if (run.first < 0 || run.first > a.places - run.count || run.count > a.places || run.begin < 0 ||
        run.end > (long long)a.table_width * a.page_size || (unsigned)run.table >= (unsigned)a.table_rows || p[5] < -1 || p[5] >= r) {
        atomicExch(a.error, ERR_RUNS);
        run.count = 0;
        return false;
    }
    run.innermost = a.own_run[run.first] == r;
    return true;
}

// ---- the schedule, in every block's shared memory: steps and lines in front of each run
struct Schedule {
    int step0[MAX_RUNS + 1], line0[MAX_RUNS + 1];
    long long warp_steps[THREADS / 32]; int warp_lines[THREADS / 32], warp_longest[THREADS / 32];
    int piece;                           // steps of a block's piece
    int start_run;                       // the run in which this block's piece starts
};

template <int FEW, int ROWS, bool IS_FEW, int KEYS>
__device__ bool make_schedule(const SharedArgs& a, Schedule& s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.heads / a.kv_heads;
    long long steps_before = 0;
    int lines_before = 0, longest = 0;
    for (int base = 0; base < a.run_count; base += THREADS) {
        const int r = base + tid;
        long long steps = 0;
        int lines = 0;
        Run run;
        RunTiles t;
        if (r < a.run_count && load_run(a, r, run) && run.count > 0 && run_tiles<FEW, ROWS, IS_FEW>(run, group, t)) {
            const int of_line = (run.end - run.begin + KEYS - 1) / KEYS;
            lines = t.tiles * a.kv_heads;
            steps = (long long)lines * of_line;
            longest = max(longest, of_line);
        }
        long long steps_upto = steps;
        int lines_upto = lines;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long su = __shfl_up_sync(0xffffffffu, steps_upto, o);
            const int lu = __shfl_up_sync(0xffffffffu, lines_upto, o);
            if (lane >= o) { steps_upto += su; lines_upto += lu; }
        }
        if (lane == 31) { s.warp_steps[warp] = steps_upto; s.warp_lines[warp] = lines_upto; }
        __syncthreads();
        for (int w = 0; w < warp; ++w) { steps_upto += s.warp_steps[w]; lines_upto += s.warp_lines[w]; }
        steps_upto += steps_before; lines_upto += lines_before;
        if (r < a.run_count) {
            s.step0[r] = (int)min(steps_upto - steps, 0x7fffffffLL);
            s.line0[r] = lines_upto - lines;
        }
        for (int w = 0; w < THREADS / 32; ++w) { steps_before += s.warp_steps[w]; lines_before += s.warp_lines[w]; }
        __syncthreads();
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) s.warp_longest[warp] = longest;
    if (tid == 0) { s.step0[a.run_count] = (int)min(steps_before, 0x7fffffffLL); s.line0[a.run_count] = lines_before; }
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) longest = max(longest, s.warp_longest[w]);
    const int blocks = gridDim.x;
    const long long piece = max((steps_before + blocks - 1) / blocks, (long long)max(LEAST_STEPS, (longest + LINE_PIECES - 1) / LINE_PIECES));
    const int room = IS_FEW ? a.few_rows : a.many_rows;
    const bool fits = steps_before < 0x7fffffffLL && ((long long)lines_before + blocks) * ROWS <= room;
    if (tid == 0) s.piece = (int)piece;
    // what the merge has to know (a piece of 0: nothing was done)
    if (blockIdx.x == 0) {
        int* table = IS_FEW ? a.few_table : a.many_table;
        if (tid == 0) { table[0] = fits ? (int)piece : 0; table[1] = fits ? (int)steps_before : 0; }
        for (int r = tid; r < a.run_count; r += THREADS) { table[2 + 2 * r] = s.step0[r]; table[3 + 2 * r] = s.line0[r]; }
    }
    if (!fits) {
        if (tid == 0) atomicExch(a.error, ERR_ROOM);
        return false;
    }
    const long long from = (long long)blockIdx.x * piece;
    if (from >= steps_before) return false;
    for (int r = tid; r < a.run_count; r += THREADS)
        if (s.step0[r] <= from && from < s.step0[r + 1]) s.start_run = r;
    __syncthreads();
    return true;
}

// ---- one step of a block's walk: KEYS keys of a line
struct Step {
    int valid, first, last;              // whether there is one; first or last of the block's stretch of the line
    int k0, kend, table, kvh;
    int place, row0, rows;               // the tile's rows are rows row0 .. of the tokens from `place` on
    int slot;                            // where the stretch's triple goes, in tiles of ROWS rows
    int outer;                           // a run whose tokens must all see all of its keys
    int stretch;                         // how many stretches the block has begun before
};

template <int FEW, int ROWS, bool IS_FEW, int KEYS>
struct Walker {
    int run_index, line, of_line, i, i_end, at, end, stretches, kend;
    Run run;
    RunTiles tiles;

    // (one thread of the block)
    __device__ void start(const SharedArgs& a, const Schedule& s) {
        at = (int)min((long long)blockIdx.x * s.piece, 0x7fffffffLL);
        end = (int)min((long long)at + s.piece, (long long)s.step0[a.run_count]);
        run_index = s.start_run;
        stretches = 0;
        enter_run(a);
        const int inside = at - s.step0[run_index];
        line = inside / of_line;
        i = inside - line * of_line;
        i_end = min(of_line, i + (end - at));
    }
    __device__ void enter_run(const SharedArgs& a) {
        load_run(a, run_index, run);
        run_tiles<FEW, ROWS, IS_FEW>(run, a.heads / a.kv_heads, tiles);
        of_line = (run.end - run.begin + KEYS - 1) / KEYS;
        line = i = 0;
    }
    __device__ void next(const SharedArgs& a, const Schedule& s, Step& out) {
        if (at >= end) { out.valid = 0; return; }
        const bool first = i == 0 || at == (int)((long long)blockIdx.x * s.piece);
        const int tile = line / a.kv_heads, group = a.heads / a.kv_heads;
        const int per_token = (tiles.rows + ROWS - 1) / ROWS;             // tiles of the run, or of one of its tokens
        const int part = tiles.per_token ? tile % per_token : tile;
        out.valid = 1; out.first = first; out.last = i + 1 == i_end;
        out.kvh = line - tile * a.kv_heads;
        out.place = run.first + (tiles.per_token ? tile / per_token : part * ROWS / group);
        out.row0 = tiles.per_token ? part * ROWS : part * ROWS % group;
        out.rows = min(ROWS, tiles.rows - part * ROWS);
        out.k0 = run.begin + i * KEYS;
        if (first) {
            kend = run.end;
            if (tiles.per_token) {
                const int token = a.order[out.place];
                if ((unsigned)token < (unsigned)a.tokens) kend = min(kend, a.positions[token] + 1);
            }
        }
        out.kend = kend; out.table = run.table; out.outer = !tiles.per_token;
        out.slot = s.line0[run_index] + line + blockIdx.x;
        out.stretch = stretches;
        ++at; ++i;
        if (i < i_end) return;
        ++stretches;
        if (at >= end) return;
        if (++line < tiles.tiles * a.kv_heads) {
            i = 0;
        } else {
            do ++run_index; while (s.step0[run_index + 1] == s.step0[run_index]);
            enter_run(a);
        }
        i_end = min(of_line, end - at);
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

// ---- what both storage types share: the ring of steps, and their keys and query rows on the way
template <typename T, int FEW, int ROWS, bool IS_FEW, int KEYS, int STAGES, int K_LD, int V_LD, int Q_LD>
struct Feed {
    static constexpr int PIECES = HD * (int)sizeof(T) / 16;               // 16-byte pieces of a head
    static constexpr int EACH = 16 / (int)sizeof(T);
    static constexpr int RECORDS = STAGES + 2, BASES = STAGES + 1;
    struct Shared {
        Schedule schedule;
        Step steps[RECORDS];
        long long key_base[BASES][KEYS];                                  // element offset of a key's row in the pages; -1: no key
    };
    const SharedArgs& a;
    Shared& sh;
    T *ks, *vs, *qs;
    Walker<FEW, ROWS, IS_FEW, KEYS> walker;                                     // thread 0's

    __device__ Feed(const SharedArgs& args, Shared& shared, T* k, T* v, T* q) : a(args), sh(shared), ks(k), vs(v), qs(q) {}

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
                const int group = a.heads / a.kv_heads;
                T* qd = qs + (size_t)(st.stretch % STAGES) * ROWS * Q_LD;
                const T* q = (const T*)a.q;
                for (int e = threadIdx.x; e < ROWS * PIECES; e += THREADS) {
                    const int r = e / PIECES, c = (e - r * PIECES) * EACH;
                    bool ok = r < st.rows;
                    long long at = 0;
                    if (ok) {
                        const int row = st.row0 + r, token = a.order[st.place + row / group];
                        ok = (unsigned)token < (unsigned)a.tokens;
                        // a shared run ends in front of its tokens
                        if (ok && st.outer && a.positions[token] + 1 < st.kend) atomicExch(a.error, ERR_RUNS);
                        if (ok) at = (long long)token * a.q_ld + (st.kvh * group + row % group) * HD + c;
                        else atomicExch(a.error, ERR_RUNS);
                    }
                    copy16(qd + r * Q_LD + c, q + at, ok);
                }
            }
        }
        copies_commit();
    }
    // Schedule and first steps; false: nothing to do.  The launch of the many rows comes first and waits for the kernel in
    // front of it.  That of the few rows reads nothing that the many's wrote, and starts when all of its blocks have waited:
    // it works beside it and waits when it is done, so that the merge behind it finds both done.
    __device__ bool start() {
        if (!IS_FEW && !a.early) grid_dependency_wait();
        const bool any = make_schedule<FEW, ROWS, IS_FEW, KEYS>(a, sh.schedule);
        if (any) {
            if (threadIdx.x == 0) {
                walker.start(a, sh.schedule);
                for (int n = 0; n <= STAGES; ++n) walker.next(a, sh.schedule, sh.steps[n]);
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
        if (threadIdx.x == 0) walker.next(a, sh.schedule, sh.steps[(n + STAGES + 1) % RECORDS]);
    }
    __device__ const Step& step(int n) const { return sh.steps[n % RECORDS]; }
};

// ------------------------------------------------------------------------------------------------ bfloat16
// WARPS_M x WARPS_K warps: warp (wm, wk) has rows 16 wm .. and, of a step, the scores of KEYS / WARPS_K keys; the warps wk
// exchange the rows' maxima and the weights through shared memory, and each sums up its share of the head's columns over
// all keys, so that a stretch's result needs no joining.
template <int WARPS_M, int WARPS_K, int STAGES>
struct MmaShape {
    static constexpr int ROWS = 16 * WARPS_M, KEYS = MMA_KEYS;
    static constexpr int LD = HD + 8;                    // padded rows: ldmatrix without bank conflicts
    static constexpr int P_LD = KEYS + 8;
    static constexpr int KPW = KEYS / WARPS_K, NT = KPW / 8;
    static constexpr int PAIRS = (HD / 16 + WARPS_K - 1) / WARPS_K;       // 16-column pieces of the head per warp
    static constexpr bool IS_FEW = WARPS_M == 1;
    using F = Feed<bf16, 16, ROWS, IS_FEW, KEYS, STAGES, LD, LD, LD>;
    static constexpr size_t TILE = (size_t)KEYS * LD * sizeof(bf16);
    static constexpr size_t Q = (size_t)ROWS * LD * sizeof(bf16);
    static constexpr size_t P = WARPS_K > 1 ? (size_t)ROWS * P_LD * sizeof(bf16) : 0;
    static constexpr size_t SMEM = STAGES * (2 * TILE + Q) + P + sizeof(typename F::Shared) + 2 * WARPS_K * ROWS * sizeof(float);
};

template <int WARPS_M, int WARPS_K, int STAGES>
__global__ void __launch_bounds__(THREADS)
shared_mma_kernel(const SharedArgs a) {
    using S = MmaShape<WARPS_M, WARPS_K, STAGES>;
    constexpr int KEYS = S::KEYS;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* ks = reinterpret_cast<bf16*>(smem);
    bf16* vs = ks + (size_t)STAGES * KEYS * S::LD;
    bf16* qs = vs + (size_t)STAGES * KEYS * S::LD;
    bf16* ps = qs + (size_t)STAGES * S::ROWS * S::LD;
    float* row_max = reinterpret_cast<float*>(ps + S::P / sizeof(bf16));  // [WARPS_K][ROWS]
    float* row_sum = row_max + WARPS_K * S::ROWS;
    typename S::F::Shared& sh = *reinterpret_cast<typename S::F::Shared*>(row_sum + WARPS_K * S::ROWS);
    typename S::F feed(a, sh, ks, vs, qs);
    if (!feed.start()) return;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = warp / WARPS_K, wk = warp % WARPS_K;
    const int g = lane >> 2, t = lane & 3;
    const int r_lo = wm * 16 + g, r_hi = r_lo + 8;
    const float sc = a.scale * LOG2E;                     // scores in base-2 units
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;
    float o[2 * S::PAIRS][4];
    constexpr bool Q_IN_REGS = HD <= 128;
    unsigned qf[Q_IN_REGS ? HD / 16 : 1][4];

    for (int n = 0; feed.step(n).valid; ++n) {
        feed.advance(n);
        const Step st = feed.step(n);
        const bf16* q_at = qs + (size_t)(st.stretch % STAGES) * S::ROWS * S::LD +
                           (wm * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * S::LD + 8 * (lane >> 4);
        if (st.first) {
            m_lo = m_hi = -INFINITY; l_lo = l_hi = 0.f;
#pragma unroll
            for (int c = 0; c < 2 * S::PAIRS; ++c) { o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f; }
            if (Q_IN_REGS) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) ldmatrix_x4(qf[k], q_at + k * 16);
            }
        }
        const bf16* kt = ks + (size_t)(n % STAGES) * KEYS * S::LD + (size_t)wk * S::KPW * S::LD;
        const bf16* vt = vs + (size_t)(n % STAGES) * KEYS * S::LD;
        // ---- scores of this warp's keys
        float s[S::NT][4];
#pragma unroll
        for (int c = 0; c < S::NT; ++c) { s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f; }
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            unsigned q4[4];
            if (Q_IN_REGS) { q4[0] = qf[k][0]; q4[1] = qf[k][1]; q4[2] = qf[k][2]; q4[3] = qf[k][3]; }
            else ldmatrix_x4(q4, q_at + k * 16);
#pragma unroll
            for (int c = 0; c < S::NT / 2; ++c) {
                unsigned b[4];
                ldmatrix_x4(b, kt + (c * 16 + (lane & 7) + 8 * (lane >> 4)) * S::LD + k * 16 + 8 * ((lane >> 3) & 1));
                mma_bf16(s[2 * c], q4, b[0], b[1]);
                mma_bf16(s[2 * c + 1], q4, b[2], b[3]);
            }
        }
        // ---- keys that are not there (behind the end; a page that is none)
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
        const long long* base = sh.key_base[n % S::F::BASES] + wk * S::KPW;
#pragma unroll
        for (int c = 0; c < S::NT; ++c) {
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
        if constexpr (WARPS_K > 1) {
            if (t == 0) { row_max[wk * S::ROWS + r_lo] = mx_lo; row_max[wk * S::ROWS + r_hi] = mx_hi; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WARPS_K; ++w) {
                mx_lo = fmaxf(mx_lo, row_max[w * S::ROWS + r_lo]);
                mx_hi = fmaxf(mx_hi, row_max[w * S::ROWS + r_hi]);
            }
        }
        const float mn_lo = fmaxf(m_lo, mx_lo), mn_hi = fmaxf(m_hi, mx_hi);
        const float base_lo = mn_lo == -INFINITY ? 0.f : mn_lo * sc, base_hi = mn_hi == -INFINITY ? 0.f : mn_hi * sc;
        const float corr_lo = exp2f(m_lo * sc - base_lo), corr_hi = exp2f(m_hi * sc - base_hi);
        m_lo = mn_lo; m_hi = mn_hi;
        float sum_lo = 0.f, sum_hi = 0.f;
#pragma unroll
        for (int c = 0; c < S::NT; ++c) {
            s[c][0] = exp2f(s[c][0] * sc - base_lo); s[c][1] = exp2f(s[c][1] * sc - base_lo);
            s[c][2] = exp2f(s[c][2] * sc - base_hi); s[c][3] = exp2f(s[c][3] * sc - base_hi);
            sum_lo += s[c][0] + s[c][1];
            sum_hi += s[c][2] + s[c][3];
        }
        l_lo = l_lo * corr_lo + sum_lo;                   // of this thread's keys; the threads' sums meet at the end
        l_hi = l_hi * corr_hi + sum_hi;
        if (__any_sync(0xffffffffu, corr_lo != 1.f || corr_hi != 1.f)) {
#pragma unroll
            for (int c = 0; c < 2 * S::PAIRS; ++c) { o[c][0] *= corr_lo; o[c][1] *= corr_lo; o[c][2] *= corr_hi; o[c][3] *= corr_hi; }
        }
        // ---- weighted values: the weights are rounded to bfloat16, as the values are; the sums l hold them unrounded
        if constexpr (WARPS_K > 1) {
#pragma unroll
            for (int c = 0; c < S::NT; ++c) {
                *reinterpret_cast<unsigned*>(ps + r_lo * S::P_LD + wk * S::KPW + c * 8 + 2 * t) = pack_bf16(s[c][0], s[c][1]);
                *reinterpret_cast<unsigned*>(ps + r_hi * S::P_LD + wk * S::KPW + c * 8 + 2 * t) = pack_bf16(s[c][2], s[c][3]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k) {
            unsigned p4[4];
            if constexpr (WARPS_K > 1) {
                ldmatrix_x4(p4, ps + (wm * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * S::P_LD + k * 16 + 8 * (lane >> 4));
            } else {
                p4[0] = pack_bf16(s[2 * k][0], s[2 * k][1]);
                p4[1] = pack_bf16(s[2 * k][2], s[2 * k][3]);
                p4[2] = pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]);
                p4[3] = pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3]);
            }
#pragma unroll
            for (int c = 0; c < S::PAIRS; ++c) {
                const int pair = wk + c * WARPS_K;
                if (HD / 16 % WARPS_K == 0 || pair < HD / 16) {
                    unsigned b[4];
                    ldmatrix_x4_trans(b, vt + (k * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * S::LD + pair * 16 + 8 * (lane >> 4));
                    mma_bf16(o[2 * c], p4, b[0], b[1]);
                    mma_bf16(o[2 * c + 1], p4, b[2], b[3]);
                }
            }
        }
        if (!st.last) continue;
        // ---- the stretch's triples
        l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1); l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
        l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1); l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
        if constexpr (WARPS_K > 1) {
            if (t == 0) { row_sum[wk * S::ROWS + r_lo] = l_lo; row_sum[wk * S::ROWS + r_hi] = l_hi; }
            __syncthreads();
            l_lo = l_hi = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS_K; ++w) { l_lo += row_sum[w * S::ROWS + r_lo]; l_hi += row_sum[w * S::ROWS + r_hi]; }
        }
        const size_t row = (S::IS_FEW ? 0 : (size_t)a.few_rows) + (size_t)st.slot * S::ROWS;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = half ? r_hi : r_lo;
            if (r >= st.rows) continue;
            float* dst = a.part_o + (row + r) * HD;
#pragma unroll
            for (int c = 0; c < 2 * S::PAIRS; ++c) {
                const int column = (wk + (c >> 1) * WARPS_K) * 16 + (c & 1) * 8 + 2 * t;
                if (HD / 16 % WARPS_K == 0 || column < HD)
                    *reinterpret_cast<float2*>(dst + column) = make_float2(o[c][2 * half], o[c][2 * half + 1]);
            }
            if (wk == 0 && t == 0) {
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
    using F = Feed<float, F32_FEW, ROWS, IS_FEW, KEYS, STAGES, K_LD, HD, HD>;
    static constexpr size_t SMEM = sizeof(float) * ((size_t)STAGES * KEYS * (K_LD + HD) + (size_t)STAGES * ROWS * HD + (size_t)ROWS * P_LD +
                                                    2 * WARPS_K * ROWS) + sizeof(typename F::Shared);
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
    typename S::F feed(a, sh, ks, vs, qs);
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

// --------------------------------------------------------------------------------------------------- merge
// A warp per (place, head): its lanes find the row's triples (each lane one, in turns of 32), the weights travel by
// shuffles, the columns are summed four per lane in the order of the triples.
constexpr int MERGE_WARPS = 4;

template <typename T, int FEW, int FEW_ROWS, int MANY_ROWS, int KEYS>
__global__ void __launch_bounds__(32 * MERGE_WARPS)
shared_merge_kernel(const SharedArgs a) {
    const int unit = blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads;
    const int place = unit / a.heads, h = unit - place * a.heads;
    int token = -1, own = -1;
    if (place < a.places) { token = a.order[place]; own = a.own_run[place]; }
    grid_dependency_wait();
    grid_dependents_go();
    if (place >= a.places) return;
    if ((unsigned)token >= (unsigned)a.tokens) {
        if (lane == 0) atomicExch(a.error, ERR_RUNS);
        return;
    }
    const int kvh = h / group, g = h - kvh * group;
    constexpr int CHUNKS = (HD / 4 + 31) / 32;
    float4 sum[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) sum[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, denom = 0.f;
    int r = own;
    if (own >= a.run_count || own < 0) r = -1;
    bool more = r >= 0;
    int skip = 0;                                         // triples of run r that earlier turns took
    while (more) {
        // ---- up to 32 triples: lane j finds the j-th
        long long mine = -1;
        int have = 0;
        while (r >= 0 && have < 32) {
            Run run;
            load_run(a, r, run);
            int count = 0;
            if (run.count > 0 && place >= run.first && place < run.first + run.count) {
                const int row_in = (run.innermost ? 0 : (place - run.first) * group) + g;
                const bool few = (run.innermost ? group : run.count * group) <= FEW;
                const int rows = few ? FEW_ROWS : MANY_ROWS;
                const int* table = few ? a.few_table : a.many_table;
                const int piece = table[0], steps = table[1], of_line = (run.end - run.begin + KEYS - 1) / KEYS;
                const int tile = (run.innermost ? (place - run.first) * ((group + rows - 1) / rows) : 0) + row_in / rows;
                const int line = tile * a.kv_heads + kvh;
                const long long from = (long long)table[2 + 2 * r] + (long long)line * of_line;
                if (piece > 0 && from + of_line <= steps) {
                    const int b0 = (int)(from / piece), b1 = (int)((from + of_line - 1) / piece);
                    count = b1 - b0 + 1;
                    const int j = lane - have + skip;
                    if (lane >= have && j < count)
                        mine = (few ? 0 : (long long)a.few_rows) + (long long)(table[3 + 2 * r] + line + b0 + j) * rows + row_in % rows;
                }
            }
            const int left = count - skip;
            if (left > 32 - have) { skip += 32 - have; have = 32; break; }
            have += left;
            skip = 0;
            const int parent = a.runs[(size_t)r * RUN_INTS + 5];
            r = parent < r ? parent : -1;
        }
        more = r >= 0;
        float m = -INFINITY, l = 0.f;
        if (mine >= 0) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + mine * 2);
            m = ml.x; l = ml.y;
        }
        const float top_new = fmaxf(top, warp_max(m));
        if (top_new == -INFINITY) continue;
        const float before = top == -INFINITY ? 0.f : expf(top - top_new);
        const float w = m == -INFINITY ? 0.f : expf(m - top_new);
        denom = denom * before + warp_sum(l * w);
        top = top_new;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) { sum[c].x *= before; sum[c].y *= before; sum[c].z *= before; sum[c].w *= before; }
        for (int j0 = 0; j0 < have; j0 += 8) {
            // eight triples' columns are asked for before the first is used
            float4 v[8][CHUNKS];
            float wj[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const long long at = __shfl_sync(0xffffffffu, mine, (j0 + j) & 31);
                wj[j] = __shfl_sync(0xffffffffu, w, (j0 + j) & 31);
                if (j0 + j >= have || at < 0) wj[j] = 0.f;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
                    if (wj[j] != 0.f && (HD / 4 % 32 == 0 || lane + 32 * c < HD / 4))
                        v[j][c] = *reinterpret_cast<const float4*>(a.part_o + at * HD + (lane + 32 * c) * 4);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (wj[j] != 0.f) {
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        sum[c].x = fmaf(wj[j], v[j][c].x, sum[c].x); sum[c].y = fmaf(wj[j], v[j][c].y, sum[c].y);
                        sum[c].z = fmaf(wj[j], v[j][c].z, sum[c].z); sum[c].w = fmaf(wj[j], v[j][c].w, sum[c].w);
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

using MmaFew = MmaShape<1, 4, 2>;
using MmaMany = MmaShape<4, 1, 2>;
constexpr int F32_FEW_M = F32_FEW / 8, F32_FEW_K = 4 / F32_FEW_M;
using F32Few = F32Shape<F32_FEW_M, F32_FEW_K, true>;
using F32Many = F32Shape<4, 1, false>;
static_assert(MmaFew::ROWS == 16 && F32Few::ROWS == F32_FEW && F32Few::JN >= 1, "tiles of few rows");

// blocks of `kernel` that the current device runs at once
template <typename K>
static int blocks_at_once(K kernel, size_t smem, int& blocks) {
    int device = 0, sms = 0, per_sm = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, THREADS, smem);
    blocks = sms * per_sm;
    return e != cudaSuccess ? (int)e : blocks > 0 ? 0 : (int)ERR_UNSUPPORTED;
}

constexpr long long TABLE_BYTES = 2 * (2 + 2 * MAX_RUNS) * 4;       // both schedules, in front of the triples
static_assert(TABLE_BYTES % 16 == 0, "the triples start on 16 bytes");
struct Launch { int few_blocks, many_blocks; };
constexpr int MAX_DEVICES = 64;

static int launch_shape(int dtype, Launch& shape) {
    static Launch known[2][MAX_DEVICES] = {};            // per process; the same whoever writes it
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (device < 0 || device >= MAX_DEVICES) return ERR_UNSUPPORTED;
    Launch& have = known[dtype == DTYPE_BF16][device];
    if (have.many_blocks == 0) {
        Launch found;
        int rc = dtype == DTYPE_BF16 ? blocks_at_once(shared_mma_kernel<1, 4, 2>, MmaFew::SMEM, found.few_blocks)
                                     : blocks_at_once(shared_f32_kernel<F32_FEW_M, F32_FEW_K, true>, F32Few::SMEM, found.few_blocks);
        if (rc == 0)
            rc = dtype == DTYPE_BF16 ? blocks_at_once(shared_mma_kernel<4, 1, 2>, MmaMany::SMEM, found.many_blocks)
                                     : blocks_at_once(shared_f32_kernel<4, 1, false>, F32Many::SMEM, found.many_blocks);
        if (rc != 0) return rc;
        have = found;
    }
    shape = have;
    return 0;
}

// Rows of triples that the two launches may need.  Innermost runs are tiled token by token, other runs of few rows have a
// tile each; the many-row tiles of the runs around a token are at most `levels` deep.
static void rows_needed(int dtype, const Launch& shape, long long places, long long runs, int heads, int kv_heads, int levels,
                        long long& few, long long& many) {
    const int few_rows = dtype == DTYPE_BF16 ? MmaFew::ROWS : F32Few::ROWS, many_rows = dtype == DTYPE_BF16 ? MmaMany::ROWS : F32Many::ROWS;
    const long long group = heads / kv_heads;
    few = ((places + runs) * kv_heads + shape.few_blocks) * few_rows;
    long long tiles = levels * ((places * group + many_rows - 1) / many_rows) + runs;
    if (group > few_rows) tiles += places * ((group + many_rows - 1) / many_rows);
    many = (tiles * kv_heads + shape.many_blocks) * many_rows;
}

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
    Launch shape;
    const int rc = launch_shape(dtype, shape);
    if (rc != 0) return rc > 0 ? -1000 - rc : rc;
    long long few, many;
    rows_needed(dtype, shape, places, runs, heads, kv_heads, levels, few, many);
    return (few + many) * (HD + 2) * 4 + TABLE_BYTES;
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
    Launch shape;
    int rc = launch_shape(dtype, shape);
    if (rc != 0) return rc;
    long long few, many;
    rows_needed(dtype, shape, places, run_count, heads, kv_heads, 0, few, many);
    const long long tables = TABLE_BYTES;
    const long long rows = (room_bytes - tables) / ((HD + 2) * 4);
    if (rows - few < many || few > 0x7fffffffLL) return ERR_BAD_ARGUMENT;
    SharedArgs a;
    a.q = q; a.q_ld = q_ld; a.k_pages = k_pages; a.v_pages = v_pages; a.page_stride = page_stride; a.page_size = page_size;
    a.num_pages = num_pages; a.block_tables = block_tables; a.table_rows = table_rows; a.table_width = table_width;
    a.positions = positions; a.tokens = tokens; a.order = order; a.places = places; a.runs = runs; a.run_count = run_count;
    a.own_run = own_run; a.out = out; a.out_ld = out_ld; a.heads = heads; a.kv_heads = kv_heads; a.scale = scale;
    a.few_table = (int*)room; a.many_table = a.few_table + 2 + 2 * MAX_RUNS;
    a.few_rows = (int)few; a.many_rows = (int)min(rows - few, 0x7fffffffLL);
    a.part_o = reinterpret_cast<float*>((unsigned char*)room + tables);
    a.part_ml = a.part_o + (few + a.many_rows) * HD;
    a.early = early; a.error = error;
    if (dtype == DTYPE_BF16) {
        rc = launch_dependent(shared_mma_kernel<4, 1, 2>, dim3(shape.many_blocks), dim3(THREADS), MmaMany::SMEM, stream, a);
        if (rc == 0) rc = launch_dependent(shared_mma_kernel<1, 4, 2>, dim3(shape.few_blocks), dim3(THREADS), MmaFew::SMEM, stream, a);
    } else {
        rc = launch_dependent(shared_f32_kernel<4, 1, false>, dim3(shape.many_blocks), dim3(THREADS), F32Many::SMEM, stream, a);
        if (rc == 0) rc = launch_dependent(shared_f32_kernel<F32_FEW_M, F32_FEW_K, true>, dim3(shape.few_blocks), dim3(THREADS), F32Few::SMEM, stream, a);
    }
    if (rc != 0) return rc;
    const dim3 grid((unsigned)(((long long)places * heads + MERGE_WARPS - 1) / MERGE_WARPS));
    return dtype == DTYPE_BF16
               ? launch_dependent(shared_merge_kernel<bf16, 16, MmaFew::ROWS, MmaMany::ROWS, MMA_KEYS>, grid, dim3(32 * MERGE_WARPS), 0, stream, a)
               : launch_dependent(shared_merge_kernel<float, F32_FEW, F32Few::ROWS, F32Many::ROWS, F32_KEYS>, grid, dim3(32 * MERGE_WARPS), 0, stream, a);
}

}  // extern "C"
