// Pages of a paged KV cache that several rows of a table may hold: forked, extended, given back, moved together and copied.
//
// refs[p] counts the rows that hold page p; 0: free.  All of it stays on the GPU: the calls read lengths, counts and tables there and
// write them there, so that a step of a search needs no answer on the host and can be captured.  What is taken is always the free page of
// the lowest number, for rows in their order, so results do not depend on the order in which blocks run: counts change by atomic
// additions, whose sum has no order, and everything else is decided from prefix sums.
//
// Work on tables is bound by latency: some hundred kilobytes, and a chain of a few dependent reads.  Prefix sums over all pages and rows are made by one
// block, or, of large caches, by one cluster, whose blocks tell one another their totals through distributed shared memory: one launch, and no second pass over a
// grid.  Launches of one call start under those in front of them.  Copies are bound by memory: 16 bytes a thread, four in flight (1.1 GB moved in 181 us, 6.3 TB/s).
#include "cg_common.cuh"

namespace cg {
namespace {

constexpr int kClusterBlocks = 8, kClusterThreads = 512, kClusterWarps = kClusterThreads / 32;
constexpr int kRowThreads = 256, kRowColumns = 1024;  // of a block that works on a row of a table
constexpr int kCopyThreads = 256, kCopyVectors = 4;
constexpr int64_t kAlonePages = 8192;  // up to here, and with a row a thread, one block does (8 rows in 2,600 pages extended: 6 us, by eight blocks 9 to 11)
constexpr int32_t kSlotsTogether = 2 * kClusterBlocks * kClusterThreads;
constexpr int64_t kMostPages = INT32_MAX - 1024;  // a warp counts on behind its last page, and a block behind its last column of a row

struct Table {
    const int32_t *entries, *lens;
    int64_t row;  // entries from one row to the next
    int32_t rows, width, page_size;
    int32_t num_pages;
    int32_t *status;
};

__device__ __forceinline__ void note(int32_t *status, int32_t what) {
    if (status) atomicOr(status, what);
}
__device__ __forceinline__ int64_t index_at(const void *p, int64_t i, int wide) {
    return wide ? __ldg(static_cast<const long long *>(p) + i) : __ldg(static_cast<const int *>(p) + i);
}
// Tokens of a row; a length that its table cannot hold is cut.
__device__ __forceinline__ int32_t length_of(const Table &t, int row) {
    const int64_t n = t.lens[row], most = static_cast<int64_t>(t.width) * t.page_size;
    if (n >= 0 && n <= most) return static_cast<int32_t>(n);
    note(t.status, CG_S_BAD_PAGE);
    return n < 0 ? 0 : static_cast<int32_t>(most);
}
__device__ __forceinline__ int32_t pages_of(int64_t tokens, int32_t page_size) { return static_cast<int32_t>((tokens + page_size - 1) / page_size); }
// A page that a row holds, or -1 for one that the cache does not have.
__device__ __forceinline__ int32_t page_at(const Table &t, int row, int column) {
    const int32_t p = t.entries[row * t.row + column];
    if (p >= 0 && p < t.num_pages) return p;
    note(t.status, CG_S_BAD_PAGE);
    return -1;
}

// ---- sums over a cluster ----------------------------------------------------------------------------
// BLOCKS of kClusterThreads threads, one or kClusterBlocks: a block alone needs no steps between blocks, of 2 us in all, and is enough for most caches.
template <int BLOCKS> __device__ __forceinline__ int cluster_rank() {
    int r = 0;
    if (BLOCKS > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Everything that the cluster's threads wrote, to whatever memory, is there for all of them afterwards.
template <int BLOCKS> __device__ __forceinline__ void cluster_barrier() {
    if (BLOCKS > 1) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
}
template <int BLOCKS> __device__ __forceinline__ int64_t of_block(const int64_t *mine, int rank) {
    if (BLOCKS == 1) return *mine;
    uint32_t at;
    int64_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}
template <class T> __device__ __forceinline__ T sum_upto(T x) {  // over the warp's lanes up to this one
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const T y = __shfl_up_sync(~0u, x, d);
        if (static_cast<int>(threadIdx.x & 31) >= d) x += y;
    }
    return x;
}
// Room of a block for the sums: its warps' numbers, its own for the other blocks, and what the blocks in front and all of them have.
struct Told {
    int64_t a[kClusterWarps], b[kClusterWarps], block[2], front[2], all[2];
};
struct Sums {  // in front of this warp, and of all warps
    int64_t a, b, all_a, all_b;
};
// Sums over the cluster's warps of two numbers of each.  One warp of a block asks the other blocks: with every warp asking for every number it took 10,000 cycles.
// A barrier of the cluster stands in it.
template <int BLOCKS> __device__ __forceinline__ Sums over_warps(int64_t a, int64_t b, Told *told) {
    static_assert(kClusterWarps <= 32 && BLOCKS <= 32, "a lane each");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) told->a[warp] = a, told->b[warp] = b;
    __syncthreads();
    const int64_t x = lane < kClusterWarps ? told->a[lane] : 0, y = lane < kClusterWarps ? told->b[lane] : 0;
    const int64_t upto_x = sum_upto(x), upto_y = sum_upto(y);
    Sums s{__shfl_sync(~0u, upto_x - x, warp), __shfl_sync(~0u, upto_y - y, warp), __shfl_sync(~0u, upto_x, 31), __shfl_sync(~0u, upto_y, 31)};
    if (BLOCKS == 1) return s;
    if (threadIdx.x == 0) told->block[0] = s.all_a, told->block[1] = s.all_b;
    cluster_barrier<BLOCKS>();
    if (warp == 0) {
        const int64_t p = lane < BLOCKS ? of_block<BLOCKS>(&told->block[0], lane) : 0, q = lane < BLOCKS ? of_block<BLOCKS>(&told->block[1], lane) : 0;
        const int64_t upto_p = sum_upto(p), upto_q = sum_upto(q);
        if (lane == cluster_rank<BLOCKS>()) told->front[0] = upto_p - p, told->front[1] = upto_q - q;
        if (lane == 31) told->all[0] = upto_p, told->all[1] = upto_q;
    }
    __syncthreads();
    s.a += told->front[0], s.b += told->front[1];
    s.all_a = told->all[0], s.all_b = told->all[1];
    return s;
}

// Steps of a warp: for small caches of four pages a lane, so that more warps have some, else of sixteen.
template <int BLOCKS> constexpr int32_t kQuads = BLOCKS > 1 ? 4 : 1;
template <int BLOCKS> constexpr int32_t kRunStep = 128 * kQuads<BLOCKS>;
// A warp's run of pages, [first, last); runs of warps and blocks follow one another.
struct Run {
    int32_t first, last;
};
template <int BLOCKS> __device__ __forceinline__ Run run_of(int32_t num_pages) {
    constexpr int kAll = BLOCKS * kClusterWarps;
    const int64_t run = ((static_cast<int64_t>(num_pages) + kAll - 1) / kAll + kRunStep<BLOCKS> - 1) / kRunStep<BLOCKS> * kRunStep<BLOCKS>;
    const int64_t first = (cluster_rank<BLOCKS>() * kClusterWarps + static_cast<int>(threadIdx.x >> 5)) * run, last = first + run;
    return Run{static_cast<int32_t>(first < num_pages ? first : num_pages), static_cast<int32_t>(last < num_pages ? last : num_pages)};
}
// The counts of a lane's pages of a step that begins at p0, four by four `apart` pages from one another; `behind` for those behind the run.  Whole steps are loaded
// without a branch in between, all at once.
template <int QUADS>
__device__ __forceinline__ void counts_of(const int32_t *refs, int32_t p, int32_t apart, const Run &run, int32_t p0, bool vectors, int32_t behind, int4 (&c)[QUADS]) {
    if (vectors && p0 <= run.last - 128 * QUADS) {
#pragma unroll
        for (int i = 0; i < QUADS; ++i) c[i] = *reinterpret_cast<const int4 *>(refs + p + i * apart);
        return;
    }
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
        const int32_t q = p + i * apart;
        c[i].x = q < run.last ? refs[q] : behind;
        c[i].y = q < run.last - 1 ? refs[q + 1] : behind;
        c[i].z = q < run.last - 2 ? refs[q + 2] : behind;
        c[i].w = q < run.last - 3 ? refs[q + 3] : behind;
    }
}
template <int QUADS> __device__ __forceinline__ int32_t zeros(const int4 (&c)[QUADS]) {
    int32_t n = 0;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) n += (c[i].x == 0) + (c[i].y == 0) + (c[i].z == 0) + (c[i].w == 0);
    return n;
}
template <int BLOCKS> __device__ __forceinline__ int32_t free_in(const int32_t *refs, const Run &run, bool vectors) {
    int32_t n = 0;
#pragma unroll 2
    for (int32_t p0 = run.first; p0 < run.last; p0 += kRunStep<BLOCKS>) {
        int4 c[kQuads<BLOCKS>];
        counts_of(refs, p0 + 4 * static_cast<int32_t>(threadIdx.x & 31), 128, run, p0, vectors, 1, c);
        n += zeros(c);
    }
    return __reduce_add_sync(~0u, n);
}

// Writes the numbers of the first free pages to `list`, in order, as many as the cluster's threads want together (`wanted` is this
// thread's), if there are so many.  Returns the sum of what the threads before this one want; free_pages: how many there are.
// Barriers of the cluster stand between its reads of the counts and its end.
template <int BLOCKS>
__device__ __forceinline__ int64_t take_free(const int32_t *refs, int32_t num_pages, int64_t wanted, int32_t *list, Told *told, int64_t *wanted_all,
                                             int64_t *free_pages) {
    const Run run = run_of<BLOCKS>(num_pages);
    const bool vectors = reinterpret_cast<uintptr_t>(refs) % 16 == 0;
    const int32_t free = free_in<BLOCKS>(refs, run, vectors);
    const int64_t upto = sum_upto(wanted);
    const Sums s = over_warps<BLOCKS>(free, __shfl_sync(~0u, upto, 31), told);
    const int32_t most = static_cast<int32_t>(s.all_b < num_pages ? s.all_b : num_pages);
    int32_t rank = static_cast<int32_t>(s.a);
    if (free && rank < most) {
        for (int32_t p0 = run.first; p0 < run.last && rank < most; p0 += kRunStep<BLOCKS>) {  // neighbouring pages a lane
            const int32_t p = p0 + 4 * kQuads<BLOCKS> * static_cast<int32_t>(threadIdx.x & 31);
            int4 c[kQuads<BLOCKS>];
            counts_of(refs, p, 4, run, p0, vectors, 1, c);
            const int32_t mine = zeros(c);
            const int32_t before = sum_upto(mine);
            int32_t at = rank + before - mine;
            const auto put = [&](int32_t count, int32_t page) {
                if (count == 0 && at < most) list[at] = page;
                at += count == 0;
            };
#pragma unroll
            for (int i = 0; i < kQuads<BLOCKS>; ++i) put(c[i].x, p + 4 * i), put(c[i].y, p + 4 * i + 1), put(c[i].z, p + 4 * i + 2), put(c[i].w, p + 4 * i + 3);
            rank += __shfl_sync(~0u, before, 31);
        }
    }
    cluster_barrier<BLOCKS>();
    *wanted_all = s.all_b, *free_pages = s.all_a;
    return s.b + upto - wanted;
}

// ---- fork ----------------------------------------------------------------------------------------------
struct Writers {  // of a page that new rows would go on writing to
    int32_t first, count;
};
struct ForkArgs {
    Table old;
    int32_t *table, *lens, *refs, *moves;  // of the new rows; moves [3][nnew]
    const void *parents;
    Writers *writers;  // [num_pages], of the pages that matter
    int32_t *list;     // [nnew]
    int32_t *copies;   // how many
    int64_t row;
    int32_t nnew, wide, release;
};

// Columns column0 + first, + step .. below column1 of a row: the new row's entries, and the counts' changes.  Where a new row holds what the old one of its place
// held, as rows of one request do in the context that they share, nothing changes and no atomic is issued.
__device__ __forceinline__ void fork_row(const ForkArgs &a, int32_t row, int32_t column0, int32_t column1, int32_t first, int32_t step) {
    int64_t parent = -1;
    if (row < a.nnew) {
        parent = index_at(a.parents, row, a.wide);
        if (parent < -1 || parent >= a.old.rows) {
            if (first == 0) note(a.old.status, CG_S_BAD_PAGE);
            parent = -1;
        }
    }
    const int32_t tokens = parent >= 0 ? length_of(a.old, static_cast<int>(parent)) : 0, need = pages_of(tokens, a.old.page_size);
    const int32_t had = a.release && row < a.old.rows ? pages_of(length_of(a.old, row), a.old.page_size) : 0;
    if (row < a.nnew && column0 == 0 && first == 0) a.lens[row] = tokens;
    const int32_t last = tokens % a.old.page_size ? need - 1 : -1;  // the column of a page that is not full
    for (int32_t j = column0 + first; j < column1; j += step) {
        const int32_t now = j < need ? page_at(a.old, static_cast<int>(parent), j) : -1, before = j < had ? page_at(a.old, row, j) : -1;
        if (row < a.nnew) a.table[row * a.row + j] = now;
        if (now != before) {
            if (now >= 0) atomicAdd(a.refs + now, 1);
            if (before >= 0) atomicAdd(a.refs + before, -1);
        }
        if (j == last && now >= 0) a.writers[now] = Writers{INT32_MAX, 0};  // the same from every row that does it
    }
}
// A block per row and 1,024 columns.
__global__ void __launch_bounds__(kRowThreads) fork_tables_kernel(const __grid_constant__ ForkArgs a) {
    let_next_launch_start();
    const int parts = a.old.width > kRowColumns ? (a.old.width + kRowColumns - 1) / kRowColumns : 1;
    const int row = blockIdx.x / parts, column0 = (blockIdx.x - row * parts) * kRowColumns;
    fork_row(a, row, column0, min(a.old.width, column0 + kRowColumns), threadIdx.x, kRowThreads);
}

// One cluster, a row a thread.  A page that is not full may be written to by one row only: the first of the new rows that hold it
// keeps it, if no other row does (it is counted more often than by these), and each of the rest gets a copy.  TABLES: small tables are made here
// too, a warp a row, which saves a launch.
template <int BLOCKS, bool TABLES>
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(kClusterThreads) fork_writers_kernel(const __grid_constant__ ForkArgs a) {
    __shared__ Told told;
    let_next_launch_start();
    if (TABLES) {
        const int32_t rows = a.release && a.old.rows > a.nnew ? a.old.rows : a.nnew;
        for (int32_t row = threadIdx.x >> 5; row < rows; row += kClusterWarps) fork_row(a, row, 0, a.old.width, threadIdx.x & 31, 32);
        __syncthreads();
    } else {
        wait_for_launch_before();
    }
    const int32_t each = (a.nnew + BLOCKS - 1) / BLOCKS, row = cluster_rank<BLOCKS>() * each + threadIdx.x;
    const bool here = threadIdx.x < each && row < a.nnew;
    int32_t tokens = 0, page = -1, part = 0, column = 0;
    if (here) {
        tokens = a.lens[row];
        part = tokens % a.old.page_size;
        column = tokens / a.old.page_size;
        if (part) page = a.table[row * a.row + column];
        if (page >= 0) {
            atomicMin(&a.writers[page].first, row);
            atomicAdd(&a.writers[page].count, 1);
        }
    }
    cluster_barrier<BLOCKS>();
    bool copied = false;
    if (page >= 0) copied = __ldcg(&a.writers[page].first) != row || __ldcg(&a.writers[page].count) != __ldcg(a.refs + page);
    int64_t all, free;
    const int64_t rank = take_free<BLOCKS>(a.refs, a.old.num_pages, copied, a.list, &told, &all, &free);
    if (copied) {
        const bool found = rank < free;
        const int32_t to = found ? __ldcg(a.list + rank) : -1;
        atomicAdd(a.refs + page, -1);
        a.table[row * a.row + column] = to;
        if (found) {
            a.refs[to] = 1;
            a.moves[rank] = page;
            a.moves[a.nnew + rank] = to;
            a.moves[2 * a.nnew + rank] = part;
        } else {  // the tokens of that page are lost
            a.lens[row] = tokens - part;
            note(a.old.status, CG_S_NO_PAGE);
        }
    }
    const int32_t made = static_cast<int32_t>(all < free ? all : free);
    for (int32_t r = made + cluster_rank<BLOCKS>() * kClusterThreads + threadIdx.x; r < a.nnew; r += BLOCKS * kClusterThreads)
        a.moves[r] = a.moves[a.nnew + r] = a.moves[2 * a.nnew + r] = -1;
    if (cluster_rank<BLOCKS>() == 0 && threadIdx.x == 0) *a.copies = made;
}

// ---- give back -----------------------------------------------------------------------------------------
struct FreeArgs {
    Table t;
    int32_t *table, *lens, *refs;
    const void *rows;  // or nullptr: all
    int32_t nfree, wide;
};
// A block per row.  A row that is named twice is given back once: its length is taken by the first.
__global__ void __launch_bounds__(kRowThreads) free_pages_kernel(const __grid_constant__ FreeArgs a) {
    __shared__ int32_t taken;
    const int64_t row = a.rows ? index_at(a.rows, blockIdx.x, a.wide) : blockIdx.x;
    if (row < 0 || row >= a.t.rows) {
        if (row != -1 && threadIdx.x == 0) note(a.t.status, CG_S_BAD_PAGE);
        return;
    }
    if (threadIdx.x == 0) taken = atomicExch(a.lens + row, 0);
    __syncthreads();
    int64_t need = pages_of(taken < 0 ? 0 : taken, a.t.page_size);
    if (taken < 0 || need > a.t.width) {
        if (threadIdx.x == 0) note(a.t.status, CG_S_BAD_PAGE);
        if (need > a.t.width) need = a.t.width;
    }
    for (int64_t j = threadIdx.x; j < need; j += kRowThreads) {
        const int32_t p = page_at(a.t, static_cast<int>(row), static_cast<int>(j));
        a.table[row * a.t.row + j] = -1;
        if (p >= 0 && atomicAdd(a.refs + p, -1) <= 0) {  // nobody held it
            atomicAdd(a.refs + p, 1);
            note(a.t.status, CG_S_BAD_PAGE);
        }
    }
}

// ---- extend --------------------------------------------------------------------------------------------
struct ExtendArgs {
    Table t;
    int32_t *table, *lens, *refs, *list;
    int32_t *firsts;        // [rows]: where a row's new tokens begin, -1 if they found no place
    const int32_t *starts;  // [rows + 1], or nullptr: a token a row
    int64_t *slots;
    int32_t ntokens;
};
struct Growth {  // of a row: its pages before, how many it gets, and where they stand in the list, or would
    int32_t before, pages;
    int64_t rank;
};
__device__ __forceinline__ int32_t start_of(const ExtendArgs &a, int row) {
    if (!a.starts) return row;
    const int32_t s = a.starts[row];
    if (s >= 0 && s <= a.ntokens) return s;
    note(a.t.status, CG_S_BAD_PAGE);
    return s < 0 ? 0 : a.ntokens;
}
// The slot of token i, whose row is found among the starts.
__device__ __forceinline__ int64_t slot_of(const ExtendArgs &a, int32_t i) {
    int32_t row = i, start = i;
    if (a.starts) {
        int32_t lo = 0, hi = a.t.rows;  // starts[lo] <= i < starts[hi], if any are
        if (i < __ldg(a.starts) || i >= __ldg(a.starts + hi)) return -1;  // a token of no row
        while (hi - lo > 1) {
            const int32_t mid = (lo + hi) / 2;
            if (__ldg(a.starts + mid) <= i) lo = mid;
            else hi = mid;
        }
        row = lo;
        start = max(0, __ldg(a.starts + row));
    }
    const int32_t first = __ldcg(a.firsts + row);
    const int64_t place = static_cast<int64_t>(first) + i - start;
    if (first < 0 || place < first || place >= __ldcg(a.lens + row)) return -1;
    const int32_t column = static_cast<int32_t>(place / a.t.page_size), p = __ldcg(a.t.entries + row * a.t.row + column);
    if (p >= 0 && p < a.t.num_pages) return static_cast<int64_t>(p) * a.t.page_size + (place - static_cast<int64_t>(column) * a.t.page_size);
    note(a.t.status, CG_S_BAD_PAGE);
    return -1;
}
// One cluster, a row a thread for the sums; then the threads of a block share its rows' new pages, and (`slots_too`) all of them the tokens.
template <int BLOCKS>
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(kClusterThreads) extend_pages_kernel(const __grid_constant__ ExtendArgs a, int slots_too) {
    __shared__ Told told;
    __shared__ Growth grown[kClusterThreads];
    let_next_launch_start();
    const int32_t S = a.t.page_size, each = (a.t.rows + BLOCKS - 1) / BLOCKS, row0 = cluster_rank<BLOCKS>() * each;
    const int32_t row = row0 + threadIdx.x;
    const bool here = threadIdx.x < each && row < a.t.rows;
    int32_t tokens = 0, asked = 0;
    int64_t wanted = 0;
    bool fits = true;
    Growth g{0, 0, 0};
    if (here) {
        asked = start_of(a, row + 1) - start_of(a, row);
        if (asked < 0) {
            note(a.t.status, CG_S_BAD_PAGE);
            asked = 0;
        }
        tokens = length_of(a.t, row);
        g.before = pages_of(tokens, S);
        const int64_t after = static_cast<int64_t>(tokens) + asked;
        wanted = (after + S - 1) / S - g.before;
        if (g.before + wanted > a.t.width) {
            note(a.t.status, CG_S_BAD_PAGE);
            fits = false, wanted = 0;
        }
    }
    int64_t all, free;
    g.rank = take_free<BLOCKS>(a.refs, a.t.num_pages, wanted, a.list, &told, &all, &free);
    if (here) {
        if (wanted > 0 && g.rank + wanted > free) {
            note(a.t.status, CG_S_NO_PAGE);
            fits = false;
        }
        if (fits && asked) a.lens[row] = tokens + asked;
        g.pages = fits ? static_cast<int32_t>(wanted) : 0;
        a.firsts[row] = fits ? tokens : -1;
        grown[threadIdx.x] = g;
    }
    __syncthreads();
    // The block's rows' pages follow one another in the list: a page a thread, its row found among theirs.
    const int32_t mine = a.t.rows - row0 < each ? a.t.rows - row0 : each;  // rows of this block, none or less behind the last
    if (mine > 0) {
        const int64_t asked_for = grown[mine - 1].rank + grown[mine - 1].pages, end = asked_for < free ? asked_for : free;
        for (int64_t r = grown[0].rank + threadIdx.x; r < end; r += kClusterThreads) {
            int32_t lo = 0, hi = mine;  // ranks rise: the last row that begins at r or in front of it
            while (hi - lo > 1) {
                const int32_t mid = (lo + hi) / 2;
                if (grown[mid].rank <= r) lo = mid;
                else hi = mid;
            }
            const Growth &x = grown[lo];
            if (r - x.rank >= x.pages) continue;  // of a row that found no place
            const int32_t p = __ldcg(a.list + r);
            a.table[(row0 + lo) * a.t.row + x.before + (r - x.rank)] = p;
            a.refs[p] = 1;
        }
    }
    if (!slots_too) return;
    cluster_barrier<BLOCKS>();
    for (int32_t i = cluster_rank<BLOCKS>() * kClusterThreads + threadIdx.x; i < a.ntokens; i += BLOCKS * kClusterThreads) a.slots[i] = slot_of(a, i);
}
__global__ void __launch_bounds__(kRowThreads) slots_kernel(const __grid_constant__ ExtendArgs a) {
    wait_for_launch_before();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
    if (i < a.ntokens) a.slots[i] = slot_of(a, static_cast<int32_t>(i));
}

// ---- compact -------------------------------------------------------------------------------------------
struct CompactArgs {
    Table t;
    int32_t *table, *refs, *places, *moves;  // moves [2][num_pages / 2]
    int32_t *copies, *before_middle;
};
__device__ __forceinline__ void compact_row(const CompactArgs &a, int32_t row, int32_t column0, int32_t column1, int32_t first, int32_t step) {
    const int32_t need = pages_of(length_of(a.t, row), a.t.page_size);
    for (int32_t j = column0 + first; j < column1 && j < need; j += step) {
        const int32_t p = page_at(a.t, row, j);
        if (p < 0) continue;
        const int32_t to = __ldcg(a.places + p);
        if (to >= 0) a.table[row * a.t.row + j] = to;
        else note(a.t.status, CG_S_BAD_PAGE);  // a page that nobody holds
    }
}
// One cluster.  With n pages held, those at n and behind go to the holes in front of n, the first to the first.  TABLES: as above.
template <int BLOCKS, bool TABLES>
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(kClusterThreads) compact_places_kernel(const __grid_constant__ CompactArgs a) {
    __shared__ Told told;
    let_next_launch_start();
    const Run run = run_of<BLOCKS>(a.t.num_pages);
    const bool vectors = reinterpret_cast<uintptr_t>(a.refs) % 16 == 0;
    const int32_t lane = threadIdx.x & 31, free = free_in<BLOCKS>(a.refs, run, vectors);
    const Sums sums = over_warps<BLOCKS>(free, run.last - run.first - free, &told);
    const int32_t n = static_cast<int32_t>(sums.all_b);  // pages held
    if (n >= run.first && n < run.last) {  // the warp whose pages n is one of: those held in front of it
        int32_t front = 0;
        for (int32_t p = run.first + lane; p < n; p += 32) front += a.refs[p] != 0;
        front = __reduce_add_sync(~0u, front);
        if (lane == 0) *a.before_middle = static_cast<int32_t>(sums.b) + front;
    }
    cluster_barrier<BLOCKS>();
    const int32_t front = n < a.t.num_pages ? __ldcg(a.before_middle) : n, made = n - front;  // holes in front of n = held pages behind
    const int32_t half = a.t.num_pages / 2;
    int32_t before = static_cast<int32_t>(sums.b);  // pages held in front of p0
    for (int32_t p0 = run.first; p0 < run.last; p0 += kRunStep<BLOCKS>) {
        const int32_t p = p0 + 4 * kQuads<BLOCKS> * lane;
        int4 c[kQuads<BLOCKS>];
        counts_of(a.refs, p, 4, run, p0, vectors, 0, c);
        const int32_t held = 4 * kQuads<BLOCKS> - zeros(c), upto = sum_upto(held);
        int32_t at = before + upto - held;
        const auto place = [&](int32_t count, int32_t q) {
            if (q >= run.last) return;
            if (count != 0 && q >= n) a.moves[at - front] = q;
            if (count == 0 && q < n) a.moves[half + q - at] = q;
            a.places[q] = count != 0 ? q : -1;
            at += count != 0;
        };
#pragma unroll
        for (int i = 0; i < kQuads<BLOCKS>; ++i) place(c[i].x, p + 4 * i), place(c[i].y, p + 4 * i + 1), place(c[i].z, p + 4 * i + 2), place(c[i].w, p + 4 * i + 3);
        before += __shfl_sync(~0u, upto, 31);
    }
    cluster_barrier<BLOCKS>();
    for (int32_t r = cluster_rank<BLOCKS>() * kClusterThreads + threadIdx.x; r < half; r += BLOCKS * kClusterThreads) {
        if (r < made) {
            const int32_t from = __ldcg(a.moves + r), to = __ldcg(a.moves + half + r);
            a.places[from] = to;
            a.refs[to] = __ldcg(a.refs + from);
            a.refs[from] = 0;
        } else {
            a.moves[r] = a.moves[half + r] = -1;
        }
    }
    if (cluster_rank<BLOCKS>() == 0 && threadIdx.x == 0) *a.copies = made;
    if (TABLES) {
        __syncthreads();
        for (int32_t row = threadIdx.x >> 5; row < a.t.rows; row += kClusterWarps) compact_row(a, row, 0, a.t.width, threadIdx.x & 31, 32);
    }
}
__global__ void __launch_bounds__(kRowThreads) compact_tables_kernel(const __grid_constant__ CompactArgs a) {
    let_next_launch_start();
    wait_for_launch_before();
    const int parts = (a.t.width + kRowColumns - 1) / kRowColumns;
    const int row = blockIdx.x / parts, column0 = (blockIdx.x - row * parts) * kRowColumns;
    compact_row(a, row, column0, column0 + kRowColumns, threadIdx.x, kRowThreads);
}

// ---- copy ----------------------------------------------------------------------------------------------
// A page as `outer` runs of `run` pieces (vectors or values) that follow one another in memory; outer index o stands for the page's
// token o, its head o, or, where neither follows the other, for head o % heads of token o / heads.
struct CopySide {
    char *data;
    int64_t layer, page, token, head;  // in elements
    int32_t runs;                      // kWhole ..
};
enum Runs { kWhole, kTokens, kHeads, kNone };
struct CopyArgs {
    CopySide sides[2];
    const void *src, *dst;
    const int32_t *tokens, *count;  // or nullptr
    int32_t *status;
    int64_t num_pages;
    int32_t ncopies, nlayers, page_size, heads, pieces;  // pieces of a head
    int32_t slices, wide;
};

// A unit is a slice of what is copied of one page of one layer's keys or values, so that pages of which little is copied are shared out as evenly as whole
// ones; a block goes through it kCopyThreads x kCopyVectors pieces at a time.  The next unit's numbers are on their way while one is copied.
struct Copy {
    int64_t from, to;
    int32_t tokens;
};
__device__ __forceinline__ Copy copy_at(const CopyArgs &a, int32_t i) {
    if (a.wide)
        return Copy{__ldcg(static_cast<const long long *>(a.src) + i), __ldcg(static_cast<const long long *>(a.dst) + i), a.tokens ? __ldcg(a.tokens + i) : a.page_size};
    return Copy{__ldcg(static_cast<const int *>(a.src) + i), __ldcg(static_cast<const int *>(a.dst) + i), a.tokens ? __ldcg(a.tokens + i) : a.page_size};
}
template <class Piece>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    wait_for_launch_before();
    const int32_t ncopies = a.count ? __ldcg(a.count) : a.ncopies, each = 2 * a.nlayers * a.slices;
    const int64_t units = static_cast<int64_t>(ncopies) * each;
    constexpr int kValues = sizeof(Piece) / 2;
    const int32_t step = static_cast<int32_t>(gridDim.x), over = step / each, rest = step - over * each;
    int32_t which_next = static_cast<int32_t>(blockIdx.x) / each, in_next = static_cast<int32_t>(blockIdx.x) - which_next * each;
    Copy next{};
    if (blockIdx.x < units) next = copy_at(a, which_next);
    for (int64_t u = blockIdx.x; u < units; u += step) {
        const int32_t in = in_next;
        const int64_t from = next.from, to = next.to;
        const int32_t tokens = next.tokens;
        which_next += over, in_next += rest;
        if (in_next >= each) in_next -= each, ++which_next;
        if (u + step < units) next = copy_at(a, which_next);
        if (from < 0 || to < 0 || from >= a.num_pages || to >= a.num_pages || tokens < 0 || tokens > a.page_size) {
            const bool padding = from == -1 || to == -1;
            if (!padding && in == 0 && threadIdx.x == 0) note(a.status, CG_S_BAD_PAGE);
            continue;
        }
        const int32_t which = in / a.slices, slice = in - which * a.slices, layer = which >> 1;
        const CopySide &s = a.sides[which & 1];
        const int32_t pieces = tokens * a.heads * a.pieces, share = ((pieces + a.slices - 1) / a.slices + 7) & ~7, first = slice * share;
        const int32_t last = first + share < pieces ? first + share : pieces;
        if (first >= last || from == to) continue;
        const int32_t run = s.runs == kWhole ? pieces : s.runs == kTokens ? a.heads * a.pieces : s.runs == kHeads ? tokens * a.pieces : a.pieces;
        const char *const src = s.data + 2 * (layer * s.layer + from * s.page);
        char *const dst = s.data + 2 * (layer * s.layer + to * s.page);
        for (int32_t e0 = first + static_cast<int32_t>(threadIdx.x); e0 < last; e0 += kCopyThreads * kCopyVectors) {
            Piece x[kCopyVectors];
            int64_t at[kCopyVectors];
#pragma unroll
            for (int v = 0; v < kCopyVectors; ++v) {
                const int32_t e = e0 + v * kCopyThreads;
                at[v] = -1;
                if (e < last) {
                    if (s.runs == kWhole) {
                        at[v] = static_cast<int64_t>(e) * kValues;
                    } else {
                        const int32_t o = e / run, rest = e - o * run;
                        const int64_t step = s.runs == kTokens ? o * s.token : s.runs == kHeads ? o * s.head : o / a.heads * s.token + o % a.heads * s.head;
                        at[v] = step + static_cast<int64_t>(rest) * kValues;
                    }
                    x[v] = *reinterpret_cast<const Piece *>(src + 2 * at[v]);
                }
            }
#pragma unroll
            for (int v = 0; v < kCopyVectors; ++v)
                if (at[v] >= 0) *reinterpret_cast<Piece *>(dst + 2 * at[v]) = x[v];
        }
    }
}

CopySide copy_side(void *data, const int64_t *s, int heads, int head_size) {
    const bool heads_follow = s[3] == head_size || heads == 1, tokens_follow = s[2] == head_size;
    const int runs = heads_follow && s[2] == static_cast<int64_t>(heads) * head_size ? kWhole : heads_follow ? kTokens : tokens_follow ? kHeads : kNone;
    return CopySide{static_cast<char *>(data), s[0], s[1], s[2], s[3], runs};
}
bool vectors(const CopySide &s) {
    return reinterpret_cast<uintptr_t>(s.data) % 16 == 0 && s.layer % 8 == 0 && s.page % 8 == 0 && s.token % 8 == 0 && s.head % 8 == 0;
}

// count: how many copies there are, on the GPU, or nullptr: ncopies; spread: they may well be as many; early: the launch in front writes what is read
// here and has let this one start
int copy_pages(const cg_copy_job &j, const int32_t *count, bool spread, bool early, cudaStream_t st) {
    if (j.ncopies == 0 || j.nlayers == 0 || j.page_size == 0) return CG_OK;
    CopyArgs a{};
    a.sides[0] = copy_side(j.pages_k, j.pages_k_strides, j.heads, j.head_size);
    a.sides[1] = copy_side(j.pages_v, j.pages_v_strides, j.heads, j.head_size);
    a.src = j.src, a.dst = j.dst, a.tokens = j.tokens, a.count = count, a.status = j.status;
    a.num_pages = j.num_pages;
    a.ncopies = j.ncopies, a.nlayers = j.nlayers, a.page_size = j.page_size, a.heads = j.heads, a.wide = j.wide;
    const bool vec = j.head_size % 8 == 0 && vectors(a.sides[0]) && vectors(a.sides[1]);
    a.pieces = vec ? j.head_size / 8 : j.head_size;
    const int64_t pieces = static_cast<int64_t>(j.page_size) * j.heads * a.pieces;
    // as many slices as give every block some units, none below what a block copies at a time
    const int64_t parts = (pieces + kCopyThreads * kCopyVectors - 1) / (kCopyThreads * kCopyVectors), most = static_cast<int64_t>(sm_count()) * 8;
    const int64_t pages = 2 * static_cast<int64_t>(j.nlayers) * j.ncopies, slices = (4 * most + pages - 1) / pages, units = pages * (slices < parts ? slices : parts);
    a.slices = static_cast<int32_t>(slices < parts ? slices : parts);
    // More blocks than run at a time make room for others as they end, so that units of unlike lengths are shared out evenly; blocks that find no unit cost a little
    // (700 parts of pages: 197 us with as many blocks as run, 181 with sixteen times as many; a large cache compacted: 208, 195 with four times and 191 with sixteen;
    // a fork, where few of the possible copies are there, is 2 us slower with four times and 10 with sixteen).
    const int64_t blocks = most * (!count ? 16 : spread && units >= 8 * most ? 4 : 1);
    const dim3 grid(static_cast<unsigned>(units < blocks ? units : blocks));
    return vec ? launch(copy_pages_kernel<uint4>, grid, kCopyThreads, 0, early, st, a) : launch(copy_pages_kernel<uint16_t>, grid, kCopyThreads, 0, early, st, a);
}

int check_copy(const cg_copy_job &j) {
    if ((reinterpret_cast<uintptr_t>(j.pages_k) | reinterpret_cast<uintptr_t>(j.pages_v)) % 2) return CG_E_ALIGN;
    if (j.ncopies < 0 || j.nlayers < 0 || j.page_size <= 0 || j.heads <= 0 || j.head_size <= 0 || j.num_pages < 0 || j.num_pages > kMostPages) return CG_E_SHAPE;
    // offsets inside a page, and units of one copy, are 32-bit numbers
    if (static_cast<int64_t>(j.heads) * j.head_size > (1 << 28) || static_cast<int64_t>(j.page_size) * j.heads * j.head_size > (1 << 30) ||
        static_cast<int64_t>(j.nlayers) * (static_cast<int64_t>(j.page_size) * j.heads * j.head_size / 1024 + 1) > (1 << 29))
        return CG_E_CAPACITY;
    return CG_OK;
}

// ---- entries -------------------------------------------------------------------------------------------
struct Workspace {  // where its parts begin
    int64_t writers, list, firsts, total;
};
Workspace workspace_of(int64_t num_pages) {
    Workspace w{};
    w.writers = 64;  // two words of counts in front
    w.list = w.writers + 8 * num_pages;
    w.firsts = w.list + 4 * num_pages;
    w.total = w.firsts + 4 * CG_MAX_REQUESTS;
    return w;
}

// Whether one block goes through a table about as fast as a grid is launched: up to two steps a warp.
bool few_entries(int64_t rows, int64_t width) { return rows * (width / 32 + 1) <= 2 * kClusterWarps; }

enum What { kFork, kFree, kExtend, kCompact };

int check_pages(const cg_pages_job *job, What what) {
    if (!job) return CG_E_NULL;
    const cg_pages_job &j = *job;
    if (j.nrows < 0 || j.width < 0 || j.page_size <= 0 || j.num_pages < 0 || j.num_pages > kMostPages || j.nnew < 0 || j.ntokens < 0) return CG_E_SHAPE;
    if (j.nrows > CG_MAX_REQUESTS || ((what == kFork || (what == kFree && j.which)) && j.nnew > CG_MAX_REQUESTS)) return CG_E_CAPACITY;
    if (static_cast<int64_t>(j.width) * j.page_size > INT32_MAX || j.width > kMostPages) return CG_E_SHAPE;
    if ((j.nrows && ((j.width && !j.table) || !j.kv_lens)) || (j.num_pages && !j.refs)) return CG_E_NULL;
    if (what == kFork && (!j.which || (j.width && !j.new_table) || !j.new_lens || !j.moves) && j.nnew) return CG_E_NULL;
    if (what == kExtend && ((!j.slots && j.ntokens) || (!j.q_starts && j.ntokens != j.nrows))) return j.q_starts || !j.slots ? CG_E_NULL : CG_E_SHAPE;
    if (what == kCompact && j.num_pages && (!j.places || (!j.moves && j.num_pages > 1))) return CG_E_NULL;
    if (what != kFree) {
        if (j.workspace_bytes < workspace_of(j.num_pages).total || !j.workspace) return CG_E_CAPACITY;
        if (reinterpret_cast<uintptr_t>(j.workspace) % 16) return CG_E_ALIGN;
    }
    return CG_OK;
}
Table table_of(const cg_pages_job &j) {
    return Table{j.table, j.kv_lens, j.table_row, j.nrows, j.width, j.page_size, static_cast<int32_t>(j.num_pages), j.status};
}
char *part_of(const cg_pages_job &j, int64_t at) { return static_cast<char *>(j.workspace) + at; }

}  // namespace
}  // namespace cg

extern "C" int64_t cg_pages_workspace(int64_t num_pages) {
    return num_pages < 0 || num_pages > cg::kMostPages ? CG_E_SHAPE : cg::workspace_of(num_pages).total;
}

extern "C" int cg_copy_pages(const cg_copy_job *job, void *stream) {
    using namespace cg;
    if (!job) return CG_E_NULL;
    const cg_copy_job &j = *job;
    if (const int rc = check_copy(j)) return rc;
    if (j.ncopies == 0 || j.nlayers == 0) return CG_OK;
    if (!j.pages_k || !j.pages_v || !j.src || !j.dst) return CG_E_NULL;
    return copy_pages(j, nullptr, true, false, static_cast<cudaStream_t>(stream));
}

extern "C" int cg_fork_pages(const cg_pages_job *job, const cg_copy_job *copy, void *stream) {
    using namespace cg;
    if (const int rc = check_pages(job, kFork)) return rc;
    const cg_pages_job &j = *job;
    if (copy) {
        if (const int rc = check_copy(*copy)) return rc;
        if (copy->nlayers && (!copy->pages_k || !copy->pages_v)) return CG_E_NULL;
        if (copy->page_size != j.page_size || copy->num_pages != j.num_pages) return CG_E_SHAPE;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Workspace w = workspace_of(j.num_pages);
    ForkArgs a{};
    a.old = table_of(j);
    a.table = j.new_table, a.lens = j.new_lens, a.refs = j.refs, a.moves = j.moves, a.parents = j.which;
    a.writers = reinterpret_cast<Writers *>(part_of(j, w.writers)), a.list = reinterpret_cast<int32_t *>(part_of(j, w.list));
    a.copies = reinterpret_cast<int32_t *>(part_of(j, 0));
    a.row = j.new_table_row;
    a.nnew = j.nnew, a.wide = j.wide, a.release = j.release;
    const int rows = j.release && j.nrows > j.nnew ? j.nrows : j.nnew, parts = j.width > kRowColumns ? (j.width + kRowColumns - 1) / kRowColumns : 1;
    if (rows == 0) return CG_OK;
    if (static_cast<int64_t>(rows) * parts > INT32_MAX) return CG_E_SHAPE;
    const bool alone = j.num_pages <= kAlonePages && j.nnew <= kClusterThreads;
    if (alone && few_entries(rows, j.width) && j.nnew) {
        if (const int rc = launch(fork_writers_kernel<1, true>, dim3(1), kClusterThreads, 0, false, st, a)) return rc;
    } else {
        if (const int rc = launch(fork_tables_kernel, dim3(rows * parts), kRowThreads, 0, false, st, a)) return rc;
        if (j.nnew == 0) return CG_OK;
        if (const int rc = alone ? launch(fork_writers_kernel<1, false>, dim3(1), kClusterThreads, 0, true, st, a)
                                 : launch(fork_writers_kernel<kClusterBlocks, false>, dim3(kClusterBlocks), kClusterThreads, 0, true, st, a))
            return rc;
    }
    if (!copy) return CG_OK;
    cg_copy_job c = *copy;
    c.src = j.moves, c.dst = j.moves + j.nnew, c.tokens = j.moves + 2 * static_cast<int64_t>(j.nnew);
    c.wide = 0, c.ncopies = j.nnew, c.status = j.status;
    return copy_pages(c, a.copies, false, true, st);
}

extern "C" int cg_free_pages(const cg_pages_job *job, void *stream) {
    using namespace cg;
    if (const int rc = check_pages(job, kFree)) return rc;
    const cg_pages_job &j = *job;
    FreeArgs a{table_of(j), j.table, j.kv_lens, j.refs, j.which, j.which ? j.nnew : j.nrows, j.wide};
    if (a.nfree == 0) return CG_OK;
    return launch(free_pages_kernel, dim3(a.nfree), kRowThreads, 0, false, static_cast<cudaStream_t>(stream), a);
}

extern "C" int cg_extend_pages(const cg_pages_job *job, void *stream) {
    using namespace cg;
    if (const int rc = check_pages(job, kExtend)) return rc;
    const cg_pages_job &j = *job;
    if (j.nrows == 0 && j.ntokens == 0) return CG_OK;
    if (j.nrows == 0) return CG_E_SHAPE;  // tokens of nobody
    const Workspace w = workspace_of(j.num_pages);
    ExtendArgs a{table_of(j), j.table, j.kv_lens, j.refs, reinterpret_cast<int32_t *>(part_of(j, w.list)), reinterpret_cast<int32_t *>(part_of(j, w.firsts)),
                 j.q_starts, j.slots, j.ntokens};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Slots of a few tokens a row are the cluster's work too, those of prompts a grid's.
    const bool together = j.ntokens <= kSlotsTogether;
    const bool alone = j.num_pages <= kAlonePages && j.nrows <= kClusterThreads && j.ntokens <= 4 * kClusterThreads;
    if (alone) return launch(extend_pages_kernel<1>, dim3(1), kClusterThreads, 0, false, st, a, 1);
    if (const int rc = launch(extend_pages_kernel<kClusterBlocks>, dim3(kClusterBlocks), kClusterThreads, 0, false, st, a, together ? 1 : 0)) return rc;
    if (together) return CG_OK;
    const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(j.ntokens) + kRowThreads - 1) / kRowThreads);
    return launch(slots_kernel, dim3(blocks), kRowThreads, 0, true, st, a);
}

extern "C" int cg_compact_pages(const cg_pages_job *job, const cg_copy_job *copy, void *stream) {
    using namespace cg;
    if (const int rc = check_pages(job, kCompact)) return rc;
    const cg_pages_job &j = *job;
    if (copy) {
        if (const int rc = check_copy(*copy)) return rc;
        if (copy->nlayers && (!copy->pages_k || !copy->pages_v)) return CG_E_NULL;
        if (copy->page_size != j.page_size || copy->num_pages != j.num_pages) return CG_E_SHAPE;
    }
    if (j.num_pages == 0) return CG_OK;
    const int64_t blocks = static_cast<int64_t>(j.nrows) * ((j.width + kRowColumns - 1) / kRowColumns);  // of a grid over the table
    if (blocks > INT32_MAX) return CG_E_SHAPE;  // before anything has moved
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int32_t *const words = reinterpret_cast<int32_t *>(part_of(j, 0));
    CompactArgs a{table_of(j), j.table, j.refs, j.places, j.moves, words, words + 1};
    const bool alone = j.num_pages <= kAlonePages, together = alone && few_entries(j.nrows, j.width);
    const int rc = together ? launch(compact_places_kernel<1, true>, dim3(1), kClusterThreads, 0, false, st, a)
                   : alone  ? launch(compact_places_kernel<1, false>, dim3(1), kClusterThreads, 0, false, st, a)
                            : launch(compact_places_kernel<kClusterBlocks, false>, dim3(kClusterBlocks), kClusterThreads, 0, false, st, a);
    if (rc) return rc;
    if (!together && j.nrows && j.width) {
        if (const int rc2 = launch(compact_tables_kernel, dim3(static_cast<unsigned>(blocks)), kRowThreads, 0, true, st, a)) return rc2;
    }
    if (!copy) return CG_OK;
    cg_copy_job c = *copy;
    c.src = j.moves, c.dst = j.moves + j.num_pages / 2, c.tokens = nullptr;
    c.wide = 0, c.ncopies = static_cast<int32_t>(j.num_pages / 2), c.status = j.status;
    return copy_pages(c, a.copies, true, true, st);
}
