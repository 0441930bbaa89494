// What the two attention kernels share: how the work of a batch is divided, and what is left where a tile is divided.
//
// A tile is up to M query rows of one request that read the same key/value head: row r of a request is token r / group, query head
// r % group of the head's group, so that a key that is read serves all of them.  A tile's work is counted in units, blocks of BK keys
// that one of its rows sees (one unit at least).  All units of a call stand in one line, (request, head, tile, block), and every
// CTA takes an equal run of it: whatever the batch's lengths, the CTAs end together.  A tile that two CTAs or more share leaves
// a maximum, a sum and a product a row from each of them in the workspace, and a second kernel joins those.  Where all tiles are short
// (`undivided`) a CTA takes the tiles that begin in its run, whole.  Lengths stay on the
// GPU, so that one captured graph serves all of them: each CTA works out its own run.
#pragma once

#include "cg_common.cuh"

namespace cg {

// The divided tile that begins in a CTA: what joins its parts needs to know of it.
struct __align__(16) Join {
    int32_t sharers;  // CTAs that have a part of it, 0: none begins here
    int32_t first, n, kv, head, t, unused[2];
};

struct AttendArgs {
    const char *q, *k, *v;
    char *out;
    float *lse;
    const int32_t *table, *kv_lens, *q_starts;
    char *parts;    // [ctas][2] rows of sums, see part_bytes
    Join *joins;    // [ctas]
    int32_t *status;
    int64_t q_token, q_head, out_token, out_head, k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
    int64_t table_row, num_pages;
    int32_t page_shift, group_shift;  // log2(page_size) and log2(group), -1 if that is no power of two
    int32_t nrequests, nrows, q_heads, heads, group, head_size, page_size, table_width, causal, window;
    int32_t undivided;  // tiles are not divided among CTAs
    float scale;    // of the scores, times log2(e)
};

constexpr float kNegInf = -INFINITY;
constexpr int64_t kMostKeys = 1 << 30;  // of a request: places of keys and of blocks behind them stay numbers of 32 bits

// bytes of one CTA's share of a tile: float sums[M][DP], then float2 (maximum, sum of weights)[M]
__host__ __device__ constexpr int64_t part_bytes(int M, int DP) { return static_cast<int64_t>(M) * (DP * 4 + 8); }

struct Lengths {
    int first, n, kv;  // first row of q, rows, keys
};
__device__ __forceinline__ Lengths lengths_of(const AttendArgs &a, int b, bool report = false) {
    Lengths r;
    int last;
    r.first = b, last = b + 1;
    if (a.q_starts) r.first = __ldg(a.q_starts + b), last = __ldg(a.q_starts + b + 1);
    r.kv = __ldg(a.kv_lens + b);
    const int64_t room = min(static_cast<int64_t>(a.table_width) * a.page_size, kMostKeys);
    const bool bad = r.first < 0 || last < r.first || last > a.nrows || r.kv < 0 || r.kv > room;
    if (bad) {
        r.first = min(max(r.first, 0), a.nrows);
        last = min(max(last, r.first), a.nrows);
        r.kv = r.kv < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(r.kv), room));
        if (report && a.status) atomicOr(a.status, CG_S_BAD_PAGE);
    }
    r.n = last - r.first;
    return r;
}

// The token of a row of a request's, and its query head, counted in its group.  (Tiles of many rows shift where they can: 8,192 tokens 590 ->
// 582 us.  The kernel for few rows has no registers for both forms: 40 requests of 250 tokens 43.2 us with them, 42.2 without.)
template <int M> __device__ __forceinline__ int token_of(const AttendArgs &a, int row) {
    return M > 16 && a.group_shift >= 0 ? row >> a.group_shift : row / a.group;
}
__device__ __forceinline__ int member_of(const AttendArgs &a, int row, int token) { return row - token * a.group; }

// keys [lo, hi) that token i of n sees.  (A place may be as low as -2^31 and a window as wide as 2^31 - 1: their difference is only taken where
// the window ends behind the first key.)
__device__ __forceinline__ int first_key(const AttendArgs &a, const Lengths &r, int i) {
    const int place = r.kv - r.n + i;
    return a.window > 0 && place >= a.window ? place - a.window + 1 : 0;
}
__device__ __forceinline__ int last_key(const AttendArgs &a, const Lengths &r, int i) {
    return a.causal ? min(r.kv, max(0, r.kv - r.n + i + 1)) : r.kv;
}

struct Tile {
    int lo, hi;          // keys that a row of the tile sees
    int block0, units;   // first block of BK keys, blocks
};
template <int M, int BK> __device__ __forceinline__ Tile tile_of(const AttendArgs &a, const Lengths &r, int t) {
    const int last = min(r.n * a.group, (t + 1) * M) - 1;
    Tile x;
    x.hi = last_key(a, r, token_of<M>(a, last));
    x.lo = min(first_key(a, r, token_of<M>(a, t * M)), x.hi);
    x.block0 = x.lo / BK;
    x.units = max(1, (x.hi + BK - 1) / BK - x.block0);
    return x;
}
template <int M> __device__ __forceinline__ int tiles_of(const AttendArgs &a, const Lengths &r) { return (r.n * a.group + M - 1) / M; }

// The part of a tile that a CTA has.
struct Piece {
    Lengths r;
    Tile tile;
    int request, head, t;
    int begin, end;      // blocks of BK keys
    bool whole, starts;  // the tile is all here; its first block is here
    int sharers;         // CTAs that share a tile that starts here
};

// A CTA's run through the line of units.  init is called by all threads of the block, with room in shared memory for
// nrequests + 1 numbers; next by any of them, as often, all with the same result.
template <int M, int BK, int COST> struct Run {
    int64_t at, to, total;
    int ctas;
    int b, h, t, tiles, skip;
    Lengths r;

    // by requests a thread (TILES false: most have one tile) or by requests a warp, tiles a lane
    template <int THREADS, bool MANY_TILES>
    __device__ __forceinline__ void init(const AttendArgs &a, int64_t *before) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        if (!MANY_TILES && a.nrequests <= 32) {  // every warp by itself, a request a lane: no memory, no barriers
            Lengths x{0, 0, 0};
            int64_t units = 0;
            if (lane < a.nrequests) {
                x = lengths_of(a, lane, blockIdx.x == 0 && warp == 0);
                const int n = tiles_of<M>(a, x);
                for (int k = 0; k < n; ++k) units += tile_of<M, BK>(a, x, k).units + COST;
            }
            int64_t end = units * a.heads;
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, end, d);
                if (lane >= d) end += o;
            }
            total = __shfl_sync(0xffffffffu, end, 31);
            share();
            if (at < to) {
                b = __popc(__ballot_sync(0xffffffffu, end <= at));  // requests that end at or in front of `at`
                const int64_t begin = __shfl_sync(0xffffffffu, end - units * a.heads, b);
                r = Lengths{__shfl_sync(0xffffffffu, x.first, b), __shfl_sync(0xffffffffu, x.n, b), __shfl_sync(0xffffffffu, x.kv, b)};
                find(a, at - begin, __shfl_sync(0xffffffffu, units, b));
            }
            return;
        }
        if (MANY_TILES) {
            for (int i = warp; i < a.nrequests; i += THREADS / 32) {
                const Lengths x = lengths_of(a, i, blockIdx.x == 0 && lane == 0);
                const int n = tiles_of<M>(a, x);
                int units = 0;
                for (int k = lane; k < n; k += 32) units += tile_of<M, BK>(a, x, k).units + COST;
                units = __reduce_add_sync(0xffffffffu, units);
                if (lane == 0) before[i + 1] = static_cast<int64_t>(units) * a.heads;
            }
        } else {
            for (int i = tid; i < a.nrequests; i += THREADS) {
                const Lengths x = lengths_of(a, i, blockIdx.x == 0);
                const int n = tiles_of<M>(a, x);
                int units = 0;
                for (int k = 0; k < n; ++k) units += tile_of<M, BK>(a, x, k).units + COST;
                before[i + 1] = static_cast<int64_t>(units) * a.heads;
            }
        }
        __syncthreads();
        if (warp == 0) {
            int64_t carry = 0;
            for (int i = 0; i < a.nrequests; i += 32) {
                int64_t s = i + lane < a.nrequests ? before[i + lane + 1] : 0;
                for (int d = 1; d < 32; d <<= 1) {
                    const int64_t o = __shfl_up_sync(0xffffffffu, s, d);
                    if (lane >= d) s += o;
                }
                s += carry;
                if (i + lane < a.nrequests) before[i + lane + 1] = s;
                carry = __shfl_sync(0xffffffffu, s, 31);
            }
            if (lane == 0) before[0] = 0;
        }
        __syncthreads();
        total = before[a.nrequests];
        share();
        if (at < to) {
            int lo = 0, hi = a.nrequests - 1;  // the last request that begins at or before `at` and has rows
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (before[mid] <= at) lo = mid;
                else hi = mid - 1;
            }
            b = lo;
            r = lengths_of(a, b);
            const int64_t of_request = before[b + 1] - before[b];
            find(a, at - before[b], of_request < INT32_MAX ? static_cast<uint32_t>(of_request) / static_cast<uint32_t>(a.heads) : of_request / a.heads);
        }
        __syncthreads();  // the numbers' memory is free again
    }

    // This CTA's run: [at, to) of `total`.
    __device__ __forceinline__ void share() {
        const int c = blockIdx.x;
        ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));
        at = to = 0;
        if (c >= ctas) return;
        if (small()) {
            at = static_cast<uint32_t>(total) * static_cast<uint32_t>(c) / static_cast<uint32_t>(ctas);
            to = static_cast<uint32_t>(total) * static_cast<uint32_t>(c + 1) / static_cast<uint32_t>(ctas);
        } else {
            at = total * c / ctas;
            to = total * (c + 1) / ctas;
        }
    }
    // whether products of a place and the number of CTAs are numbers of 32 bits (a 64-bit division takes a hundred instructions)
    __device__ __forceinline__ bool small() const { return total < (1 << 20) && ctas < (1 << 11); }

    // Head, tile and blocks in it of place `rest` of request b, whose lengths are in r; by a warp.
    __device__ __forceinline__ void find(const AttendArgs &a, int64_t rest, int64_t per_head) {
        const int lane = threadIdx.x & 31;
        tiles = tiles_of<M>(a, r);
        h = static_cast<int>(rest < INT32_MAX && per_head < INT32_MAX ? static_cast<uint32_t>(rest) / static_cast<uint32_t>(per_head) : rest / per_head);
        rest -= h * per_head;
        for (int first = 0;; first += 32) {  // 32 tiles at a time: how many end at or in front of `rest`
            int s = first + lane < tiles ? tile_of<M, BK>(a, r, first + lane).units + COST : 0;
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, s, d);
                if (lane >= d) s += o;
            }
            const int n = __popc(__ballot_sync(0xffffffffu, s <= rest && first + lane < tiles));
            const int gone = __shfl_sync(0xffffffffu, s, n ? n - 1 : 0);
            t = first + n;
            if (n) rest -= gone;
            if (n < 32) break;
        }
        skip = static_cast<int>(rest);
        if (a.undivided && skip) {  // the tile that begins in front of this run is another's
            at += tile_of<M, BK>(a, r, t).units + COST - skip;
            skip = 0;
            ++t;
        }
    }

    __device__ __forceinline__ bool next(const AttendArgs &a, Piece &p) {
        while (at < to) {
            while (t >= tiles) {
                t = 0;
                if (++h >= a.heads) {
                    h = 0;
                    do {
                        if (++b >= a.nrequests) {  // (lengths that change under way)
                            at = to;
                            return false;
                        }
                        r = lengths_of(a, b);
                        tiles = tiles_of<M>(a, r);
                    } while (tiles == 0);
                }
            }
            p.tile = tile_of<M, BK>(a, r, t);
            const int length = p.tile.units + COST, left = length - skip;
            const int take = a.undivided ? left : static_cast<int>(min(static_cast<int64_t>(left), to - at));
            const int begin = max(0, skip - COST), end = max(0, skip + take - COST);
            p.r = r;
            p.request = b, p.head = h, p.t = t;
            p.begin = p.tile.block0 + begin;
            p.end = p.tile.block0 + end;
            p.starts = begin == 0;
            p.whole = p.starts && end == p.tile.units;
            p.sharers = 0;
            if (p.starts && !p.whole) {
                const int last = small() ? static_cast<int>((static_cast<uint32_t>(at + left) * static_cast<uint32_t>(ctas) - 1) / static_cast<uint32_t>(total))
                                         : static_cast<int>(((at + left) * ctas - 1) / total);
                p.sharers = last - static_cast<int>(blockIdx.x) + 1;
            }
            at += take;
            skip = 0;
            ++t;
            if (end > begin) return true;
        }
        return false;
    }
};

// the page of a request that a key is in, counted from its first, and the key's place in it
__device__ __forceinline__ int page_index(const AttendArgs &a, int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size; }
__device__ __forceinline__ int place_in_page(const AttendArgs &a, int key) { return a.page_shift >= 0 ? key & (a.page_size - 1) : key % a.page_size; }

// Where a page of a request lies, or -1.
__device__ __forceinline__ int page_of(const AttendArgs &a, int b, int index) {
    const int page = __ldg(a.table + b * a.table_row + index);
    if (page >= 0 && page < a.num_pages) return page;
    if (a.status) atomicOr(a.status, CG_S_BAD_PAGE);
    return -1;
}

// 2^x to 2 units of the last place (0 for -infinity); a weight that is too small for a normal number is 0
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// times in about milliseconds, as bar_wait compares them
__device__ __forceinline__ uint32_t beat_of(uint64_t ns) { return static_cast<uint32_t>(ns >> 20); }
__device__ __forceinline__ void beat(volatile int *failed) { failed[1] = static_cast<int>(beat_of(now_ns())); }

// A lane's values of a row of a head, DP / 32 side by side.
template <int DP> __device__ __forceinline__ void load_mine(const AttendArgs &a, uint64_t row, bool there, uint32_t (&x)[DP / 64]) {
    const int col = (threadIdx.x & 31) * (DP / 32);
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) x[c] = there && col < a.head_size ? __ldg(reinterpret_cast<const unsigned int *>(row) + col / 2 + c) : 0u;
}
template <int DT> __device__ __forceinline__ float half_of(uint32_t pair, int upper) { return Half16<DT>::to_float(static_cast<uint16_t>(pair >> (16 * upper))); }

// One row over keys [k0, k1) by a warp, straight from memory: for rows that do not see a key of their tile whose values are not finite,
// since a weight of zero does not keep those out of a product.  Eight keys on their way at a time.  sums[i] is value lane * (DP / 32) + i of the
// head.
template <int DT, int DP>
__device__ __forceinline__ void slow_row(const AttendArgs &a, const Lengths &r, int b, int head, int row, int k0, int k1, volatile int *failed,
                                      float (&sums)[DP / 32], float &top, float &total) {
    constexpr int kKeys = 8;
    const int lane = threadIdx.x & 31, token = row / a.group;
    uint32_t x[DP / 64];
    load_mine<DP>(a, reinterpret_cast<uint64_t>(a.q + (r.first + token) * a.q_token + (head * a.group + member_of(a, row, token)) * a.q_head), true, x);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) sums[i] = 0.0f;
    top = kNegInf, total = 0.0f;
    k0 = max(k0, first_key(a, r, token)), k1 = min(k1, last_key(a, r, token));
#pragma unroll 1
    for (int j0 = k0; j0 < k1; j0 += 32) {
        const int j = j0 + lane, page = j < k1 ? page_of(a, b, page_index(a, j)) : -1, in_page = place_in_page(a, j);
        const uint64_t k = reinterpret_cast<uint64_t>(a.k + page * a.k_page + in_page * a.k_token + head * a.k_head);
        const uint64_t v = reinterpret_cast<uint64_t>(a.v + page * a.v_page + in_page * a.v_token + head * a.v_head);
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
#pragma unroll 1
        for (int n = 0; n < 32 && j0 + n < k1; n += kKeys) {
            uint32_t y[kKeys][DP / 64], z[kKeys][DP / 64];
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                load_mine<DP>(a, __shfl_sync(0xffffffffu, k, n + i), there >> (n + i) & 1, y[i]);
                load_mine<DP>(a, __shfl_sync(0xffffffffu, v, n + i), there >> (n + i) & 1, z[i]);
            }
            float s[kKeys], now = top;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                s[i] = 0.0f;
                if (there >> (n + i) & 1) {
#pragma unroll
                    for (int c = 0; c < DP / 32; ++c) s[i] += half_of<DT>(x[c / 2], c & 1) * half_of<DT>(y[i][c / 2], c & 1);
                }
                for (int d = 16; d; d >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
                s[i] = j0 + n + i < k1 ? s[i] * a.scale : kNegInf;
                now = fmaxf(now, s[i]);
            }
            const float base = now == kNegInf ? 0.0f : now, keep = exp2_approx(top - base);
            total *= keep;
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) sums[c] *= keep;
#pragma unroll
            for (int i = 0; i < kKeys; ++i) {
                const float w = exp2_approx(s[i] - base);
                total += w;
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) sums[c] += (there >> (n + i) & 1) ? w * half_of<DT>(z[i][c / 2], c & 1) : 0.0f;
            }
            top = now;
        }
        if (lane == 0) beat(failed);  // (others of the block wait for this row)
    }
}

// Which of a warp's `rows` (a bit a lane; a lane's row sees [lo, hi)) have to be done again, because a key that they do not see has values in
// [k0, k1) or [k2, k3) that are not finite.  Where a row sees a value of the same column that is no number, its result is that in any
// case: a cache full of them costs one look at the blocks that not all rows see.  (A call: in line, 8,192
// tokens of 32 heads took as long or 10 us longer, as the kernel's code came to lie.)
template <int DT, int DP>
__device__ __noinline__ uint32_t rows_again(const AttendArgs &a, int b, int head, uint32_t rows, int lo, int hi, int k0, int k1, int k2, int k3) {
    constexpr int kMine = DP / 32;  // columns of a lane
    constexpr uint32_t kExponent = DT == CG_F16 ? 0x7C00u : 0x7F80u, kAll = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    int bad0[kMine], bad1[kMine], nan0[kMine], nan1[kMine];  // the first and last keys
#pragma unroll
    for (int c = 0; c < kMine; ++c) bad0[c] = nan0[c] = INT32_MAX, bad1[c] = nan1[c] = -1;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int to = part ? k3 : k1;
#pragma unroll 1
        for (int j0 = part ? k2 : k0; j0 < to; j0 += 32) {
            const int j = j0 + lane, page = j < to ? page_of(a, b, page_index(a, j)) : -1;
            const uint64_t v = reinterpret_cast<uint64_t>(a.v + page * a.v_page + place_in_page(a, j) * a.v_token + head * a.v_head);
            const uint32_t there = __ballot_sync(kAll, page >= 0);
#pragma unroll 8
            for (int n = 0; n < 32; ++n) {
                uint32_t x[kMine / 2];
                load_mine<DP>(a, __shfl_sync(kAll, v, n), there >> n & 1, x);
#pragma unroll
                for (int c = 0; c < kMine; ++c) {
                    const uint32_t u = x[c / 2] >> (16 * (c % 2)) & 0x7FFFu;
                    if (u >= kExponent) bad0[c] = min(bad0[c], j0 + n), bad1[c] = j0 + n;
                    if (u > kExponent) nan0[c] = min(nan0[c], j0 + n), nan1[c] = j0 + n;
                }
            }
        }
    }
    uint32_t again = 0;
    for (; rows; rows &= rows - 1) {
        const int i = __ffs(rows) - 1, first = __shfl_sync(kAll, lo, i), behind = __shfl_sync(kAll, hi, i);
        bool yes = false;
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
            const bool hidden = bad0[c] < first || bad1[c] >= behind;
            const bool none = (nan0[c] >= first && nan0[c] < behind) || (nan1[c] >= first && nan1[c] < behind);
            yes = yes || (hidden && !none);
        }
        if (__any_sync(kAll, yes)) again |= 1u << i;
    }
    return again;
}

constexpr uint64_t kGiveUpNs = 10ull * 1000 * 1000 * 1000;  // a wait takes microseconds
// ---- barriers in shared memory --------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
// Whether the phase ended.  If it does not within kGiveUpNs, or another wait of the block gave up, the block is told to end, and says so in the
// status.  Behind the word that tells stands the time (see beat) at which the block was last at work on something long, rows done again or a
// piece of many keys: the wait goes on while that is recent.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *failed) {
    uint64_t start = 0;
#pragma unroll 1
    for (uint32_t n = 1; !bar_try(bar, parity); ++n) {
        if (n & 255) continue;
        if (*failed) return false;
        const uint64_t now = now_ns();
        if (!start) start = now;
        if (now - start > kGiveUpNs) {
            if (beat_of(now) - static_cast<uint32_t>(failed[1]) > beat_of(kGiveUpNs)) *failed = 1;
            start = now;
        }
    }
    return true;
}
// the same for a whole warp, with one result
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *failed) { return __all_sync(0xffffffffu, bar_wait(bar, parity, failed)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ Join join_of(const AttendArgs &a, int c) {
    Join j;
    const int4 *from = reinterpret_cast<const int4 *>(a.joins + c);
    reinterpret_cast<int4 *>(&j)[0] = __ldcg(from), reinterpret_cast<int4 *>(&j)[1] = __ldcg(from + 1);
    return j;
}
__device__ __forceinline__ Join join_for(const Piece &p) { return Join{p.sharers, p.r.first, p.r.n, p.r.kv, p.head, p.t, {0, 0}}; }

// Values col .. col + 3 of row `at` of a request and key/value head, from a joined maximum, sum of weights and sums.
template <int DT>
__device__ __forceinline__ void store_joined(const AttendArgs &a, const Lengths &r, int at, int kv_head, int col, float top, float total, float4 sum) {
    const int token = at / a.group, head = kv_head * a.group + member_of(a, at, token);
    const bool sees = last_key(a, r, token) > first_key(a, r, token);
    const float inv = 1.0f / total;
    if (col < a.head_size) {
        const uint16_t h[4] = {Half16<DT>::from_float(sum.x * inv), Half16<DT>::from_float(sum.y * inv), Half16<DT>::from_float(sum.z * inv),
                               Half16<DT>::from_float(sum.w * inv)};
        const uint2 y = make_uint2(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16);
        *reinterpret_cast<uint2 *>(a.out + (r.first + token) * a.out_token + head * a.out_head + 2 * col) = sees ? y : make_uint2(0u, 0u);
    }
    if (a.lse && col == 0)
        a.lse[static_cast<int64_t>(r.first + token) * a.q_heads + head] =
            sees ? ((top == kNegInf ? 0.0f : top) + log2f(total)) * 0.693147180559945f : kNegInf;
}

// Joins what the CTAs of a divided tile of many rows have left.  Block (i, j): 64 rows of the tile that begins in CTA i, a row a thread,
// four 16-byte pieces of it, of four CTAs on their way together: one request's rows over a long context are in dozens.  Sums are stored
// [DP / 4][M][4], as a kernel with a row a thread writes them side by side.
template <int DT, int M, int DP>
__global__ void __launch_bounds__(64 * (DP / 16)) combine_kernel(const __grid_constant__ AttendArgs a) {
    wait_for_launch_before();
    const int c = blockIdx.x, row = blockIdx.y * 64 + threadIdx.x % 64, piece0 = threadIdx.x / 64 * 4;
    const Join join = join_of(a, c);
    if (join.sharers == 0) return;
    const Lengths r{join.first, join.n, join.kv};
    const int64_t at = static_cast<int64_t>(join.t) * M + row;
    if (at >= static_cast<int64_t>(r.n) * a.group) return;
    float top = kNegInf, total = 0.0f;
    float4 sum[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < join.sharers; i += 4) {
        float2 ml[4];
        float4 x[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            ml[n] = make_float2(kNegInf, 0.0f);
            const char *p = a.parts + (2 * (c + i + n) + (i + n == 0)) * part_bytes(M, DP);
            if (i + n < join.sharers) ml[n] = __ldcg(reinterpret_cast<const float2 *>(p + M * DP * 4) + row);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[n][k] = i + n < join.sharers ? __ldcg(reinterpret_cast<const float4 *>(p) + (piece0 + k) * M + row) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float now = fmaxf(top, ml[n].x), base = now == kNegInf ? 0.0f : now;
            const float keep = exp2_approx(top - base), w = exp2_approx(ml[n].x - base);
            total = total * keep + ml[n].y * w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                sum[k].x = sum[k].x * keep + x[n][k].x * w, sum[k].y = sum[k].y * keep + x[n][k].y * w;
                sum[k].z = sum[k].z * keep + x[n][k].z * w, sum[k].w = sum[k].w * keep + x[n][k].w * w;
            }
            top = now;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) store_joined<DT>(a, r, static_cast<int>(at), join.head, 4 * (piece0 + k), top, total, sum[k]);
}

// cg_attend_tiles.cu
int launch_attend_tiles(const AttendArgs &a, int dtype, int ctas, cudaStream_t st);
constexpr int kTileRows = 256, kTileKeys = 128, kTileCost = 2;

}  // namespace cg
