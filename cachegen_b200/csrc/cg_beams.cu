// The best continuations of a request's beams: of all (beam, token) the k with the largest
//     score[beam] + x[beam, token] - log sum_w exp x[beam, w],
// in falling order, equal ones by beam and token.
//
// rows_kernel reads the logits once.  Every thread keeps its largest value and the sum of exponentials against it, and a block keeps a
// value that k of its logits reach: only what lies above that can be among the best, and is written down with its token.  A block's first
// tile gives the value (the k-th largest of its threads' largest), what is written down raises it.  It is bound by memory, and by the
// instructions of the sum: per logit one conversion, half a maximum, and halves of subtraction, product, exponential's own and addition.
//
// choose_kernel joins the blocks' sums of a row, sorts what they wrote down, row by row (there the order is the logits' own), and takes the
// best of the rows' heads k times.  Which of two rows' heads is better depends on both rows' sums, and those, in 32 bits, are known to
// kRowError.  Where two heads are closer than that, the sums of the rows in question are worked out again in 64 bits, from the logits, by all
// blocks of the request's cluster, and the best are taken again: what comes out is ordered by the values in 64 bits.
#include "cg_common.cuh"

#include <math_constants.h>

namespace cg {
namespace {

constexpr int kLogitF32 = CG_LOGITS_F32;
constexpr int kRowThreads = 256, kVectors = 4;             // of rows_kernel; 16-byte vectors of a thread in a tile
constexpr int kTileVectors = kRowThreads * kVectors;
constexpr int kHeld = 1024, kHeldSoft = kHeld / 2;         // candidates of a block, and from how many on it sorts out
constexpr int kChooseBlocks = 8;                           // of a request's cluster
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTilesPerPart = 4;
constexpr int kChooseWarps = 8, kMostChooseWarps = 16, kSorted = 512, kMostList = 4096;
// Relative error of a row's sum in 32 bits, and so the absolute one of its logarithm.  A term exp(-u) is 2 to the power of a product: the
// difference u is off by 2^-24 of itself, the constant by 2^-26, the product by 2^-24, in all 2^-22.8 u; u on average, weighted with the terms, is
// below 17 for up to 2^24 tokens (n terms of one size u beside the largest weigh n u exp(-u) / (1 + n exp(-u))): 2.3e-6.  The power itself: 2^-22.
// A thread's sum is made of 8 additions to each of four accumulators and three to join them a tile, and is carried from tile to tile: at most
// (12 + kTilesPerPart) 2^-24; from there on sums are 64 bits wide.  Moved to a new maximum it takes another product and power, kTilesPerPart + 1
// times at most with the block's: 2^-21.4 each.  In all below 2.3e-6 + 0.3e-6 + 1.0e-6 + 1.8e-6.
constexpr double kRowError = 6e-6;

struct Part {  // what a block found in its part of a row
    double sum;          // of exp(x - top)
    float top, least;    // the largest logit, and one that k logits of the part reach (-infinity if there are no k)
    int32_t count, pad;  // candidates
};
struct Candidate {
    float x;
    int32_t token;
};
struct BeamArgs {
    const void *logits;
    const float *scores;
    float *out;
    int32_t *tokens, *parents;
    Part *parts;             // [rows][nparts]
    Candidate *candidates;   // [rows][nparts][room]
    int64_t row_stride;
    int32_t beams, vocab, k, nparts, part_vectors, room, list_room, sort_room;
};

// A float's bits in an order in which they compare as numbers without a sign; 0 and -0 are the same.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 of_pair(uint64_t p) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(p));
    return d;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int DT> struct Logits;
template <> struct Logits<CG_BF16> {
    using Value = uint16_t;
    static constexpr int kPer = 8;
    static constexpr uint32_t kNone = 0xFF80FF80u;  // -infinity
    static __device__ __forceinline__ float to_float(uint16_t b) { return Half16<CG_BF16>::to_float(b); }
    static __device__ __forceinline__ float2 two(const uint32_t *w, int i) { return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)); }
    static __device__ __forceinline__ float most(const uint32_t *w) {
        const auto at = [&](int i) { return *reinterpret_cast<const __nv_bfloat162 *>(w + i); };
        const __nv_bfloat162 m = __hmax2(__hmax2(at(0), at(1)), __hmax2(at(2), at(3)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
template <> struct Logits<CG_F16> {
    using Value = uint16_t;
    static constexpr int kPer = 8;
    static constexpr uint32_t kNone = 0xFC00FC00u;
    static __device__ __forceinline__ float to_float(uint16_t b) { return Half16<CG_F16>::to_float(b); }
    static __device__ __forceinline__ float2 two(const uint32_t *w, int i) { return __half22float2(*reinterpret_cast<const __half2 *>(w + i)); }
    static __device__ __forceinline__ float most(const uint32_t *w) {
        const auto at = [&](int i) { return *reinterpret_cast<const __half2 *>(w + i); };
        const __half2 m = __hmax2(__hmax2(at(0), at(1)), __hmax2(at(2), at(3)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
template <> struct Logits<kLogitF32> {
    using Value = uint32_t;
    static constexpr int kPer = 4;
    static constexpr uint32_t kNone = 0xFF800000u;
    static __device__ __forceinline__ float to_float(uint32_t b) { return __uint_as_float(b); }
    static __device__ __forceinline__ float2 two(const uint32_t *w, int i) { return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])); }
    static __device__ __forceinline__ float most(const uint32_t *w) {
        return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])), fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
    }
};

// A row's logits in 16-byte vectors of memory: vector v has the tokens v * kPer - shift and on.
template <int DT> struct Row {
    using L = Logits<DT>;
    const typename L::Value *data;
    int32_t vocab, shift;
    __device__ __forceinline__ Row(const BeamArgs &a, int64_t row)
        : data(static_cast<const typename L::Value *>(a.logits) + row * a.row_stride), vocab(a.vocab),
          shift(static_cast<int32_t>(reinterpret_cast<uintptr_t>(data) % 16 / sizeof(typename L::Value))) {}
    __device__ __forceinline__ int32_t vectors() const { return (shift + vocab + L::kPer - 1) / L::kPer; }
    __device__ __forceinline__ int32_t token(int32_t v, int e) const { return v * L::kPer + e - shift; }
    __device__ __forceinline__ float at(int32_t token) const { return L::to_float(data[token]); }
    __device__ __forceinline__ uint4 load(int32_t v) const {
        const int32_t first = v * L::kPer - shift;
        uint4 x;
        if (first >= 0 && first <= vocab - L::kPer) {
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(data + first));
            return x;
        }
        uint32_t w[4];  // the row's ends
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = L::kNone;
#pragma unroll
        for (int e = 0; e < L::kPer; ++e) {
            const int32_t t = first + e;
            if (t < 0 || t >= vocab) continue;
            const uint32_t b = __ldg(data + t);
            if (L::kPer == 4) w[e & 3] = b;
            else w[e / 2] = e & 1 ? (w[e / 2] & 0xFFFFu) | b << 16 : (w[e / 2] & 0xFFFF0000u) | b;
        }
        x = make_uint4(w[0], w[1], w[2], w[3]);
        return x;
    }
};
template <int DT> __device__ __forceinline__ float value_of(const uint4 &x, int e) {
    const float2 two = Logits<DT>::two(reinterpret_cast<const uint32_t *>(&x), e / 2);
    return e & 1 ? two.y : two.x;
}

struct Shared {
    Candidate held[kHeld];
    int32_t nheld, sums[2][kRowThreads / 32];
    float tops[kRowThreads / 32];
    double parts[kRowThreads / 32];
};
// Sum over the block; `turn` alternates.
__device__ __forceinline__ int32_t block_sum(Shared &s, int32_t x, int turn) {
    const int32_t w = __reduce_add_sync(~0u, x);
    if (threadIdx.x % 32 == 0) s.sums[turn & 1][threadIdx.x / 32] = w;
    __syncthreads();
    int32_t all = 0;
#pragma unroll
    for (int i = 0; i < kRowThreads / 32; ++i) all += s.sums[turn & 1][i];
    return all;
}

// Keeps exactly the k first of `n` candidates and the elements that `more` goes through, by value and then by token (or all, if there are fewer
// than k), bit by bit: what comes last is only met where values are equal by the hundred or rise along a row.  more(f) calls f(value, token).
// Returns what k of them reach, or -infinity.
template <class More>
__device__ __noinline__ float keep_first(Shared &s, int32_t n, int32_t k, More more) {
    Candidate mine[kHeld / kRowThreads];
#pragma unroll
    for (int i = 0; i < kHeld / kRowThreads; ++i) {
        const int32_t at = i * kRowThreads + threadIdx.x;
        mine[i] = at < n ? s.held[at] : Candidate{-CUDART_INF_F, 0};
    }
    const auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kHeld / kRowThreads; ++i)
            if (mine[i].x > -CUDART_INF_F) f(ordered(mine[i].x), mine[i].token);
        more([&](float x, int32_t token) {
            if (x > -CUDART_INF_F) f(ordered(x), token);
        });
    };
    int turn = 0;
    uint32_t least = 0;  // the largest that k of them reach; 0: there are fewer
    for (int bit = 31; bit >= 0; --bit) {
        int32_t c = 0;
        each([&](uint32_t key, int32_t) { c += key >= (least | 1u << bit); });
        if (block_sum(s, c, turn++) >= k) least |= 1u << bit;
    }
    int32_t above = 0;
    each([&](uint32_t key, int32_t) { above += key > least; });
    const int32_t wanted = k - block_sum(s, above, turn++);
    uint32_t last = 0;  // the token up to which `wanted` of the equal ones lie
    if (least) {
        for (int bit = 30; bit >= 0; --bit) {
            int32_t c = 0;
            const uint32_t below = last | 1u << bit;
            each([&](uint32_t key, int32_t token) { c += key == least && static_cast<uint32_t>(token) < below; });
            if (block_sum(s, c, turn++) < wanted) last |= 1u << bit;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) s.nheld = 0;
    __syncthreads();
    each([&](uint32_t key, int32_t token) {
        if (key > least || (key == least && static_cast<uint32_t>(token) <= last)) s.held[atomicAdd(&s.nheld, 1)] = Candidate{from_ordered(key), token};
    });
    __syncthreads();
    return least ? from_ordered(least) : -CUDART_INF_F;
}

// A value that k of the block's keys reach, to 16 bits; 0 if there are fewer of them (above that of -infinity).  key(i), i < N: a thread's.
template <int N, class Key>
__device__ __forceinline__ uint32_t reached(int32_t k, Key key) {
    uint32_t mine[N], least = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        mine[i] = key(i);
        if (mine[i] <= ordered(-CUDART_INF_F)) mine[i] = 0;
    }
    for (int bit = 31; bit >= 16; --bit) {
        int32_t c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __syncthreads_count(mine[i] >= (least | 1u << bit));
        if (c >= k) {
            least |= 1u << bit;
            if (c == k) break;
        }
    }
    return least;
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const __grid_constant__ BeamArgs a) {
    using L = Logits<DT>;
    __shared__ Shared s;
    const int32_t row = blockIdx.x / a.nparts, part = blockIdx.x - row * a.nparts, tid = threadIdx.x, k = a.k;
    let_next_launch_start();
    Part *const out = a.parts + blockIdx.x;
    const float score = __ldg(a.scores + row);
    if (!(fabsf(score) < CUDART_INF_F)) {  // a beam that has not begun
        if (tid == 0) *out = Part{0.0, -CUDART_INF_F, -CUDART_INF_F, 0, 0};
        return;
    }
    const Row<DT> x(a, row);
    const int32_t all = x.vectors(), from = min(all, part * a.part_vectors), to = min(all, from + a.part_vectors);
    if (tid == 0) s.nheld = 0;
    float top = -CUDART_INF_F, sum = 0.0f, least = -CUDART_INF_F;
    int32_t n = 0;
    const uint64_t scale = pair_of(kLog2e, kLog2e);
    uint4 next[kVectors];
    const auto fetch = [&](int32_t v0) {
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
            const int32_t v = v0 + u * kRowThreads + tid;
            next[u] = v < to ? x.load(v) : make_uint4(L::kNone, L::kNone, L::kNone, L::kNone);
        }
    };
    fetch(from);
    for (int32_t v0 = from; v0 < to; v0 += kTileVectors) {
        uint4 now[kVectors];
        float most[kVectors];
#pragma unroll
        for (int u = 0; u < kVectors; ++u) now[u] = next[u];
        if (v0 + kTileVectors < to) fetch(v0 + kTileVectors);
#pragma unroll
        for (int u = 0; u < kVectors; ++u) most[u] = L::most(reinterpret_cast<const uint32_t *>(&now[u]));
        const float tile = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        const float higher = fmaxf(top, tile);
        if (higher > -CUDART_INF_F) {
            const uint64_t minus = pair_of(-higher, -higher);
            uint64_t acc[2] = {pair_of(__fmul_rn(sum, power2(__fmul_rn(__fsub_rn(top, higher), kLog2e))), 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll
            for (int u = 0; u < kVectors; ++u) {
#pragma unroll
                for (int i = 0; i < L::kPer / 2; ++i) {
                    const float2 two = L::two(reinterpret_cast<const uint32_t *>(&now[u]), i);
                    const float2 y = of_pair(pair_mul(pair_add(pair_of(two.x, two.y), minus), scale));
                    acc[i & 1] = pair_add(acc[i & 1], pair_of(power2(y.x), power2(y.y)));
                }
            }
            const float2 both = of_pair(pair_add(acc[0], acc[1]));
            sum = __fadd_rn(both.x, both.y);
            top = higher;
        }
        // candidates: of the first tile what reaches the k-th largest of the threads' largest, of the others what lies above what k logits
        // in front of it reach
        const bool first = v0 == from;
        if (first) {
            const uint32_t key = reached<1>(k, [&](int) { return ordered(tile); });
            least = key ? from_ordered(key) : -CUDART_INF_F;
        }
        const auto above = [&](float y) { return first ? y >= least && y > -CUDART_INF_F : y > least; };
        const bool any = above(tile);
        if (any) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u) {
                if (!above(most[u])) continue;
#pragma unroll
                for (int e = 0; e < L::kPer; ++e) {
                    const float y = value_of<DT>(now[u], e);
                    if (above(y)) {
                        const int32_t at = atomicAdd(&s.nheld, 1);
                        if (at < kHeld) s.held[at] = Candidate{y, x.token(v0 + u * kRowThreads + tid, e)};
                    }
                }
            }
        }
        if (__syncthreads_or(any)) {
            const int32_t found = s.nheld;
            if (found > kHeld) {  // what was held in front of this tile is whole
                uint4 copy[kVectors];  // (what is handed on by address would never be in registers)
#pragma unroll
                for (int u = 0; u < kVectors; ++u) copy[u] = now[u];
                const int32_t token0 = x.token(v0 + tid, 0);
                least = keep_first(s, n, k, [&](auto f) {
#pragma unroll
                    for (int u = 0; u < kVectors; ++u)
#pragma unroll
                        for (int e = 0; e < L::kPer; ++e) f(value_of<DT>(copy[u], e), token0 + u * kRowThreads * L::kPer + e);
                });
            } else if (found > kHeldSoft) {
                least = keep_first(s, found, k, [](auto) {});
            }
            n = found > kHeldSoft ? s.nheld : found;
            __syncthreads();
        }
    }
    // raised by what is held, or cut to k
    if (n > k) {
        const uint32_t key = reached<kHeldSoft / kRowThreads>(k, [&](int i) {
            const int32_t at = i * kRowThreads + tid;
            return at < n ? ordered(s.held[at].x) : 0u;
        });
        if (key) least = fmaxf(least, from_ordered(key));
        int32_t left = 0;
#pragma unroll
        for (int i = 0; i < kHeldSoft / kRowThreads; ++i) {
            const int32_t at = i * kRowThreads + tid;
            left += __syncthreads_count(at < n && s.held[at].x >= least);
        }
        if (left > a.room) {  // equal ones
            least = keep_first(s, n, k, [](auto) {});
            n = s.nheld;
        }
    }
    // the block's sum
    const int lane = tid % 32, warp = tid / 32;
    float high = top;
#pragma unroll
    for (int d = 16; d; d /= 2) high = fmaxf(high, __shfl_xor_sync(~0u, high, d));
    if (lane == 0) s.tops[warp] = high;
    const bool odd = sum != sum || top == CUDART_INF_F;  // NaN or infinity among the logits
    const bool again = __syncthreads_or(odd);
#pragma unroll
    for (int i = 0; i < kRowThreads / 32; ++i) high = fmaxf(high, s.tops[i]);
    double mine = 0.0;
    if (again) {
        for (int32_t v = from + tid; v < to; v += kRowThreads) {
            for (int e = 0; e < L::kPer; ++e) {
                const int32_t t = x.token(v, e);
                if (t < 0 || t >= a.vocab) continue;
                const float y = x.at(t);
                if (high == CUDART_INF_F) mine += y == CUDART_INF_F;
                else if (y > -CUDART_INF_F) mine += power2(__fmul_rn(__fsub_rn(y, high), kLog2e));
            }
        }
    } else if (high > -CUDART_INF_F) {
        mine = __fmul_rn(sum, power2(__fmul_rn(__fsub_rn(top, high), kLog2e)));
    }
#pragma unroll
    for (int d = 16; d; d /= 2) mine += __shfl_xor_sync(~0u, mine, d);
    if (lane == 0) s.parts[warp] = mine;
    if (tid == 0) s.nheld = 0;
    __syncthreads();
    for (int32_t at = tid; at < n; at += kRowThreads) {
        const Candidate c = s.held[at];
        if (c.x >= least) a.candidates[static_cast<int64_t>(blockIdx.x) * a.room + atomicAdd(&s.nheld, 1)] = c;
    }
    __syncthreads();
    if (tid == 0) {
        double sum_all = 0.0;
        for (int i = 0; i < kRowThreads / 32; ++i) sum_all += s.parts[i];
        *out = Part{sum_all, high, least, s.nheld, 0};
    }
}

// ---- choose ------------------------------------------------------------------------------------------------
__device__ __forceinline__ int choose_rank() {
    int r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_block(const void *mine, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(mine)), "r"(rank));
    return at;
}
__device__ __forceinline__ uint32_t word_of_block(const uint32_t *mine, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at_block(mine, rank)) : "memory");
    return v;
}
__device__ __forceinline__ double double_of_block(const double *mine, int rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at_block(mine, rank)) : "memory");
    return v;
}

// Candidates as one number: by value, then the lower token first.
__device__ __forceinline__ uint64_t key_of(const Candidate &c) { return static_cast<uint64_t>(ordered(c.x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(c.token)); }

// One warp: a row's candidates that reach `least`, those of all its blocks, sorted; the first k to `to`.  Returns how many.
__device__ int32_t sort_row(const BeamArgs &a, int32_t row, float least, uint64_t *room, uint64_t *to) {
    const int lane = threadIdx.x % 32;
    const Part *const parts = a.parts + static_cast<int64_t>(row) * a.nparts;
    const Candidate *const candidates = a.candidates + static_cast<int64_t>(row) * a.nparts * a.room;
    const auto each = [&](auto f) {  // f(whether there is one, its key), by all lanes together
        for (int32_t p = 0; p < a.nparts; ++p) {
            const int32_t count = __ldcg(&parts[p].count);
            for (int32_t i0 = 0; i0 < count; i0 += 32) {
                Candidate c{-CUDART_INF_F, 0};
                if (i0 + lane < count) {
                    const float2 w = __ldcg(reinterpret_cast<const float2 *>(candidates + static_cast<int64_t>(p) * a.room + i0 + lane));
                    c = Candidate{w.x, __float_as_int(w.y)};
                }
                f(c.x >= least && c.x > -CUDART_INF_F, key_of(c));
            }
        }
    };
    int32_t n = 0;
    each([&](bool there, uint64_t key) {
        const uint32_t who = __ballot_sync(~0u, there);
        const int32_t at = n + __popc(who & ((1u << lane) - 1u));
        if (there && at < a.sort_room) room[at] = key;
        n += __popc(who);
    });
    if (n > a.sort_room) {  // many equal ones: the k-th key, bit by bit, then only what reaches it (keys differ)
        uint64_t kth = 0;
        for (int bit = 63; bit >= 0; --bit) {
            int32_t c = 0;
            each([&](bool there, uint64_t key) { c += __popc(__ballot_sync(~0u, there && key >= (kth | 1ull << bit))); });
            if (c >= a.k) kth |= 1ull << bit;
        }
        n = 0;
        each([&](bool there, uint64_t key) {
            const uint32_t who = __ballot_sync(~0u, there && key >= kth);
            const int32_t at = n + __popc(who & ((1u << lane) - 1u));
            if (who >> lane & 1) room[at] = key;
            n += __popc(who);
        });
    }
    int32_t size = 32;
    while (size < n) size *= 2;
    for (int32_t i = n + lane; i < size; i += 32) room[i] = 0;
    __syncwarp();
    for (int32_t run = 2; run <= size; run *= 2) {
        for (int32_t d = run / 2; d; d /= 2) {
            for (int32_t i = lane; i < size / 2; i += 32) {
                const int32_t lo = i / d * 2 * d + i % d, hi = lo + d;
                const uint64_t p = room[lo], q = room[hi];
                if ((p < q) == ((lo & run) == 0)) room[lo] = q, room[hi] = p;
            }
            __syncwarp();
        }
    }
    const int32_t kept = n < a.k ? n : a.k;
    for (int32_t i = lane; i < kept; i += 32) to[i] = room[i];
    return kept;
}

// A continuation of a request: its score, and what decides between equal ones, the beam, the logit and the token in one number.
struct Choice {
    double total;
    uint64_t rest;
    __device__ __forceinline__ int32_t beam() const { return 255 - static_cast<int32_t>(rest >> 56); }
    __device__ __forceinline__ int32_t token() const { return 0xFFFFFF - static_cast<int32_t>(rest & 0xFFFFFF); }
    __device__ __forceinline__ float x() const { return from_ordered(static_cast<uint32_t>(rest >> 24)); }
    __device__ __forceinline__ bool before(const Choice &o) const { return total > o.total || (total == o.total && rest > o.rest); }
};
__device__ __forceinline__ uint64_t rest_of(int32_t beam, float x, int32_t token) {
    return static_cast<uint64_t>(255 - beam) << 56 | static_cast<uint64_t>(ordered(x)) << 24 | static_cast<uint64_t>(0xFFFFFF - token);
}
__device__ __forceinline__ uint64_t ordered_double(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(__dadd_rn(x, 0.0)));
    return u >> 63 ? ~u : u | 1ull << 63;
}

// How room in shared memory is divided; K beams, W warps
struct ChooseRoom {
    double *base, *sums;      // [K]: score - log sum exp(x - top); a block's share of a sum
    Choice *list, *sorted;    // [list_room], [kSorted]; in their place, where these are too small,
    uint64_t *best, *sorting; // [K][k], [W][sort_room]
    float *top;               // [K]
    int32_t *count;           // [K]
    uint32_t *near;           // [K]: whether the sum is wanted in 64 bits; near[K]: whether any is
    static __host__ __device__ size_t lists(const BeamArgs &a, int warps) {
        const size_t usual = sizeof(Choice) * (static_cast<size_t>(a.list_room) + kSorted);
        const size_t other = sizeof(uint64_t) * (static_cast<size_t>(a.beams) * a.k + static_cast<size_t>(warps) * a.sort_room);
        return (usual > other ? usual : other) + 15 & ~static_cast<size_t>(15);
    }
    static size_t bytes(const BeamArgs &a, int warps) { return lists(a, warps) + a.beams * (2 * sizeof(double) + 3 * sizeof(float)) + sizeof(float); }
    __device__ ChooseRoom(char *at, const BeamArgs &a, int warps) {
        list = reinterpret_cast<Choice *>(at);
        sorted = list + a.list_room;
        best = reinterpret_cast<uint64_t *>(at);
        sorting = best + static_cast<int64_t>(a.beams) * a.k;
        base = reinterpret_cast<double *>(at + lists(a, warps));
        sums = base + a.beams;
        top = reinterpret_cast<float *>(sums + a.beams);
        count = reinterpret_cast<int32_t *>(top + a.beams);
        near = reinterpret_cast<uint32_t *>(count + a.beams);
    }
};

// x against the row's largest, so that logits of any size leave the scores their digits; where that is infinite, those that are share the row.
__device__ __forceinline__ double entering(float x, float top) {
    if (top < CUDART_INF_F) return static_cast<double>(x) - top;
    return x == CUDART_INF_F ? 0.0 : -CUDART_INF;
}

// One warp: the best of the heads of the rows' sorted candidates, k times.  doubt: marks rows whose heads are too close for sums in 32 bits.
__device__ bool take_best(const BeamArgs &a, const ChooseRoom &r, int32_t request, bool doubt) {
    const int lane = threadIdx.x % 32;
    const int32_t mine = (a.beams - lane + 31) / 32;  // rows lane, lane + 32, ...: their heads, a byte each
    uint64_t heads = 0;
    bool doubtful = false;
    float *const out = a.out + static_cast<int64_t>(request) * a.k;
    int32_t *const tokens = a.tokens + static_cast<int64_t>(request) * a.k, *const parents = a.parents + static_cast<int64_t>(request) * a.k;
    const auto head_of = [&](int32_t j) {
        const int32_t row = lane + 32 * j, at = static_cast<int32_t>(heads >> 8 * j & 0xFF);
        return at < r.count[row] ? r.base[row] + entering(from_ordered(static_cast<uint32_t>(r.best[row * a.k + at] >> 32)), r.top[row]) : -CUDART_INF;
    };
    for (int32_t i = 0; i < a.k; ++i) {
        double best = -CUDART_INF;
        int32_t which = 0;
        for (int32_t j = 0; j < mine; ++j) {
            const double v = head_of(j);
            if (v > best) best = v, which = j;
        }
        double most = best;
        int32_t row = best > -CUDART_INF ? lane + 32 * which : INT32_MAX;
#pragma unroll
        for (int d = 16; d; d /= 2) {
            const double v = __shfl_xor_sync(~0u, most, d);
            const int32_t w = __shfl_xor_sync(~0u, row, d);
            if (v > most || (v == most && w < row)) most = v, row = w;
        }
        if (!(most > -CUDART_INF)) {  // nothing is left
            for (int32_t rest = i + lane; rest < a.k; rest += 32) out[rest] = -CUDART_INF_F, tokens[rest] = -1, parents[rest] = -1;
            break;
        }
        if (doubt) {
            bool near = false;
            for (int32_t j = 0; j < mine; ++j)
                if (lane + 32 * j != row && head_of(j) >= most - 2.0 * kRowError) r.near[lane + 32 * j] = 1, near = true;
            if (__any_sync(~0u, near)) {
                doubtful = true;
                if (lane == 0) r.near[row] = 1;
            }
        }
        if (row % 32 == lane) {
            const int32_t j = row / 32;
            const uint64_t key = r.best[row * a.k + static_cast<int32_t>(heads >> 8 * j & 0xFF)];
            out[i] = static_cast<float>(most);
            tokens[i] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
            parents[i] = request * a.beams + row;
            heads += 1ull << 8 * j;
        }
    }
    __syncwarp();
    return doubtful;
}

// The block puts n continuations in order: each counts those in front of it.
__device__ __forceinline__ void sort_list(const Choice *list, Choice *sorted, int32_t n) {
    for (int32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const Choice mine = list[i];
        int32_t place = 0;
        for (int32_t j = 0; j < n; ++j) place += list[j].before(mine);
        sorted[place] = mine;
    }
    __syncthreads();
}
__device__ __forceinline__ void write_sorted(const BeamArgs &a, const Choice *sorted, int32_t request, int32_t n) {
    for (int32_t i = threadIdx.x; i < a.k; i += blockDim.x) {
        const int64_t at = static_cast<int64_t>(request) * a.k + i;
        const bool there = i < n;
        const Choice c = sorted[there ? i : 0];
        a.out[at] = there ? static_cast<float>(c.total) : -CUDART_INF_F;
        a.tokens[at] = there ? c.token() : -1;
        a.parents[at] = there ? request * a.beams + c.beam() : -1;
    }
}
// The continuations that may be among the best, in *list; returns how many there are, more than `kSorted` if that is no use.  A bound that k of
// one row reach drops most of them while they are read, the k-th largest of what is left (by the upper half of its bits) nearly all of the others; both with
// room for what 32-bit sums are off.  *sorted is as large as kSorted.
__device__ __forceinline__ int32_t gather_choices(const BeamArgs &a, const ChooseRoom &r, int32_t request, int32_t *counts, Choice **list, Choice **sorted) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    double bound = -CUDART_INF;
    for (int32_t i = lane; i < a.beams; i += 32) bound = fmax(bound, r.sums[i]);
#pragma unroll
    for (int d = 16; d; d /= 2) bound = fmax(bound, __shfl_xor_sync(~0u, bound, d));
    bound -= 2.0 * kRowError;
    const int32_t pairs = a.beams * a.nparts;
    const int64_t first = static_cast<int64_t>(request) * pairs;
    for (int32_t p0 = warp; p0 < pairs; p0 += 32 * warps) {
        const int32_t mine = p0 + lane * warps;
        int32_t count = 0;
        if (mine < pairs) {
            const Part *const part = a.parts + first + mine;
            const int32_t beam = mine / a.nparts;
            const float top = __ldcg(&part->top);
            count = __ldcg(&part->count);
            if (!(r.base[beam] + entering(top, r.top[beam]) >= bound)) count = 0;
        }
        for (uint32_t left = __ballot_sync(~0u, count > 0); left; left &= left - 1) {
            const int from = __ffs(left) - 1, pair = p0 + from * warps, beam = pair / a.nparts;
            const int32_t n = __shfl_sync(~0u, count, from);
            const float2 *const candidates = reinterpret_cast<const float2 *>(a.candidates + (first + pair) * a.room);
            for (int32_t i = lane; i < n; i += 32) {
                const float2 c = __ldcg(candidates + i);
                const double total = r.base[beam] + entering(c.x, r.top[beam]);
                if (total >= bound && total > -CUDART_INF) {
                    const int32_t at = atomicAdd(&counts[0], 1);
                    if (at < a.list_room) r.list[at] = Choice{total, rest_of(beam, c.x, __float_as_int(c.y))};
                }
            }
        }
    }
    __syncthreads();
    const int32_t n = counts[0];
    if (n > a.list_room) return INT32_MAX;
    if (n <= 2 * a.k + 32) return n;
    uint32_t least = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t want = least | 1u << bit;
        int32_t c = 0;
        for (int32_t i = threadIdx.x; i < n; i += blockDim.x) c += ordered_double(r.list[i].total) >> 32 >= want;
        c = __reduce_add_sync(~0u, c);
        int32_t *const sum = counts + 1 + bit % 3;  // one is filled, one is read, one is set back
        if (lane == 0 && c) atomicAdd(sum, c);
        __syncthreads();
        if (*sum >= a.k) least = want;
        if (threadIdx.x == 0) counts[1 + (bit + 1) % 3] = 0;
    }
    const uint64_t u = static_cast<uint64_t>(least) << 32;
    bound = __longlong_as_double(static_cast<long long>(u >> 63 ? u & ~(1ull << 63) : ~u)) - 2.0 * kRowError;
    if (threadIdx.x == 0) counts[0] = 0;
    __syncthreads();
    for (int32_t i = threadIdx.x; i < n; i += blockDim.x) {
        if (r.list[i].total < bound) continue;
        const int32_t at = atomicAdd(&counts[0], 1);
        if (at < kSorted) r.sorted[at] = r.list[i];
    }
    __syncthreads();
    *list = r.sorted, *sorted = r.list;
    return counts[0];
}

// A cluster a request.  Its first block chooses; the others wait to be asked for sums in 64 bits.
template <int DT>
__global__ void __cluster_dims__(kChooseBlocks, 1, 1) __launch_bounds__(kMostChooseWarps * 32) choose_kernel(const __grid_constant__ BeamArgs a) {
    extern __shared__ __align__(16) char room[];
    __shared__ double warps_sums[16];
    __shared__ int32_t counts[4];
    const int rank = choose_rank(), lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const int32_t request = blockIdx.x / kChooseBlocks;
    const ChooseRoom r(room, a, warps);
    Choice *list = r.list, *sorted = r.sorted;
    int32_t n = 0;
    if (rank == 0) {
        for (int32_t i = threadIdx.x; i <= a.beams; i += blockDim.x) r.near[i] = 0;
        if (threadIdx.x < 4) counts[threadIdx.x] = 0;
        wait_for_launch_before();
        for (int32_t i = warp; i < a.beams; i += warps) {
            const int32_t row = request * a.beams + i;
            const Part *const parts = a.parts + static_cast<int64_t>(row) * a.nparts;
            float top = -CUDART_INF_F, least = -CUDART_INF_F;
            for (int32_t p = lane; p < a.nparts; p += 32) top = fmaxf(top, __ldcg(&parts[p].top)), least = fmaxf(least, __ldcg(&parts[p].least));
#pragma unroll
            for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, d)), least = fmaxf(least, __shfl_xor_sync(~0u, least, d));
            double sum = 0.0;
            for (int32_t p = lane; p < a.nparts; p += 32) {
                const float high = __ldcg(&parts[p].top);
                if (high == top) sum += __ldcg(&parts[p].sum);
                else if (high > -CUDART_INF_F && top < CUDART_INF_F) sum += __ldcg(&parts[p].sum) * exp(static_cast<double>(high) - top);
            }
#pragma unroll
            for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == 0) {
                const bool any = top > -CUDART_INF_F;
                const double base = any ? static_cast<double>(__ldg(a.scores + row)) - log(sum) : -CUDART_INF;
                r.top[i] = top;
                r.base[i] = base;
                r.sums[i] = any && least > -CUDART_INF_F ? base + entering(least, top) : -CUDART_INF;
            }
        }
        __syncthreads();
        n = gather_choices(a, r, request, counts, &list, &sorted);
        if (n <= kSorted) {
            sort_list(list, sorted, n);
            for (int32_t i = threadIdx.x; i + 1 < n; i += blockDim.x) {
                const Choice &p = sorted[i], &q = sorted[i + 1];
                if (p.total - q.total <= 2.0 * kRowError && p.beam() != q.beam() && (i < a.k || sorted[a.k - 1].total - p.total <= 2.0 * kRowError))
                    r.near[p.beam()] = r.near[q.beam()] = r.near[a.beams] = 1;
            }
            __syncthreads();
            if (!r.near[a.beams]) write_sorted(a, sorted, request, n);
        } else {  // many equal ones: row by row
            for (int32_t i = warp; i < a.beams; i += warps) {
                const int32_t row = request * a.beams + i;
                float least = -CUDART_INF_F;
                for (int32_t p = lane; p < a.nparts; p += 32) least = fmaxf(least, __ldcg(&a.parts[static_cast<int64_t>(row) * a.nparts + p].least));
#pragma unroll
                for (int d = 16; d; d /= 2) least = fmaxf(least, __shfl_xor_sync(~0u, least, d));
                const int32_t found = r.top[i] > -CUDART_INF_F ? sort_row(a, row, least, r.sorting + warp * a.sort_room, r.best + i * a.k) : 0;
                if (lane == 0) r.count[i] = found;
            }
            __syncthreads();
            if (warp == 0 && take_best(a, r, request, true) && lane == 0) r.near[a.beams] = 1;
        }
    }
    cluster_barrier();
    const bool again = word_of_block(r.near + a.beams, 0);
    if (again) {
        wait_for_launch_before();
        for (int32_t i = 0; i < a.beams; ++i) {
            if (!word_of_block(r.near + i, 0)) continue;  // (the same for all threads)
            const float top = __uint_as_float(word_of_block(reinterpret_cast<const uint32_t *>(r.top + i), 0));
            double sum = 0.0;
            if (top < CUDART_INF_F) {
                const Row<DT> x(a, static_cast<int64_t>(request) * a.beams + i);
                for (int32_t t = rank * blockDim.x + threadIdx.x; t < a.vocab; t += kChooseBlocks * blockDim.x) {
                    const float y = x.at(t);
                    if (y > -CUDART_INF_F) sum += exp(static_cast<double>(y) - top);
                }
            }
#pragma unroll
            for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
            __syncthreads();
            if (lane == 0) warps_sums[warp] = sum;
            __syncthreads();
            if (threadIdx.x == 0) {
                sum = 0.0;
                for (int w = 0; w < warps; ++w) sum += warps_sums[w];
                r.sums[i] = sum;
            }
        }
        cluster_barrier();
        if (rank == 0) {
            for (int32_t i = threadIdx.x; i < a.beams; i += blockDim.x) {
                if (!r.near[i] || r.top[i] == CUDART_INF_F) continue;
                double sum = 0.0;
                for (int b = 0; b < kChooseBlocks; ++b) sum += double_of_block(r.sums + i, b);
                r.base[i] = static_cast<double>(__ldg(a.scores + static_cast<int64_t>(request) * a.beams + i)) - log(sum);
            }
            __syncthreads();
            if (n > kSorted) {
                if (warp == 0) take_best(a, r, request, false);
            } else {
                for (int32_t i = threadIdx.x; i < n; i += blockDim.x) {
                    Choice &c = list[i];
                    c.total = r.base[c.beam()] + entering(c.x(), r.top[c.beam()]);
                }
                __syncthreads();
                sort_list(list, sorted, n);
                write_sorted(a, sorted, request, n);
            }
        }
    }
    cluster_barrier();  // nobody reads another block's memory any more
}

struct Sizes {
    int32_t nparts, part_vectors, room;
    int64_t parts_bytes, total;
};
int64_t row_vectors(const cg_beam_job &j) {
    const int per = j.dtype == kLogitF32 ? 4 : 8;
    return (static_cast<int64_t>(j.vocab) + 2 * (per - 1)) / per;  // the row may begin inside a vector
}
// Parts of a row: at most four tiles long, so that a part's end is not far and the bound on the sums' errors holds; shorter as long as
// that fills the GPU, but not below a tile.
Sizes sizes_of(const cg_beam_job &j, int sms) {
    Sizes z{};
    const int64_t vectors = row_vectors(j), tiles = (vectors + kTileVectors - 1) / kTileVectors, rows = static_cast<int64_t>(j.nrequests) * j.beams;
    int64_t parts = (8 * static_cast<int64_t>(sms) + rows - 1) / rows;
    if (parts > tiles) parts = tiles;
    if (parts < (tiles + kTilesPerPart - 1) / kTilesPerPart) parts = (tiles + kTilesPerPart - 1) / kTilesPerPart;
    z.part_vectors = static_cast<int32_t>((tiles + parts - 1) / parts * kTileVectors);
    z.nparts = static_cast<int32_t>((vectors + z.part_vectors - 1) / z.part_vectors);
    z.room = 4 * j.k > 64 ? 4 * j.k : 64;
    z.parts_bytes = (rows * z.nparts * static_cast<int64_t>(sizeof(Part)) + 15) / 16 * 16;
    z.total = z.parts_bytes + rows * z.nparts * z.room * static_cast<int64_t>(sizeof(Candidate));
    return z;
}

int check_job(const cg_beam_job *job) {
    if (!job) return CG_E_NULL;
    const cg_beam_job &j = *job;
    if (j.dtype != CG_F16 && j.dtype != CG_BF16 && j.dtype != kLogitF32) return CG_E_DTYPE;
    if (j.nrequests < 0 || j.beams <= 0 || j.vocab <= 0 || j.k <= 0 || j.vocab > CG_MAX_VOCAB) return CG_E_SHAPE;
    if (j.beams > CG_MAX_BEAMS || j.k > CG_MAX_CHOICES || j.beams * j.k > CG_MAX_BEAM_CHOICES || static_cast<int64_t>(j.nrequests) * j.beams > (1 << 20))
        return CG_E_CAPACITY;
    return CG_OK;
}

template <int DT>
int run(BeamArgs &a, int32_t nrequests, cudaStream_t st) {
    const int64_t blocks = static_cast<int64_t>(nrequests) * a.beams * a.nparts;
    if (blocks > INT32_MAX) return CG_E_CAPACITY;
    const int warps = a.beams > kChooseWarps ? kMostChooseWarps : kChooseWarps;
    const size_t smem = ChooseRoom::bytes(a, warps);
    if (const int rc = allow_smem(choose_kernel<DT>, smem)) return rc;
    if (const int rc = launch(rows_kernel<DT>, dim3(static_cast<unsigned>(blocks)), kRowThreads, 0, false, st, a)) return rc;
    return launch(choose_kernel<DT>, dim3(static_cast<unsigned>(nrequests) * kChooseBlocks), warps * 32, smem, true, st, a);
}

}  // namespace
}  // namespace cg

extern "C" int64_t cg_beam_workspace(const cg_beam_job *job) {
    if (const int rc = cg::check_job(job)) return rc;
    return job->nrequests ? cg::sizes_of(*job, cg::sm_count()).total : 0;
}

extern "C" int cg_beam_select(const cg_beam_job *job, void *stream) {
    using namespace cg;
    if (const int rc = check_job(job)) return rc;
    const cg_beam_job &j = *job;
    if (j.nrequests == 0) return CG_OK;
    if (!j.logits || !j.scores || !j.out_scores || !j.tokens || !j.parents) return CG_E_NULL;
    const Sizes z = sizes_of(j, sm_count());
    if (!j.workspace || j.workspace_bytes < z.total) return CG_E_CAPACITY;
    if (reinterpret_cast<uintptr_t>(j.workspace) % 16 || reinterpret_cast<uintptr_t>(j.logits) % (j.dtype == kLogitF32 ? 4 : 2)) return CG_E_ALIGN;
    int sort_room = 64;
    while (sort_room < 4 * j.k && sort_room < 512) sort_room *= 2;
    const int list_room = 4 * j.beams * j.k < kSorted ? kSorted : 4 * j.beams * j.k < kMostList ? 4 * j.beams * j.k : kMostList;
    BeamArgs a{j.logits, j.scores, j.out_scores, j.tokens, j.parents, static_cast<Part *>(j.workspace),
               reinterpret_cast<Candidate *>(static_cast<char *>(j.workspace) + z.parts_bytes), j.row_stride,
               j.beams, j.vocab, j.k, z.nparts, z.part_vectors, z.room, list_room, sort_room};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (j.dtype == CG_F16) return run<CG_F16>(a, j.nrequests, st);
    if (j.dtype == CG_BF16) return run<CG_BF16>(a, j.nrequests, st);
    return run<kLogitF32>(a, j.nrequests, st);
}
