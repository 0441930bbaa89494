// The best continuations of a request's beams: of all (beam, token) the k with the largest
//     score[beam] + x[beam, token] - log sum_w exp x[beam, w],
// in falling order, equal ones by beam and token.
//
// rows_kernel reads the logits once.  All rows' tiles of 16 KB stand in one line, and every block takes a run of it; what it has of one row is a
// part.  A thread keeps its largest value and a sum of exponentials.  k of a part's logits reach the k-th largest of its threads' largest; what does not
// reach it cannot be among the best, and the rest, little more than k, is read again and written down with its token.  Bound by memory (131 MB of 16-bit logits in
// 33 us, 4.0 TB/s): of these, loads alone are 26, ends of parts, 2 us each, 5, and exponentials 2.  Blocks that take half as much have
// more ends: 39 us; tiles asked for two ahead, or through shared memory, leave room for fewer warps: 37 to 39.
//
// choose_kernel joins a row's parts, drops what is below a bound that k continuations of one row reach, and puts the rest in order.  Which of two rows'
// continuations is better depends on both rows' sums, and those, in 32 bits, are known to kRowError.  Where neighbours of different rows are closer than
// that, the sums of their rows are worked out again in 64 bits, from the logits, by all blocks of the request's cluster, and the order is made again: what
// comes out is ordered by the values in 64 bits.  (Of 60 steps of 16 requests with 16 beams and 32 choices six had such neighbours, of 60 of 64 with 8 beams
// and 16 choices none; it takes about 25 us.)  Otherwise choosing is a chain of short steps behind the last row, 6 to 10 us, bound by latency, and its code is read for
// the first time in every launch: loops are kept short (four loads in flight and unrolled comparisons took a request of four beams from 12.0 to 13.8 us).
#include "cg_common.cuh"

#include <math_constants.h>

#include <cstddef>

namespace cg {
namespace {

constexpr int kLogitF32 = CG_LOGITS_F32;
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32, kVectors = 4;  // of rows_kernel; 16-byte vectors of a thread in a tile
constexpr int kTileVectors = kRowThreads * kVectors;
constexpr int kRowBlocks = 4;                              // on an SM, of 64 registers a thread (three: 36 us for 131 MB, six, which spill: 37, four: 34)
constexpr int kTilesPerPart = 16, kTileRoom = 512;         // a part's tiles, and how many of its threads' tiles may have candidates
constexpr int kChooseBlocks = 8;                           // of a request's cluster
constexpr int kChooseWarps = 8, kMostChooseWarps = 16, kSorted = 512, kSortedAtOnce = 192, kBins = 256, kMostList = 4096;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMostPlain = 32768.0f;                     // logits from -kMostPlain to here are summed the quick way
// Relative error of a row's sum in 32 bits, and so the absolute one of its logarithm.  A term is 2 to the power y = x log2(e) - c, c whole and at most 9 below
// the thread's largest: with u = top - x, y is at most 1.45 u + 9 and off by 2^-24 of itself, so the term by 2^-24 (u + 6.3).  u on average, weighted with
// the terms, is below 17 for up to 2^24 tokens (n terms of one size u beside the largest weigh n u exp(-u) / (1 + n exp(-u))): 1.4e-6.  log2(e) is off by
// 2^-26 of itself, which for the largest term is known and taken out; for the others 1.4e-8 u: 0.3e-6.  A thread all of whose logits are below -kMostPlain takes
// that instead of its largest: its terms are what they are, or 0, and weigh nothing, since the part's largest is above (or the part is summed again).  (Against
// masks such as -1e10 c would be off by what is lost in x log2(e), some hundreds, and the power infinite.)  The power itself: 2^-22.  A thread's sum is 8 additions to each of
// four accumulators, two to join them and one a tile, the warp's and the block's 8 more: 34 2^-24 or 2.1e-6, with factors that are whole powers of two.  Parts' sums are
// taken to their largest, and joined, with two powers and a logarithm of 32 bits: 2^-21 and 2^-23.  In all below 1.4e-6 + 0.3e-6 + 0.3e-6 + 2.1e-6 + 0.6e-6.
constexpr double kRowError = 5e-6;

struct alignas(16) Part {  // what a block found in its part of a row
    double sum;             // of exp(x - top)
    float top, least;       // the largest logit, and one that k logits of the part reach (-infinity if there are no k)
    int32_t count, pad[3];  // candidates
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
    int32_t beams, vocab, k, room, list_room, sort_room;
    // All rows' tiles stand in one line, every block takes block_tiles of them; its tiles of one row are `cuts` parts (most of one are empty).
    int32_t row_tiles, block_tiles, cuts, line, nparts;  // nparts: room of a row
    __device__ __forceinline__ int32_t first_block(int32_t row) const { return row * row_tiles / block_tiles; }
    __device__ __forceinline__ int32_t parts_of(int32_t row) const { return (((row + 1) * row_tiles - 1) / block_tiles - first_block(row) + 1) * cuts; }
};

// whether a beam with this score has begun; NaN has not
__device__ __forceinline__ bool begun(float score) { return fabsf(score) < CUDART_INF_F; }
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
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// 2^y for y < 1000, and log(x) for x > 0, to 2^-22 and 2^-23: 32-bit functions of what is left when whole powers of two are taken out.
__device__ __forceinline__ double quick_power2(double y) {
    if (!(y > -1000.0)) return 0.0;
    const double n = rint(y);
    return static_cast<double>(power2(static_cast<float>(y - n))) * __hiloint2double((1023 + static_cast<int>(n)) << 20, 0);
}
__device__ __forceinline__ double quick_log(double x) {
    const int high = __double2hiint(x);
    const float m = static_cast<float>(__hiloint2double((high & 0xFFFFF) | 1023 << 20, __double2loint(x)));
    return ((high >> 20) - 1023) * 0.69314718055994531 + logf(m);
}
// A sum of numbers up to 1, to 2^-84 each, whose result does not depend on the order of additions: rows of the same logits in another order have the same.
struct Wide {
    uint64_t low, high;
    __device__ __forceinline__ void add(const Wide &o) {
        low += o.low;
        high += o.high + (low < o.low);
    }
    static __device__ __forceinline__ Wide of(double x) {  // x = m 2^(e - 52), and m 2^(e + 32) is what counts 2^-84
        const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x)), m = (u & 0xFFFFFFFFFFFFFull) | 1ull << 52;
        const int shift = static_cast<int>(u >> 52) - 1023 + 32;
        if (shift > 0) return Wide{m << shift, m >> (64 - shift)};
        return Wide{shift > -64 ? m >> -shift : 0, 0};
    }
    __device__ __forceinline__ double value() const { return (static_cast<double>(high) * 0x1p64 + static_cast<double>(low)) * 0x1p-84; }
};
// 2 to the power of a whole number that is not positive; 0 for what a float does not hold
__device__ __forceinline__ float whole_power2(float n) { return n < -126.0f ? 0.0f : __int_as_float((127 + static_cast<int>(n)) << 23); }

template <int DT> struct Logits;
template <> struct Logits<CG_BF16> {
    using Value = uint16_t;
    static constexpr int kPer = 8;
    static constexpr uint32_t kNone = 0xFF80FF80u;  // -infinity
    static __device__ __forceinline__ float to_float(uint16_t b) { return Half16<CG_BF16>::to_float(b); }
    static __device__ __forceinline__ float2 two(const uint32_t *w, int i) { return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)); }
    template <int WORDS> static __device__ __forceinline__ float most(const uint32_t *w) {
        __nv_bfloat162 m[2] = {*reinterpret_cast<const __nv_bfloat162 *>(w), *reinterpret_cast<const __nv_bfloat162 *>(w + 1)};
#pragma unroll
        for (int i = 2; i < WORDS; ++i) m[i & 1] = __hmax2(m[i & 1], *reinterpret_cast<const __nv_bfloat162 *>(w + i));
        const __nv_bfloat162 both = __hmax2(m[0], m[1]);
        return fmaxf(__low2float(both), __high2float(both));
    }
};
template <> struct Logits<CG_F16> {
    using Value = uint16_t;
    static constexpr int kPer = 8;
    static constexpr uint32_t kNone = 0xFC00FC00u;
    static __device__ __forceinline__ float to_float(uint16_t b) { return Half16<CG_F16>::to_float(b); }
    static __device__ __forceinline__ float2 two(const uint32_t *w, int i) { return __half22float2(*reinterpret_cast<const __half2 *>(w + i)); }
    template <int WORDS> static __device__ __forceinline__ float most(const uint32_t *w) {
        __half2 m[2] = {*reinterpret_cast<const __half2 *>(w), *reinterpret_cast<const __half2 *>(w + 1)};
#pragma unroll
        for (int i = 2; i < WORDS; ++i) m[i & 1] = __hmax2(m[i & 1], *reinterpret_cast<const __half2 *>(w + i));
        const __half2 both = __hmax2(m[0], m[1]);
        return fmaxf(__low2float(both), __high2float(both));
    }
};
template <> struct Logits<kLogitF32> {
    using Value = uint32_t;
    static constexpr int kPer = 4;
    static constexpr uint32_t kNone = 0xFF800000u;
    static __device__ __forceinline__ float to_float(uint32_t b) { return __uint_as_float(b); }
    static __device__ __forceinline__ float2 two(const uint32_t *w, int i) { return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])); }
    template <int WORDS> static __device__ __forceinline__ float most(const uint32_t *w) {
        float m[2] = {__uint_as_float(w[0]), __uint_as_float(w[1])};
#pragma unroll
        for (int i = 2; i < WORDS; ++i) m[i & 1] = fmaxf(m[i & 1], __uint_as_float(w[i]));
        return fmaxf(m[0], m[1]);
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
    // whether vectors from .. to - 1 lie in the row as a whole
    __device__ __forceinline__ bool whole(int32_t from, int32_t to) const { return from * L::kPer >= shift && to * L::kPer - shift <= vocab; }
    __device__ __forceinline__ uint4 load_whole(int32_t v) const {
        uint4 x;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(data + (v * L::kPer - shift)));
        return x;
    }
    __device__ __forceinline__ uint4 load(int32_t v) const { return whole(v, v + 1) ? load_whole(v) : load_part(data, vocab, v * L::kPer - shift); }
    static __device__ __noinline__ uint4 load_part(const typename L::Value *data, int32_t vocab, int32_t first) {
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
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <int DT> __device__ __forceinline__ float value_of(const uint4 &x, int e) {
    const float2 two = Logits<DT>::two(reinterpret_cast<const uint32_t *>(&x), e / 2);
    return e & 1 ? two.y : two.x;
}

struct Shared {
    float most[kTilesPerPart][kRowThreads];   // of a thread's tiles the largest logit
    uint4 alone[kVectors][kRowThreads];       // a part's tile that is its only one
    uint16_t tiles[kTileRoom];                // tile * kRowThreads + thread of those that have candidates
    int32_t ntiles, found;
    float tops[kRowWarps], sums[kRowWarps], bases[kRowWarps];  // a warp's sum is sums * 2 ^ bases
    alignas(8) int32_t digits[256];           // also of the threads the largest logits' keys
    int32_t digit, left;
    bool again;                               // a sum that the quick way does not give
};

// What k of the block's keys (s.digits, 0 for none) reach.  The first is for one warp: of the eight keys of a lane it looks at the largest two (k <= 16: the
// largest) alone, and returns the k-th largest of these: a few more than k of all keys reach it.  (Bit by bit over all keys: four beams of 32,000 logits 7.1 us
// instead of 5.7.)  0: there are not so many.  The second is for all threads, and exact; the same for all.
__device__ __forceinline__ uint32_t kth_of_lanes(const Shared &s, int32_t k) {
    const int lane = threadIdx.x % 32;
    uint32_t high = 0, second = 0;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) {
        const uint32_t x = static_cast<uint32_t>(s.digits[i * 32 + lane]);
        second = max(second, min(high, x)), high = max(high, x);
    }
    int32_t before = 0, before_second = 0;  // keys in front of this lane's, those of lower lanes first among equal ones
    if (k <= 16) {
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
            const uint32_t x = __shfl_sync(~0u, high, i);
            before += x > high || (x == high && i < lane);
        }
        second = 0, before_second = INT32_MAX;
    } else {
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
            const uint32_t x = __shfl_sync(~0u, high, i), y = __shfl_sync(~0u, second, i);
            before += (x > high || (x == high && i < lane)) + (y > high || (y == high && i < lane));
            before_second += (x > second || (x == second && i <= lane)) + (y > second || (y == second && i < lane));
        }
    }
    const uint32_t mine = before == k - 1 ? high : before_second == k - 1 ? second : 0;
    return __reduce_max_sync(~0u, mine);
}
constexpr int kMostOfLanes = 40;  // the largest k for the first: behind it lanes' third keys would be missed
__device__ __noinline__ uint32_t kth_of_all(Shared &s, int32_t k) {
    const uint32_t mine = static_cast<uint32_t>(s.digits[threadIdx.x]);
    int32_t before = 0;
#pragma unroll 4
    for (int i = 0; i < kRowThreads; ++i) {
        const uint32_t x = static_cast<uint32_t>(s.digits[i]);
        before += x > mine || (x == mine && i < static_cast<int>(threadIdx.x));
    }
    if (before == k - 1) s.left = static_cast<int32_t>(mine);
    __syncthreads();
    return static_cast<uint32_t>(s.left);
}

// The digit, of those counted from `first` on in steps of `step`, at which their sum reaches s.left, which becomes what is left for it.
__device__ __forceinline__ int32_t digit_of(Shared &s, int first, int step) {
    __syncthreads();
    if (threadIdx.x == 0) {
        int32_t left = s.left, d = first;
        while (left > s.digits[d] && d + step >= 0 && d + step < 256) left -= s.digits[d], d += step;
        s.digit = d, s.left = left;
    }
    __syncthreads();
    return s.digit;
}
// Writes exactly the k first of a part's logits, by value and then by token: read again digit by digit.  For parts where many are
// equal; there are more than k.
template <int DT>
__device__ __noinline__ float write_first(Shared &s, const Row<DT> x, int32_t from, int32_t to, int32_t k, Candidate *out) {
    using L = Logits<DT>;
    const auto each = [&](auto f) {  // f(key, place in the part), for all but -infinity and NaN
        for (int32_t v = from + threadIdx.x; v < to; v += kRowThreads) {
            const uint4 w = x.load(v);
            for (int e = 0; e < L::kPer; ++e) {
                const float y = value_of<DT>(w, e);
                if (y > -CUDART_INF_F) f(ordered(y), static_cast<uint32_t>((v - from) * L::kPer + e));
            }
        }
    };
    const auto count = [&](auto digit) {  // digit(key, place): -1 for those that do not count
        __syncthreads();
        for (int d = threadIdx.x; d < 256; d += kRowThreads) s.digits[d] = 0;
        __syncthreads();
        int32_t same = -1, times = 0;  // neighbours are often the same
        each([&](uint32_t key, uint32_t place) {
            const int32_t d = digit(key, place);
            if (d != same) {
                if (same >= 0) atomicAdd(&s.digits[same], times);
                same = d, times = 0;
            }
            ++times;
        });
        if (same >= 0) atomicAdd(&s.digits[same], times);
    };
    __syncthreads();
    if (threadIdx.x == 0) s.left = k, s.found = 0;
    uint32_t least = 0, last = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        count([&](uint32_t key, uint32_t) { return shift < 24 && (key ^ least) >> (shift + 8) ? -1 : static_cast<int32_t>(key >> shift & 255); });
        least |= static_cast<uint32_t>(digit_of(s, 255, -1)) << shift;
    }
    static_assert(kTilesPerPart * kTileVectors * 8 <= 1 << 24, "three digits");
    for (int shift = 16; shift >= 0; shift -= 8) {
        count([&](uint32_t key, uint32_t place) { return key != least || (place ^ last) >> (shift + 8) ? -1 : static_cast<int32_t>(place >> shift & 255); });
        last |= static_cast<uint32_t>(digit_of(s, 0, 1)) << shift;
    }
    each([&](uint32_t key, uint32_t place) {
        if (key > least || (key == least && place <= last)) out[atomicAdd(&s.found, 1)] = Candidate{from_ordered(key), x.token(from, 0) + static_cast<int32_t>(place)};
    });
    __syncthreads();
    return from_ordered(least);
}

__device__ __forceinline__ float of_warps(const Shared &s) {
    float high = s.tops[0];
#pragma unroll
    for (int i = 1; i < kRowWarps; ++i) high = fmaxf(high, s.tops[i]);
    return high;
}
// A part's sum where there are infinities, NaN or logits that are too large: of ones for the infinite logits, or without the NaN.
template <int DT>
__device__ __noinline__ double sum_again(Shared &s, const Row<DT> x, int32_t from, int32_t to) {
    const float high = of_warps(s);
    double mine = 0.0;
    for (int32_t v = from + threadIdx.x; v < to; v += kRowThreads) {
        const uint4 w = x.load(v);
        for (int e = 0; e < Logits<DT>::kPer; ++e) {
            const float y = value_of<DT>(w, e);
            if (high == CUDART_INF_F) mine += y == CUDART_INF_F;
            else if (y > -CUDART_INF_F) mine += power2(__fmul_rn(__fsub_rn(y, high), kLog2e));
        }
    }
    double *const parts = reinterpret_cast<double *>(s.digits);  // (no longer in use)
    static_assert(sizeof(s.digits) >= kRowWarps * sizeof(double) && offsetof(Shared, digits) % sizeof(double) == 0, "room for the warps' sums");
#pragma unroll
    for (int d = 16; d; d /= 2) mine += __shfl_xor_sync(~0u, mine, d);
    __syncthreads();
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = mine;
    __syncthreads();
    double whole = 0.0;
    for (int i = 0; i < kRowWarps; ++i) whole += parts[i];
    return whole;
}

// A block's tiles in the line, each asked for while the one in front of it is worked on, across the ends of rows too.
template <int DT> struct Line {
    using L = Logits<DT>;
    uint4 next[kVectors];
    const uint4 *from;   // this thread's first vector of the tile that is asked for next
    int32_t at, end, v0;  // that tile in the line, and its first vector in its row
    int32_t row, shift;
    bool there;

    __device__ __forceinline__ void begin_row(const BeamArgs &a) {
        there = begun(__ldg(a.scores + row));
        const Row<DT> x(a, row);
        shift = x.shift;
        from = reinterpret_cast<const uint4 *>(x.data - x.shift) + (v0 + static_cast<int32_t>(threadIdx.x));
    }
    __device__ __forceinline__ Line(const BeamArgs &a, int32_t first, int32_t last) : at(first), end(last), row(first / a.row_tiles) {
        v0 = (first - row * a.row_tiles) * kTileVectors;
        begin_row(a);
        ask(a);
    }
    __device__ __forceinline__ void ask(const BeamArgs &a) {
        if (at >= end) return;
        if (there) {
            if (v0 * L::kPer >= shift && (v0 + kTileVectors) * L::kPer - shift <= a.vocab) {
#pragma unroll
                for (int u = 0; u < kVectors; ++u)
                    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(next[u].x), "=r"(next[u].y), "=r"(next[u].z), "=r"(next[u].w)
                                 : "l"(from + u * kRowThreads));
            } else {  // the row's ends, and nothing behind them
                const Row<DT> x(a, row);
#pragma unroll
                for (int u = 0; u < kVectors; ++u) next[u] = x.load(v0 + u * kRowThreads + static_cast<int32_t>(threadIdx.x));
            }
        }
        ++at, v0 += kTileVectors, from += kTileVectors;
        if (at < end && at == (row + 1) * a.row_tiles) {
            ++row, v0 = 0;
            begin_row(a);
        }
    }
};

// The next `tiles` tiles of the line, vectors from .. to - 1 of a row, by the block.
template <int DT>
__device__ __forceinline__ void do_part(const BeamArgs &a, Shared &s, Line<DT> &line, const Row<DT> &x, int32_t from, int32_t to, int32_t tiles, Part *out,
                                        Candidate *candidates) {
    using L = Logits<DT>;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    float top = -CUDART_INF_F, sum = 0.0f, base = 0.0f;
    const uint64_t scale = pair_of(kLog2e, kLog2e);
#pragma unroll 1
    for (int32_t tile = 0; tile < tiles; ++tile) {
        uint4 now[kVectors];
#pragma unroll
        for (int u = 0; u < kVectors; ++u) now[u] = line.next[u];
        line.ask(a);
        if (tiles == 1) {
#pragma unroll
            for (int u = 0; u < kVectors; ++u) s.alone[u][tid] = now[u];
        }
        const float m = L::template most<4 * kVectors>(reinterpret_cast<const uint32_t *>(now));
        s.most[tile][tid] = m;
        top = fmaxf(top, m);
        const float want = fmaxf(__fmul_rn(m, kLog2e), -kMostPlain * kLog2e);
        if (want > base + 8.0f || sum == 0.0f) {
            const float next = rintf(want);
            sum = sum == 0.0f ? 0.0f : __fmul_rn(sum, whole_power2(base - next));
            base = next;
        }
        const uint64_t minus = pair_of(-base, -base);
        uint64_t acc[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll
        for (int u = 0; u < kVectors; ++u) {
#pragma unroll
            for (int i = 0; i < L::kPer / 2; ++i) {
                const float2 two = L::two(reinterpret_cast<const uint32_t *>(&now[u]), i);
                const float2 y = of_pair(pair_fma(pair_of(two.x, two.y), scale, minus));
                acc[i & 1] = pair_add(acc[i & 1], pair_of(power2(y.x), power2(y.y)));
            }
        }
        const float2 both = of_pair(pair_add(acc[0], acc[1]));
        sum = __fadd_rn(sum, __fadd_rn(both.x, both.y));
    }
    const bool odd = (!(sum < CUDART_INF_F) && top > -CUDART_INF_F) || top > kMostPlain;
    const uint32_t key = ordered(top);
    const float high = from_ordered(__reduce_max_sync(~0u, key));
    const float warp_base = from_ordered(__reduce_max_sync(~0u, sum > 0.0f ? ordered(base) : 0x00800000u));
    float warp_sum = sum > 0.0f ? __fmul_rn(sum, whole_power2(base - warp_base)) : 0.0f;
#pragma unroll
    for (int d = 16; d; d /= 2) warp_sum = __fadd_rn(warp_sum, __shfl_xor_sync(~0u, warp_sum, d));
    if (lane == 0) s.tops[warp] = high, s.sums[warp] = warp_sum, s.bases[warp] = warp_base;
    s.digits[tid] = static_cast<int32_t>(top > -CUDART_INF_F ? key : 0);
    if (tid == 0) s.found = s.ntiles = 0;
    const bool odd_ones = __syncthreads_or(odd);
    // Candidates: what reaches the k-th largest of the threads' largest, or all if fewer than k threads have one.  One warp finds it, another joins the
    // warps' sums meanwhile.
    if (warp == 0) {
        const uint32_t reach = a.k <= kMostOfLanes ? kth_of_lanes(s, a.k) : 0;
        if (lane == 0) s.left = static_cast<int32_t>(reach);
    }
    if (warp == 1) {
        const float top_here = lane < kRowWarps ? s.tops[lane] : -CUDART_INF_F, sum_here = lane < kRowWarps ? s.sums[lane] : 0.0f;
        const float base_here = sum_here > 0.0f ? s.bases[lane % kRowWarps] : -CUDART_MAX_NORMAL_F;
        const float all_top = from_ordered(__reduce_max_sync(~0u, ordered(top_here))), all_base = from_ordered(__reduce_max_sync(~0u, ordered(base_here)));
        float whole = sum_here > 0.0f ? __fmul_rn(sum_here, whole_power2(base_here - all_base)) : 0.0f;
#pragma unroll
        for (int d = kRowWarps / 2; d; d /= 2) whole = __fadd_rn(whole, __shfl_xor_sync(~0u, whole, d));
        if (lane == 0) {
            s.again = odd_ones || (all_top < -kMostPlain && all_top > -CUDART_INF_F);
            out->top = all_top;
            out->sum = whole > 0.0f ? whole * quick_power2(all_base - static_cast<double>(kLog2e) * all_top) : 0.0;
        }
    }
    __syncthreads();
    uint32_t least_key = static_cast<uint32_t>(s.left);
    if (!least_key) {  // (the same for all threads, which read it before it changes)
        __syncthreads();
        least_key = kth_of_all(s, a.k);
    }
    float least = least_key ? from_ordered(least_key) : -CUDART_INF_F;
    const auto fits = [&](float y) { return y >= least && y > -CUDART_INF_F; };
    if (fits(top)) {
#pragma unroll 4
        for (int t = 0; t < tiles; ++t) {
            if (!fits(s.most[t][tid])) continue;
            const int32_t at = atomicAdd(&s.ntiles, 1);
            if (at < kTileRoom) s.tiles[at] = static_cast<uint16_t>(t * kRowThreads + tid);
        }
    }
    __syncthreads();
    // Tiles that have some are read again, from the L2 cache, a vector a thread.
    const int32_t ntiles = min(s.ntiles, kTileRoom);
    for (int32_t i = tid; i < kVectors * ntiles; i += kRowThreads) {
        const int32_t at = s.tiles[i / kVectors], u = i % kVectors, thread = at % kRowThreads, v = from + at / kRowThreads * kTileVectors + u * kRowThreads + thread;
        if (v >= to) continue;
        const uint4 w = tiles == 1 ? s.alone[u][thread] : x.load(v);
        if (!fits(L::template most<4>(reinterpret_cast<const uint32_t *>(&w)))) continue;
#pragma unroll
        for (int e = 0; e < L::kPer; ++e) {
            const float y = value_of<DT>(w, e);
            if (!fits(y)) continue;
            const int32_t place = atomicAdd(&s.found, 1);
            if (place < a.room) candidates[place] = Candidate{y, x.token(v, e)};
        }
    }
    __syncthreads();
    if (s.found > a.room || s.ntiles > kTileRoom) least = write_first<DT>(s, x, from, to, a.k, candidates);  // (the same for all threads)
    if (s.again) {
        const double whole = sum_again<DT>(s, x, from, to);
        if (tid == 0) out->sum = whole;
    }
    if (tid == 0) out->least = least, out->count = s.found;
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads, kRowBlocks) rows_kernel(const __grid_constant__ BeamArgs a) {
    __shared__ Shared s;
    let_next_launch_start();
    int32_t at = static_cast<int32_t>(blockIdx.x) * a.block_tiles, row = at / a.row_tiles, cut = 0;
    const int32_t end = min(a.line, at + a.block_tiles);
    Line<DT> line(a, at, end);
    while (at < end) {
        const int32_t first = row * a.row_tiles, row_end = min(end, first + a.row_tiles), to = min(row_end, at + kTilesPerPart);
        const int64_t part = static_cast<int64_t>(row) * a.nparts + (static_cast<int32_t>(blockIdx.x) - a.first_block(row)) * a.cuts + cut;
        if (begun(__ldg(a.scores + row))) {
            const Row<DT> x(a, row);
            do_part<DT>(a, s, line, x, (at - first) * kTileVectors, min(x.vectors(), (to - first) * kTileVectors), to - at, a.parts + part,
                        a.candidates + part * a.room);
        } else {
            for (int32_t i = at; i < to; ++i) line.ask(a);  // (nothing of these has been asked for)
            if (threadIdx.x == 0) a.parts[part] = Part{0.0, -CUDART_INF_F, -CUDART_INF_F, 0, {}};
        }
        at = to, ++cut;
        if (at == row_end) {
            if (threadIdx.x == 0)
                for (int32_t i = 1; cut + i <= a.cuts; ++i) a.parts[part + i] = Part{0.0, -CUDART_INF_F, -CUDART_INF_F, 0, {}};
            ++row, cut = 0;
        }
        if (at < end) __syncthreads();  // (what the block has in common is written to again)
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
__device__ __forceinline__ Wide wide_of_block(const Wide *mine, int rank) {
    Wide v;
    asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(v.low), "=l"(v.high) : "r"(at_block(mine, rank)) : "memory");
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
        for (int32_t p = 0; p < a.parts_of(row); ++p) {
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
    uint64_t key;  // the score, in an order in which numbers without a sign compare
    uint64_t rest;
    __device__ __forceinline__ double total() const { return __longlong_as_double(static_cast<long long>(key >> 63 ? key & ~(1ull << 63) : ~key)); }
    __device__ __forceinline__ int32_t beam() const { return 255 - static_cast<int32_t>(rest >> 56); }
    __device__ __forceinline__ int32_t token() const { return 0xFFFFFF - static_cast<int32_t>(rest & 0xFFFFFF); }
    __device__ __forceinline__ float x() const { return from_ordered(static_cast<uint32_t>(rest >> 24)); }
};
__device__ __forceinline__ uint64_t rest_of(int32_t beam, float x, int32_t token) {
    return static_cast<uint64_t>(255 - beam) << 56 | static_cast<uint64_t>(ordered(x)) << 24 | static_cast<uint64_t>(0xFFFFFF - token);
}
__device__ __forceinline__ uint64_t ordered_double(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(__dadd_rn(x, 0.0)));
    return u >> 63 ? ~u : u | 1ull << 63;
}

// A list of them, keys and rests apart: sorting reads the keys.
struct Choices {
    uint64_t *keys, *rests;
    __device__ __forceinline__ Choice at(int32_t i) const { return Choice{keys[i], rests[i]}; }
    __device__ __forceinline__ void put(int32_t i, const Choice &c) const { keys[i] = c.key, rests[i] = c.rest; }
};

// How room in shared memory is divided; K beams, W warps
struct ChooseRoom {
    double *base, *bounds;    // [K]: score - log sum exp(x - top); what k continuations of the row reach
    Wide *wides, *of_warps;   // [K]: a block's share of a sum; [kMostChooseWarps]
    Choices list, sorted;     // [list_room], [kSorted]; in their place, where these are too small,
    uint64_t *best, *sorting; // [K][k], [W][sort_room]
    float *top;               // [K]
    int32_t *count;           // [K]
    uint32_t *near;           // [K]: whether the sum is wanted in 64 bits; near[K]: whether any is
    int32_t *places;          // [kSorted]
    static __host__ __device__ size_t lists(const BeamArgs &a, int warps) {
        const size_t usual = sizeof(Choice) * (static_cast<size_t>(a.list_room) + kSorted);
        const size_t other = sizeof(uint64_t) * (static_cast<size_t>(a.beams) * a.k + static_cast<size_t>(warps) * a.sort_room);
        return (usual > other ? usual : other) + 15 & ~static_cast<size_t>(15);
    }
    static size_t bytes(const BeamArgs &a, int warps) { return lists(a, warps) + a.beams * (sizeof(Wide) + 2 * sizeof(double) + 3 * sizeof(float)) + sizeof(float) * (1 + kSorted) + sizeof(Wide) * kMostChooseWarps; }
    __device__ ChooseRoom(char *at, const BeamArgs &a, int warps) {
        list.keys = reinterpret_cast<uint64_t *>(at);
        list.rests = list.keys + a.list_room;
        sorted.keys = list.rests + a.list_room;
        sorted.rests = sorted.keys + kSorted;
        best = reinterpret_cast<uint64_t *>(at);
        sorting = best + static_cast<int64_t>(a.beams) * a.k;
        wides = reinterpret_cast<Wide *>(at + lists(a, warps));
        of_warps = wides + a.beams;
        base = reinterpret_cast<double *>(of_warps + kMostChooseWarps);
        bounds = base + a.beams;
        top = reinterpret_cast<float *>(bounds + a.beams);
        count = reinterpret_cast<int32_t *>(top + a.beams);
        near = reinterpret_cast<uint32_t *>(count + a.beams);
        places = reinterpret_cast<int32_t *>(near + a.beams + 1);
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

// The block puts n continuations in order: it counts those in front of each, which several threads share, by their keys; rests are looked at where keys are the
// same.  places: [kSorted], zeros before and after.
__device__ __forceinline__ void sort_list(const Choices &list, const Choices &sorted, int32_t n, int32_t *places) {
    if (n == 0) return;
    int team = 1;
    while (2 * team * n <= static_cast<int>(blockDim.x)) team *= 2;
    const int32_t each = blockDim.x / team, share = ((n + team - 1) / team + 1) & ~1;
    for (int32_t i0 = 0; i0 < n; i0 += each) {
        const int32_t i = i0 + threadIdx.x % each, first = threadIdx.x / each * share, last = min(n, first + share);
        if (i < n && first < last) {
            const uint64_t mine = list.keys[i];
            int32_t place = 0, same = 0;
            int32_t j = first;
#pragma unroll 2
            for (; j < last - 1; j += 2) {  // (first is even)
                const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(list.keys + j);
                place += (two.x > mine) + (two.y > mine);
                same += (two.x == mine) + (two.y == mine);
            }
            if (j < last) place += list.keys[j] > mine, same += list.keys[j] == mine;
            if (same > (i >= first && i < last)) {
                const uint64_t rest = list.rests[i];
                for (j = first; j < last; ++j) place += list.keys[j] == mine && list.rests[j] > rest;
            }
            if (place) atomicAdd(&places[i], place);
        }
    }
    __syncthreads();
    for (int32_t i = threadIdx.x; i < n; i += blockDim.x) {
        sorted.put(places[i], list.at(i));
        places[i] = 0;
    }
    __syncthreads();
}
__device__ __forceinline__ void write_sorted(const BeamArgs &a, const Choices &sorted, int32_t request, int32_t n) {
    for (int32_t i = threadIdx.x; i < a.k; i += blockDim.x) {
        const int64_t at = static_cast<int64_t>(request) * a.k + i;
        const bool there = i < n;
        const Choice c = sorted.at(there ? i : 0);
        a.out[at] = there ? static_cast<float>(c.total()) : -CUDART_INF_F;
        a.tokens[at] = there ? c.token() : -1;
        a.parents[at] = there ? request * a.beams + c.beam() : -1;
    }
}
// The continuations that may be among the best, in *list; returns how many there are, more than `kSorted` if that is no use.  A bound that k of
// one row reach drops most of them while they are read; where that leaves many, they are counted in bins, and all behind the bin of the k-th and the next one are
// dropped.  Both leave room for what 32-bit sums are off.  *sorted is as large as kSorted.
__device__ __forceinline__ int32_t gather_choices(const BeamArgs &a, const ChooseRoom &r, int32_t request, int32_t *counts, Choices *list, Choices *sorted) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    double bound = -CUDART_INF;
    for (int32_t i = 0; i < a.beams; ++i) bound = fmax(bound, r.bounds[i]);
    bound -= 2.0 * kRowError;
    const int32_t pairs = a.beams * a.nparts;  // of a beam and a part of its row
    const int64_t first = static_cast<int64_t>(request) * pairs;
    for (int32_t p0 = warp; p0 < pairs; p0 += 32 * warps) {
        // of each lane's pair the candidates that may do, and those of the lanes in front
        const int32_t mine = p0 + lane * warps, my_beam = mine / a.nparts;
        int32_t count = 0;
        if (mine < pairs && mine - my_beam * a.nparts < a.parts_of(request * a.beams + my_beam)) {
            const Part *const part = a.parts + first + mine;
            const float top = part->top;
            count = part->count;
            if (!(r.base[my_beam] + entering(top, r.top[my_beam]) >= bound)) count = 0;
        }
        int32_t upto = count;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int32_t y = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += y;
        }
        const int32_t all = __shfl_sync(~0u, upto, 31);
#pragma unroll 1
        for (int32_t i0 = 0; i0 < all; i0 += 32) {
            const int32_t i = i0 + lane;
            int owner = 0;  // the first lane whose candidates end behind i
#pragma unroll
            for (int d = 16; d; d /= 2)
                if (__shfl_sync(~0u, upto, owner + d - 1) <= i) owner += d;
            const int32_t before = __shfl_sync(~0u, upto, owner) - __shfl_sync(~0u, count, owner), pair = p0 + owner * warps;
            if (i >= all) continue;
            const int32_t beam = pair / a.nparts;
            const float2 c = __ldcg(reinterpret_cast<const float2 *>(a.candidates + (first + pair) * a.room + (i - before)));
            const double total = r.base[beam] + entering(c.x, r.top[beam]);
            if (!(total >= bound && total > -CUDART_INF)) continue;
            const int32_t at = atomicAdd(&counts[0], 1);
            if (at < a.list_room) r.list.put(at, Choice{ordered_double(total), rest_of(beam, c.x, __float_as_int(c.y))});
        }
    }
    __syncthreads();
    const int32_t n = counts[0];
    if (n > a.list_room) return INT32_MAX;
    if (n <= kSortedAtOnce) return n;
    if (!(bound > -CUDART_INF)) {  // no row's part had k: from the least of the list on
        uint32_t least = ~0u;
        for (int32_t i = threadIdx.x; i < n; i += blockDim.x) least = min(least, static_cast<uint32_t>(r.list.keys[i] >> 32));
        least = __reduce_min_sync(~0u, least);
        if (lane == 0) atomicMin(reinterpret_cast<uint32_t *>(&counts[1]), least);
        __syncthreads();
        bound = Choice{static_cast<uint64_t>(static_cast<uint32_t>(counts[1])) << 32, 0}.total();
    }
    double high = -CUDART_INF;  // the best of the rows' largest: there x - top is 0
    for (int32_t i = 0; i < a.beams; ++i) high = fmax(high, r.base[i]);
    const float width = static_cast<float>(high - bound) * (1.0f / kBins), a_bin = 1.0f / width;
    if (!(width > 1e-4f && width < 1e30f)) return n;
    static_assert(1e-4 > 16.0 * kRowError, "a bin is wider than what sums are off");
    const auto bin = [&](const Choice &c) { return min(kBins - 1, static_cast<int32_t>(static_cast<float>(c.total() - bound) * a_bin)); };
    for (int32_t i = threadIdx.x; i < n; i += blockDim.x) atomicAdd(&r.places[bin(r.list.at(i))], 1);
    __syncthreads();
    if (warp == 0) {  // the bin in which the k-th stands, counted from the last
        constexpr int kEach = kBins / 32;
        int32_t mine = 0;
        for (int32_t i = 0; i < kEach; ++i) mine += r.places[kBins - 1 - lane * kEach - i];
        int32_t upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int32_t y = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += y;
        }
        if (upto >= a.k && upto - mine < a.k) {
            int32_t left = a.k - (upto - mine), at = kBins - 1 - lane * kEach;
            while (left > r.places[at]) left -= r.places[at--];  // (ends in this lane's share)
            counts[1] = at;
        }
    }
    if (threadIdx.x == 0) counts[0] = 0;
    __syncthreads();
    const int32_t first_bin = counts[1] - 1;  // one bin more than is counted, wider than what sums are off
    for (int32_t i = threadIdx.x; i < kBins; i += blockDim.x) r.places[i] = 0;
    for (int32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const Choice c = r.list.at(i);
        if (bin(c) < first_bin) continue;
        const int32_t at = atomicAdd(&counts[0], 1);
        if (at < kSorted) r.sorted.put(at, c);
    }
    __syncthreads();
    *list = r.sorted, *sorted = r.list;
    return counts[0];
}

// A cluster a request.  Its first block chooses; the others wait to be asked for sums in 64 bits.
template <int DT>
__global__ void __cluster_dims__(kChooseBlocks, 1, 1) __launch_bounds__(kMostChooseWarps * 32) choose_kernel(const __grid_constant__ BeamArgs a) {
    extern __shared__ __align__(16) char room[];
    __shared__ int32_t counts[2];
    const int rank = choose_rank(), lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const int32_t request = blockIdx.x / kChooseBlocks;
    const ChooseRoom r(room, a, warps);
    Choices list = r.list, sorted = r.sorted;
    int32_t n = 0;
    if (rank == 0) {
        for (int32_t i = threadIdx.x; i <= a.beams; i += blockDim.x) r.near[i] = 0;
        for (int32_t i = threadIdx.x; i < kSorted; i += blockDim.x) r.places[i] = 0;
        if (threadIdx.x == 0) counts[0] = 0, counts[1] = -1;  // how many; a bin, or the upper half of a score's key
        wait_for_launch_before();
        for (int32_t i = warp; i < a.beams; i += warps) {
            const int32_t row = request * a.beams + i;
            const Part *const parts = a.parts + static_cast<int64_t>(row) * a.nparts;
            const int32_t nparts = a.parts_of(row);
            float top = -CUDART_INF_F, least = -CUDART_INF_F;
            for (int32_t p = lane; p < nparts; p += 32) top = fmaxf(top, parts[p].top), least = fmaxf(least, parts[p].least);
            top = from_ordered(__reduce_max_sync(~0u, ordered(top))), least = from_ordered(__reduce_max_sync(~0u, ordered(least)));
            double sum = 0.0;
            for (int32_t p = lane; p < nparts; p += 32) {
                const float high = parts[p].top;
                if (high == top) sum += parts[p].sum;
                else if (high > -CUDART_INF_F && top < CUDART_INF_F) sum += parts[p].sum * quick_power2((static_cast<double>(high) - top) * 1.4426950408889634);
            }
#pragma unroll
            for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == 0) {
                const bool any = top > -CUDART_INF_F;
                const double base = any ? static_cast<double>(__ldg(a.scores + row)) - quick_log(sum) : -CUDART_INF;
                r.top[i] = top;
                r.base[i] = base;
                r.bounds[i] = any && least > -CUDART_INF_F ? base + entering(least, top) : -CUDART_INF;
            }
        }
        __syncthreads();
        n = gather_choices(a, r, request, counts, &list, &sorted);
        if (n <= kSorted) {
            sort_list(list, sorted, n, r.places);
            for (int32_t i = threadIdx.x; i + 1 < n; i += blockDim.x) {
                const Choice p = sorted.at(i), q = sorted.at(i + 1);
                if (p.total() - q.total() <= 2.0 * kRowError && p.beam() != q.beam() && (i < a.k || sorted.at(a.k - 1).total() - p.total() <= 2.0 * kRowError))
                    r.near[p.beam()] = r.near[q.beam()] = r.near[a.beams] = 1;
            }
            __syncthreads();
            if (!r.near[a.beams]) write_sorted(a, sorted, request, n);
        } else {  // many equal ones: row by row
            for (int32_t i = warp; i < a.beams; i += warps) {
                const int32_t row = request * a.beams + i;
                float least = -CUDART_INF_F;
                for (int32_t p = lane; p < a.parts_of(row); p += 32) least = fmaxf(least, __ldcg(&a.parts[static_cast<int64_t>(row) * a.nparts + p].least));
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
            Wide sum{0, 0};
            const Row<DT> x(a, static_cast<int64_t>(request) * a.beams + i);
            for (int32_t t = rank * blockDim.x + threadIdx.x; t < a.vocab; t += kChooseBlocks * blockDim.x) {
                const float y = x.at(t);
                if (top == CUDART_INF_F ? y == top : y > -CUDART_INF_F) sum.add(Wide::of(top == CUDART_INF_F ? 1.0 : exp(static_cast<double>(y) - top)));
            }
#pragma unroll
            for (int d = 16; d; d /= 2) sum.add(Wide{__shfl_xor_sync(~0u, sum.low, d), __shfl_xor_sync(~0u, sum.high, d)});
            __syncthreads();
            if (lane == 0) r.of_warps[warp] = sum;
            __syncthreads();
            if (threadIdx.x == 0) {
                sum = Wide{0, 0};
                for (int w = 0; w < warps; ++w) sum.add(r.of_warps[w]);
                r.wides[i] = sum;
            }
        }
        cluster_barrier();
        if (rank == 0) {
            for (int32_t i = threadIdx.x; i < a.beams; i += blockDim.x) {
                if (!r.near[i]) continue;
                Wide sum{0, 0};
                for (int b = 0; b < kChooseBlocks; ++b) sum.add(wide_of_block(r.wides + i, b));
                r.base[i] = static_cast<double>(__ldg(a.scores + static_cast<int64_t>(request) * a.beams + i)) - log(sum.value());
            }
            __syncthreads();
            if (n > kSorted) {
                if (warp == 0) take_best(a, r, request, false);
            } else {
                for (int32_t i = threadIdx.x; i < n; i += blockDim.x) {
                    const Choice c = list.at(i);
                    list.keys[i] = ordered_double(r.base[c.beam()] + entering(c.x(), r.top[c.beam()]));
                }
                __syncthreads();
                sort_list(list, sorted, n, r.places);
                write_sorted(a, sorted, request, n);
            }
        }
    }
    cluster_barrier();  // nobody reads another block's memory any more
}

struct Sizes {
    int32_t row_tiles, block_tiles, cuts, line, nparts, room;
    int64_t parts_bytes, total;
};
// A line that is longer than numbers of 32 bits has a total of -1.
Sizes sizes_of(const cg_beam_job &j, int sms) {
    Sizes z{};
    const int per = j.dtype == kLogitF32 ? 4 : 8;
    const int64_t vectors = (static_cast<int64_t>(j.vocab) + 2 * (per - 1)) / per;  // a row may begin inside a vector
    const int64_t tiles = (vectors + kTileVectors - 1) / kTileVectors, rows = static_cast<int64_t>(j.nrequests) * j.beams, line = rows * tiles;
    // Equal runs of the line cross the ends of rows, and every end of a part costs time.  Where whole rows, or equal parts of them, keep nearly all blocks busy they are what a
    // block takes: 512 rows of 16 tiles by 512 blocks 32.7 us, by 586 with 14 tiles each 34.7; 256 rows of 17 tiles by 256 blocks 30.0, by 544 23.9.
    const int64_t blocks = static_cast<int64_t>(sms) * kRowBlocks, nearly = blocks * 17 / 20;
    int64_t each = (line + blocks - 1) / blocks;
    if (rows <= blocks) {
        for (int64_t parts = blocks / rows; parts >= 1 && rows * parts >= nearly; --parts)
            if (tiles % parts == 0) {
                each = tiles / parts;
                break;
            }
    } else {
        const int64_t of_block = (rows + blocks - 1) / blocks;
        if ((rows + of_block - 1) / of_block >= nearly) each = of_block * tiles;
    }
    if (line > INT32_MAX / 2 || each > INT32_MAX / 2) {
        z.total = -1;
        return z;
    }
    z.row_tiles = static_cast<int32_t>(tiles), z.block_tiles = static_cast<int32_t>(each), z.line = static_cast<int32_t>(line);
    z.cuts = static_cast<int32_t>(((each < tiles ? each : tiles) + kTilesPerPart - 1) / kTilesPerPart);
    z.nparts = static_cast<int32_t>((tiles + each - 2) / each + 1) * z.cuts;
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
    if (j.beams > CG_MAX_BEAMS || j.k > CG_MAX_CHOICES || j.beams * j.k > CG_MAX_BEAM_CHOICES || static_cast<int64_t>(j.nrequests) * j.beams > CG_MAX_BEAM_ROWS)
        return CG_E_CAPACITY;
    return CG_OK;
}

template <int DT>
int run(BeamArgs &a, int32_t nrequests, cudaStream_t st) {
    const int64_t blocks = (static_cast<int64_t>(a.line) + a.block_tiles - 1) / a.block_tiles;
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
    if (job->nrequests == 0) return 0;
    const int64_t total = cg::sizes_of(*job, cg::sm_count()).total;
    return total < 0 ? CG_E_CAPACITY : total;
}

extern "C" int cg_beam_select(const cg_beam_job *job, void *stream) {
    using namespace cg;
    if (const int rc = check_job(job)) return rc;
    const cg_beam_job &j = *job;
    if (j.nrequests == 0) return CG_OK;
    if (!j.logits || !j.scores || !j.out_scores || !j.tokens || !j.parents) return CG_E_NULL;
    const Sizes z = sizes_of(j, sm_count());
    if (z.total < 0) return CG_E_CAPACITY;
    if (!j.workspace || j.workspace_bytes < z.total) return CG_E_CAPACITY;
    if (reinterpret_cast<uintptr_t>(j.workspace) % 16 || reinterpret_cast<uintptr_t>(j.logits) % (j.dtype == kLogitF32 ? 4 : 2)) return CG_E_ALIGN;
    int sort_room = 64;
    while (sort_room < 4 * j.k && sort_room < 512) sort_room *= 2;
    const int list_room = 4 * j.beams * j.k < kSorted ? kSorted : 4 * j.beams * j.k < kMostList ? 4 * j.beams * j.k : kMostList;
    BeamArgs a{j.logits, j.scores, j.out_scores, j.tokens, j.parents, static_cast<Part *>(j.workspace),
               reinterpret_cast<Candidate *>(static_cast<char *>(j.workspace) + z.parts_bytes), j.row_stride,
               j.beams, j.vocab, j.k, z.room, list_room, sort_room, z.row_tiles, z.block_tiles, z.cuts, z.line, z.nparts};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (j.dtype == CG_F16) return run<CG_F16>(a, j.nrequests, st);
    if (j.dtype == CG_BF16) return run<CG_BF16>(a, j.nrequests, st);
    return run<kLogitF32>(a, j.nrequests, st);
}
