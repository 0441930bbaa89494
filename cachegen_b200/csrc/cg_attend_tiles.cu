// Attention over a paged KV cache for many query rows a key/value head: chunks of new tokens and whole prompts.
//
// Here the products bound the kernel, so they go to the tensor cores' own memory: a CTA has up to 256 query rows, two halves of 128,
// whose scores S and results O are accumulators in tensor memory (128 columns each: all 512), and whose weights P overwrite
// the scores they came from.  While one half's softmax works on its scores, the tensor cores work on the other's:
//
//     warps 0-3, 4-7   softmax of one half each: a thread has a row, so there are no exchanges for maxima and sums
//     warps 8-11       copies of Q, K and V to shared memory through the page table
//     warp 12          one thread issues the products: S = Q K^T from shared memory, O += P V with P from tensor memory
//     warp 13          works out which piece of which tile is next, for all of them
//
// A tile of at most 128 rows is worked on by both halves all the same: they take its blocks of keys in turn, and the first adds the second's
// sums to its own at the end (49 rows over up to 27,300 keys of 18 requests: 113 us, by one half 133).
//
// A row's maximum is only raised when a score is more than 2^8 times beyond it in weight: weights up to 2^8 (in fp16 2^15, see kLift) lose nothing as
// 16-bit or 32-bit floats, and O, which has to be multiplied in tensor memory for every raise, is then left alone in nearly every block.
// (Two halves of queries in turn, scores and weights in tensor memory, and a maximum that lags behind are published methods for such tensor cores.)
//
// Keys and values come by TMA, a box of up to 32 tokens of one page at a time, where pages allow it (8, 16 or a multiple of 32 tokens) and
// all 32 are seen; else by 16-byte asynchronous copies: pages may have any size, a block's last keys may lie in the middle of one, and
// what lies behind them has to arrive as zeros (a weight of zero does not keep NaN out of a product).
//
// 8,192 tokens of 32 heads: 589 us, 933 TFLOP/s with the power cap (1,050 in a cold run); 256 tokens over 16,384 keys, 64 / 8 heads: 149 us.
// A block of 128 keys takes 3,050 cycles for 256 rows: a half's weights take 1,750 and its products 1,180, and the halves take turns; the
// products alone would take 2,048.  Loops stay loops and one thread issues the products: the roles' code shares the instruction
// caches, and unrolled it took twice the time.
#include "cg_attend.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace cg {
namespace {

constexpr int kTileThreads = 512;
constexpr int kTileStages128 = 5;  // K or V tiles of 128 keys x 128 values

__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes;
}

// ---- TMA ----------------------------------------------------------------------------------------
struct PageMaps {  // of keys and values [pages, heads, page_size, head_size]; rows 0: TMA cannot read these pages
    CUtensorMap k, v;
    int32_t rows;  // tokens of a box
};
__device__ __forceinline__ void tma_box(uint32_t to, const CUtensorMap *map, int value, int token, int head, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(map),
                 "r"(value), "r"(token), "r"(head), "r"(page), "r"(bar) : "memory");
}

// ---- tensor memory and products ---------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t dst, int columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, int columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// (descriptors by their lower halves: one addition moves an operand)
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nmov.b64 x, {%1, %3};\nmov.b64 y, {%2, %3};\nsetp.ne.u32 p, %5, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(add ? 1 : 0) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 y;\nmov.b64 y, {%2, %3};\nsetp.ne.u32 p, %5, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(add ? 1 : 0) : "memory");
}
// an operand in shared memory, rows (of queries, of keys) of 64 values that are swizzled in groups of 8 rows, 1024 bytes; `panel`: bytes
// from 64 values of a row to the next 64, where they are the operand's outer axis
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t panel) { return ((addr >> 4) & 0x3FFF) | ((panel >> 4) & 0x3FFF) << 16; }
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
// 32-bit sums of products of 16-bit values, 128 rows, n columns; b_outer: the second operand's rows are the summed axis
__host__ __device__ constexpr uint32_t product(int dtype, int n, bool b_outer) {
    const uint32_t type = dtype == CG_BF16 ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | (b_outer ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}

__device__ __forceinline__ void tmem_load32(uint32_t (&x)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]),
                   "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]),
                   "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]),
                   "=r"(x[31]) : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&x)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]),
                   "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15]), "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&x)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::"r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]),
                   "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15]), "r"(x[16]), "r"(x[17]), "r"(x[18]), "r"(x[19]), "r"(x[20]),
                   "r"(x[21]), "r"(x[22]), "r"(x[23]), "r"(x[24]), "r"(x[25]), "r"(x[26]), "r"(x[27]), "r"(x[28]), "r"(x[29]), "r"(x[30]),
                   "r"(x[31]), "r"(at) : "memory");
}
// (the registers are named so that nothing reads them in front of the wait)
__device__ __forceinline__ void tmem_load_wait(uint32_t (&x)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]), "+r"(x[10]),
                   "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]), "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]),
                   "+r"(x[21]), "+r"(x[22]), "+r"(x[23]), "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]), "+r"(x[30]),
                   "+r"(x[31]) :: "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- pairs of 32-bit floats, as one instruction takes them ------------------------------------------------
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ float2 parts_of(uint64_t p) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int DT> __device__ __forceinline__ uint32_t round_pair(float lo, float hi) {
    uint32_t w;
    if (DT == CG_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
// 32 scores to weights 2^(s * scale + down), rounded to 16 bits for the product: off by half a step each.  Those of fp16 are 2^7 times what they
// are of bf16, so up to 2^15 with a maximum that lags behind by 2^8: its step stops shrinking at 2^-14.  So half a step holds
// down to 2^-21 of the largest; what is below 2^-32 is 0, of n keys n 2^-32 together.  The sum of weights is as many times larger.
template <int DT> constexpr float kLift = DT == CG_F16 ? 7.0f : 0.0f;
template <int DT> __device__ __forceinline__ void weigh(const uint32_t (&x)[32], uint64_t scale, uint64_t down, uint32_t (&w)[16], uint64_t (&sum)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 y = parts_of(pair_fma(pair_of(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale, down));
        const float w0 = exp2_approx(y.x), w1 = exp2_approx(y.y);
        sum[i & 1] = pair_add(sum[i & 1], pair_of(w0, w1));
        w[i] = round_pair<DT>(w0, w1);
    }
}

// ---- shared memory ------------------------------------------------------------------------------
// Q [2 halves][DP / 64 panels][128 rows][128 bytes], then the ring of K and V tiles [DP / 64][128 keys][128 bytes]; the 16-byte piece p of a
// row lies at p ^ row % 8, which is the swizzle that the products expect.
template <int DP> constexpr int kTileBytes = 128 * DP * 2;
template <int DP> constexpr int kTileStages = kTileStages128 * 128 / DP;
template <int DP> constexpr int kBarsAt = (2 + kTileStages<DP>)*kTileBytes<DP>;
template <int DP> constexpr int kTilesSmem = kBarsAt<DP> + 512 + 1024 + 1024;  // and what it takes to begin at a multiple of 1024
enum { kQFull, kQEmpty, kSFull, kPFull = kSFull + 2, kOFull = kPFull + 4, kPieceFull = kOFull + 2, kPieceEmpty = kPieceFull + 2,
       kJoinReady = kPieceEmpty + 2, kJoinDone, kKvFull };  // two each of S, O and pieces; P: the first 96 keys' weights of a
// half, then the others'

// A piece as the scheduling warp hands it to the others, 48 bytes.
struct __align__(16) Parcel {
    int32_t first, n, kv, request;
    int32_t head, t, begin, end;  // no blocks: there are no more pieces
    int32_t lo, hi, starts, whole;
};

template <int DT, int DP>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tiles_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ PageMaps maps) {
    extern __shared__ unsigned char raw[];
    constexpr int kStages = kTileStages<DP>, kPieces = DP / 8, kRowsAtOnce = 32 / kPieces;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (known to be the same in a warp)
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    unsigned char *mem = raw + (base - smem_addr(raw));
    const uint32_t tiles_at = base + 2 * kTileBytes<DP>, bars = base + kBarsAt<DP>;
    const auto bar = [&](int i) { return bars + 8 * i; };
    const auto full = [&](int s) { return bar(kKvFull + s); };
    const auto empty = [&](int s) { return bar(kKvFull + kStages + s); };
    static_assert(8 * (kKvFull + 2 * kStages) <= 320, "room for the barriers");
    volatile int *words = reinterpret_cast<volatile int *>(mem + kBarsAt<DP> + 320);  // tensor memory, failed, bar_wait's clock
    Parcel *parcels = reinterpret_cast<Parcel *>(mem + kBarsAt<DP> + 384);  // [2]
    volatile int *failed = words + 1;

    Run<kTileRows, kTileKeys, kTileCost> run;  // (of warp 13; all find their run together)
    if (tid == 0 && maps.rows) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    run.template init<kTileThreads, true>(a, reinterpret_cast<int64_t *>(mem));
    let_next_launch_start();
    if (tid == 0) {
        bar_init(bar(kQFull), 4);
        bar_init(bar(kQEmpty), 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(kSFull + i), 1);
            bar_init(bar(kPFull + 2 * i), 4);
            bar_init(bar(kPFull + 2 * i + 1), 4);
            bar_init(bar(kOFull + i), 1);
            bar_init(bar(kPieceFull + i), 1);
            bar_init(bar(kPieceEmpty + i), 13);  // warps that read it
        }
        bar_init(bar(kJoinReady), 4);
        bar_init(bar(kJoinDone), 4);
        for (int s = 0; s < kStages; ++s) bar_init(full(s), 4), bar_init(empty(s), 1);
        failed[0] = failed[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) tmem_alloc(base + kBarsAt<DP> + 320, 512);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (TMA writes where `run` has had its numbers)
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = words[0];
    // columns: S (and P) of the halves, then O
    const auto s_at = [&](int half) { return tmem + 128 * half; };
    const auto o_at = [&](int half) { return tmem + 256 + 128 * half; };
    float2 *join_ml = reinterpret_cast<float2 *>(mem + kBarsAt<DP> + 512);  // [128]: maxima and sums of the second half
    // the next piece: every warp reads it for itself
    Parcel p;
    int pieces = 0;
    const auto next_piece = [&]() {
        if (!warp_wait(bar(kPieceFull + (pieces & 1)), pieces >> 1 & 1, failed)) return false;
        const int4 *from = reinterpret_cast<const int4 *>(parcels + (pieces & 1));
        int4 *to = reinterpret_cast<int4 *>(&p);
        to[0] = from[0], to[1] = from[1], to[2] = from[2];
        __syncwarp();
        if (lane == 0) bar_arrive(bar(kPieceEmpty + (pieces & 1)));
        ++pieces;
        return p.end > p.begin;
    };

    if (warp < 8) {
        // ================================================================ softmax: a row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int half = warp >> 2, in_half = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_mine = s_at(half) + lanes, o_mine = o_at(half) + lanes;
        uint32_t s_phase = 0, o_phase = 0, join_phase = 0;
        bool ok = true;
        while (ok && next_piece()) {
            const Lengths r{p.first, p.n, p.kv};
            const int blocks = p.end - p.begin, row0 = p.t * kTileRows, rows = min(kTileRows, r.n * a.group - row0);
            const bool both = rows <= 128;  // both halves have the same rows, and every second block each
            const int step = both ? 2 : 1, first = both ? half : 0, top_row = both ? 0 : half * 128, row = top_row + in_half;
            if (first >= blocks) continue;
            const bool there = row < rows;
            const int token = there ? token_of<kTileRows>(a, row0 + row) : 0, head = p.head * a.group + (there ? member_of(a, row0 + row, token) : 0);
            // (rows behind the last see everything: they ask for no masks)
            const int lo = there ? first_key(a, r, token) : 0, hi = there ? last_key(a, r, token) : INT32_MAX;
            const int half_lo = first_key(a, r, token_of<kTileRows>(a, row0 + min(rows, top_row + 128) - 1));
            const int half_hi = last_key(a, r, token_of<kTileRows>(a, row0 + top_row));
            const bool any_masked = p.begin * kTileKeys < half_lo || p.end * kTileKeys > half_hi;
            float m = kNegInf, l = 0.0f;
            for (int j = first; j < blocks; j += step) {
                const int key = (p.begin + j) * kTileKeys;
                ok = warp_wait(bar(kSFull + half), s_phase, failed);
                s_phase ^= 1;
                if (!ok) break;
                fence_after();
                const bool masked = key < half_lo || key + kTileKeys > half_hi;  // for one of the half's rows
                uint32_t x[4][32];
                tmem_load32(x[0], s_mine);
                tmem_load32(x[1], s_mine + 32);
                tmem_load_wait(x[0]);
                tmem_load_wait(x[1]);
                tmem_load32(x[2], s_mine + 64);
                tmem_load32(x[3], s_mine + 96);
                const uint32_t from = key - lo, count = max(0, hi - lo);  // key + i is seen: from + i < count, without signs
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) x[i / 32][i % 32] = from + i < count ? x[i / 32][i % 32] : __float_as_uint(kNegInf);
                }
                float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                for (int i = 0; i < 64; i += 2) top[i / 2 & 3] = max3(top[i / 2 & 3], __uint_as_float(x[i / 32][i % 32]), __uint_as_float(x[i / 32][i % 32 + 1]));
                tmem_load_wait(x[2]);
                tmem_load_wait(x[3]);
                if (masked) {
#pragma unroll
                    for (int i = 64; i < 128; ++i) x[i / 32][i % 32] = from + i < count ? x[i / 32][i % 32] : __float_as_uint(kNegInf);
                }
#pragma unroll
                for (int i = 64; i < 128; i += 2) top[i / 2 & 3] = max3(top[i / 2 & 3], __uint_as_float(x[i / 32][i % 32]), __uint_as_float(x[i / 32][i % 32 + 1]));
                const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale;
                const bool raise = high > m + 8.0f || (m == kNegInf && high > m);
                if (__any_sync(0xffffffffu, raise)) {
                    const float keep = raise ? (m == kNegInf ? 0.0f : exp2_approx(m - high)) : 1.0f;
                    if (raise) m = high;
                    l *= keep;
                    if (j > first) {  // the products of the block before are done: this block's scores came behind them
#pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t y[32];
                            tmem_load32(y, o_mine + 32 * c);
                            tmem_load_wait(y);
#pragma unroll
                            for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * keep);
                            tmem_store32(o_mine + 32 * c, y);
                        }
                    }
                }
                const float base = m == kNegInf ? 0.0f : kLift<DT> - m;
                const uint64_t scale = pair_of(a.scale, a.scale), down = pair_of(base, base);
                uint64_t sum[2] = {0, 0};
                // (weights take half the columns of the scores that they come from: these have been read)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
                    weigh<DT>(x[c], scale, down, w, sum);
                    tmem_store16(s_mine + 16 * c, w);
                    if (c >= 2) {  // the products begin with three quarters of the weights, while the last are worked out
                        tmem_store_wait();
                        fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(bar(kPFull + 2 * half + c - 2));
                    }
                }
                const float2 s0 = parts_of(sum[0]), s1 = parts_of(sum[1]);
                l += (s0.x + s0.y) + (s1.x + s1.y);
            }
            m -= kLift<DT>;  // what the sums are relative to
            ok = ok && warp_wait(bar(kOFull + half), o_phase, failed);
            o_phase ^= 1;
            if (!ok) break;
            fence_after();
            if (both && blocks > 1) {  // the first half adds the second's sums to its own
                if (half) {
                    join_ml[in_half] = make_float2(m, l);
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(kJoinReady));
                    ok = warp_wait(bar(kJoinDone), join_phase, failed);
                    join_phase ^= 1;
                    continue;
                }
                ok = warp_wait(bar(kJoinReady), join_phase, failed);
                join_phase ^= 1;
                if (!ok) break;
                fence_after();
                const float2 ml = join_ml[in_half];
                const float high = fmaxf(m, ml.x), base = high == kNegInf ? 0.0f : high;
                const float mine = exp2_approx(m - base), other = exp2_approx(ml.x - base);
                l = l * mine + ml.y * other;
                m = high;
#pragma unroll 1
                for (int c = 0; c < DP / 32; ++c) {
                    uint32_t y[32], z[32];
                    tmem_load32(y, o_mine + 32 * c);
                    tmem_load32(z, o_mine + 128 + 32 * c);
                    tmem_load_wait(y);
                    tmem_load_wait(z);
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * mine + __uint_as_float(z[i]) * other);
                    tmem_store32(o_mine + 32 * c, y);
                }
                tmem_store_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(kJoinDone));
            }
            char *part = a.parts + (2 * blockIdx.x + (p.starts ? 1 : 0)) * part_bytes(kTileRows, DP);
            float2 *part_ml = reinterpret_cast<float2 *>(part + kTileRows * DP * 4);
            const bool sees = hi > lo;
            bool odd = false;
            const float inv = sees ? 1.0f / l : 0.0f;
            const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | a.out_token | a.out_head) & 31) == 0;
            char *to = a.out + (r.first + token) * a.out_token + head * a.out_head;
            uint32_t y[32];
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                tmem_load32(y, o_mine + 32 * c);
                tmem_load_wait(y);
                if (any_masked) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) odd = odd || (y[i] & 0x7F800000u) == 0x7F800000u;
                }
                if (there && p.whole) {
                    // 32 bytes at a time where they are aligned: a thread's row is its own, and halves of a sector take as long
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t h[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            h[k] = round_pair<DT>(__uint_as_float(y[16 * i + 2 * k]) * inv, __uint_as_float(y[16 * i + 2 * k + 1]) * inv);
                            if (!sees) h[k] = 0;
                        }
                        char *at = to + 2 * (32 * c + 16 * i);
                        const int left = a.head_size - (32 * c + 16 * i);
                        if (wide && left >= 16) {
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]), "r"(h[4]),
                                         "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                        } else {
                            if (left >= 8) *reinterpret_cast<uint4 *>(at) = make_uint4(h[0], h[1], h[2], h[3]);
                            if (left >= 16) *reinterpret_cast<uint4 *>(at + 16) = make_uint4(h[4], h[5], h[6], h[7]);
                        }
                    }
                } else if (there) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4 *>(part + ((8 * c + i) * kTileRows + row) * 16) = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                }
            }
            if (there && p.whole && a.lse)
                a.lse[static_cast<int64_t>(r.first + token) * a.q_heads + head] = sees ? (m + log2f(l)) * 0.693147180559945f : kNegInf;
            if (there && !p.whole) part_ml[row] = make_float2(m, l);
            // A value that is not finite, of a key that some rows do not see, is in all rows' sums: those rows are done again, from memory.
            // (Such keys lie in front of half_lo or from half_hi on; the blocks at these borders have keys that most rows see.)
            uint32_t again = __ballot_sync(0xffffffffu, odd && there);
            if (again) {
                const int k0 = max(p.lo, p.begin * kTileKeys), k3 = min(p.hi, p.end * kTileKeys);
                const int k1 = half_lo > k0 ? min(k3, (half_lo / kTileKeys + 1) * kTileKeys) : k0;
                const int k2 = half_hi < k3 ? max(k1, max(half_hi - 1, 0) / kTileKeys * kTileKeys) : k3;
                again = rows_again<DT, DP>(a, p.request, p.head, again, lo, hi, k0, k1, k2, k3);
            }
            for (; again; again &= again - 1) {
                const int i = top_row + 32 * (warp & 3) + __ffs(again) - 1;
                __syncwarp();  // (the row has been written once)
                float x[DP / 32], top, total;
                slow_row<DT, DP>(a, r, p.request, p.head, row0 + i, p.begin * kTileKeys, p.end * kTileKeys, failed, x, top, total);
                const int tok = token_of<kTileRows>(a, row0 + i), hd = p.head * a.group + member_of(a, row0 + i, tok);
                const bool any = last_key(a, r, tok) > first_key(a, r, tok);
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    const int d = lane * (DP / 32) + c;
                    if (!p.whole) reinterpret_cast<float *>(part)[(d / 4 * kTileRows + i) * 4 + d % 4] = x[c];
                    else if (d < a.head_size)
                        reinterpret_cast<uint16_t *>(a.out + (r.first + tok) * a.out_token + hd * a.out_head)[d] = any ? Half16<DT>::from_float(x[c] / total) : 0;
                }
                if (lane == 0 && !p.whole) part_ml[i] = make_float2(top, total);
                if (lane == 0 && p.whole && a.lse)
                    a.lse[static_cast<int64_t>(r.first + tok) * a.q_heads + hd] = any ? (top + log2f(total)) * 0.693147180559945f : kNegInf;
            }
            fence_before();  // O has been read: the next piece's products follow an arrival of this warp
        }
    } else if (warp < 12) {
        // ================================================================ copies
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        const int w = warp - 8, piece = lane % kPieces;
        // A tile of copies is told of when kLag more have been begun.  Products may need the tile behind the first that is not free yet: the
        // ring has to hold both and kLag more.
        constexpr int kLag = 2;
        static_assert(kStages >= kLag + 2, "the products would wait for a tile that waits for them");
        const uint32_t at_piece = static_cast<uint32_t>(piece / 8) * 16384;
        const bool box_lane = maps.rows && lane % maps.rows == 0;  // the lane of a box's first token
        const int box_bytes = 32 * DP * 2;
        int stage = 0, untold = 0, q_phase = 0;  // of the next tile; tiles by copies, the last ones begun, that have not been told of
        uint32_t phase = 1;                      // (a barrier's phase before its first is over)
        bool ok = true, first_piece = true;
        const auto tell_first = [&]() {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            const int at = stage - untold;
            if (lane == 0) bar_arrive(full(at < 0 ? at + kStages : at));
            --untold;
        };
        const auto tell_all = [&]() {
            if (!untold) return;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            while (untold) tell_first();
        };
        // where this lane's pieces of a tile go: rows 2 i + lane / 16 (of DP 64: 4 i + lane / 8) of the warp's 32
        constexpr int kOrders = 8 / kRowsAtOnce;  // of a row's pieces, which repeat every 8 rows
        uint32_t place[kOrders];
#pragma unroll
        for (int i = 0; i < kOrders; ++i) {
            const int row = i * kRowsAtOnce + lane / kPieces;
            place[i] = at_piece + (32 * w + row) * 128 + (((piece & 7) ^ (row & 7)) << 4);
        }
        const bool in_head = 8 * piece < a.head_size;
        const auto copy_rows = [&](uint32_t tile, const char *at, bool there) {  // lane i: where row 32 w + i lies
            const uint32_t rows_there = __ballot_sync(0xffffffffu, there);
            const uint64_t where = reinterpret_cast<uint64_t>(at);
#pragma unroll
            for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
                const int src = i * kRowsAtOnce + lane / kPieces;
                const uint64_t from = __shfl_sync(0xffffffffu, where, src);
                const bool copy = in_head && (rows_there >> src & 1);
                const uint32_t dst = tile + place[i % kOrders] + i / kOrders * 1024;
                const uint64_t where_from = copy ? from + 16 * piece : reinterpret_cast<uint64_t>(a.q);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(where_from), "r"(copy ? 16 : 0) : "memory");
            }
        };
        while (ok && next_piece()) {
            const Lengths r{p.first, p.n, p.kv};
            const int blocks = p.end - p.begin, row0 = p.t * kTileRows, rows = min(kTileRows, r.n * a.group - row0);
            const auto page_for = [&](int j) {
                const int key = (p.begin + j) * kTileKeys + 32 * w + lane;
                return j < blocks && key >= p.lo && key < p.hi ? page_of(a, p.request, page_index(a, key)) : -1;
            };
            const auto copy_queries = [&]() {
#pragma unroll 1
                for (int half = 0; half < (rows > 128 ? 2 : 1); ++half) {
                    const int row = half * 128 + 32 * w + lane;
                    const bool there = row < rows;
                    const int token = there ? token_of<kTileRows>(a, row0 + row) : 0, head = p.head * a.group + (there ? member_of(a, row0 + row, token) : 0);
                    copy_rows(base + half * kTileBytes<DP>, a.q + (r.first + token) * a.q_token + head * a.q_head, there);
                }
            };
            int page = page_for(0);
            if (first_piece) copy_queries();  // while the table is read
            tell_all();  // what the products of the piece before need
            // Tiles in the order in which products use them: keys and values of a block after the other; with both halves on the same rows the
            // next block's keys in front of a block's values.
            const int behind = rows <= 128 ? 1 : 0;
            int in_page = 0, here = -1, in_page_before = 0, here_before = -1;
#pragma unroll 1
            for (int j = 0; ok && j < blocks + behind; ++j) {
                in_page_before = in_page, here_before = here;
                in_page = place_in_page(a, (p.begin + j) * kTileKeys + 32 * w + lane), here = page;
                page = page_for(j + 1);
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    if (kv ? j < behind : j >= blocks) continue;
                    const int at_page = kv && behind ? here_before : here, at_token = kv && behind ? in_page_before : in_page;
                    const bool boxes = maps.rows && __all_sync(0xffffffffu, at_page >= 0);
                    if (boxes) tell_all();
                    if (!(ok = warp_wait(empty(stage), phase, failed))) break;
                    const uint32_t tile = tiles_at + stage * kTileBytes<DP>;
                    if (boxes) {
                        if (lane == 0) bar_expect(full(stage), box_bytes);
                        __syncwarp();
                        if (box_lane) {
#pragma unroll
                            for (int panel = 0; panel < DP / 64; ++panel)
                                tma_box(tile + panel * 16384 + (32 * w + lane) * 128, kv ? &maps.v : &maps.k, 64 * panel, at_token, p.head, at_page, full(stage));
                        }
                    } else {
                        const char *at = kv ? a.v + at_page * a.v_page + at_token * a.v_token + p.head * a.v_head
                                            : a.k + at_page * a.k_page + at_token * a.k_token + p.head * a.k_head;
                        copy_rows(tile, at, at_page >= 0);
                        asm volatile("cp.async.commit_group;" ::: "memory");
                        ++untold;
                    }
                    if (++stage == kStages) stage = 0, phase ^= 1;
                    if (untold > kLag) {
                        asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
                        tell_first();
                    }
                }
                if (!ok || j > 0) continue;
                // the queries of all pieces but the first, behind the first block's tiles: once the last products with the ones before are done
                if (!first_piece) {
                    if (!(ok = warp_wait(bar(kQEmpty), q_phase, failed))) break;
                    q_phase ^= 1;
                    copy_queries();
                }
                first_piece = false;
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(bar(kQFull));
                while (untold) tell_first();
            }
        }
        if (ok) tell_all();
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ================================================================ products
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 12) {
            // the whole warp goes through the same steps, so that operands stay in uniform registers; one thread issues
            constexpr uint32_t qk = product(DT, kTileKeys, false), pv = product(DT, DP, true);
            constexpr uint32_t kTile = kTileBytes<DP> >> 4;  // in units of a descriptor's address
            const uint32_t q_desc = operand(base, 16), k_desc = operand(tiles_at, 16), v_desc = operand(tiles_at, 16384);
            const bool issues = elect_one();
            uint32_t p_phase = 0, q_phase = 0, stage = 0, phase = 0;  // of the tile that is waited for next
            bool ok = true;
            const auto scores = [&](int half, uint32_t at) {
                const uint32_t q = q_desc + half * kTile, k = k_desc + at * kTile;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) mma_ss(s_at(half), q + (i / 4) * 1024 + (i % 4) * 2, k + (i / 4) * 1024 + (i % 4) * 2, kOperandHigh, qk, i > 0);
            };
            const auto tile_there = [&]() {  // its stage, when it is there
                const uint32_t at = stage;
                ok = warp_wait(full(at), phase, failed);
                if (++stage == kStages) stage = 0, phase ^= 1;
                return at;
            };
            while (ok && next_piece()) {
                const int blocks = p.end - p.begin, rows = min(kTileRows, p.n * a.group - p.t * kTileRows), halves = rows > 128 ? 2 : 1;
                if (!(ok = warp_wait(bar(kQFull), q_phase, failed))) break;
                q_phase ^= 1;
                uint32_t k_stage = tile_there(), v_stage = 0;
                if (!ok) break;
                fence_after();
                if (halves == 1) {  // both halves on the same rows
                    const auto begin = [&](int half, uint32_t at, bool last) {  // scores of one block
                        if (!issues) return;
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i)
                            mma_ss(s_at(half), q_desc + (i / 4) * 1024 + (i % 4) * 2, k_desc + at * kTile + (i / 4) * 1024 + (i % 4) * 2, kOperandHigh, qk, i > 0);
                        commit(bar(kSFull + half));
                        commit(empty(at));
                        if (last) commit(bar(kQEmpty));
                    };
                    begin(0, k_stage, blocks == 1);
                    if (blocks > 1) {
                        k_stage = tile_there();
                        if (ok) fence_after(), begin(1, k_stage, blocks == 2);
                    }
#pragma unroll 1
                    for (int j = 0; ok && j < blocks; ++j) {
                        const int half = j & 1;
                        const bool more = j + 2 < blocks;
                        if ((j & 1023) == 1023) beat(failed);  // (warp 13 waits for the length of a piece)
                        v_stage = tile_there();
                        if (!ok || !(ok = warp_wait(bar(kPFull + 2 * half), p_phase >> half & 1, failed)) ||
                            !(ok = warp_wait(bar(kPFull + 2 * half + 1), p_phase >> half & 1, failed)))
                            break;
                        p_phase ^= 1 << half;
                        fence_after();
                        if (issues) {
#pragma unroll
                            for (int k = 0; k < kTileKeys / 16; ++k)
                                mma_ts(o_at(half), s_at(half) + 8 * k, v_desc + v_stage * kTile + k * 128, kOperandHigh, pv, j > 1 || k > 0);
                            if (!more) commit(bar(kOFull + half));
                            commit(empty(v_stage));
                        }
                        if (more) {
                            k_stage = tile_there();
                            if (ok) fence_after(), begin(half, k_stage, j + 3 == blocks);
                        }
                        __syncwarp();
                    }
                    continue;
                }
                if (issues) {
                    scores(0, k_stage);
                    commit(bar(kSFull));
                    scores(1, k_stage);
                    commit(bar(kSFull + 1));
                    commit(empty(k_stage));
                    if (blocks == 1) commit(bar(kQEmpty));
                }
#pragma unroll 1
                for (int j = 0; j < blocks; ++j) {
                    const bool more = j + 1 < blocks;
                    if ((j & 1023) == 1023) beat(failed);
                    v_stage = tile_there();
                    if (ok && more) k_stage = tile_there();  // (ahead of the weights, which all that follows waits for)
                    if (!ok) break;
                    const uint32_t v = v_desc + v_stage * kTile;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!(ok = warp_wait(bar(kPFull + 2 * half), p_phase >> half & 1, failed))) break;
                        fence_after();
                        if (issues) {
#pragma unroll
                            for (int k = 0; k < 6; ++k) mma_ts(o_at(half), s_at(half) + 8 * k, v + k * 128, kOperandHigh, pv, j > 0 || k > 0);
                        }
                        if (!(ok = warp_wait(bar(kPFull + 2 * half + 1), p_phase >> half & 1, failed))) break;
                        p_phase ^= 1 << half;
                        fence_after();
                        if (issues) {
#pragma unroll
                            for (int k = 6; k < kTileKeys / 16; ++k) mma_ts(o_at(half), s_at(half) + 8 * k, v + k * 128, kOperandHigh, pv, true);
                            if (more) scores(half, k_stage);
                            commit(bar(more ? kSFull + half : kOFull + half));
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (issues) {
                        commit(empty(v_stage));
                        if (more) commit(empty(k_stage));
                        if (j + 2 == blocks) commit(bar(kQEmpty));
                    }
                    __syncwarp();
                }
            }
        }
        if (warp == 13) {
            Join join{};
            Piece x;
            bool more = true;
            for (int i = 0; more; ++i) {
                more = run.next(a, x);
                if (more && x.sharers) join = join_for(x);
                if (i >= 2 && !warp_wait(bar(kPieceEmpty + (i & 1)), (i / 2 - 1) & 1, failed)) break;
                if (lane == 0) {
                    Parcel &to = parcels[i & 1];
                    to = more ? Parcel{x.r.first, x.r.n, x.r.kv, x.request, x.head, x.t, x.begin, x.end, x.tile.lo, x.tile.hi, x.starts, x.whole} : Parcel{};
                    bar_arrive(bar(kPieceFull + (i & 1)));
                }
                __syncwarp();
            }
            if (lane == 0 && a.joins) a.joins[blockIdx.x] = join;
        }
        __syncwarp();
    }
    // every product has been waited for (its O read), or the block has given up on one: what is on its way then takes microseconds
    if (*failed) {
        if (lane == 0 && a.status) atomicOr(a.status, CG_S_TIMEOUT);
        for (const uint64_t start = now_ns(); now_ns() - start < 1000000;) {}
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 12) tmem_free(tmem, 512);
}

// Maps of the pages, where TMA can read them: its boxes are whole runs of 8 rows in shared memory, and sizes and strides have limits.
bool map_pages(const AttendArgs &a, int dtype, PageMaps &maps) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }();
    const int rows = a.page_size % 32 == 0 ? 32 : a.page_size;
    if (!encode || (rows != 32 && rows != 16 && rows != 8) || a.num_pages == 0) return false;
    const cuuint64_t sizes[4] = {static_cast<cuuint64_t>(a.head_size), static_cast<cuuint64_t>(a.page_size), static_cast<cuuint64_t>(a.heads),
                                 static_cast<cuuint64_t>(a.num_pages)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, steps[4] = {1, 1, 1, 1};
    const auto one = [&](CUtensorMap &map, const char *at, int64_t token, int64_t head, int64_t page) {
        cuuint64_t strides[3] = {static_cast<cuuint64_t>(token), static_cast<cuuint64_t>(head), static_cast<cuuint64_t>(page)};
        for (int i = 0; i < 3; ++i) {
            if (sizes[i + 1] == 1) strides[i] = 16;  // never used
            if (strides[i] == 0 || strides[i] % 16 || strides[i] >= 1ull << 40) return false;
        }
        const CUtensorMapDataType type = dtype == CG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        return encode(&map, type, 4, const_cast<char *>(at), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (!one(maps.k, a.k, a.k_token, a.k_head, a.k_page) || !one(maps.v, a.v, a.v_token, a.v_head, a.v_page)) return false;
    maps.rows = rows;
    return true;
}

template <int DT, int DP> int launch_tiles(const AttendArgs &a, int ctas, cudaStream_t st) {
    constexpr int smem = kTilesSmem<DP>;
    PageMaps maps{};
    if (!map_pages(a, DT, maps)) maps.rows = 0;
    int rc = allow_smem(attend_tiles_kernel<DT, DP>, smem);
    if (rc) return rc;
    rc = launch(attend_tiles_kernel<DT, DP>, dim3(ctas), kTileThreads, smem, false, st, a, maps);
    if (rc || !a.joins) return rc;
    return launch(combine_kernel<DT, kTileRows, DP>, dim3(ctas, kTileRows / 64), 64 * (DP / 16), 0, true, st, a);
}

}  // namespace

int launch_attend_tiles(const AttendArgs &a, int dtype, int ctas, cudaStream_t st) {
    if (a.head_size <= 64) return dtype == CG_F16 ? launch_tiles<CG_F16, 64>(a, ctas, st) : launch_tiles<CG_BF16, 64>(a, ctas, st);
    return dtype == CG_F16 ? launch_tiles<CG_F16, 128>(a, ctas, st) : launch_tiles<CG_BF16, 128>(a, ctas, st);
}

}  // namespace cg
