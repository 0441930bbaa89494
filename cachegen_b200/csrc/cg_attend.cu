// Attention over a paged KV cache: the entry point, and the kernel for few query rows a key/value head (single tokens, drafts).
//
// With up to 16 rows a head every cached value is used for few products and the kernel's time is that of reading the cache
// once.  So a block is there to keep loads in flight: four warps walk through 16 keys at a time each, every one with a warp of its own
// that copies keys and values to a ring for it, and no barrier of the block; the warps' sums are joined when the block's piece of
// the tile ends, while the next piece's keys are on their way.  Copies are 16 bytes a lane, asynchronous: pages may have any size and
// strides.  (A bulk copy a row is one instruction for 32 rows, but took 2,400 cycles to issue where these take 500.)  Products are
// m16n8k16 on fragments in registers: tcgen05 takes 64 rows at least, its accumulator would have to come back from tensor memory for each
// 16 keys, and at 16 rows the products take less than a fifth of the time that the keys take to arrive.
//
// A step of 64 requests of up to 4,096 tokens (32 / 8 heads, 753 MB): 150 us, 5.0 TB/s; the blocks read at 6.0 while they run.  One request of
// 32,768 tokens (134 MB): 37 us, of which 6 pass before keys flow and 6 while 37 blocks' parts of each head are joined.
#include "cg_attend.cuh"

namespace cg {
namespace {

constexpr int kRowsM = 16, kWarps = 4, kStages = 3, kChunk = 16;
constexpr int kRowsBK = kWarps * kChunk, kRowsCost = 1;

template <int DT>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (DT == CG_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or zeros where there is nothing to read; and an arrival at a barrier when the thread's copies so far are there
__device__ __forceinline__ void copy16(uint32_t to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_behind_copies(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void sync_weighing_warps() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int DT> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    return Half16<DT>::from_float(lo) | static_cast<uint32_t>(Half16<DT>::from_float(hi)) << 16;
}
// whether one of two 16-bit floats is infinite or no number
template <int DT> __device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t e = DT == CG_F16 ? 0x7C00u : 0x7F80u;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// Shared memory: kWarps rings of kStages stages of 16 keys, then 16 values; rows are 16 bytes longer than their 2 * DP, so that the
// eight rows of a matrix lie in different banks.  Then room for a part of the warps' sums, their maxima and sums of weights, a word that
// says whether values that are not finite were met where rows see unlike keys, one that says that a wait was given up, one for bar_wait's
// clock, and the stages' barriers.  Two blocks share an SM.
template <int DP> constexpr int kRowBytes2 = 2 * DP + 16;
template <int DP> constexpr int kStageBytes = 2 * kChunk * kRowBytes2<DP>;
template <int DP> constexpr int kRingBytes = kStages * kStageBytes<DP>;
constexpr int most_of(int x, int y) { return x > y ? x : y; }
constexpr int kSumFloats = 16 * 36;  // of a warp: 16 rows of 32 values, 8 of 64 or 4 of 128, four more between rows
template <int DP> constexpr int kSumsAt = most_of(kWarps * kRingBytes<DP>, (CG_MAX_REQUESTS + 1) * 8 + 8);
template <int DP> constexpr int kMlAt = kSumsAt<DP> + kWarps * kSumFloats * 4;
template <int DP> constexpr int kAttendSmem = kMlAt<DP> + kWarps * kRowsM * 8 + 16 + 16 * kWarps * kStages;
static_assert(2 * (kAttendSmem<128> + 1024) <= 228 * 1024, "two blocks an SM");

// Weights are numbers up to 1, rounded to the cache's type for the second product.  Those of fp16 are 2^15 times that: its step stops
// shrinking at 2^-14 and what is below 2^-25 is 0, where a million such weights beside a large one are 3 % of the result.  So they are off by half a
// step down to 2^-29 of the largest; those below 2^-40 are 0, of n keys n 2^-40 together.  The sum of weights is as many times larger.
template <int DT> constexpr float kLift = DT == CG_F16 ? 15.0f : 0.0f;

template <int DT, int DP>
__global__ void __launch_bounds__(kWarps * 64, 2) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    float2(*row_ml)[kRowsM] = reinterpret_cast<float2(*)[kRowsM]>(smem + kMlAt<DP>);  // [kWarps]
    volatile int &row_odd = *reinterpret_cast<volatile int *>(smem + kMlAt<DP> + kWarps * kRowsM * 8);
    constexpr int kSteps = DP / 16, kRow = kRowBytes2<DP>;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, (tid >> 5) % kWarps, 0);
    const bool copies = tid >= kWarps * 32;
    const uint32_t ring = smem_addr(smem) + warp * kRingBytes<DP>;
    volatile int *failed = &row_odd + 1;
    const uint32_t full = smem_addr(smem) + kMlAt<DP> + kWarps * kRowsM * 8 + 16 + 16 * kStages * warp, empty = full + 8 * kStages;

    Run<kRowsM, kRowsBK, kRowsCost> run;
    run.template init<kWarps * 64, false>(a, reinterpret_cast<int64_t *>(smem));
    let_next_launch_start();
    if (tid == 0) row_odd = 0, failed[0] = failed[1] = 0;
    if (!copies && lane == 0) {
        for (int i = 0; i < kStages; ++i) bar_init(full + 8 * i, 32), bar_init(empty + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    uint32_t stage = 0, phase = 0;  // of the next chunk, of all pieces
    bool ok = true;
    Piece p;
    if (copies) {
        // ================================================================ keys and values to the ring of warp `warp`
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");  // 128 threads of 56 and 128 of 200 registers: the 256 x 128 of the launch
        constexpr int kPieces = DP / 8, kRowsAtOnce = 32 / kPieces;  // 16-byte pieces of a row; rows that a warp copies with one instruction
        const int piece = lane % kPieces, in_head = 8 * piece < a.head_size ? 16 : 0;
        const uint32_t place = ring + lane / kPieces * kRow + 16 * piece;
        bool round = false;  // whether the stages have been used
        while (ok && run.next(a, p)) {
            const int nchunks = p.end - p.begin, key0 = p.begin * kRowsBK + warp * kChunk + (lane & 15);
            const char *const keys = a.k + p.head * a.k_head + 16 * piece, *const values = a.v + p.head * a.v_head + 16 * piece;
            const auto page_for = [&](int chunk) {  // lanes i and 16 + i: of key i
                const int key = key0 + chunk * kRowsBK;
                return chunk < nchunks && key >= p.tile.lo && key < p.tile.hi ? page_of(a, p.request, page_index(a, key)) : -1;
            };
            int page = page_for(0);
#pragma unroll 1
            for (int chunk = 0; chunk < nchunks; ++chunk) {
                const int in_page = place_in_page(a, key0 + chunk * kRowsBK);
                // lanes below 16 have the keys' places, the others the values'
                const int64_t at = lane < 16 ? page * a.k_page + in_page * a.k_token : page * a.v_page + in_page * a.v_token;
                const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
                page = page_for(chunk + 1);
                if (round && !(ok = warp_wait(empty + 8 * stage, phase ^ 1, failed))) break;
                const uint32_t to = place + stage * kStageBytes<DP>;
#pragma unroll
                for (int i = 0; i < kChunk / kRowsAtOnce; ++i) {
                    const int row = i * kRowsAtOnce + lane / kPieces;
                    const int64_t k_at = __shfl_sync(0xffffffffu, at, row), v_at = __shfl_sync(0xffffffffu, at, 16 + row);
                    const int bytes = there >> row & 1 ? in_head : 0;
                    copy16(to + i * kRowsAtOnce * kRow, bytes ? keys + k_at : a.q, bytes);
                    copy16(to + (kChunk + i * kRowsAtOnce) * kRow, bytes ? values + v_at : a.q, bytes);
                }
                arrive_behind_copies(full + 8 * stage);
                if (++stage == kStages) stage = 0, phase ^= 1, round = true;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int g = lane >> 2, q2 = 2 * (lane & 3);
    Join join{};
    uint32_t qf[kSteps][4];
    const auto queries = [&](const Piece &x) {  // as fragments
        const int rows = min(kRowsM, x.r.n * a.group - x.t * kRowsM);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = g + 8 * i, at = x.t * kRowsM + row, token = token_of<kRowsM>(a, at);
            const char *q = a.q + (x.r.first + token) * a.q_token + (x.head * a.group + member_of(a, at, token)) * a.q_head + 2 * q2;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int k = 0; k < 2; ++k) qf[s][i + 2 * k] = 0u;
            if (row < rows) {
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (DP == a.head_size || 16 * s + 8 * k < a.head_size)
                            qf[s][i + 2 * k] = __ldg(reinterpret_cast<const unsigned int *>(q + 2 * (16 * s + 8 * k)));
            }
        }
    };
    bool more = run.next(a, p);
    if (more) queries(p);
    while (more) {
        const Lengths r = p.r;
        const int rows = min(kRowsM, r.n * a.group - p.t * kRowsM), row0 = p.t * kRowsM;
        int lo[2], hi[2];  // the keys that this thread's two rows see
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = g + 8 * i, token = token_of<kRowsM>(a, row0 + row);
            lo[i] = row < rows ? first_key(a, r, token) : 0;
            hi[i] = row < rows ? last_key(a, r, token) : 0;
        }
        // chunks inside [all_lo, all_hi) are seen by all rows
        const int first_token = token_of<kRowsM>(a, row0), last_token = token_of<kRowsM>(a, row0 + rows - 1);
        const int all_lo = first_key(a, r, last_token), all_hi = last_key(a, r, first_token);
        const bool mixed = last_token != first_token;  // whether rows see unlike keys (what none sees is zero)
        const int nchunks = p.end - p.begin;
        const int key0 = p.begin * kRowsBK + warp * kChunk;

        float o[kSteps * 2][4], m[2] = {kNegInf, kNegInf}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kSteps * 2; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][k] = 0.0f;
        bool odd = false;
        // this lane's row of the four matrices of an ldmatrix
        const uint32_t k_row = ((lane & 7) + ((lane >> 4) << 3)) * kRow + (((lane >> 3) & 1) << 4), v_row = (kChunk + (lane & 15)) * kRow + ((lane >> 4) << 4);
#pragma unroll 1
        for (int chunk = 0; chunk < nchunks; ++chunk) {
            ok = ok && warp_wait(full + 8 * stage, phase, failed);
            if (!ok) break;
            const uint32_t at = ring + stage * kStageBytes<DP>;
            float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                ldmatrix4(b, at + k_row + 32 * k);
                mma16816<DT>(s[0], qf[k], b[0], b[1]);
                mma16816<DT>(s[1], qf[k], b[2], b[3]);
            }
            const int key = key0 + chunk * kRowsBK;
            const bool all = key >= all_lo && key + kChunk <= all_hi;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[i][k] *= a.scale;
            if (!all) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int j = key + 8 * i + q2 + (k & 1);
                        if (j < lo[k >> 1] || j >= hi[k >> 1]) s[i][k] = kNegInf;
                    }
            }
            float top[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                top[i] = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float now = fmaxf(m[i], top[i]), keep = now == kNegInf ? 1.0f : exp2_approx(m[i] - now);
                    m[i] = now;
                    l[i] *= keep;
#pragma unroll
                    for (int k = 0; k < kSteps * 2; ++k) o[k][2 * i] *= keep, o[k][2 * i + 1] *= keep;
                }
            }
            const float base[2] = {m[0] == kNegInf ? 0.0f : m[0] - kLift<DT>, m[1] == kNegInf ? 0.0f : m[1] - kLift<DT>};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s[i][k] = exp2_approx(s[i][k] - base[k >> 1]);
                    l[k >> 1] += s[i][k];
                }
            const uint32_t w[4] = {pack_pair<DT>(s[0][0], s[0][1]), pack_pair<DT>(s[0][2], s[0][3]),
                                   pack_pair<DT>(s[1][0], s[1][1]), pack_pair<DT>(s[1][2], s[1][3])};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                ldmatrix4_trans(b, at + v_row + 32 * k);
                if (!all && mixed) odd = odd || not_finite2<DT>(b[0]) || not_finite2<DT>(b[1]) || not_finite2<DT>(b[2]) || not_finite2<DT>(b[3]);
                mma16816<DT>(o[2 * k], w, b[0], b[1]);
                mma16816<DT>(o[2 * k + 1], w, b[2], b[3]);
            }
            __syncwarp();
            if (lane == 0) bar_arrive(empty + 8 * stage);
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
        Piece next;
        more = run.next(a, next);
        if (more) queries(next);  // on their way while this piece ends
        // ---- the warps' sums become one
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            m[i] -= kLift<DT>;  // what the sums are relative to
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if ((lane & 3) == 0) row_ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
        }
        if (odd) row_odd = 1;
        sync_weighing_warps();
        const bool slow = row_odd;
        float keep[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = kNegInf;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) top = fmaxf(top, row_ml[k][g + 8 * i].x);
            keep[i] = top == kNegInf ? 1.0f : exp2_approx(m[i] - top);
        }
        const int width = rows <= 4 ? DP : rows <= 8 ? 64 : 32;  // values of a row at a time
        float *const sums = reinterpret_cast<float *>(smem + kSumsAt<DP>);  // [kWarps][rows][width + 4]
        char *part = a.parts + (2 * blockIdx.x + (p.starts ? 1 : 0)) * part_bytes(kRowsM, DP);
        if (!slow) {
#pragma unroll
            for (int first = 0; first < DP; first += 32) {
                if (first % width) continue;
                if (first) sync_weighing_warps();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (g + 8 * i >= rows) break;
                    float *to = sums + warp * kSumFloats + (g + 8 * i) * (width + 4) + q2;
#pragma unroll
                    for (int k = 0; k < kSteps * 2; ++k) {
                        if (first / 8 + k >= kSteps * 2 || 8 * k >= width) break;
                        *reinterpret_cast<float2 *>(to + 8 * k) = make_float2(o[first / 8 + k][2 * i] * keep[i], o[first / 8 + k][2 * i + 1] * keep[i]);
                    }
                }
                sync_weighing_warps();
                for (int i = tid; i < rows * (width / 4); i += kWarps * 32) {
                    const int row = i / (width / 4), col = 4 * (i % (width / 4));
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float top = kNegInf, total = 0.0f;
#pragma unroll
                    for (int k = 0; k < kWarps; ++k) {
                        const float4 y = *reinterpret_cast<const float4 *>(sums + k * kSumFloats + row * (width + 4) + col);
                        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                        top = fmaxf(top, row_ml[k][row].x);
                    }
                    const float base = top == kNegInf ? 0.0f : top;
#pragma unroll
                    for (int k = 0; k < kWarps; ++k) total += exp2_approx(row_ml[k][row].x - base) * row_ml[k][row].y;
                    if (p.whole) {
                        store_joined<DT>(a, r, row0 + row, p.head, first + col, top, total, x);
                    } else {
                        *reinterpret_cast<float4 *>(part + (row * DP + first + col) * 4) = x;
                        if (first + col == 0) reinterpret_cast<float2 *>(part + kRowsM * DP * 4)[row] = make_float2(top, total);
                    }
                }
            }
        } else {
            for (int row = warp; row < rows; row += kWarps) {
                float x[DP / 32], top, total;
                slow_row<DT, DP>(a, r, p.request, p.head, row0 + row, p.begin * kRowsBK, p.end * kRowsBK, failed, x, top, total);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) sums[warp * kSumFloats + lane * (DP / 32) + i] = x[i];
                __syncwarp();
                if (4 * lane < DP) {
                    const float4 y = *reinterpret_cast<const float4 *>(sums + warp * kSumFloats + 4 * lane);
                    if (p.whole) store_joined<DT>(a, r, row0 + row, p.head, 4 * lane, top, total, y);
                    else *reinterpret_cast<float4 *>(part + (row * DP + 4 * lane) * 4) = y;
                }
                if (lane == 0 && !p.whole) reinterpret_cast<float2 *>(part + kRowsM * DP * 4)[row] = make_float2(top, total);
                __syncwarp();
            }
        }
        if (p.sharers) join = join_for(p);
        if (slow) sync_weighing_warps();  // (all have read the word)
        if (tid == 0) row_odd = 0;
        sync_weighing_warps();
        p = next;
    }
    if (tid == 0 && a.joins) a.joins[blockIdx.x] = join;
    if (tid == 0 && *failed && a.status) atomicOr(a.status, CG_S_TIMEOUT);
}

constexpr int kJoinThreads = 1024;
// Joins what the CTAs of a divided tile have left.  Block i: the tile that begins in CTA i, if one does that is divided.  One long request
// alone has few tiles, and each is divided among dozens of CTAs: the parts are spread over the block's threads.
template <int DT, int DP>
__global__ void __launch_bounds__(kJoinThreads) combine_rows_kernel(const __grid_constant__ AttendArgs a) {
    __shared__ float4 sums[kJoinThreads];
    __shared__ float2 tops[kJoinThreads];
    wait_for_launch_before();
    const int c = blockIdx.x, tid = threadIdx.x;
    const Join join = join_of(a, c);
    if (join.sharers == 0) return;
    const Lengths r{join.first, join.n, join.kv};
    const int rows = min(kRowsM, r.n * a.group - join.t * kRowsM), items = rows * (DP / 4), lanes = kJoinThreads / items;
    const int item = tid % items, part = tid / items, row = item / (DP / 4), col = 4 * (item % (DP / 4));
    float top = kNegInf, total = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](float2 ml, float4 x) {
        const float now = fmaxf(top, ml.x), base = now == kNegInf ? 0.0f : now;
        const float keep = exp2_approx(top - base), w = exp2_approx(ml.x - base);
        total = total * keep + ml.y * w;
        sum.x = sum.x * keep + x.x * w, sum.y = sum.y * keep + x.y * w, sum.z = sum.z * keep + x.z * w, sum.w = sum.w * keep + x.w * w;
        top = now;
    };
    if (part < lanes) {
#pragma unroll 4
        for (int i = part; i < join.sharers; i += lanes) {
            const char *p = a.parts + (2 * (c + i) + (i == 0)) * part_bytes(kRowsM, DP);
            add(__ldcg(reinterpret_cast<const float2 *>(p + kRowsM * DP * 4) + row), __ldcg(reinterpret_cast<const float4 *>(p) + item));
        }
        sums[tid] = sum;
        tops[tid] = make_float2(top, total);
    }
    __syncthreads();
    if (part != 0) return;
    for (int i = 1; i < lanes; ++i) add(tops[i * items + item], sums[i * items + item]);
    store_joined<DT>(a, r, join.t * kRowsM + row, join.head, col, top, total, sum);
}

template <int DT, int DP>
int launch_attend_rows(const AttendArgs &a, int ctas, cudaStream_t st) {
    constexpr int smem = kAttendSmem<DP>;
    int rc = allow_smem(attend_rows_kernel<DT, DP>, smem);
    if (rc) return rc;
    rc = launch(attend_rows_kernel<DT, DP>, dim3(ctas), kWarps * 64, smem, false, st, a);
    if (rc || !a.joins) return rc;
    return launch(combine_rows_kernel<DT, DP>, dim3(ctas), kJoinThreads, 0, true, st, a);
}

// Tiles of at most so many units stay whole: what a second kernel takes to join parts, 4 to 5 us, is more than these units take.  (40 requests
// of 250 tokens of 32 heads: 41 us, divided 44; 400 rows over 300 keys of two requests: 18 us, divided 23.  With eight units one request of
// 400 tokens takes 13.7 us instead of 10.3.)
constexpr int kUndividedUnits = 4;

// What a call launches, from what the host knows: the tensors' sizes.
struct Plan {
    bool tiles;      // the kernel for many rows
    int ctas, dp;
    bool undivided;  // no tile is divided among CTAs
    int64_t bytes;   // of the workspace: 0 if no tile is divided
};

int plan_of(const cg_attention_job &j, Plan &p) {
    if (j.dtype != CG_F16 && j.dtype != CG_BF16) return CG_E_DTYPE;
    if (j.nrequests < 0 || j.nrows < 0 || j.heads <= 0 || j.q_heads <= 0 || j.q_heads % j.heads || j.head_size <= 0 || j.page_size <= 0 ||
        j.table_width < 0 || j.num_pages < 0 || j.num_pages > INT32_MAX || j.window < 0 || j.max_q < 0 || j.head_size > 128 ||
        static_cast<int64_t>(j.nrows) * j.q_heads > INT32_MAX - 512 || (!j.q_starts && j.nrows != j.nrequests))
        return CG_E_SHAPE;
    if (j.head_size % 8) return CG_E_ALIGN;
    if (j.nrequests > CG_MAX_REQUESTS) return CG_E_CAPACITY;
    const int64_t group = j.q_heads / j.heads;
    const int most = !j.q_starts ? 1 : j.max_q > 0 ? j.max_q : j.nrows;
    // More rows than one tile of the kernel for few would read the keys several times: 16 requests of 4,000 tokens with 20 rows a head take 59 us
    // with the kernel for many and 91 with that for few, with 16 rows 58 and 57, with 4 rows 59 and 54.  (Its maxima are those of
    // unscaled scores: a scale that is not positive is the other kernel's.)
    p.tiles = most * group > kRowsM && j.scale > 0.0f;
    p.dp = j.head_size > 64 ? 128 : 64;
    const int M = p.tiles ? kTileRows : kRowsM, BK = p.tiles ? kTileKeys : kRowsBK;
    const int64_t keys = static_cast<int64_t>(j.table_width) * j.page_size;
    const int64_t per_tile = keys <= BK ? 1 : (keys + BK - 1) / BK;                              // units of a tile, at most
    if ((static_cast<int64_t>(j.nrows) * group / M + 1) * (per_tile + kTileCost) > INT32_MAX) return CG_E_CAPACITY;  // a request's units a head
    const int64_t tiles = (static_cast<int64_t>(j.nrows) * group / M + j.nrequests) * j.heads;  // at most
    const int64_t slots = static_cast<int64_t>(sm_count()) * (p.tiles ? 1 : 2);
    p.ctas = static_cast<int>(per_tile > slots || tiles * per_tile > slots ? slots : tiles * per_tile);
    p.undivided = per_tile <= kUndividedUnits;
    p.bytes = !p.undivided ? p.ctas * (2 * part_bytes(M, p.dp) + static_cast<int64_t>(sizeof(Join))) : 0;
    return CG_OK;
}

}  // namespace
}  // namespace cg

extern "C" int64_t cg_paged_attention_workspace(const cg_attention_job *job) {
    if (!job) return CG_E_NULL;
    if (job->nrows == 0 || job->nrequests == 0) return 0;
    cg::Plan p;
    const int rc = cg::plan_of(*job, p);
    return rc ? rc : p.bytes;
}

extern "C" int cg_paged_attention(const cg_attention_job *job, void *stream) {
    using namespace cg;
    if (!job) return CG_E_NULL;
    const cg_attention_job &j = *job;
    Plan p;
    int rc = plan_of(j, p);
    if (rc) return rc;
    if (j.nrows == 0 || j.nrequests == 0) return CG_OK;
    if (!j.q || !j.out || !j.kv_lens || (j.table_width && (!j.table || !j.pages_k || !j.pages_v))) return CG_E_NULL;
    for (const int64_t s : {j.q_strides[0], j.q_strides[1], j.out_strides[0], j.out_strides[1], j.pages_k_strides[0], j.pages_k_strides[1],
                            j.pages_k_strides[2], j.pages_v_strides[0], j.pages_v_strides[1], j.pages_v_strides[2]})
        if (s % 8) return CG_E_ALIGN;
    for (const void *x : {j.q, static_cast<const void *>(j.out), j.pages_k, j.pages_v, static_cast<const void *>(j.workspace)})
        if (reinterpret_cast<uintptr_t>(x) % 16) return CG_E_ALIGN;
    if (p.bytes && (!j.workspace || j.workspace_bytes < p.bytes)) return CG_E_CAPACITY;
    AttendArgs a{};
    a.q = static_cast<const char *>(j.q), a.k = static_cast<const char *>(j.pages_k), a.v = static_cast<const char *>(j.pages_v);
    a.out = static_cast<char *>(j.out), a.lse = j.lse;
    a.table = j.table, a.kv_lens = j.kv_lens, a.q_starts = j.q_starts, a.status = j.status;
    if (p.bytes) {
        a.parts = static_cast<char *>(j.workspace);
        a.joins = reinterpret_cast<Join *>(a.parts + p.bytes - p.ctas * static_cast<int64_t>(sizeof(Join)));
    }
    a.q_token = 2 * j.q_strides[0], a.q_head = 2 * j.q_strides[1], a.out_token = 2 * j.out_strides[0], a.out_head = 2 * j.out_strides[1];
    a.k_page = 2 * j.pages_k_strides[0], a.k_token = 2 * j.pages_k_strides[1], a.k_head = 2 * j.pages_k_strides[2];
    a.v_page = 2 * j.pages_v_strides[0], a.v_token = 2 * j.pages_v_strides[1], a.v_head = 2 * j.pages_v_strides[2];
    a.table_row = j.table_row, a.num_pages = j.num_pages;
    a.nrequests = j.nrequests, a.nrows = j.nrows, a.q_heads = j.q_heads, a.heads = j.heads, a.group = j.q_heads / j.heads;
    a.head_size = j.head_size, a.page_size = j.page_size, a.table_width = j.table_width, a.causal = j.causal, a.window = j.window;
    a.undivided = p.undivided;
    const auto log2_of = [](int n) { return n & (n - 1) ? -1 : __builtin_ctz(static_cast<unsigned>(n)); };
    a.page_shift = log2_of(j.page_size), a.group_shift = log2_of(a.group);
    a.scale = j.scale * 1.44269504088896340736f;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.tiles) return launch_attend_tiles(a, j.dtype, p.ctas, st);
    if (p.dp == 64) return j.dtype == CG_F16 ? launch_attend_rows<CG_F16, 64>(a, p.ctas, st) : launch_attend_rows<CG_BF16, 64>(a, p.ctas, st);
    return j.dtype == CG_F16 ? launch_attend_rows<CG_F16, 128>(a, p.ctas, st) : launch_attend_rows<CG_BF16, 128>(a, p.ctas, st);
}
