// Attention over a paged KV cache: the entry point, and the kernel for few query rows a key/value head (single tokens, drafts).
//
// With up to 16 rows a head every cached value is used for few products and the kernel's time is that of reading the cache
// once.  So a block is there to keep loads in flight: each of its warps walks through 16 keys at a time of its own, with its own
// ring of asynchronous copies and no barrier of the block, and the warps' sums are joined when the block's piece of the
// tile ends.  Products are m16n8k16 on fragments in registers: tcgen05 takes 64 rows at least, its accumulator would have to come back from
// tensor memory for each 16 keys, and at 16 rows the products take less than a fifth of the time that the keys take to arrive.
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
// 16 bytes, or zeros where there is nothing to read
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int DT> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    return Half16<DT>::from_float(lo) | static_cast<uint32_t>(Half16<DT>::from_float(hi)) << 16;
}
// whether one of two 16-bit floats is infinite or no number
template <int DT> __device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t e = DT == CG_F16 ? 0x7C00u : 0x7F80u;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// Shared memory: kWarps rings of kStages stages of 16 keys, then 16 values; rows of 2 * DP bytes, 16-byte pieces in an order
// (piece ^ row % 8) in which eight rows' pieces of a matrix lie in different banks.  Where the piece ends the same memory holds the warps' sums.
template <int DP> constexpr int kRingBytes = kStages * 2 * kChunk * DP * 2;
// Behind it: the warps' maxima and sums, and a word that says whether values that are not finite were met where rows see unlike keys.
constexpr int most_of(int x, int y) { return x > y ? x : y; }
template <int DP> constexpr int kMlAt = most_of(kWarps * kRingBytes<DP>, most_of(kWarps * kRowsM * (DP + 4) * 4, (CG_MAX_REQUESTS + 1) * 8 + 8));
template <int DP> constexpr int kAttendSmem = kMlAt<DP> + kWarps * kRowsM * 8 + 16;

template <int DT, int DP>
__global__ void __launch_bounds__(kWarps * 32, 2) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    float2(*row_ml)[kRowsM] = reinterpret_cast<float2(*)[kRowsM]>(smem + kMlAt<DP>);  // [kWarps]
    volatile int &row_odd = *reinterpret_cast<volatile int *>(smem + kMlAt<DP> + kWarps * kRowsM * 8);
    constexpr int kPieces = DP / 8, kSteps = DP / 16;  // 16-byte pieces of a row; 16-value steps
    constexpr int kRowsAtOnce = 32 / kPieces;          // rows that a warp copies with one instruction
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, q2 = 2 * (lane & 3);
    const uint32_t ring = smem_addr(smem) + warp * kRingBytes<DP>;

    Run<kRowsM, kRowsBK, kRowsCost> run;
    run.template init<kWarps * 32, false>(a, reinterpret_cast<int64_t *>(smem));
    let_next_launch_start();
    int4 join = make_int4(0, 0, 0, 0);
    if (tid == 0) row_odd = 0;
    Piece p;
    while (run.next(a, p)) {
        const Lengths r = p.r;
        const int rows = min(kRowsM, r.n * a.group - p.t * kRowsM), row0 = p.t * kRowsM;
        // ---- this thread's two rows: the keys that they see, and the queries as fragments
        int lo[2], hi[2];
        uint32_t qf[kSteps][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = g + 8 * i, at = row0 + row, token = at / a.group;
            const bool there = row < rows;
            lo[i] = there ? first_key(a, r, token) : 0;
            hi[i] = there ? last_key(a, r, token) : 0;
            const char *q = a.q + (r.first + token) * a.q_token + (p.head * a.group + at % a.group) * a.q_head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int d = 16 * s + 8 * k + q2;
                    qf[s][i + 2 * k] = there && d < a.head_size ? __ldg(reinterpret_cast<const unsigned int *>(q + 2 * d)) : 0u;
                }
        }
        // chunks inside [all_lo, all_hi) are seen by all rows
        const int all_lo = first_key(a, r, (row0 + rows - 1) / a.group), all_hi = last_key(a, r, row0 / a.group);
        const int nchunks = p.end - p.begin;
        const int key0 = p.begin * kRowsBK + warp * kChunk;

        // ---- copies: lane i (and i + 16) knows where key i of the chunk lies
        const auto page_for = [&](int chunk) {
            const int key = key0 + chunk * kRowsBK + (lane & 15);
            return chunk < nchunks && key >= p.tile.lo && key < p.tile.hi ? page_of(a, p.request, key / a.page_size) : -1;
        };
        int page = page_for(0);
        const auto fetch = [&](int chunk) {
            if (chunk < nchunks) {
                const int key = key0 + chunk * kRowsBK + (lane & 15), in_page = key % a.page_size;
                const int64_t at_k = page * a.k_page + in_page * a.k_token + p.head * a.k_head;
                const int64_t at_v = page * a.v_page + in_page * a.v_token + p.head * a.v_head;
                const bool there = page >= 0;
                const uint32_t to = ring + chunk % kStages * (2 * kChunk * DP * 2);
                const int piece = lane % kPieces;
#pragma unroll
                for (int i = 0; i < kChunk / kRowsAtOnce; ++i) {
                    const int row = i * kRowsAtOnce + lane / kPieces;
                    const int64_t from_k = __shfl_sync(0xffffffffu, at_k, row), from_v = __shfl_sync(0xffffffffu, at_v, row);
                    const bool copy = __shfl_sync(0xffffffffu, there, row) && 8 * piece < a.head_size;
                    const uint32_t dst = to + row * (2 * DP) + ((piece ^ (row & 7)) << 4);
                    copy16(dst, copy ? a.k + from_k + 16 * piece : a.k, copy);
                    copy16(dst + kChunk * DP * 2, copy ? a.v + from_v + 16 * piece : a.v, copy);
                }
            }
            copies_end_group();
            page = page_for(chunk + 1);
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) fetch(i);

        float o[kSteps * 2][4], m[2] = {kNegInf, kNegInf}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kSteps * 2; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][k] = 0.0f;
        bool odd = false;
        // this lane's row and piece of the four matrices of an ldmatrix
        const int k_row = (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
        const int v_row = lane & 15, v_piece = lane >> 4;
        for (int chunk = 0; chunk < nchunks; ++chunk) {
            copies_wait<kStages - 2>();
            __syncwarp();
            const uint32_t k_at = ring + chunk % kStages * (2 * kChunk * DP * 2), v_at = k_at + kChunk * DP * 2;
            float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                ldmatrix4(b, k_at + k_row * (2 * DP) + (((2 * k + k_piece) ^ (k_row & 7)) << 4));
                mma16816<DT>(s[0], qf[k], b[0], b[1]);
                mma16816<DT>(s[1], qf[k], b[2], b[3]);
            }
            const int key = key0 + chunk * kRowsBK;
            const bool all = key >= all_lo && key + kChunk <= all_hi;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = key + 8 * i + q2 + (k & 1);
                    s[i][k] = all || (j >= lo[k >> 1] && j < hi[k >> 1]) ? s[i][k] * a.scale : kNegInf;
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
            const float base[2] = {m[0] == kNegInf ? 0.0f : m[0], m[1] == kNegInf ? 0.0f : m[1]};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s[i][k] = exp2_approx(s[i][k] - base[k >> 1]);
                    l[k >> 1] += s[i][k];
                }
            // weights are between 0 and 1 and rounded to the cache's type for the product: off by half a step each, without bias
            const uint32_t w[4] = {pack_pair<DT>(s[0][0], s[0][1]), pack_pair<DT>(s[0][2], s[0][3]),
                                   pack_pair<DT>(s[1][0], s[1][1]), pack_pair<DT>(s[1][2], s[1][3])};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                ldmatrix4_trans(b, v_at + v_row * (2 * DP) + (((2 * k + v_piece) ^ (v_row & 7)) << 4));
                if (!all) odd = odd || not_finite2<DT>(b[0]) || not_finite2<DT>(b[1]) || not_finite2<DT>(b[2]) || not_finite2<DT>(b[3]);
                mma16816<DT>(o[2 * k], w, b[0], b[1]);
                mma16816<DT>(o[2 * k + 1], w, b[2], b[3]);
            }
            __syncwarp();
            fetch(chunk + kStages - 1);
        }
        copies_wait<0>();
        // ---- the warps' sums become one
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if ((lane & 3) == 0) row_ml[warp][g + 8 * i] = make_float2(m[i], l[i]);
        }
        if (odd) row_odd = 1;
        __syncthreads();
        float *sums = reinterpret_cast<float *>(smem);  // [kWarps][kRowsM][DP + 4]
        const bool slow = row_odd;
        if (!slow) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = kNegInf;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) top = fmaxf(top, row_ml[k][g + 8 * i].x);
                const float keep = top == kNegInf ? 1.0f : exp2_approx(m[i] - top);
                float *to = sums + (warp * kRowsM + g + 8 * i) * (DP + 4) + q2;
#pragma unroll
                for (int k = 0; k < kSteps * 2; ++k) *reinterpret_cast<float2 *>(to + 8 * k) = make_float2(o[k][2 * i] * keep, o[k][2 * i + 1] * keep);
            }
        } else {
            for (int row = warp; row < rows; row += kWarps) {
                float x[DP / 32], top, total;
                slow_row<DT, DP>(a, r, p.request, p.head, row0 + row, p.begin * kRowsBK, p.end * kRowsBK, x, top, total);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) sums[row * (DP + 4) + lane + 32 * i] = x[i];
                if (lane == 0) row_ml[0][row] = make_float2(top, total);
            }
        }
        __syncthreads();
        const int nparts = slow ? 1 : kWarps;
        char *part = a.parts + (2 * blockIdx.x + (p.starts ? 1 : 0)) * part_bytes(kRowsM, DP);
        for (int i = tid; i < rows * (DP / 4); i += kWarps * 32) {
            const int row = i / (DP / 4), col = 4 * (i % (DP / 4));
            float4 x = *reinterpret_cast<const float4 *>(sums + row * (DP + 4) + col);
            float top = row_ml[0][row].x;
            for (int k = 1; k < nparts; ++k) {
                const float4 y = *reinterpret_cast<const float4 *>(sums + (k * kRowsM + row) * (DP + 4) + col);
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                top = fmaxf(top, row_ml[k][row].x);
            }
            const float base = top == kNegInf ? 0.0f : top;
            float total = 0.0f;
            for (int k = 0; k < nparts; ++k) total += exp2_approx(row_ml[k][row].x - base) * row_ml[k][row].y;
            if (p.whole) {
                const int at = row0 + row, token = at / a.group, head = p.head * a.group + at % a.group;
                const bool sees = last_key(a, r, token) > first_key(a, r, token);
                const float inv = 1.0f / total;
                if (col < a.head_size) {
                    const uint2 y = make_uint2(pack_pair<DT>(x.x * inv, x.y * inv), pack_pair<DT>(x.z * inv, x.w * inv));
                    *reinterpret_cast<uint2 *>(a.out + (r.first + token) * a.out_token + head * a.out_head + 2 * col) = sees ? y : make_uint2(0u, 0u);
                }
                if (a.lse && col == 0)
                    a.lse[static_cast<int64_t>(r.first + token) * a.q_heads + head] = sees ? (base + log2f(total)) * 0.693147180559945f : kNegInf;
            } else {
                *reinterpret_cast<float4 *>(part + i * 16) = x;
                if (col == 0) reinterpret_cast<float2 *>(part + kRowsM * DP * 4)[row] = make_float2(top, total);
            }
        }
        if (p.sharers) join = make_int4(p.request, p.head, p.t, p.sharers);
        if (tid == 0) row_odd = 0;  // (read by all in front of the barrier before)
        __syncthreads();
    }
    if (tid == 0 && a.joins) a.joins[blockIdx.x] = join;
}

template <int DT, int DP>
int launch_attend_rows(const AttendArgs &a, int ctas, cudaStream_t st) {
    constexpr int smem = kAttendSmem<DP>;
    int rc = allow_smem(attend_rows_kernel<DT, DP>, smem);
    if (rc) return rc;
    rc = launch(attend_rows_kernel<DT, DP>, dim3(ctas), kWarps * 32, smem, false, st, a);
    if (rc || !a.joins) return rc;
    return launch(combine_kernel<DT, kRowsM, DP, false>, dim3(ctas, kRowsM * (DP / 4) / 256), 256, 0, true, st, a);
}

// What a call launches, from what the host knows: the tensors' sizes.
struct Plan {
    bool tiles;      // the kernel for many rows
    int ctas, dp;
    int64_t bytes;   // of the workspace: 0 if no tile can be divided
};

int plan_of(const cg_attention_job &j, Plan &p) {
    if (j.dtype != CG_F16 && j.dtype != CG_BF16) return CG_E_DTYPE;
    if (j.nrequests < 0 || j.nrows < 0 || j.heads <= 0 || j.q_heads <= 0 || j.q_heads % j.heads || j.head_size <= 0 || j.page_size <= 0 ||
        j.table_width < 0 || j.num_pages < 0 || j.num_pages > INT32_MAX || j.window < 0 || j.max_q < 0 || j.head_size > 128 ||
        static_cast<int64_t>(j.nrows) * j.q_heads > INT32_MAX || (!j.q_starts && j.nrows != j.nrequests))
        return CG_E_SHAPE;
    if (j.head_size % 8) return CG_E_ALIGN;
    if (j.nrequests > CG_MAX_REQUESTS) return CG_E_CAPACITY;
    const int64_t group = j.q_heads / j.heads;
    const int most = !j.q_starts ? 1 : j.max_q > 0 ? j.max_q : j.nrows;
    p.tiles = most * group > kRowsM && j.scale > 0.0f;  // (its maxima are those of unscaled scores)
    p.dp = j.head_size > 64 ? 128 : 64;
    const int M = p.tiles ? kTileRows : kRowsM, BK = p.tiles ? kTileKeys : kRowsBK;
    const int64_t keys = static_cast<int64_t>(j.table_width) * j.page_size;
    const int64_t per_tile = keys <= BK ? 1 : (keys + BK - 1) / BK;                              // units of a tile, at most
    const int64_t tiles = (static_cast<int64_t>(j.nrows) * group / M + j.nrequests) * j.heads;  // at most
    const int64_t slots = static_cast<int64_t>(sm_count()) * (p.tiles ? 1 : 2);
    p.ctas = static_cast<int>(per_tile > slots || tiles * per_tile > slots ? slots : tiles * per_tile);
    p.bytes = per_tile > 1 ? p.ctas * (2 * part_bytes(M, p.dp) + static_cast<int64_t>(sizeof(int4))) : 0;
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
        a.joins = reinterpret_cast<int4 *>(a.parts + p.bytes - p.ctas * static_cast<int64_t>(sizeof(int4)));
    }
    a.q_token = 2 * j.q_strides[0], a.q_head = 2 * j.q_strides[1], a.out_token = 2 * j.out_strides[0], a.out_head = 2 * j.out_strides[1];
    a.k_page = 2 * j.pages_k_strides[0], a.k_token = 2 * j.pages_k_strides[1], a.k_head = 2 * j.pages_k_strides[2];
    a.v_page = 2 * j.pages_v_strides[0], a.v_token = 2 * j.pages_v_strides[1], a.v_head = 2 * j.pages_v_strides[2];
    a.table_row = j.table_row, a.num_pages = j.num_pages;
    a.nrequests = j.nrequests, a.nrows = j.nrows, a.q_heads = j.q_heads, a.heads = j.heads, a.group = j.q_heads / j.heads;
    a.head_size = j.head_size, a.page_size = j.page_size, a.table_width = j.table_width, a.causal = j.causal, a.window = j.window;
    a.scale = j.scale * 1.44269504088896340736f;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.tiles) return launch_attend_tiles(a, j.dtype, p.ctas, st);
    if (p.dp == 64) return j.dtype == CG_F16 ? launch_attend_rows<CG_F16, 64>(a, p.ctas, st) : launch_attend_rows<CG_BF16, 64>(a, p.ctas, st);
    return j.dtype == CG_F16 ? launch_attend_rows<CG_F16, 128>(a, p.ctas, st) : launch_attend_rows<CG_BF16, 128>(a, p.ctas, st);
}
