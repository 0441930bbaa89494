// Rows of 16-bit values on their way into or out of a paged KV cache, rotated by their positions as they pass.
//
// One kernel moves all of it: the heads of a token are read from a dense array or from the token's slot of the cache, the
// rotated ones are turned, and they are written to the other side.  Every byte is read once and written once, so memory bounds
// it: a block's work is laid out to keep 16-byte accesses of neighbouring threads side by side and two of a thread's rows in
// flight.
//
// The angle of pair i at position p is p * w_i.  In 32-bit floats that loses what matters from some thousands of positions on
// (an angle of 10^5 is known to 0.008), and a table of cosines costs 512 bytes a token to read and has a last position.
// Here w_i / (2 pi) is a 64-bit binary fraction of a turn and p * w_i a 64-bit integer product: what overflows is whole
// turns.  After 2^20 positions the fraction is off by less than 2^-36 turns; its upper 32 bits, as a float, by 2^-25 half turns.
// Each block works out the cosines and sines of its tokens once, in shared memory, for all heads and layers that it moves.
#include "cg_common.cuh"

namespace cg {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kMostHead = 512;
constexpr int kMostCount = INT32_MAX - 512;  // of tokens and of layers: a block counts on to the end of its share, up to 256 behind the last

// One of the up to three arrays of rows: queries, keys, values.  A side with `paged` set is addressed by slots.
struct MoveSide {
    char *data;
    int64_t layer, page, token, head;  // strides in elements
};
struct MoveRows {
    MoveSide src, dst;
    int32_t heads, turned, src_paged, dst_paged;
};
struct MoveArgs {
    MoveRows rows[3];
    const void *positions, *slots;
    const uint64_t *turns;
    int32_t *status;
    int64_t num_slots, pos_layer;
    int32_t nlayers, ntokens, head_size, rot, page_size, wide_positions, wide_slots;
    int32_t tokens_per_block, head_lanes, layers_per_block, token_blocks, heads, back;
};

__device__ __forceinline__ int64_t index_at(const void *p, int64_t i, int wide) {
    return wide ? __ldg(static_cast<const long long *>(p) + i) : __ldg(static_cast<const int *>(p) + i);
}

__device__ __forceinline__ char *row_of(const MoveSide &s, bool paged, int layer, int token, int64_t page, int in_page, int head) {
    const int64_t at = layer * s.layer + head * s.head + (paged ? page * s.page + in_page * s.token : token * s.token);
    return s.data + 2 * at;
}

template <int DT> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    return make_float2(Half16<DT>::to_float(static_cast<uint16_t>(w)), Half16<DT>::to_float(static_cast<uint16_t>(w >> 16)));
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    return Half16<DT>::from_float(a) | static_cast<uint32_t>(Half16<DT>::from_float(b)) << 16;
}

// The 16 values of a thread's piece of a head, in two vectors: half layout, values lo + i and hi + i are pair i; interleaved,
// values 2i and 2i + 1 of the 16 in a row.
template <int DT, bool INTERLEAVED>
__device__ __forceinline__ void turn16(uint4 &lo, uint4 &hi, const float2 (&cs)[8]) {
    uint32_t *a = reinterpret_cast<uint32_t *>(&lo), *b = reinterpret_cast<uint32_t *>(&hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = unpack2<DT>(a[i]), y = unpack2<DT>(b[i]);
        if (INTERLEAVED) {
            a[i] = pack2<DT>(x.x * cs[i].x - x.y * cs[i].y, x.y * cs[i].x + x.x * cs[i].y);
            b[i] = pack2<DT>(y.x * cs[4 + i].x - y.y * cs[4 + i].y, y.y * cs[4 + i].x + y.x * cs[4 + i].y);
        } else {
            a[i] = pack2<DT>(x.x * cs[2 * i].x - y.x * cs[2 * i].y, x.y * cs[2 * i + 1].x - y.y * cs[2 * i + 1].y);
            b[i] = pack2<DT>(y.x * cs[2 * i].x + x.x * cs[2 * i].y, y.y * cs[2 * i + 1].x + x.y * cs[2 * i + 1].y);
        }
    }
}

// Threads: x = piece of a head (16 values; VEC false: 32 lanes that walk over a head value by value, for sizes, strides or
// addresses that 16-byte accesses cannot take), y = token of the block, then head lane.  A thread stays with its token, so its
// cosines stay in registers while it goes through the token's heads of all the block's layers.
template <int DT, bool INTERLEAVED, bool VEC>
__global__ void __launch_bounds__(kMoveThreads) move_rows_kernel(const __grid_constant__ MoveArgs a) {
    extern __shared__ float2 turned[];  // [tokens_per_block][rot / 2]
    const int half = a.rot / 2, nthreads = blockDim.x * blockDim.y;
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;
    const int block_y = blockIdx.x / a.token_blocks, token0 = (blockIdx.x - block_y * a.token_blocks) * a.tokens_per_block;
    const int mine = threadIdx.y / a.head_lanes, token = token0 + mine;
    const int layer1 = min(a.nlayers, (block_y + 1) * a.layers_per_block);
    bool active = token < a.ntokens;
    int64_t slot = 0;
    if (a.slots && active) slot = index_at(a.slots, token, a.wide_slots);  // on its way while cosines are worked out
    // cosines are shared by the block's layers unless every layer has positions of its own; then a block has one layer
    const int64_t pos0 = static_cast<int64_t>(block_y) * a.layers_per_block * a.pos_layer;
    for (int i = tid; i < a.tokens_per_block * half; i += nthreads) {
        const int t = i / half;
        if (token0 + t < a.ntokens) {
            const uint64_t p = static_cast<uint64_t>(index_at(a.positions, pos0 + token0 + t, a.wide_positions));
            const int32_t part = static_cast<int32_t>((p * __ldg(a.turns + (i - t * half))) >> 32);
            float s, c;
            sincospif(static_cast<float>(part) * 0x1p-31f, &s, &c);
            turned[i] = make_float2(c, a.back ? -s : s);
        }
    }
    int64_t page = 0;
    int in_page = 0;
    if (a.slots && active) {
        if (slot < 0 || slot >= a.num_slots) {  // a token of padding, or one that the cache has no place for
            if (slot != -1 && a.status && threadIdx.x == 0) atomicOr(a.status, CG_S_BAD_PAGE);
            active = false;
        } else {
            page = slot / a.page_size;
            in_page = static_cast<int>(slot - page * a.page_size);
        }
    }
    const int head_lane = threadIdx.y - mine * a.head_lanes;
    int layer = block_y * a.layers_per_block, h = head_lane;
    const float2 *cs_row = turned + mine * half;
    // the array and head of (h of all arrays' heads); moves on by head_lanes
    const auto find = [&](int &which, int &head) {
        while (h >= a.heads) h -= a.heads, ++layer;
        head = h;
        which = 0;
        if (head >= a.rows[0].heads) head -= a.rows[0].heads, which = 1;
        if (which == 1 && head >= a.rows[1].heads) head -= a.rows[1].heads, which = 2;
    };
    if (VEC) {
        const int j = threadIdx.x;
        const bool turns = 16 * j < a.rot;
        const int lo = 2 * (turns && !INTERLEAVED ? 8 * j : 16 * j), hi = turns && !INTERLEAVED ? lo + a.rot : lo + 16;  // bytes
        float2 cs[8];
        constexpr int kFlight = 2;  // rows of a thread in flight
        for (bool first = true;; first = false) {
            char *to[kFlight];
            uint4 x[kFlight], y[kFlight];
            bool turn[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u, h += a.head_lanes) {
                int which, head;
                find(which, head);
                to[u] = nullptr;
                if (active && layer < layer1) {
                    const MoveRows &r = a.rows[which];
                    const char *from = row_of(r.src, r.src_paged, layer, token, page, in_page, head);
                    x[u] = *reinterpret_cast<const uint4 *>(from + lo);
                    y[u] = *reinterpret_cast<const uint4 *>(from + hi);
                    to[u] = row_of(r.dst, r.dst_paged, layer, token, page, in_page, head);
                    turn[u] = turns && r.turned;
                }
            }
            if (first && half) {  // the cosines are there, the first rows on their way
                __syncthreads();
                if (turns) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) cs[i] = cs_row[8 * j + i];
                }
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                if (!to[u]) return;
                if (turn[u]) turn16<DT, INTERLEAVED>(x[u], y[u], cs);
                *reinterpret_cast<uint4 *>(to[u] + lo) = x[u];
                *reinterpret_cast<uint4 *>(to[u] + hi) = y[u];
            }
        }
    } else {
        if (half) __syncthreads();
        if (!active) return;
        for (;; h += a.head_lanes) {
            int which, head;
            find(which, head);
            if (layer >= layer1) return;
            const MoveRows &r = a.rows[which];
            const uint16_t *from = reinterpret_cast<const uint16_t *>(row_of(r.src, r.src_paged, layer, token, page, in_page, head));
            uint16_t *to = reinterpret_cast<uint16_t *>(row_of(r.dst, r.dst_paged, layer, token, page, in_page, head));
            const int pairs = r.turned ? half : 0;
            for (int e = threadIdx.x; e < a.head_size - pairs; e += blockDim.x) {
                if (e < pairs) {  // one thread has both values of a pair: rows may be turned in place
                    const int i0 = INTERLEAVED ? 2 * e : e, i1 = INTERLEAVED ? 2 * e + 1 : half + e;
                    const float x = Half16<DT>::to_float(from[i0]), y = Half16<DT>::to_float(from[i1]);
                    const float2 cs = cs_row[e];
                    to[i0] = Half16<DT>::from_float(x * cs.x - y * cs.y);
                    to[i1] = Half16<DT>::from_float(y * cs.x + x * cs.y);
                } else {
                    to[e + pairs] = from[e + pairs];
                }
            }
        }
    }
}

bool vectors(const MoveSide &s) {
    return reinterpret_cast<uintptr_t>(s.data) % 16 == 0 && s.layer % 8 == 0 && s.page % 8 == 0 && s.token % 8 == 0 && s.head % 8 == 0;
}

template <int DT>
int launch_move(MoveArgs &a, bool interleaved, cudaStream_t st) {
    bool vec = a.head_size % 16 == 0 && a.rot % 16 == 0;
    a.heads = 0;
    for (const MoveRows &r : a.rows) {
        a.heads += r.heads;
        if (r.heads) vec = vec && vectors(r.src) && vectors(r.dst);
    }
    const int pieces = vec ? a.head_size / 16 : 32, lanes = kMoveThreads / pieces;
    // Few tokens: a block each, all lanes on its heads, for the shortest time.  Many: a thread goes through up to sixteen rows, so that
    // its cosines and its slot are worked out once for them: four tokens a block, then layers, as long as the blocks fill
    // every SM twice.  (1,999 tokens of 32 + 32 heads: 22.9 us by fours, 26.4 one by one; 1,999 keys of 32 layers of 8 heads: 48 us
    // with eight layers a block, 80 with one.)
    const int64_t blocks = static_cast<int64_t>(sm_count()) * 8;
    const int64_t rows = static_cast<int64_t>(a.ntokens) * a.heads * a.nlayers;
    a.tokens_per_block = lanes >= 4 && rows / (4 * lanes) >= blocks ? 4 : 1;
    // (a block of few heads has more tokens, so that it has threads)
    const int room = lanes / a.heads < a.ntokens ? lanes / a.heads : a.ntokens;
    if (a.tokens_per_block < room) a.tokens_per_block = room;
    a.head_lanes = lanes / a.tokens_per_block;
    if (a.head_lanes > a.heads) a.head_lanes = a.heads;  // (idle lanes would only wait)
    a.layers_per_block = 1;
    if (a.pos_layer == 0) {
        const int64_t per_layer = (a.heads + a.head_lanes - 1) / a.head_lanes, groups = (a.ntokens + a.tokens_per_block - 1) / a.tokens_per_block;
        while (a.layers_per_block < a.nlayers && a.layers_per_block * per_layer < 16 && groups * (a.nlayers / (2 * a.layers_per_block)) >= blocks)
            a.layers_per_block *= 2;
    }
    const int64_t gx = (static_cast<int64_t>(a.ntokens) + a.tokens_per_block - 1) / a.tokens_per_block;
    const int64_t gy = (static_cast<int64_t>(a.nlayers) + a.layers_per_block - 1) / a.layers_per_block;
    if (gx * gy > INT32_MAX) return CG_E_SHAPE;
    a.token_blocks = static_cast<int>(gx);
    const dim3 grid(static_cast<unsigned>(gx * gy)), block(pieces, a.head_lanes * a.tokens_per_block);
    const size_t smem = sizeof(float2) * a.tokens_per_block * (a.rot / 2);
    if (vec) {
        if (interleaved) move_rows_kernel<DT, true, true><<<grid, block, smem, st>>>(a);
        else move_rows_kernel<DT, false, true><<<grid, block, smem, st>>>(a);
    } else {
        if (interleaved) move_rows_kernel<DT, true, false><<<grid, block, smem, st>>>(a);
        else move_rows_kernel<DT, false, false><<<grid, block, smem, st>>>(a);
    }
    return check_launch();
}

enum Direction { kTurn, kAppend, kGather };

MoveSide dense_side(const void *p, const int64_t *s) {
    return MoveSide{static_cast<char *>(const_cast<void *>(p)), s[0], 0, s[1], s[2]};
}
MoveSide paged_side(const void *p, const int64_t *s) {
    return MoveSide{static_cast<char *>(const_cast<void *>(p)), s[0], s[1], s[2], s[3]};
}

int move(const cg_rows_job *job, Direction way, cudaStream_t st) {
    if (!job) return CG_E_NULL;
    const cg_rows_job &j = *job;
    if (j.dtype != CG_F16 && j.dtype != CG_BF16) return CG_E_DTYPE;
    if (j.nlayers < 0 || j.nlayers > kMostCount || j.ntokens < 0 || j.ntokens > kMostCount || j.heads < 0 || j.q_heads < 0 ||
        j.head_size <= 0 || j.head_size > kMostHead || static_cast<int64_t>(j.heads) * 2 + j.q_heads > 65536)
        return CG_E_SHAPE;
    if (j.rotary_dims < 0 || j.rotary_dims > j.head_size || j.rotary_dims % 2) return CG_E_SHAPE;
    if (j.nlayers == 0 || j.ntokens == 0) return CG_OK;
    if (j.rotary_dims && (!j.positions || !j.turns)) return CG_E_NULL;
    MoveArgs a{};
    a.positions = j.positions;
    a.turns = j.turns;
    a.nlayers = j.nlayers;
    a.ntokens = j.ntokens;
    a.head_size = j.head_size;
    a.rot = j.rotary_dims;
    a.wide_positions = j.wide_positions;
    a.pos_layer = j.pos_layer;
    a.back = way == kGather ? 1 : j.inverse;
    a.page_size = 1;
    if (way == kTurn) {
        if (j.heads == 0) return CG_OK;
        if (!j.k || !j.k_out) return CG_E_NULL;
        a.rows[1] = MoveRows{dense_side(j.k, j.k_strides), dense_side(j.k_out, j.k_out_strides), j.heads, 1, 0, 0};
    } else {
        if (j.heads == 0 || !j.k || !j.v || !j.pages_k || !j.pages_v || !j.slots) return j.heads ? CG_E_NULL : CG_E_SHAPE;
        if (j.page_size <= 0 || j.num_pages < 0 || j.pos_layer) return CG_E_SHAPE;
        a.slots = j.slots;
        a.wide_slots = j.wide_slots;
        a.status = j.status;
        a.page_size = j.page_size;
        a.num_slots = j.num_pages * j.page_size;
        const MoveSide k = dense_side(j.k, j.k_strides), v = dense_side(j.v, j.v_strides);
        const MoveSide pk = paged_side(j.pages_k, j.pages_k_strides), pv = paged_side(j.pages_v, j.pages_v_strides);
        if (way == kAppend) {
            a.rows[1] = MoveRows{k, pk, j.heads, 1, 0, 1};
            a.rows[2] = MoveRows{v, pv, j.heads, 0, 0, 1};
            if (j.q_heads) {
                if (!j.q || !j.q_out) return CG_E_NULL;
                if (j.nlayers != 1) return CG_E_SHAPE;
                a.rows[0] = MoveRows{dense_side(j.q, j.q_strides), dense_side(j.q_out, j.q_out_strides), j.q_heads, 1, 0, 0};
            }
        } else {
            a.rows[1] = MoveRows{pk, k, j.heads, 1, 1, 0};
            a.rows[2] = MoveRows{pv, v, j.heads, 0, 1, 0};
        }
    }
    for (MoveRows &r : a.rows) r.turned = r.turned && a.rot;
    return j.dtype == CG_F16 ? launch_move<CG_F16>(a, j.interleaved, st) : launch_move<CG_BF16>(a, j.interleaved, st);
}

}  // namespace
}  // namespace cg

extern "C" int cg_rotary(const cg_rows_job *job, void *stream) {
    return cg::move(job, cg::kTurn, static_cast<cudaStream_t>(stream));
}
extern "C" int cg_append_paged(const cg_rows_job *job, void *stream) {
    return cg::move(job, cg::kAppend, static_cast<cudaStream_t>(stream));
}
extern "C" int cg_gather_paged(const cg_rows_job *job, void *stream) {
    return cg::move(job, cg::kGather, static_cast<cudaStream_t>(stream));
}
