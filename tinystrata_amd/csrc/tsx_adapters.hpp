// tsx_adapters.hpp - what the adapters' forward and backward kernels share: the tiles of a launch, the arguments and their
// checks.
#pragma once

#include <algorithm>

#include "tsx_common.hpp"
#include "tsx_device.hpp"

namespace tsx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

constexpr int kMaxRank = 256;

// The tiles of a launch: `extra` blocks for every chunk of kChunk rows, for the rows of the 16-row tiles that name more than
// one adapter (first: they have the ids to read before they know their rows), then the 16-row tiles as the rows stand.
constexpr int kChunk = 4096, kMaxAdapters = 4096;
struct Tiles {
    int64_t plain;  // a multiple of 8: a run of tiles for each XCD
    int extra, chunks;
    Tiles(int64_t rows, int n, int most) : plain((rows + 127) / 128 * 8), chunks((int) ((rows + kChunk - 1) / kChunk)) {
        // a class of c rows takes ceil(c / 16) tiles; there are at most n + 1 classes and as many as rows.  Past `most` of them
        // a block takes a further tile (a chunk of one adapter costs each of its blocks a look at the ids)
        const int64_t r = std::min<int64_t>(rows, kChunk);
        extra = n == 0 || r < 2 ? 0 : (int) std::min<int64_t>(std::min(r / 16 + std::min<int64_t>(n + 1, r), r), most);
    }
    int64_t blocks() const { return plain + (int64_t) extra * chunks; }
};
struct Tile {
    int cur;      // the adapter, or -1: rows without one
    int64_t row;  // of lane l: row l % 16 of the tile, -1 past the last
};
// The block's tile number `round`.  count: n + 1 ints of LDS.  False: it has none.  Every thread of the block calls
template <int WAVES>
__device__ __forceinline__ bool find_tile(Tile& t, const int32_t* ids, int64_t rows, int n, int regroup, int extra, int round,
                                          int* count, int tid) {
    constexpr int NT = 64 * WAVES, R = kChunk / NT, SEGS = kChunk / 64;
    static_assert(SEGS == 64, "one segment a lane");
    __shared__ int s_sum[WAVES], s_seg[SEGS], s_row[16], s_class, s_first;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto class_of = [&](int64_t j) {  // 0 .. n - 1, n for none, -1 past the rows (an unconditional load: eight in flight)
        const int id = ids[min(j, rows - 1)];
        return j >= rows ? -1 : id < 0 || id >= n ? n : id;
    };
    if ((int) blockIdx.x >= regroup) {
        if (round > 0) return false;
        // neighbouring tiles on one XCD (blocks go round them), whose L2 then holds the matrices of few adapters
        const int q = blockIdx.x - regroup, per = (gridDim.x - regroup) / 8;
        t.row = ((int64_t) (q % 8) * per + q / 8) * 16 + (lane & 15);
        const int c = class_of(t.row), first = __builtin_amdgcn_readfirstlane(c);
        if (first < 0) return false;
        if (c < 0) t.row = -1;
        t.cur = first == n ? -1 : first;
        return __ballot(c >= 0 && c != first) == 0;
    }
    const int64_t base = (int64_t) (blockIdx.x / extra) * kChunk;
    const int mine = blockIdx.x % extra + round * extra;
    if (mine >= kChunk) return false;
    if (rows <= 64) {
        // a decode step: every wave has all rows on its lanes, and finds each lane's class mates from one ballot per bit of a
        // class, with no barrier (64 mixed rows, 2048 -> 512, rank 16: 11.1 us for 15.0 the long way)
        const int c = class_of(lane), lead = __shfl(c, lane & 48, 64);
        const uint64_t other = __ballot(c >= 0 && c != lead), below = (1ull << lane) - 1;
        const bool ours = c >= 0 && ((other >> (lane & 48)) & 0xFFFFu) != 0;
        uint64_t mates = __ballot(ours);
        if (!mates) return false;
        for (int bit = 0; n >> bit; ++bit) {
            const uint64_t set = __ballot(c >> bit & 1);
            mates &= c >> bit & 1 ? set : ~set;
        }
        const int before = __builtin_popcountll(mates & below), k = (__builtin_popcountll(mates) + 15) / 16;
        const bool leads = ours && before == 0;
        int at = 0;  // tiles of the classes that a lower lane leads
#pragma unroll
        for (int q = 1; q <= 4; ++q) at += __builtin_popcountll(__ballot(leads && k >= q) & below);
        const uint64_t hit = __ballot(leads && mine >= at && mine < at + k);
        if (!hit) return false;
        const int lane0 = __builtin_ctzll(hit), cls = __builtin_amdgcn_readlane(c, lane0);
        const int to = before - 16 * (mine - __builtin_amdgcn_readlane(at, lane0));  // its place in the tile
        const bool in = ours && c == cls && to >= 0 && to < 16;
        const int got = __builtin_amdgcn_ds_permute(4 * (in ? to : 63), in ? lane + 1 : 0);  // 0 where none writes
        t.row = (int64_t) __shfl(got, lane & 15, 64) - 1;
        t.cur = cls == n ? -1 : cls;
        return true;
    }
    int c[R];
    bool some = false;
#pragma unroll
    for (int r = 0; r < R; ++r) c[r] = class_of(base + r * NT + tid);
#pragma unroll
    for (int r = 0; r < R; ++r) {  // the rows of tiles of one class are not ours
        const int first = __shfl(c[r], lane & 48, 64);
        const uint64_t other = __ballot(c[r] >= 0 && c[r] != first);
        if (((other >> (lane & 48)) & 0xFFFFu) == 0) c[r] = -1;
        some |= c[r] >= 0;
    }
    if (!__syncthreads_or(some)) return false;
    for (int q = tid; q <= n; q += NT) count[q] = 0;
    if (tid < 16) s_row[tid] = -1;
    if (tid == 0) s_class = -2;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (c[r] >= 0) atomicAdd(&count[c[r]], 1);
    __syncthreads();
    // the classes' tiles, in class order: which class tile `mine` belongs to, and which of it
    const int per = (n + NT) / NT, q0 = tid * per, q1 = min(q0 + per, n + 1);
    int own = 0;
    for (int q = q0; q < q1; ++q) own += (count[q] + 15) / 16;
    int incl = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
    }
    if (lane == 63) s_sum[wave] = incl;
    __syncthreads();
    int at = incl - own;
    for (int w = 0; w < wave; ++w) at += s_sum[w];
    if (mine >= at && mine < at + own) {
        for (int q = q0; q < q1; ++q) {
            const int k = (count[q] + 15) / 16;
            if (mine < at + k) {
                s_class = q;
                s_first = 16 * (mine - at);
                break;
            }
            at += k;
        }
    }
    __syncthreads();
    const int cls = s_class, first = s_first;
    if (cls < 0) return false;
    // its rows in row order: ranks from ballots, the segments of 64 rows in order
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint64_t b = __ballot(c[r] == cls);
        if (lane == 0) s_seg[r * WAVES + wave] = __builtin_popcountll(b);
    }
    __syncthreads();
    int before = s_seg[lane];
    const int self = before;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(before, o, 64);
        if (lane >= o) before += v;
    }
    before -= self;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint64_t b = __ballot(c[r] == cls);
        const int rank = __builtin_amdgcn_readlane(before, r * WAVES + wave) + __builtin_popcountll(b & ((1ull << lane) - 1));
        if (c[r] == cls && rank >= first && rank < first + 16) s_row[rank - first] = r * NT + tid;
    }
    __syncthreads();
    const int got = s_row[lane & 15];
    t.row = got < 0 ? -1 : base + got;
    t.cur = __builtin_amdgcn_readfirstlane(cls == n ? -1 : cls);
    return true;
}

struct AdArgs {
    const void* a;
    const void* b;
    int64_t a_stride, b_stride;  // in values
    const float* scale;
    const int32_t* ids;
    const float* x;
    const float* base;
    float* y;
    const float* dy;
    const float* dbase;
    float* dx;
    float* u;
    float* v;
    int64_t ld_x, ld_base, ld_y, ld_dy, ld_dbase, ld_dx, rows;
    int n, rank, n_in, n_out, cols, regroup, extra;  // cols: output columns per block; regroup: blocks of all chunks
};
template <int T> __device__ __forceinline__ const void* matrix_at(const void* p, int64_t values) {
    return (const char*) p + values * (T == TSX_F32 ? 4 : 2);
}

inline size_t elem_size(int type) { return type == TSX_F32 ? 4 : 2; }

inline int check_adapters(const char* what, const tsx_adapters* p, int64_t rows) {
    TSX_REQUIRE(p, "%s: no adapters", what);
    if (p->type != TSX_F32 && p->type != TSX_F16 && p->type != TSX_BF16) {
        set_error("%s: matrices of type %d (fp32, fp16 or bf16)", what, p->type);
        return TSX_ERR_UNSUPPORTED;
    }
    if (p->n > kMaxAdapters) {
        set_error("%s: %d adapters (at most %d)", what, p->n, kMaxAdapters);
        return TSX_ERR_UNSUPPORTED;
    }
    if (p->rank < 1 || p->rank > kMaxRank || p->n_in < 1 || p->n_out < 1 || p->n_in > (1 << 24) || p->n_out > (1 << 24)) {
        set_error("%s: rank %d, %d -> %d not supported (rank 1..256, sizes 1..2^24)", what, p->rank, p->n_in, p->n_out);
        return TSX_ERR_UNSUPPORTED;
    }
    const size_t z = elem_size(p->type);
    TSX_REQUIRE(p->n >= 0 && rows >= 0 && rows <= INT32_MAX, "%s: n >= 0, rows 0..2^31 - 1", what);
    TSX_REQUIRE(p->n == 0 || (p->a && p->b && aligned(p->a, z) && aligned(p->b, z)), "%s: a and b aligned to their type", what);
    TSX_REQUIRE(p->n <= 1 || (p->a_stride >= (int64_t) p->rank * p->n_in && p->b_stride >= (int64_t) p->rank * p->n_out),
                "%s: adapters overlap (a_stride, b_stride)", what);
    TSX_REQUIRE(aligned(p->scale, 4), "%s: scale 4-byte aligned", what);
    return TSX_OK;
}
inline bool quads(const float* p, int64_t ld, int cols) { return cols % 4 == 0 && ld % 4 == 0 && aligned(p, 16); }
// every quad of the matrices is one load
inline bool matrix_quads(const tsx_adapters* p) {
    const size_t z = 4 * elem_size(p->type);
    return p->rank % 4 == 0 && p->n_in % 4 == 0 && p->n_out % 4 == 0 && p->a_stride % 4 == 0 && p->b_stride % 4 == 0 &&
           aligned(p->a, z) && aligned(p->b, z);
}
// columns per block: the blocks of one tile of rows repeat its first product, so a tile is split only as far as it takes to
// give every CU a block
inline int columns_per_block(int64_t tiles, int cols, int least) {
    const int64_t want = std::max<int64_t>(1, 256 / tiles), per = (cols + want - 1) / want;
    return (int) ((std::max<int64_t>(per, least) + least - 1) / least * least);
}
inline void fill(AdArgs& k, const tsx_adapters* p, const int32_t* ids, int64_t rows, const Tiles& t) {
    k.a = p->a, k.b = p->b, k.a_stride = p->a_stride, k.b_stride = p->b_stride, k.scale = p->scale, k.ids = ids;
    k.regroup = t.extra * t.chunks, k.extra = t.extra;
    k.rows = rows, k.n = p->n, k.rank = p->rank, k.n_in = p->n_in, k.n_out = p->n_out;
}

}  // namespace
}  // namespace tsx
