// tsx_adapters.hip - low-rank adapters of many requests beside a projection on gfx950, and their gradients:
// tsx_moe_adapters, tsx_moe_adapters_backward.
//
//   y[j] = base[j] + s[a] B[a] (A[a] x[j]),  a = ids[j];   u = A x,  v = s B^T dy:
//   dx = dbase + A^T v,  dA[a] = sum over a's rows of v x^T,  dB[a] = sum of dy (s u)^T.
//
// x, y and the gradients are fp32 as everywhere in this library, the matrices fp32, fp16 or bf16; the products run on
// v_mfma_f32_16x16x4_f32, whose operands are fp32, so nothing is rounded below 32 bits.  The rank is small, so the rows of x
// and y are most of the bytes and each is moved once: a block takes 16 rows, forms their u with its waves sharing the
// contraction (one sum in LDS), and expands it at once, u staying in the registers in the layout that the second product
// reads: the accumulator of u holds ranks 4 g .. 4 g + 3 of row l % 16 in lane l = 16 g + .., and an operand holds row
// l % 16, k = g, so accumulator register e is the operand of the step over ranks 4 g + e, with no exchange between lanes.
//
// A block works for one adapter.  Sixteen rows that lie together and name one adapter (a prompt's rows, one token) are a tile
// as they stand; the others (a mixed batch, the edges between requests) are regrouped, kChunk rows at a time, by further
// blocks that each read the chunk's ids and work out which rows are theirs: no table is built ahead, so one launch does.
#include "tsx_common.hpp"
#include "tsx_device.hpp"

#include <algorithm>

namespace tsx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

constexpr int kMaxRank = 256;

// eight consecutive values of type T as stored, and as floats
struct __attribute__((aligned(8))) Raw16 {  // one 16-byte load of an 8-byte aligned address
    uint32_t w[4];
};
template <int T> struct Oct {
    Raw16 v;
    __device__ __forceinline__ float at(int c) const {
        const uint32_t w = v.w[c / 2], h = c & 1 ? w >> 16 : w & 0xFFFFu;
        return T == TSX_F16 ? h2f((uint16_t) h) : __builtin_bit_cast(float, h << 16);
    }
};
template <> struct Oct<TSX_F32> {
    f32x4 v[2];
    __device__ __forceinline__ float at(int c) const { return v[c / 4][c % 4]; }
};
template <int T> __device__ __forceinline__ float value_at(const void* p, int64_t e) {
    if (T == TSX_F32) return ((const float*) p)[e];
    const uint16_t h = ((const uint16_t*) p)[e];
    return T == TSX_F16 ? h2f(h) : __builtin_bit_cast(float, (uint32_t) h << 16);
}
// floats e .. e + 3 of p, those from `left` on as 0.  VEC: e and the rows lie on 16-byte boundaries, left is a multiple of 4
template <bool VEC> __device__ __forceinline__ f32x4 load_quad(const float* p, int64_t e, int left) {
    f32x4 q = {0.f, 0.f, 0.f, 0.f};
    if constexpr (VEC) {
        if (left > 0) q = *(const f32x4*) (p + e);
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < left) q[c] = p[e + c];
    }
    return q;
}
template <bool VEC> __device__ __forceinline__ void store_quad(float* p, int64_t e, int left, const f32x4& d) {
    if constexpr (VEC) {
        if (left > 0) *(f32x4*) (p + e) = d;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < left) p[e + c] = d[c];
    }
}
// values e .. e + 7 of p, those from `left` on as 0.  VEC: e on a multiple of 4 values, the array on one, left a multiple of 4
template <int T, bool VEC> __device__ __forceinline__ Oct<T> load_oct(const void* p, int64_t e, int left) {
    Oct<T> q;
    if constexpr (T == TSX_F32) {
        q.v[0] = load_quad<VEC>((const float*) p, e, left);
        q.v[1] = load_quad<VEC>((const float*) p, e + 4, left - 4);
    } else {
        const uint16_t* h = (const uint16_t*) p + e;
        q.v = Raw16{{0u, 0u, 0u, 0u}};
        if constexpr (VEC) {
            if (left >= 8) {
                q.v = *(const Raw16*) h;
            } else if (left > 0) {
                const uint2 w = *(const uint2*) h;
                q.v.w[0] = w.x, q.v.w[1] = w.y;
            }
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < left) q.v.w[c / 2] |= (uint32_t) h[c] << (c & 1 ? 16 : 0);
        }
    }
    return q;
}
// the four values e .. e + 3 as floats
template <int T, bool VEC> __device__ __forceinline__ f32x4 load_four(const void* p, int64_t e, int left) {
    if constexpr (T == TSX_F32) return load_quad<VEC>((const float*) p, e, left);
    const uint16_t* h = (const uint16_t*) p + e;
    uint32_t w[2] = {0u, 0u};
    if constexpr (VEC) {
        if (left > 0) {
            const uint2 v = *(const uint2*) h;
            w[0] = v.x, w[1] = v.y;
        }
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < left) w[c / 2] |= (uint32_t) h[c] << (c & 1 ? 16 : 0);
    }
    f32x4 o;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t v = c & 1 ? w[c / 2] >> 16 : w[c / 2] & 0xFFFFu;
        o[c] = T == TSX_F16 ? h2f((uint16_t) v) : __builtin_bit_cast(float, v << 16);
    }
    return o;
}

// acc[rt] += the [16 ranks][K] tiles of w (row-major [rank][K]) times x^T over the chunks of 32 columns that are this wave's:
// lane l = 16 g + i holds rank 16 rt + i of w, row i of x, and columns 8 g .. 8 g + 7 of the chunk (any order of the columns
// will do as long as both operands have the same).  The blocks start `turn` chunks apart: rows are a power of two apart as
// often as not, and blocks that walk them in step would meet in the same memory channels.
template <int T, int RT, bool VEC, int WAVES>
__device__ __forceinline__ void contract_rows(f32x4 (&acc)[RT], const void* w, int rank, const float* x, int K, int wave,
                                              int lane, int turn) {
    constexpr int UN = RT == 1 ? 4 : RT <= 4 ? 2 : 1;  // chunks in flight
    const int i = lane & 15, g = lane >> 4, chunks = (K + 31) / 32;
    turn %= chunks;
    for (int c0 = UN * wave; c0 < chunks; c0 += UN * WAVES) {
        Oct<TSX_F32> xv[UN];
        Oct<T> wv[UN][RT];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            int c = c0 + u + turn;
            c -= c >= chunks ? chunks : 0;
            const int k = 32 * c + 8 * g, left = c0 + u < chunks ? K - k : 0;
            xv[u] = load_oct<TSX_F32, VEC>(x, k, left);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int r = 16 * rt + i;
                wv[u][rt] = load_oct<T, VEC>(w, (int64_t) r * K + k, r < rank ? left : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma(wv[u][rt].at(e), xv[u].at(e), acc[rt]);
    }
}
// the same with w row-major [K][rank]: a lane's values are a column apart, 16 lanes' lie together
template <int T, int RT, bool VEC, int WAVES>
__device__ __forceinline__ void contract_cols(f32x4 (&acc)[RT], const void* w, int rank, const float* x, int K, int wave,
                                              int lane, int turn) {
    constexpr int UN = RT == 1 ? 2 : 1;
    const int i = lane & 15, g = lane >> 4, chunks = (K + 31) / 32;
    turn %= chunks;
    for (int c0 = UN * wave; c0 < chunks; c0 += UN * WAVES) {
        Oct<TSX_F32> xv[UN];
        float wv[UN][RT][8];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            int c = c0 + u + turn;
            c -= c >= chunks ? chunks : 0;
            const int k = 32 * c + 8 * g, left = c0 + u < chunks ? K - k : 0;
            xv[u] = load_oct<TSX_F32, VEC>(x, k, left);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = 16 * rt + i;
                    wv[u][rt][e] = r < rank && e < left ? value_at<T>(w, (int64_t) (k + e) * rank + r) : 0.f;
                }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma(wv[u][rt][e], xv[u].at(e), acc[rt]);
    }
}

// the waves' sums added up in wave order, times s, in every wave; lds: (WAVES + 1) * RT * 1 KiB.  Ranks past the last are 0
// (an infinite column times the zeros that fill the operand up has left a NaN there)
template <int RT, int WAVES>
__device__ __forceinline__ void sum_waves(f32x4 (&acc)[RT], float s, int rank, f32x4* lds, int wave, int lane) {
    __syncthreads();  // the last use of lds is over
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) lds[(wave * RT + rt) * 64 + lane] = acc[rt];
    __syncthreads();
    f32x4* total = lds + WAVES * RT * 64;
    for (int q = threadIdx.x; q < RT * 64; q += WAVES * 64) {
        f32x4 t = lds[q];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) t += lds[w * RT * 64 + q];
        const int r = 16 * (q >> 6) + 4 * ((q >> 4) & 3);
#pragma unroll
        for (int c = 0; c < 4; ++c) t[c] = r + c < rank ? t[c] * s : 0.f;
        total[q] = t;
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) acc[rt] = total[rt * 64 + lane];
}

// The tiles of a launch: first the 16-row tiles as the rows stand, then `extra` tiles for every chunk of kChunk rows, for the
// rows of the tiles that name more than one adapter.
constexpr int kChunk = 4096, kMaxAdapters = 4096;
struct Tiles {
    int64_t plain;
    int extra, chunks;
    Tiles(int64_t rows, int n) : plain((rows + 15) / 16), chunks((int) ((rows + kChunk - 1) / kChunk)) {
        // a class of c rows takes ceil(c / 16) tiles; there are at most n + 1 classes and as many as rows
        const int64_t r = std::min<int64_t>(rows, kChunk);
        extra = n == 0 || r < 2 ? 0 : (int) std::min(r / 16 + std::min<int64_t>(n + 1, r), r);
    }
    int64_t blocks() const { return plain + (int64_t) extra * chunks; }
};
struct Tile {
    int cur;      // the adapter, or -1: rows without one
    int64_t row;  // of lane l: row l % 16 of the tile, -1 past the last
};
// count: n + 1 ints of LDS.  False: the block has no tile.  Every thread of the block calls
template <int WAVES>
__device__ __forceinline__ bool find_tile(Tile& t, const int32_t* ids, int64_t rows, int n, int64_t plain, int extra, int* count) {
    constexpr int NT = 64 * WAVES, R = kChunk / NT, SEGS = kChunk / 64;
    static_assert(SEGS == 64, "one segment a lane");
    __shared__ int s_sum[WAVES], s_seg[SEGS], s_row[16], s_class, s_first;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto class_of = [&](int64_t j) {  // 0 .. n - 1, n for none, -1 past the rows
        if (j >= rows) return -1;
        const int id = ids[j];
        return id < 0 || id >= n ? n : id;
    };
    if ((int64_t) blockIdx.x < plain) {
        t.row = (int64_t) blockIdx.x * 16 + (lane & 15);
        const int c = class_of(t.row), first = __builtin_amdgcn_readfirstlane(c);
        if (c < 0) t.row = -1;
        t.cur = first == n ? -1 : first;
        return __ballot(c >= 0 && c != first) == 0;
    }
    const int64_t e = (int64_t) blockIdx.x - plain, base = e / extra * kChunk;
    const int mine = (int) (e % extra);
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
    t.cur = cls == n ? -1 : cls;
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
    int64_t ld_x, ld_base, ld_y, ld_dy, ld_dbase, ld_dx, rows, plain;
    int n, rank, n_in, n_out, cols, extra;  // cols: output columns per block
};
template <int T> __device__ __forceinline__ const void* matrix_at(const void* p, int64_t values) {
    return (const char*) p + values * (T == TSX_F32 ? 4 : 2);
}

template <int RT> constexpr int waves_for() { return RT <= 4 ? 8 : 4; }

template <int T, int RT, bool VEC>
__global__ void __launch_bounds__(64 * waves_for<RT>()) adapters_kernel(AdArgs p) {
    constexpr int WAVES = waves_for<RT>();
    extern __shared__ int s_count[];
    __shared__ f32x4 lds[(WAVES + 1) * RT * 64];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    if (!find_tile<WAVES>(t, p.ids, p.rows, p.n, p.plain, p.extra, s_count)) return;
    if (t.cur < 0 && p.base == p.y) return;  // in place: rows without an adapter stay
    const bool mine = t.row >= 0;
    const int64_t at = mine ? t.row : __shfl(t.row, 0, 64);
    const int c0 = blockIdx.y * p.cols, c1 = min(c0 + p.cols, p.n_out);
    const float* base = p.base ? p.base + at * p.ld_base : nullptr;
    float* y = p.y + at * p.ld_y;
    f32x4 u[RT] = {};
    if (t.cur >= 0) {
        contract_rows<T, RT, VEC, WAVES>(u, matrix_at<T>(p.a, t.cur * p.a_stride), p.rank, p.x + at * p.ld_x, p.n_in, wave, lane,
                                         (int) blockIdx.x * 5);
        sum_waves<RT, WAVES>(u, p.scale ? p.scale[t.cur] : 1.f, p.rank, lds, wave, lane);
    }
    const void* b = t.cur >= 0 ? matrix_at<T>(p.b, t.cur * p.b_stride) : nullptr;
    // the block's columns, 16 a product: a run of them for every wave, four products at a time
    const int tiles = (c1 - c0 + 15) / 16, run = (tiles + WAVES - 1) / WAVES, t1 = min(tiles, (wave + 1) * run);
    constexpr int UN = RT <= 2 ? 4 : RT <= 4 ? 2 : 1;
    for (int t0 = wave * run; t0 < t1; t0 += UN) {
        f32x4 d[UN], w[UN][RT];
#pragma unroll
        for (int q = 0; q < UN; ++q) {
            const int m = c0 + 16 * (t0 + q), left = t0 + q < t1 ? c1 - m : 0;
            d[q] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (base && mine) d[q] = load_quad<VEC>(base, m + 4 * g, left - 4 * g);
            if (t.cur >= 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const int r = 16 * rt + 4 * g;
                    w[q][rt] = load_four<T, VEC>(b, (int64_t) (m + i) * p.rank + r, i < left ? p.rank - r : 0);
                }
            }
        }
        if (t.cur >= 0) {
            f32x4 sum[UN] = {};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int q = 0; q < UN; ++q) sum[q] = mfma(w[q][rt][e], u[rt][e], sum[q]);
#pragma unroll
            for (int q = 0; q < UN; ++q) d[q] += sum[q];
        }
        if (mine) {
#pragma unroll
            for (int q = 0; q < UN; ++q) {
                const int m = c0 + 16 * (t0 + q) + 4 * g;
                store_quad<VEC>(y, m, t0 + q < t1 ? c1 - m : 0, d[q]);
            }
        }
    }
}

// The backward's row half: s u and v of every row with an adapter (into u and v, [rows][16 RT], ranks past the last as 0), and
// dx.
template <int T, int RT, bool VEC>
__global__ void __launch_bounds__(64 * waves_for<RT>()) adapters_back_rows_kernel(AdArgs p) {
    constexpr int WAVES = waves_for<RT>();
    extern __shared__ int s_count[];
    __shared__ f32x4 lds[(WAVES + 1) * RT * 64];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    if (!find_tile<WAVES>(t, p.ids, p.rows, p.n, p.plain, p.extra, s_count)) return;
    const bool mine = t.row >= 0;
    const int64_t at = mine ? t.row : __shfl(t.row, 0, 64);
    const int c0 = blockIdx.y * p.cols, c1 = min(c0 + p.cols, p.n_in);
    f32x4 v[RT] = {};
    if (t.cur >= 0) {
        const float s = p.scale ? p.scale[t.cur] : 1.f;
        if (p.u && blockIdx.y == 0) {
            f32x4 u[RT] = {};
            contract_rows<T, RT, VEC, WAVES>(u, matrix_at<T>(p.a, t.cur * p.a_stride), p.rank, p.x + at * p.ld_x, p.n_in, wave,
                                             lane, (int) blockIdx.x * 5);
            sum_waves<RT, WAVES>(u, s, p.rank, lds, wave, lane);
            if (wave == 0 && mine) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) *(f32x4*) (p.u + t.row * (16 * RT) + 16 * rt + 4 * g) = u[rt];
            }
        }
        contract_cols<T, RT, VEC, WAVES>(v, matrix_at<T>(p.b, t.cur * p.b_stride), p.rank, p.dy + at * p.ld_dy, p.n_out, wave,
                                         lane, (int) blockIdx.x * 5);
        sum_waves<RT, WAVES>(v, s, p.rank, lds, wave, lane);
        if (p.v && blockIdx.y == 0 && wave == 0 && mine) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) *(f32x4*) (p.v + t.row * (16 * RT) + 16 * rt + 4 * g) = v[rt];
        }
    }
    if (!p.dx || (t.cur < 0 && p.dbase == p.dx)) return;
    const float* dbase = p.dbase ? p.dbase + at * p.ld_dbase : nullptr;
    float* dx = p.dx + at * p.ld_dx;
    const void* a = t.cur >= 0 ? matrix_at<T>(p.a, t.cur * p.a_stride) : nullptr;
    // 64 columns: lane i's four columns 4 i .. of a rank give four products, whose accumulators hold columns 16 g + 4 r + q:
    // four in a row for every r
    for (int n0 = c0 + 64 * wave; n0 < c1; n0 += 64 * WAVES) {
        f32x4 d[4] = {}, old[4] = {};
        if (dbase && mine) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int col = n0 + 16 * g + 4 * r;
                old[r] = load_quad<VEC>(dbase, col, c1 - col);
            }
        }
        if (t.cur >= 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                f32x4 w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 16 * rt + 4 * g + e, n = n0 + 4 * i;
                    w[e] = load_four<T, VEC>(a, (int64_t) r * p.n_in + n, r < p.rank ? c1 - n : 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int q = 0; q < 4; ++q) d[q] = mfma(w[e][q], v[rt][e], d[q]);
            }
        }
        if (!mine) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int col = n0 + 16 * g + 4 * r;
            store_quad<VEC>(dx, col, c1 - col, f32x4{d[0][r], d[1][r], d[2][r], d[3][r]} + old[r]);
        }
    }
}

// The backward's weight half: a block takes 64 columns of one adapter's dA (x: columns of x, coefficients v) or dB (columns
// of dy, coefficients s u) and 16 RT ranks of it.  It lists the adapter's rows itself, kChunk ids at a time, and its waves
// share them, four rows a step: lane l = 16 g + i holds coefficient i of row g and columns 4 i .. 4 i + 3 of it, four products.
// The sums of the waves meet in LDS, in wave order.  An adapter without rows gets zeros.
struct AdSumArgs {
    const float* x;
    const float* dy;
    const float* u;
    const float* v;
    const int32_t* ids;
    float* da;
    float* db;
    int64_t ld_x, ld_dy, rows;
    int n_in, n_out, rank, ldu, tiles_a, tiles_b;
};
template <int RT, bool VEC>
__global__ void __launch_bounds__(512) adapters_back_sum_kernel(AdSumArgs p) {
    constexpr int WAVES = 8, R = kChunk / 512;
    __shared__ f32x4 lds[WAVES * RT * 64];
    __shared__ int s_row[kChunk], s_seg[64];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ad = blockIdx.y, r0 = blockIdx.z * 16 * RT;
    const bool is_a = (int) blockIdx.x < p.tiles_a;
    const int n0 = 64 * (is_a ? blockIdx.x : blockIdx.x - p.tiles_a), K = is_a ? p.n_in : p.n_out, n = n0 + 4 * i;
    const float* src = is_a ? p.x : p.dy;
    const int64_t ld = is_a ? p.ld_x : p.ld_dy;
    const float* coef = (is_a ? p.v : p.u) + r0;
    f32x4 acc[4][RT] = {};
    constexpr int UN = RT <= 2 ? 4 : 2;
    for (int64_t base = 0; base < p.rows; base += kChunk) {
        int id[R];
        uint64_t hit[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t j = base + r * 512 + threadIdx.x;
            id[r] = j < p.rows ? p.ids[j] : -1;
        }
        __syncthreads();  // the last chunk's list is used up
#pragma unroll
        for (int r = 0; r < R; ++r) {
            hit[r] = __ballot(id[r] == ad);
            if (lane == 0) s_seg[r * WAVES + wave] = __builtin_popcountll(hit[r]);
        }
        __syncthreads();
        int incl = s_seg[lane];
        const int self = incl;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(incl, o, 64);
            if (lane >= o) incl += t;
        }
        const int before = incl - self, hi = __builtin_amdgcn_readlane(incl, 63);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int at = __builtin_amdgcn_readlane(before, r * WAVES + wave);
            if (id[r] == ad) s_row[at + __builtin_popcountll(hit[r] & ((1ull << lane) - 1))] = r * 512 + threadIdx.x;
        }
        __syncthreads();
        for (int j0 = 4 * UN * wave; j0 < hi; j0 += 4 * UN * WAVES) {
            f32x4 xv[UN];
            float cv[UN][RT];
#pragma unroll
            for (int s = 0; s < UN; ++s) {
                const int j = j0 + 4 * s + g;
                const bool in = j < hi;
                const int64_t row = base + (in ? s_row[j] : 0);
                xv[s] = load_quad<VEC>(src + row * ld, n, in ? K - n : 0);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) cv[s][rt] = in ? coef[row * p.ldu + 16 * rt + i] : 0.f;
            }
#pragma unroll
            for (int s = 0; s < UN; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        acc[q][rt] = is_a ? mfma(cv[s][rt], xv[s][q], acc[q][rt]) : mfma(xv[s][q], cv[s][rt], acc[q][rt]);
        }
    }
    // dA's accumulators hold rank 4 g + r of column 4 i + q, dB's column 4 (4 g + r) + q of rank i
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) lds[(wave * RT + rt) * 64 + lane] = acc[q][rt];
        __syncthreads();
        for (int s = threadIdx.x; s < RT * 64; s += 64 * WAVES) {
            f32x4 t = lds[s];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) t += lds[w * RT * 64 + s];
            const int rt = s >> 6, si = s & 15, sg = (s >> 4) & 3;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (is_a) {
                    const int k = r0 + 16 * rt + 4 * sg + r, c = n0 + 4 * si + q;
                    if (k < p.rank && c < K) p.da[((int64_t) ad * p.rank + k) * K + c] = t[r];
                } else {
                    const int k = r0 + 16 * rt + si, c = n0 + 4 * (4 * sg + r) + q;
                    if (k < p.rank && c < K) p.db[((int64_t) ad * K + c) * p.rank + k] = t[r];
                }
            }
        }
    }
}

inline size_t elem_size(int type) { return type == TSX_F32 ? 4 : 2; }

int check_adapters(const char* what, const tsx_adapters* p, int64_t rows) {
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
bool matrix_quads(const tsx_adapters* p) {
    const size_t z = 4 * elem_size(p->type);
    return p->rank % 4 == 0 && p->n_in % 4 == 0 && p->n_out % 4 == 0 && p->a_stride % 4 == 0 && p->b_stride % 4 == 0 &&
           aligned(p->a, z) && aligned(p->b, z);
}
// columns per block: the blocks of one tile of rows repeat its first product, so a tile is split only as far as it takes to
// give every CU a block
int columns_per_block(int64_t tiles, int cols, int least) {
    const int64_t want = std::max<int64_t>(1, 512 / tiles), per = (cols + want - 1) / want;
    return (int) ((std::max<int64_t>(per, least) + least - 1) / least * least);
}
void fill(AdArgs& k, const tsx_adapters* p, const int32_t* ids, int64_t rows) {
    k.a = p->a, k.b = p->b, k.a_stride = p->a_stride, k.b_stride = p->b_stride, k.scale = p->scale, k.ids = ids;
    const Tiles t(rows, p->n);
    k.plain = t.plain, k.extra = t.extra;
    k.rows = rows, k.n = p->n, k.rank = p->rank, k.n_in = p->n_in, k.n_out = p->n_out;
}

template <int T, int RT, bool VEC> void launch_forward(const AdArgs& k, dim3 grid, hipStream_t st) {
    adapters_kernel<T, RT, VEC><<<grid, 64 * waves_for<RT>(), k.extra ? (size_t) (k.n + 1) * 4 : 0, st>>>(k);
}
template <int T, int RT, bool VEC> void launch_back_rows(const AdArgs& k, dim3 grid, hipStream_t st) {
    adapters_back_rows_kernel<T, RT, VEC><<<grid, 64 * waves_for<RT>(), k.extra ? (size_t) (k.n + 1) * 4 : 0, st>>>(k);
}
template <bool BACK, int T, int RT> void launch_vec(bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    if constexpr (BACK) vec ? launch_back_rows<T, RT, true>(k, grid, st) : launch_back_rows<T, RT, false>(k, grid, st);
    else vec ? launch_forward<T, RT, true>(k, grid, st) : launch_forward<T, RT, false>(k, grid, st);
}
template <bool BACK, int T> void launch_rank(bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    if (k.rank <= 16) launch_vec<BACK, T, 1>(vec, k, grid, st);
    else if (k.rank <= 32) launch_vec<BACK, T, 2>(vec, k, grid, st);
    else if (k.rank <= 64) launch_vec<BACK, T, 4>(vec, k, grid, st);
    else if (k.rank <= 128) launch_vec<BACK, T, 8>(vec, k, grid, st);
    else launch_vec<BACK, T, 16>(vec, k, grid, st);
}
template <bool BACK> void launch(int type, bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    if (type == TSX_F32) launch_rank<BACK, TSX_F32>(vec, k, grid, st);
    else if (type == TSX_F16) launch_rank<BACK, TSX_F16>(vec, k, grid, st);
    else launch_rank<BACK, TSX_BF16>(vec, k, grid, st);
}

template <int RT, bool VEC> void launch_sum(const AdSumArgs& k, dim3 grid, hipStream_t st) {
    adapters_back_sum_kernel<RT, VEC><<<grid, 512, 0, st>>>(k);
}

// the backward's scratch: u and v
size_t back_values(const tsx_adapters* p, int64_t rows) {
    const int rt = p->rank <= 16 ? 1 : p->rank <= 32 ? 2 : p->rank <= 64 ? 4 : p->rank <= 128 ? 8 : 16;
    return ((size_t) rows * 16 * rt * 4 + 255) / 256 * 256 / 4;
}

}  // namespace
}  // namespace tsx

using namespace tsx;

extern "C" {

TSX_API int tsx_moe_adapters(const tsx_adapters* p, const int32_t* ids, const float* x, int64_t ld_x, const float* base,
                             int64_t ld_base, float* y, int64_t ld_y, int64_t rows, void* stream) {
    if (const int rc = check_adapters("tsx_moe_adapters", p, rows)) return rc;
    if (rows == 0) return TSX_OK;
    TSX_REQUIRE(ids && x && y && aligned(ids, 4) && aligned(x, 4) && aligned(base, 4) && aligned(y, 4),
                "tsx_moe_adapters: ids, x, y (and base) 4-byte aligned");
    TSX_REQUIRE(ld_x >= p->n_in && ld_y >= p->n_out && (!base || ld_base >= p->n_out) && (base != y || ld_base == ld_y),
                "tsx_moe_adapters: rows as long as their columns; in place with one ld");
    AdArgs k{};
    fill(k, p, ids, rows);
    k.x = x, k.ld_x = ld_x, k.base = base, k.ld_base = ld_base, k.y = y, k.ld_y = ld_y;
    const Tiles t(rows, p->n);
    const bool vec = matrix_quads(p) && quads(x, ld_x, 4) && quads(y, ld_y, 4) && (!base || quads(base, ld_base, 4));
    k.cols = columns_per_block(t.plain, p->n_out, 128);
    launch<false>(p->type, vec, k, dim3((unsigned) t.blocks(), (unsigned) ((p->n_out + k.cols - 1) / k.cols)), (hipStream_t) stream);
    return launch_status("tsx_moe_adapters");
}

TSX_API size_t tsx_moe_adapters_scratch_bytes(const tsx_adapters* p, int64_t rows) {
    if (!p || p->n < 0 || rows < 0 || p->rank < 1 || p->rank > kMaxRank) return 0;
    return 2 * back_values(p, rows) * 4;
}

TSX_API int tsx_moe_adapters_backward(const tsx_adapters* p, const int32_t* ids, const float* x, int64_t ld_x, const float* dy,
                                      int64_t ld_dy, const float* dbase, int64_t ld_dbase, float* dx, int64_t ld_dx,
                                      float* da, float* db, int64_t rows, void* scratch, void* stream) {
    if (const int rc = check_adapters("tsx_moe_adapters_backward", p, rows)) return rc;
    TSX_REQUIRE(rows == 0 || (ids && x && dy && scratch), "tsx_moe_adapters_backward: ids, x, dy, scratch");
    TSX_REQUIRE(aligned(ids, 4) && aligned(x, 4) && aligned(dy, 4) && aligned(dbase, 4) && aligned(dx, 4) && aligned(da, 4) &&
                    aligned(db, 4) && aligned(scratch, 256),
                "tsx_moe_adapters_backward: buffers 4-byte aligned, scratch 256-byte aligned");
    TSX_REQUIRE(rows == 0 || (ld_x >= p->n_in && ld_dy >= p->n_out && (!dx || ld_dx >= p->n_in) &&
                              (!dbase || ld_dbase >= p->n_in) && (!dbase || dbase != dx || ld_dbase == ld_dx)),
                "tsx_moe_adapters_backward: rows as long as their columns; in place with one ld");
    const hipStream_t st = (hipStream_t) stream;
    float* u = (float*) scratch;
    float* v = u + back_values(p, rows);
    const bool sums = p->n > 0 && (da || db);
    if (rows) {
        AdArgs k{};
        fill(k, p, ids, rows);
        k.x = x, k.ld_x = ld_x, k.dy = dy, k.ld_dy = ld_dy, k.dbase = dbase, k.ld_dbase = ld_dbase, k.dx = dx, k.ld_dx = ld_dx;
        k.u = sums && db ? u : nullptr;
        k.v = sums && da ? v : nullptr;
        const bool vec = matrix_quads(p) && quads(x, ld_x, 4) && quads(dy, ld_dy, 4) && (!dx || quads(dx, ld_dx, 4)) &&
                         (!dbase || quads(dbase, ld_dbase, 4));
        const Tiles t(rows, p->n);
        k.cols = dx ? columns_per_block(t.plain, p->n_in, 512) : p->n_in;
        launch<true>(p->type, vec, k, dim3((unsigned) t.blocks(), (unsigned) ((p->n_in + k.cols - 1) / k.cols)), st);
        if (const int rc = launch_status("tsx_moe_adapters_backward")) return rc;
    }
    if (sums) {
        AdSumArgs k{};
        k.x = x, k.ld_x = ld_x, k.dy = dy, k.ld_dy = ld_dy, k.u = u, k.v = v, k.ids = ids, k.rows = rows;
        k.da = da, k.db = db, k.n_in = p->n_in, k.n_out = p->n_out, k.rank = p->rank;
        k.ldu = p->rank <= 16 ? 16 : p->rank <= 32 ? 32 : p->rank <= 64 ? 64 : p->rank <= 128 ? 128 : 256;
        k.tiles_a = da ? (p->n_in + 63) / 64 : 0, k.tiles_b = db ? (p->n_out + 63) / 64 : 0;
        const bool vec = quads(x, ld_x, p->n_in) && quads(dy, ld_dy, p->n_out);
        const int rt = p->rank <= 16 ? 1 : p->rank <= 32 ? 2 : 4;
        const dim3 grid((unsigned) (k.tiles_a + k.tiles_b), (unsigned) p->n, (unsigned) ((p->rank + 16 * rt - 1) / (16 * rt)));
        if (rt == 1) vec ? launch_sum<1, true>(k, grid, st) : launch_sum<1, false>(k, grid, st);
        else if (rt == 2) vec ? launch_sum<2, true>(k, grid, st) : launch_sum<2, false>(k, grid, st);
        else vec ? launch_sum<4, true>(k, grid, st) : launch_sum<4, false>(k, grid, st);
        return launch_status("tsx_moe_adapters_backward");
    }
    return TSX_OK;
}

}  // extern "C"
