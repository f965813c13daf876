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
// The rows of a block may belong to several requests: it takes the distinct adapters of its 16 rows in turn, each for its own
// rows.  Rows of a request lie together in a prompt, so that is mostly one or two; a mixed batch reads the adapters that it
// names, which is what it has to.
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

// four consecutive values of type T as stored, and as floats
template <int T> struct Quad {
    uint2 v;
    __device__ __forceinline__ float at(int c) const {
        const uint32_t w = c < 2 ? v.x : v.y, h = c & 1 ? w >> 16 : w & 0xFFFFu;
        return T == TSX_F16 ? h2f((uint16_t) h) : __builtin_bit_cast(float, h << 16);
    }
};
template <> struct Quad<TSX_F32> {
    float4 v;
    __device__ __forceinline__ float at(int c) const { return c == 0 ? v.x : c == 1 ? v.y : c == 2 ? v.z : v.w; }
};
template <int T> __device__ __forceinline__ float value_at(const void* p, int64_t e) {
    if (T == TSX_F32) return ((const float*) p)[e];
    const uint16_t h = ((const uint16_t*) p)[e];
    return T == TSX_F16 ? h2f(h) : __builtin_bit_cast(float, (uint32_t) h << 16);
}
template <int T> __device__ __forceinline__ uint32_t bits_at(const void* p, int64_t e) { return ((const uint16_t*) p)[e]; }
// values e .. e + 3 at p, those from `left` on as 0.  VEC: one load (e on a multiple of four values of an aligned array whose
// rows are too, so left is 4 or more, or 0 or less)
template <int T, bool VEC> __device__ __forceinline__ Quad<T> load_quad(const void* p, int64_t e, int left) {
    Quad<T> q;
    if constexpr (T == TSX_F32) {
        q.v = float4{0.f, 0.f, 0.f, 0.f};
        const float* f = (const float*) p + e;
        if constexpr (VEC) {
            if (left > 0) q.v = *(const float4*) f;
        } else {
            if (left > 0) q.v.x = f[0];
            if (left > 1) q.v.y = f[1];
            if (left > 2) q.v.z = f[2];
            if (left > 3) q.v.w = f[3];
        }
    } else {
        q.v = uint2{0u, 0u};
        if constexpr (VEC) {
            if (left > 0) q.v = *(const uint2*) ((const uint16_t*) p + e);
        } else {
            if (left > 0) q.v.x = bits_at<T>(p, e);
            if (left > 1) q.v.x |= bits_at<T>(p, e + 1) << 16;
            if (left > 2) q.v.y = bits_at<T>(p, e + 2);
            if (left > 3) q.v.y |= bits_at<T>(p, e + 3) << 16;
        }
    }
    return q;
}
template <bool VEC> __device__ __forceinline__ void store_quad(float* p, int64_t e, int left, const f32x4& d) {
    if constexpr (VEC) {
        if (left > 0) *(float4*) (p + e) = float4{d[0], d[1], d[2], d[3]};
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < left) p[e + c] = d[c];
    }
}

// acc[rt] += the [16 ranks][K] tiles of w (row-major [rank][K]) times x^T over the chunks of 16 columns that are this wave's:
// lane l = 16 g + i holds rank 16 rt + i of w, row i of x, and columns 4 g .. 4 g + 3 of the chunk
template <int T, int RT, bool VEC, int WAVES>
__device__ __forceinline__ void contract_rows(f32x4 (&acc)[RT], const void* w, int rank, const float* x, int K, int wave,
                                              int lane) {
    constexpr int UN = RT == 1 ? 8 : RT == 2 ? 4 : 2;  // chunks in flight
    const int i = lane & 15, g = lane >> 4;
    for (int c0 = 16 * UN * wave; c0 < K; c0 += 16 * UN * WAVES) {
        Quad<TSX_F32> xv[UN];
        Quad<T> wv[UN][RT];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int k = c0 + 16 * u + 4 * g;
            xv[u] = load_quad<TSX_F32, VEC>(x, k, K - k);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int r = 16 * rt + i;
                wv[u][rt] = load_quad<T, VEC>(w, (int64_t) r * K + k, r < rank ? K - k : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma(wv[u][rt].at(e), xv[u].at(e), acc[rt]);
    }
}
// the same with w row-major [K][rank]: a lane's four values are a column apart, 16 lanes' lie together
template <int T, int RT, bool VEC, int WAVES>
__device__ __forceinline__ void contract_cols(f32x4 (&acc)[RT], const void* w, int rank, const float* x, int K, int wave,
                                              int lane) {
    constexpr int UN = RT == 1 ? 4 : 2;
    const int i = lane & 15, g = lane >> 4;
    for (int c0 = 16 * UN * wave; c0 < K; c0 += 16 * UN * WAVES) {
        Quad<TSX_F32> xv[UN];
        float wv[UN][RT][4];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int k = c0 + 16 * u + 4 * g;
            xv[u] = load_quad<TSX_F32, VEC>(x, k, K - k);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 16 * rt + i;
                    wv[u][rt][e] = r < rank && k + e < K ? value_at<T>(w, (int64_t) (k + e) * rank + r) : 0.f;
                }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
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

// the distinct adapters of 16 rows, one by one: every wave of a block takes the same steps
struct RowIds {
    int id;         // of row lane & 15: -1 for none, -2 past the last row
    uint32_t left;  // rows not taken yet
    __device__ __forceinline__ RowIds(const int32_t* ids, int64_t row, int64_t rows, int n) {
        id = -2;
        if (row < rows) {
            id = ids[row];
            if (id < 0 || id >= n) id = -1;
        }
        left = (uint32_t) __ballot(id != -2) & 0xFFFFu;
    }
    __device__ __forceinline__ int next() {  // left != 0
        const int cur = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
        left &= ~(uint32_t) __ballot(id == cur);
        return cur;
    }
};

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
    int n, rank, n_in, n_out, cols;  // cols: output columns per block
};
template <int T> __device__ __forceinline__ const void* matrix_at(const void* p, int64_t values) {
    return (const char*) p + values * (T == TSX_F32 ? 4 : 2);
}

template <int RT> constexpr int waves_for() { return RT <= 4 ? 8 : 4; }

template <int T, int RT, bool VEC>
__global__ void __launch_bounds__(64 * waves_for<RT>()) adapters_kernel(AdArgs p) {
    constexpr int WAVES = waves_for<RT>();
    __shared__ f32x4 lds[(WAVES + 1) * RT * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int64_t row = (int64_t) blockIdx.x * 16 + i, at = std::min(row, p.rows - 1);
    const int c0 = blockIdx.y * p.cols, c1 = min(c0 + p.cols, p.n_out);
    const float* x = p.x + at * p.ld_x;
    const float* base = p.base ? p.base + at * p.ld_base : nullptr;
    float* y = p.y + at * p.ld_y;
    RowIds ids(p.ids, row, p.rows, p.n);
    while (ids.left) {
        const int cur = ids.next();
        const bool mine = ids.id == cur;
        f32x4 u[RT] = {};
        if (cur >= 0) {
            contract_rows<T, RT, VEC, WAVES>(u, matrix_at<T>(p.a, cur * p.a_stride), p.rank, x, p.n_in, wave, lane);
            sum_waves<RT, WAVES>(u, p.scale ? p.scale[cur] : 1.f, p.rank, lds, wave, lane);
        } else if (p.base == p.y) {
            continue;  // in place: rows without an adapter stay
        }
        const void* b = cur >= 0 ? matrix_at<T>(p.b, cur * p.b_stride) : nullptr;
        for (int m0 = c0 + 16 * wave; m0 < c1; m0 += 16 * WAVES) {
            const int m = m0 + i, col = m0 + 4 * g;
            f32x4 d = {};
            Quad<TSX_F32> old = {};
            if (base && mine) old = load_quad<TSX_F32, VEC>(base, col, c1 - col);
            if (cur >= 0) {
                Quad<T> w[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const int r = 16 * rt + 4 * g;
                    w[rt] = load_quad<T, VEC>(b, (int64_t) m * p.rank + r, m < c1 ? p.rank - r : 0);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d = mfma(w[rt].at(e), u[rt][e], d);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c] += old.at(c);
            if (mine) store_quad<VEC>(y, col, c1 - col, d);
        }
    }
}

// The backward's row half: s u and v of every row with an adapter (into u and v, [rows][16 RT], ranks past the last as 0), and
// dx.
template <int T, int RT, bool VEC>
__global__ void __launch_bounds__(64 * waves_for<RT>()) adapters_back_rows_kernel(AdArgs p) {
    constexpr int WAVES = waves_for<RT>();
    __shared__ f32x4 lds[(WAVES + 1) * RT * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int64_t row = (int64_t) blockIdx.x * 16 + i, at = std::min(row, p.rows - 1);
    const int c0 = blockIdx.y * p.cols, c1 = min(c0 + p.cols, p.n_in);
    const float* dbase = p.dbase ? p.dbase + at * p.ld_dbase : nullptr;
    float* dx = p.dx ? p.dx + at * p.ld_dx : nullptr;
    RowIds ids(p.ids, row, p.rows, p.n);
    while (ids.left) {
        const int cur = ids.next();
        const bool mine = ids.id == cur;
        f32x4 v[RT] = {};
        if (cur >= 0) {
            const float s = p.scale ? p.scale[cur] : 1.f;
            if (p.u && blockIdx.y == 0) {
                f32x4 u[RT] = {};
                contract_rows<T, RT, VEC, WAVES>(u, matrix_at<T>(p.a, cur * p.a_stride), p.rank, p.x + at * p.ld_x, p.n_in,
                                                 wave, lane);
                sum_waves<RT, WAVES>(u, s, p.rank, lds, wave, lane);
                if (wave == 0 && mine) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) *(f32x4*) (p.u + row * (16 * RT) + 16 * rt + 4 * g) = u[rt];
                }
            }
            contract_cols<T, RT, VEC, WAVES>(v, matrix_at<T>(p.b, cur * p.b_stride), p.rank, p.dy + at * p.ld_dy, p.n_out,
                                             wave, lane);
            sum_waves<RT, WAVES>(v, s, p.rank, lds, wave, lane);
            if (p.v && blockIdx.y == 0 && wave == 0 && mine) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) *(f32x4*) (p.v + row * (16 * RT) + 16 * rt + 4 * g) = v[rt];
            }
        }
        if (!dx || (cur < 0 && p.dbase == p.dx)) continue;
        const void* a = cur >= 0 ? matrix_at<T>(p.a, cur * p.a_stride) : nullptr;
        // 64 columns: lane i's four columns 4 i .. of a rank give four products, whose accumulators hold columns
        // 16 g + 4 r + q: four in a row for every r
        for (int n0 = c0 + 64 * wave; n0 < c1; n0 += 64 * WAVES) {
            f32x4 d[4] = {};
            if (cur >= 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    Quad<T> w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 16 * rt + 4 * g + e, n = n0 + 4 * i;
                        w[e] = load_quad<T, VEC>(a, (int64_t) r * p.n_in + n, r < p.rank ? c1 - n : 0);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int q = 0; q < 4; ++q) d[q] = mfma(w[e].at(q), v[rt][e], d[q]);
                }
            }
            if (!mine) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int col = n0 + 16 * g + 4 * r;
                Quad<TSX_F32> old = {};
                if (dbase) old = load_quad<TSX_F32, VEC>(dbase, col, c1 - col);
                const f32x4 o = {d[0][r] + old.at(0), d[1][r] + old.at(1), d[2][r] + old.at(2), d[3][r] + old.at(3)};
                store_quad<VEC>(dx, col, c1 - col, o);
            }
        }
    }
}

// The backward's weight half: a block takes 64 columns of one adapter's dA (x: columns of x, coefficients v) or dB (columns
// of dy, coefficients s u) and 16 RT ranks of it, its waves sharing the adapter's rows (`order`, bounds[a] .. bounds[a + 1]),
// four rows a step: lane l = 16 g + i holds coefficient i of row g and columns 4 i .. 4 i + 3 of it, four products.  The sums
// of the waves meet in LDS, in wave order.  An adapter without rows gets zeros.
struct AdSumArgs {
    const float* x;
    const float* dy;
    const float* u;
    const float* v;
    const int32_t* bounds;
    const int32_t* order;
    float* da;
    float* db;
    int64_t ld_x, ld_dy;
    int n_in, n_out, rank, ldu, tiles_a, tiles_b;
};
template <int RT, bool VEC>
__global__ void __launch_bounds__(512) adapters_back_sum_kernel(AdSumArgs p) {
    constexpr int WAVES = 8;
    __shared__ f32x4 lds[WAVES * RT * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int ad = blockIdx.y, r0 = blockIdx.z * 16 * RT;
    const bool is_a = (int) blockIdx.x < p.tiles_a;
    const int n0 = 64 * (is_a ? blockIdx.x : blockIdx.x - p.tiles_a), K = is_a ? p.n_in : p.n_out, n = n0 + 4 * i;
    const float* src = is_a ? p.x : p.dy;
    const int64_t ld = is_a ? p.ld_x : p.ld_dy;
    const float* coef = (is_a ? p.v : p.u) + r0;
    const int lo = p.bounds[ad], hi = p.bounds[ad + 1];
    f32x4 acc[4][RT] = {};
    constexpr int UN = RT <= 2 ? 4 : 2;
    for (int j0 = lo + 4 * UN * wave; j0 < hi; j0 += 4 * UN * WAVES) {
        Quad<TSX_F32> xv[UN];
        float cv[UN][RT];
#pragma unroll
        for (int s = 0; s < UN; ++s) {
            const int j = j0 + 4 * s + g;
            const bool in = j < hi;
            const int64_t row = in ? p.order[j] : 0;
            xv[s] = load_quad<TSX_F32, VEC>(src + row * ld, n, in ? K - n : 0);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) cv[s][rt] = in ? coef[row * p.ldu + 16 * rt + i] : 0.f;
        }
#pragma unroll
        for (int s = 0; s < UN; ++s)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[q][rt] = is_a ? mfma(cv[s][rt], xv[s].at(q), acc[q][rt]) : mfma(xv[s].at(q), cv[s][rt], acc[q][rt]);
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
    k.rows = rows, k.n = p->n, k.rank = p->rank, k.n_in = p->n_in, k.n_out = p->n_out;
}

template <int T, int RT, bool VEC> void launch_forward(const AdArgs& k, dim3 grid, hipStream_t st) {
    adapters_kernel<T, RT, VEC><<<grid, 64 * waves_for<RT>(), 0, st>>>(k);
}
template <int T, int RT, bool VEC> void launch_back_rows(const AdArgs& k, dim3 grid, hipStream_t st) {
    adapters_back_rows_kernel<T, RT, VEC><<<grid, 64 * waves_for<RT>(), 0, st>>>(k);
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

// the backward's scratch: the rows sorted by adapter, then u and v
struct BackScratch {
    size_t bounds, order, tok, rinv, most, u, v, bytes;
    int ldu;
};
BackScratch back_scratch(const tsx_adapters* p, int64_t rows) {
    BackScratch s;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t o = at;
        at += (n + 255) / 256 * 256;
        return o;
    };
    const int rt = p->rank <= 16 ? 1 : p->rank <= 32 ? 2 : p->rank <= 64 ? 4 : p->rank <= 128 ? 8 : 16;
    s.ldu = 16 * rt;
    s.bounds = take(((size_t) p->n + 1) * 4);
    s.order = take((size_t) rows * 4);
    s.tok = take((size_t) rows * 4);
    s.rinv = take((size_t) rows * 4);
    s.most = take(4);
    s.u = take((size_t) rows * s.ldu * 4);
    s.v = take((size_t) rows * s.ldu * 4);
    s.bytes = at;
    return s;
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
    const int64_t tiles = (rows + 15) / 16;
    const bool vec = matrix_quads(p) && quads(x, ld_x, 4) && quads(y, ld_y, 4) && (!base || quads(base, ld_base, 4));
    k.cols = columns_per_block(tiles, p->n_out, 128);
    launch<false>(p->type, vec, k, dim3((unsigned) tiles, (unsigned) ((p->n_out + k.cols - 1) / k.cols)), (hipStream_t) stream);
    return launch_status("tsx_moe_adapters");
}

TSX_API size_t tsx_moe_adapters_scratch_bytes(const tsx_adapters* p, int64_t rows) {
    if (!p || p->n < 0 || rows < 0 || p->rank < 1 || p->rank > kMaxRank) return 0;
    return back_scratch(p, rows).bytes;
}

TSX_API int tsx_moe_adapters_backward(const tsx_adapters* p, const int32_t* ids, const float* x, int64_t ld_x, const float* dy,
                                      int64_t ld_dy, const float* dbase, int64_t ld_dbase, float* dx, int64_t ld_dx,
                                      float* da, float* db, int64_t rows, void* scratch, void* stream) {
    if (const int rc = check_adapters("tsx_moe_adapters_backward", p, rows)) return rc;
    if (p->n > kMaxExperts) {
        set_error("tsx_moe_adapters_backward: %d adapters (at most 512)", p->n);
        return TSX_ERR_UNSUPPORTED;
    }
    TSX_REQUIRE(scratch && (rows == 0 || (ids && x && dy)), "tsx_moe_adapters_backward: ids, x, dy, scratch");
    TSX_REQUIRE(aligned(ids, 4) && aligned(x, 4) && aligned(dy, 4) && aligned(dbase, 4) && aligned(dx, 4) && aligned(da, 4) &&
                    aligned(db, 4) && aligned(scratch, 256),
                "tsx_moe_adapters_backward: buffers 4-byte aligned, scratch 256-byte aligned");
    TSX_REQUIRE(rows == 0 || (ld_x >= p->n_in && ld_dy >= p->n_out && (!dx || ld_dx >= p->n_in) &&
                              (!dbase || ld_dbase >= p->n_in) && (!dbase || dbase != dx || ld_dbase == ld_dx)),
                "tsx_moe_adapters_backward: rows as long as their columns; in place with one ld");
    const hipStream_t st = (hipStream_t) stream;
    const BackScratch s = back_scratch(p, rows);
    char* w = (char*) scratch;
    const bool sums = p->n > 0 && (da || db);
    if (sums) {  // (no rows: the sort reads no id)
        const int rc = tsx_moe_route_sort(rows ? ids : (const int32_t*) w, (int) rows, 1, p->n, (int32_t*) (w + s.bounds),
                                          (int32_t*) (w + s.order), (int32_t*) (w + s.tok), (int32_t*) (w + s.rinv),
                                          (int32_t*) (w + s.most), stream);
        if (rc) return rc;
    }
    if (rows) {
        AdArgs k{};
        fill(k, p, ids, rows);
        k.x = x, k.ld_x = ld_x, k.dy = dy, k.ld_dy = ld_dy, k.dbase = dbase, k.ld_dbase = ld_dbase, k.dx = dx, k.ld_dx = ld_dx;
        k.u = sums && db ? (float*) (w + s.u) : nullptr;
        k.v = sums && da ? (float*) (w + s.v) : nullptr;
        const bool vec = matrix_quads(p) && quads(x, ld_x, 4) && quads(dy, ld_dy, 4) && (!dx || quads(dx, ld_dx, 4)) &&
                         (!dbase || quads(dbase, ld_dbase, 4));
        const int64_t tiles = (rows + 15) / 16;
        k.cols = dx ? columns_per_block(tiles, p->n_in, 512) : p->n_in;
        launch<true>(p->type, vec, k, dim3((unsigned) tiles, (unsigned) ((p->n_in + k.cols - 1) / k.cols)), st);
        if (const int rc = launch_status("tsx_moe_adapters_backward")) return rc;
    }
    if (sums) {
        AdSumArgs k{};
        k.x = x, k.ld_x = ld_x, k.dy = dy, k.ld_dy = ld_dy, k.u = (const float*) (w + s.u), k.v = (const float*) (w + s.v);
        k.bounds = (const int32_t*) (w + s.bounds), k.order = (const int32_t*) (w + s.order), k.da = da, k.db = db;
        k.n_in = p->n_in, k.n_out = p->n_out, k.rank = p->rank, k.ldu = s.ldu;
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
