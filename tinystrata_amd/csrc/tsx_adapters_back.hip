// tsx_adapters_back.hip - the gradients of the low-rank adapters (tsx_adapters.hip) on gfx950: tsx_moe_adapters_backward.
//
//   u = A x,  v = s B^T dy:   dx = dbase + A^T v,  dA[a] = sum over a's rows of v x^T,  dB[a] = sum of dy (s u)^T.
//
// Two launches: the rows' (u, v and dx, a tile of 16 rows of one adapter a block, tsx_adapters.hpp) and the weights' (a piece of
// dA or dB a block).  Every product runs on v_mfma_f32_16x16x4_f32, whose operands are fp32: nothing is rounded below 32 bits.
// The accumulator of v holds ranks 4 g .. 4 g + 3 of row l % 16 in lane l = 16 g + .., and an operand holds row l % 16, k = g,
// so accumulator register e is the operand of the step over ranks 4 g + e, with no exchange between lanes.
#include "tsx_adapters.hpp"

namespace tsx {
namespace {

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

// acc[rt] += the tiles of 16 ranks of w times x^T over the chunks of 32 columns that are this wave's: lane l = 16 g + i holds
// rank 16 rt + i of w, row i of x, and columns 8 g .. 8 g + 7 of the chunk (any order of the columns will do as long as both
// operands have the same).  COLS: w is row-major [K][rank], a lane's values a column apart and 16 lanes' together; else it is
// row-major [rank][K].  The blocks start `turn` chunks apart: rows are a power of two apart as often as not, and blocks that
// walk them in step would meet in the same memory channels.  Whole chunks are loaded without a condition, UN at a time (a load
// that may not be made is one at a time, with a wait behind each: dx of 4096 rows 512 -> 2048, rank 16, bf16 took 31.8 us for
// 19.8 so); a rank past the last repeats it, which sum_waves leaves out.
template <int T, int RT, bool VEC, int WAVES, bool COLS>
__device__ __forceinline__ void contract(f32x4 (&acc)[RT], const void* w, int rank, const float* x, int K, int wave, int lane,
                                         int turn) {
    constexpr int UN = RT == 1 ? 4 : RT <= 4 ? 2 : 1;
    const int i = lane & 15, g = lane >> 4, chunks = (K + 31) / 32, whole = VEC ? K / 32 : 0;
    int c0 = UN * wave;
    if constexpr (VEC) {
        turn = whole ? turn % whole : 0;
        for (; c0 + UN <= whole; c0 += UN * WAVES) {
            Oct<TSX_F32> xv[UN];
            Oct<T> wv[COLS ? 1 : UN][RT];
            float wc[COLS ? UN : 1][RT][8];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                int c = c0 + u + turn;
                c -= c >= whole ? whole : 0;
                const int k = 32 * c + 8 * g;
                xv[u] = load_oct<TSX_F32, true>(x, k, 8);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const int r = min(16 * rt + i, rank - 1);
                    if constexpr (COLS) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) wc[u][rt][e] = value_at<T>(w, (int64_t) (k + e) * rank + r);
                    } else {
                        wv[u][rt] = load_oct<T, true>(w, (int64_t) r * K + k, 8);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        acc[rt] = mfma(COLS ? wc[COLS ? u : 0][rt][e] : wv[COLS ? 0 : u][rt].at(e), xv[u].at(e), acc[rt]);
        }
    }
    for (; c0 < chunks; c0 += UN * WAVES) {  // the last columns; all where quads are not aligned
#pragma unroll 1
        for (int c1 = c0; c1 < min(c0 + UN, chunks); ++c1) {
            const int c = c1 < whole ? (c1 + turn) % whole : c1, k = 32 * c + 8 * g;
            const Oct<TSX_F32> xv = load_oct<TSX_F32, VEC>(x, k, K - k);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int r = 16 * rt + i;
                Oct<T> wv;
                if constexpr (!COLS) wv = load_oct<T, VEC>(w, (int64_t) r * K + k, r < rank ? K - k : 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float f;
                    if constexpr (COLS) f = r < rank && k + e < K ? value_at<T>(w, (int64_t) (k + e) * rank + r) : 0.f;
                    else f = wv.at(e);
                    acc[rt] = mfma(f, xv.at(e), acc[rt]);
                }
            }
        }
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

template <int RT> constexpr int waves_for() { return RT <= 4 ? 8 : 4; }

// The backward's row half: s u and v of every row with an adapter (into u and v, [rows][16 RT], ranks past the last as 0), and
// dx.  u shares no operand with the rest: the last blocks of a tile form it beside the others (300 rows 2048 -> 512, rank 32,
// fp32: the whole backward 22.6 us, 27.0 one after the other).
template <int T, int RT, bool VEC>
__global__ void __launch_bounds__(64 * waves_for<RT>()) adapters_back_rows_kernel(AdArgs p) {
    constexpr int WAVES = waves_for<RT>();
    extern __shared__ int s_count[];
    __shared__ f32x4 lds[(WAVES + 1) * RT * 64];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    if (!find_tile<WAVES>(t, p.ids, p.rows, p.n, p.regroup, p.extra, 0, s_count, threadIdx.x)) return;
    const bool mine = t.row >= 0;
    const int64_t first = __shfl(t.row, 0, 64);  // (every lane takes part)
    const int64_t at = mine ? t.row : first;
    const int c0 = blockIdx.y * p.cols, c1 = min(c0 + p.cols, p.n_in);
    f32x4 v[RT] = {};
    if (t.cur >= 0) {
        const float s = p.scale ? p.scale[t.cur] : 1.f;
        if (p.u && blockIdx.y == gridDim.y - 1) {
            f32x4 u[RT] = {};
            contract<T, RT, VEC, WAVES, false>(u, matrix_at<T>(p.a, t.cur * p.a_stride), p.rank, p.x + at * p.ld_x, p.n_in, wave,
                                             lane, (int) blockIdx.x * 5);
            sum_waves<RT, WAVES>(u, s, p.rank, lds, wave, lane);
            if (wave == 0 && mine) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) *(f32x4*) (p.u + t.row * (16 * RT) + 16 * rt + 4 * g) = u[rt];
            }
            return;
        }
        contract<T, RT, VEC, WAVES, true>(v, matrix_at<T>(p.b, t.cur * p.b_stride), p.rank, p.dy + at * p.ld_dy, p.n_out, wave,
                                         lane, (int) blockIdx.x * 5);
        sum_waves<RT, WAVES>(v, s, p.rank, lds, wave, lane);
        if (p.v && blockIdx.y == 0 && wave == 0 && mine) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) *(f32x4*) (p.v + t.row * (16 * RT) + 16 * rt + 4 * g) = v[rt];
        }
    }
    if (!p.dx || (t.cur < 0 && p.dbase == p.dx) || c0 >= p.n_in) return;
    const float* dbase = p.dbase ? p.dbase + at * p.ld_dbase : nullptr;
    float* dx = p.dx + at * p.ld_dx;
    const void* a = t.cur >= 0 ? matrix_at<T>(p.a, t.cur * p.a_stride) : nullptr;
    // 64 columns: lane i's four columns 4 i .. of a rank give four products, whose accumulators hold columns 16 g + 4 r + q:
    // four in a row for every r
    for (int n0 = c0 + 64 * wave; n0 < c1; n0 += 64 * WAVES) {
        f32x4 d[4] = {}, old[4] = {};
        const bool whole = VEC && n0 + 64 <= c1;  // loads without a condition, as above (a row that is not one reads the first)
        if (dbase) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int col = n0 + 16 * g + 4 * r;
                old[r] = whole ? load_quad<VEC>(dbase, col, 4) : load_quad<VEC>(dbase, col, c1 - col);
            }
        }
        if (t.cur >= 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                f32x4 w[4];
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 16 * rt + 4 * g + e;
                        w[e] = load_four<T, VEC>(a, (int64_t) min(r, p.rank - 1) * p.n_in + n0 + 4 * i, 4);
                        if (r >= p.rank) w[e] = f32x4{0.f, 0.f, 0.f, 0.f};  // (v is 0 there, but the last rank may be infinite)
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 16 * rt + 4 * g + e, n = n0 + 4 * i;
                        w[e] = load_four<T, VEC>(a, (int64_t) r * p.n_in + n, r < p.rank ? c1 - n : 0);
                    }
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

constexpr int kSumBlocks = 512, kSumRows = 256;  // see sum_parts

// The backward's weight half: a block takes 64 columns of one adapter's dA (x: columns of x, coefficients v) or dB (columns
// of dy, coefficients s u) and 16 RT ranks of it.  It lists the adapter's rows itself, kChunk ids at a time, and its waves
// share them, four rows a step: lane l = 16 g + i holds RT coefficients of row g and columns 4 i .. 4 i + 3 of it, four
// products a tile.  The sums of the waves meet in LDS, in wave order.  An adapter without rows gets zeros.
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
    int parts;       // blocks that share an adapter's rows
    int64_t apart;   // values from one block's sums to the next one's
    bool wide_a, wide_b;  // four columns of dA, RT ranks of dB are one store
};
template <int RT, bool VEC>
__global__ void __launch_bounds__(512) adapters_back_sum_kernel(AdSumArgs p) {
    constexpr int WAVES = 8, R = kChunk / 512;
    __shared__ f32x4 lds[WAVES * 4 * RT * 64];
    __shared__ int s_seg[64];
    int* s_row = (int*) lds;  // kChunk rows; the sums come after them
    static_assert(sizeof(lds) >= kChunk * sizeof(int), "");
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ad = blockIdx.y, part = blockIdx.z % p.parts, r0 = blockIdx.z / p.parts * 16 * RT;
    const bool is_a = (int) blockIdx.x < p.tiles_a;
    const int n0 = 64 * (is_a ? blockIdx.x : blockIdx.x - p.tiles_a), K = is_a ? p.n_in : p.n_out, n = n0 + 4 * i;
    const float* src = is_a ? p.x : p.dy;
    const int64_t ld = is_a ? p.ld_x : p.ld_dy;
    const float* coef = (is_a ? p.v : p.u) + r0 + RT * i;  // tile rt: ranks RT i + rt
    f32x4 acc[4][RT] = {};
    // steps in flight (4096 rows 512 -> 2048, rank 16, 8 adapters: the whole backward 34.7 us, with eight 36.9, with sixteen 40.7)
    constexpr int UN = 4;
    using Coef = float __attribute__((ext_vector_type(RT)));
    for (int64_t base = 0; base < p.rows; base += kChunk) {
        int id[R];
        uint64_t hit[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t j = base + r * 512 + threadIdx.x;
            id[r] = p.ids[min(j, p.rows - 1)];
            id[r] = j < p.rows ? id[r] : -1;
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
        for (int j0 = 4 * UN * (wave + WAVES * part); j0 < hi; j0 += 4 * UN * WAVES * p.parts) {
            f32x4 xv[UN];
            Coef cv[UN];
#pragma unroll
            for (int s = 0; s < UN; ++s) {
                const int j = j0 + 4 * s + g;
                const int64_t row = base + s_row[min(j, hi - 1)];  // (past the last: it again, without a condition, and 0 below)
                xv[s] = VEC ? load_quad<VEC>(src + row * ld, min(n, K - 4), 4) : load_quad<VEC>(src + row * ld, n, K - n);
                cv[s] = *(const Coef*) (coef + row * p.ldu);
            }
#pragma unroll
            for (int s = 0; s < UN; ++s) {
                const bool in = j0 + 4 * s + g < hi;
#pragma unroll
                for (int c = 0; c < 4; ++c) xv[s][c] = in ? xv[s][c] : 0.f;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) cv[s][rt] = in ? cv[s][rt] : 0.f;
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
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) lds[((wave * 4 + q) * RT + rt) * 64 + lane] = acc[q][rt];
    __syncthreads();
    auto total = [&](int q, int rt, int value) {  // value: 4 lane + r of the accumulators
        const float* v = (const float*) (lds + (q * RT + rt) * 64) + value;
        float t = *v;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) t += v[w * 4 * RT * 256];
        return t;
    };
    const int si = (threadIdx.x >> 2) & 15, sg = (threadIdx.x >> 6) & 3, r = threadIdx.x & 3;  // a value of an accumulator
    if (is_a) {  // rank RT (4 g + r) + rt of columns 4 i + q
        for (int rt = threadIdx.x >> 8; rt < RT; rt += 2) {
            const int k = r0 + RT * (4 * sg + r) + rt, c = n0 + 4 * si;
            f32x4 t;
#pragma unroll
            for (int q = 0; q < 4; ++q) t[q] = total(q, rt, threadIdx.x & 255);
            if (k < p.rank) {
                float* out = p.da + part * p.apart + ((int64_t) ad * p.rank + k) * K;
                if (p.wide_a) store_quad<true>(out, c, K - c, t);
                else store_quad<false>(out, c, K - c, t);
            }
        }
    } else {  // ranks RT i + rt of column 4 (4 g + r) + q
        for (int q = threadIdx.x >> 8; q < 4; q += 2) {
            const int k = r0 + RT * si, c = n0 + 4 * (4 * sg + r) + q;
            Coef t;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) t[rt] = total(q, rt, threadIdx.x & 255);
            if (c < K) {
                float* out = p.db + part * p.apart + ((int64_t) ad * K + c) * p.rank + k;
                if (p.wide_b) {
                    if (k < p.rank) *(Coef*) out = t;
                } else {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (k + rt < p.rank) out[rt] = t[rt];
                }
            }
        }
    }
}

// the blocks that shared an adapter's rows, added up in their order
__global__ void __launch_bounds__(256) adapters_back_join_kernel(const float* sums, int parts, int64_t apart, float* da,
                                                                 int64_t na, float* db) {
    const int64_t e = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (e >= apart) return;
    float t = sums[e];
    for (int q = 1; q < parts; ++q) t += sums[q * apart + e];
    (e < na ? da[e] : db[e - na]) = t;
}

template <int T, int RT> void launch_vec(bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    const size_t count = k.extra ? (size_t) (k.n + 1) * 4 : 0;
    if (vec) adapters_back_rows_kernel<T, RT, true><<<grid, 64 * waves_for<RT>(), count, st>>>(k);
    else adapters_back_rows_kernel<T, RT, false><<<grid, 64 * waves_for<RT>(), count, st>>>(k);
}
template <int T> void launch_rank(bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    if (k.rank <= 16) launch_vec<T, 1>(vec, k, grid, st);
    else if (k.rank <= 32) launch_vec<T, 2>(vec, k, grid, st);
    else if (k.rank <= 64) launch_vec<T, 4>(vec, k, grid, st);
    else if (k.rank <= 128) launch_vec<T, 8>(vec, k, grid, st);
    else launch_vec<T, 16>(vec, k, grid, st);
}
template <int RT, bool VEC> void launch_sum(const AdSumArgs& k, dim3 grid, hipStream_t st) {
    adapters_back_sum_kernel<RT, VEC><<<grid, 512, 0, st>>>(k);
}

// tiles of 16 ranks that a row's u and v are stored in, and that a block of the sums takes of them
inline int stored_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : rank <= 128 ? 8 : 16; }
inline int sum_tiles(int rank) { return std::min(stored_tiles(rank), 4); }
// the backward's scratch: u and v, then the sums of blocks that share rows
inline size_t back_values(const tsx_adapters* p, int64_t rows) {
    return ((size_t) rows * 16 * stored_tiles(p->rank) * 4 + 255) / 256 * 256 / 4;
}
// Blocks that share an adapter's rows: few adapters make few blocks, each with many rows to walk.  Parts
// cost a third launch (4 us) and a pass over their sums: one adapter of 4096 rows 512 -> 2048, rank 16, takes 33.7 us for 56.6
// whole, of 1024 rows 21.5 for 24.0; two of 256 rows each 22.3 for 21.5, so a part keeps kSumRows rows; blocks past two a CU
// gain nothing (1024 of them: 8 adapters of 512 rows 45.0 us for 41.0 whole)
inline int sum_parts(const tsx_adapters* p, int64_t rows) {
    if (p->n < 1 || p->n_in < 1 || p->n_out < 1) return 1;
    const int rt = sum_tiles(p->rank);
    const int64_t tiles = ((int64_t) p->n_in + 63) / 64 + ((int64_t) p->n_out + 63) / 64;
    const int64_t blocks = tiles * p->n * ((p->rank + 16 * rt - 1) / (16 * rt));
    return (int) std::max<int64_t>(1, std::min<int64_t>({kSumBlocks / blocks, rows / p->n / kSumRows, 16}));
}
inline int64_t sum_values(const tsx_adapters* p) { return (int64_t) p->n * p->rank * ((int64_t) p->n_in + p->n_out); }

}  // namespace
}  // namespace tsx

using namespace tsx;

extern "C" {

TSX_API size_t tsx_moe_adapters_scratch_bytes(const tsx_adapters* p, int64_t rows) {
    if (!p || p->n < 0 || rows < 0 || p->rank < 1 || p->rank > kMaxRank) return 0;
    const int parts = sum_parts(p, rows);
    return 2 * back_values(p, rows) * 4 + (parts > 1 ? (size_t) parts * sum_values(p) * 4 : 0);
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
    TSX_REQUIRE(!dx || (dx != x && dx != dy),
                "tsx_moe_adapters_backward: x and dy are read by other blocks than those that write dx");
    const hipStream_t st = (hipStream_t) stream;
    float* u = (float*) scratch;
    float* v = u + back_values(p, rows);
    const bool sums = p->n > 0 && (da || db);
    if (rows) {
        AdArgs k{};
        const Tiles t(rows, p->n, INT32_MAX);
        TSX_REQUIRE(grid_fits(t.blocks(), 512), "tsx_moe_adapters_backward: too many rows");
        fill(k, p, ids, rows, t);
        k.x = x, k.ld_x = ld_x, k.dy = dy, k.ld_dy = ld_dy, k.dbase = dbase, k.ld_dbase = ld_dbase, k.dx = dx, k.ld_dx = ld_dx;
        k.u = sums && db ? u : nullptr;
        k.v = sums && da ? v : nullptr;
        const bool vec = matrix_quads(p) && quads(x, ld_x, 4) && quads(dy, ld_dy, 4) && (!dx || quads(dx, ld_dx, 4)) &&
                         (!dbase || quads(dbase, ld_dbase, 4));
        k.cols = dx ? columns_per_block((rows + 15) / 16, p->n_in, 512) : p->n_in;
        const dim3 grid((unsigned) t.blocks(), (unsigned) ((p->n_in + k.cols - 1) / k.cols + (k.u ? 1 : 0)));
        if (p->type == TSX_F32) launch_rank<TSX_F32>(vec, k, grid, st);
        else if (p->type == TSX_F16) launch_rank<TSX_F16>(vec, k, grid, st);
        else launch_rank<TSX_BF16>(vec, k, grid, st);
        if (const int rc = launch_status("tsx_moe_adapters_backward")) return rc;
    }
    if (sums) {
        AdSumArgs k{};
        k.x = x, k.ld_x = ld_x, k.dy = dy, k.ld_dy = ld_dy, k.u = u, k.v = v, k.ids = ids, k.rows = rows;
        k.da = da, k.db = db, k.n_in = p->n_in, k.n_out = p->n_out, k.rank = p->rank;
        k.ldu = 16 * stored_tiles(p->rank);
        k.tiles_a = da ? (p->n_in + 63) / 64 : 0, k.tiles_b = db ? (p->n_out + 63) / 64 : 0;
        const bool vec = quads(x, ld_x, p->n_in) && quads(dy, ld_dy, p->n_out);
        const int rt = sum_tiles(p->rank);
        const int64_t na = da ? (int64_t) p->n * p->rank * p->n_in : 0, nb = db ? (int64_t) p->n * p->rank * p->n_out : 0;
        float* sums = v + back_values(p, rows);
        k.parts = sum_parts(p, rows), k.apart = na + nb;
        if (k.parts > 1) k.da = sums, k.db = sums + na;
        k.wide_a = p->n_in % 4 == 0 && k.apart % 4 == 0 && aligned(k.da, 16);
        k.wide_b = p->rank % rt == 0 && k.apart % rt == 0 && aligned(k.db, 4 * rt);
        const dim3 grid((unsigned) (k.tiles_a + k.tiles_b), (unsigned) p->n,
                        (unsigned) ((p->rank + 16 * rt - 1) / (16 * rt) * k.parts));
        if (rt == 1) vec ? launch_sum<1, true>(k, grid, st) : launch_sum<1, false>(k, grid, st);
        else if (rt == 2) vec ? launch_sum<2, true>(k, grid, st) : launch_sum<2, false>(k, grid, st);
        else vec ? launch_sum<4, true>(k, grid, st) : launch_sum<4, false>(k, grid, st);
        if (k.parts > 1)
            adapters_back_join_kernel<<<(unsigned) ((k.apart + 255) / 256), 256, 0, st>>>(sums, k.parts, k.apart, da, na, db);
        return launch_status("tsx_moe_adapters_backward");
    }
    return TSX_OK;
}

}  // extern "C"
