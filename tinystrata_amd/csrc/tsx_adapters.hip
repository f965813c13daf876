// tsx_adapters.hip - low-rank adapters of many requests beside a projection on gfx950: tsx_moe_adapters (its gradients:
// tsx_adapters_back.hip).
//
//   y[j] = base[j] + s[a] B[a] u,  u = A[a] x[j],  a = ids[j]
//
// x, y and the gradients are fp32 as everywhere in this library, the matrices fp32, fp16 or bf16, and nothing is rounded below
// 32 bits: fp32 and fp16 matrices are multiplied by v_mfma_f32_16x16x4_f32, bf16 ones by v_mfma_f32_16x16x32_bf16 with the
// other operand in three bf16 parts.  The rank is small, so the rows of x and y are most of the bytes and each is moved once: a
// block takes 16 rows, forms their u with its waves sharing the contraction (one sum in LDS), and expands it at once.
//
// A matrix instruction has a row on every lane of sixteen, so operands loaded from memory as it wants them would name 64
// places a load: they took a block's share of the cache from 64 to 16 bytes a clock.  Every operand is therefore loaded in row
// order, into registers while the chunk before it is multiplied, and turned round in a piece of LDS that its wave alone uses.
//
// A block works for one adapter.  Sixteen rows that lie together and name one adapter (a prompt's rows, one token) are a tile
// as they stand; the others (a mixed batch, the edges between requests) are regrouped, kChunk rows at a time, by further
// blocks that each read the chunk's ids and work out which rows are theirs: no table is built ahead, so one launch does.
#include "tsx_adapters.hpp"

namespace tsx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int T> struct Elem { using type = uint16_t; };
template <> struct Elem<TSX_F32> { using type = float; };
template <int T> using elem_t = typename Elem<T>::type;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int T> struct FourOf { using type = u32x2; };
template <> struct FourOf<TSX_F32> { using type = f32x4; };
template <int T> using four_t = typename FourOf<T>::type;  // four consecutive values as stored
// 16 bytes at an address that is only 8-byte aligned: one load all the same
struct __attribute__((aligned(8))) Raw16 {
    float w[4];
};
__device__ __forceinline__ f32x4 load_raw(const void* p) {
    const Raw16 r = *(const Raw16*) p;
    return f32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
}
// eight consecutive values of type T as stored, and as floats
template <int T> struct Oct {
    uint32_t w[4];
    __device__ __forceinline__ float at(int c) const {
        const uint32_t h = c & 1 ? w[c / 2] >> 16 : w[c / 2] & 0xFFFFu;
        return T == TSX_F16 ? h2f((uint16_t) h) : __builtin_bit_cast(float, h << 16);
    }
};
template <> struct Oct<TSX_F32> {
    float w[8];
    __device__ __forceinline__ float at(int c) const { return w[c]; }
};
template <int T> __device__ __forceinline__ Oct<T> lds_oct(const elem_t<T>* p) {  // p on a multiple of 16 bytes
    Oct<T> o;
    const f32x4 lo = *(lds_ptr<const f32x4>) p;
    if constexpr (T == TSX_F32) {
        const f32x4 hi = *(lds_ptr<const f32x4>) (p + 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) o.w[c] = lo[c], o.w[4 + c] = hi[c];
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float f = lo[c];  // (the cast of a vector's element itself reads its first)
            o.w[c] = __builtin_bit_cast(uint32_t, f);
        }
    }
    return o;
}
// A wave's LDS accesses run in order; this keeps the compiler's in order too where lanes read what others wrote (and as other
// types: its scheduler may take a 16-bit store and a 16-byte load to be of different objects)
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    asm volatile("" ::: "memory");
}

// A float as three bf16 that add up to it: the leading eight bits of its significand, the next eight, the rest.  Products with
// a bf16 are then exact in the three terms, and v_mfma_f32_16x16x32_bf16 takes half the time of one fp32 instruction for eight
// times its columns.  (An infinity minus itself leaves a NaN in the lower terms: the callers look for that.)
struct Parts {
    uint32_t w[3][4];
};
__device__ __forceinline__ Parts split(const Oct<TSX_F32>& x) {
    Parts p;
#pragma unroll
    for (int c = 0; c < 8; c += 2) {
        uint32_t a = __builtin_bit_cast(uint32_t, x.w[c]), b = __builtin_bit_cast(uint32_t, x.w[c + 1]);
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            p.w[t][c / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);  // the upper halves, a's lower
            if (t == 2) break;
            const float ra = __builtin_bit_cast(float, a) - __builtin_bit_cast(float, a & 0xFFFF0000u);
            const float rb = __builtin_bit_cast(float, b) - __builtin_bit_cast(float, b & 0xFFFF0000u);
            a = __builtin_bit_cast(uint32_t, ra);
            b = __builtin_bit_cast(uint32_t, rb);
        }
    }
    return p;
}
__device__ __forceinline__ f32x4 mfma_bf16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// How a block is made for type T and 16 RT ranks: its waves, and the LDS values of a wave's own piece
template <int T, int RT> struct Shape {
    static constexpr int kSize = T == TSX_F32 ? 4 : 2;
    static constexpr int kWaves = RT <= 4 ? 8 : RT <= 8 ? 4 : 2;
    static constexpr int kStep = 32 * ((RT + 1) / 2);          // ranks, in whole steps of a product over ranks
    static constexpr int kXPitch = 36;                         // floats of a row of a chunk of 32 columns of x
    static constexpr int kRowPitch = 32 + 16 / kSize;          // values of a row of a chunk of A
    static constexpr int kOutPitch = kStep + 16 / kSize;       // values of a column's ranks of B for B u
    static constexpr int kX = 16 * kXPitch * 4;                // bytes of a chunk of x
    static constexpr int kUPitch = kStep + 4;                  // floats of a row of u
    static constexpr int max(int a, int b) { return a > b ? a : b; }
    static constexpr int kOwn = max(kX + 16 * RT * kRowPitch * kSize, 16 * kOutPitch * kSize);
    static constexpr int kSum = kWaves * RT * 1024;            // the waves' sums lie where their pieces did
    static constexpr int kLds = max(kWaves * kOwn, kSum);
};

// acc[rt] += wv[rt] times xv^T over 32 columns (lane l = 16 g + i holds row i of an operand and columns 8 g .. 8 g + 7; any order
// of the columns will do as long as both operands have the same).  SPLIT: the bf16 instructions on the three parts of x
template <int T, int RT, bool SPLIT>
__device__ __forceinline__ void multiply_chunk(f32x4 (&acc)[RT], const Oct<T> (&wv)[RT], const Oct<TSX_F32>& xv) {
    if constexpr (SPLIT) {
        const Parts q = split(xv);
#pragma unroll
        for (int t = 2; t >= 0; --t)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma_bf16(wv[rt].w, q.w[t], acc[rt]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma(wv[rt].at(e), xv.at(e), acc[rt]);
    }
}
// The wave's share of `count` pieces: pieces UN wave + u, UN waves apart.  put(r) takes a piece from registers to LDS and use(c)
// works on it there; the registers are loaded with the piece UN further on in between
template <int UN, typename Reg, typename Load, typename Put, typename Use>
__device__ __forceinline__ void in_turn(int count, int first, int step, const Load& load, const Put& put, const Use& use) {
    Reg r[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
        if (first + u < count) load(r[u], first + u);
#pragma unroll 1
    for (int c = first; c < count; c += step) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (c + u >= count) break;
            put(r[u]);
            if (c + step + u < count) load(r[u], c + step + u);
            wave_lds_order();
            use(c + u);
            wave_lds_order();
        }
    }
}

// The rows of a tile as lanes load and store them: lane l takes the 16-byte pieces l % 8 of rows l / 8 and l / 8 + 8 of a chunk
// of 32 floats
struct RowPair {
    const float* p[2];
    __device__ __forceinline__ RowPair(const float* base, int64_t row, int64_t ld, int lane) {
#pragma unroll
        for (int h = 0; h < 2; ++h) p[h] = base + __shfl(row, lane / 8 + 8 * h, 64) * ld + 4 * (lane % 8);
    }
    __device__ __forceinline__ void load(f32x4 (&v)[2], int col) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h] = *(const f32x4*) (p[h] + col);
    }
    __device__ __forceinline__ void load_some(f32x4 (&v)[2], int col, int left) const {  // `left`: values from this lane's on
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) v[h][c] = c < left ? p[h][col + c] : 0.f;
    }
    static __device__ __forceinline__ void put(float* lds, const f32x4 (&v)[2], int lane) {
#pragma unroll
        for (int h = 0; h < 2; ++h) *(lds_ptr<f32x4>) (lds + (lane / 8 + 8 * h) * 36 + 4 * (lane % 8)) = v[h];
    }
};

// acc[rt] += the [16 ranks][K] tiles of w (row-major [rank][K]) times x^T over the chunks of 32 columns that are this wave's
// (a rank past the last repeats it: sum_waves leaves it out).  The blocks start `turn` chunks apart: rows are a power of two
// apart as often as not, and blocks that walk them in step would meet in the same memory channels.  VEC: quads of values are
// aligned everywhere
template <int T, int RT, bool VEC, bool SPLIT>
__device__ __forceinline__ void contract_rows(f32x4 (&acc)[RT], const void* w, int rank, const RowPair& x, int K, char* lds,
                                              int wave, int lane, int turn) {
    using S = Shape<T, RT>;
    using E = elem_t<T>;
    constexpr int PIECE = 16 / S::kSize, PER = 32 / PIECE, LOADS = 16 * RT * PER / 64;  // 16-byte pieces a row, loads a chunk
    // chunks in flight besides the one that is multiplied: what four waves a SIMD leave registers for (rank 64, bf16, 4096 rows
    // 2048 -> 1024 in segments: 27.1 us, with two 31.9; rank 16: 22.8, with one 25.6, with four 23.2)
    constexpr int UN = RT == 1 ? 2 : 1;
    float* lx = (float*) lds;
    E* lw = (E*) (lds + S::kX);
    const int i = lane & 15, g = lane >> 4, col = lane % PER * PIECE;
    auto multiply = [&]() {
        const Oct<TSX_F32> xv = lds_oct<TSX_F32>(lx + 36 * i + 8 * g);
        Oct<T> wv[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) wv[rt] = lds_oct<T>(lw + (16 * rt + i) * S::kRowPitch + 8 * g);
        multiply_chunk<T, RT, SPLIT>(acc, wv, xv);
    };
    const int whole = VEC ? K / 32 : 0;
    if constexpr (VEC) {
        struct Reg {
            f32x4 x[2];
            f32x4 w[LOADS];
        };
        turn = whole ? turn % whole : 0;
        int64_t at[LOADS];
#pragma unroll
        for (int t = 0; t < LOADS; ++t) at[t] = (int64_t) min((lane + 64 * t) / PER, rank - 1) * K + col;
        in_turn<UN, Reg>(
            whole, UN * wave, UN * S::kWaves,
            [&](Reg& r, int c) {
                c += turn;
                c -= c >= whole ? whole : 0;
                x.load(r.x, 32 * c);
#pragma unroll
                for (int t = 0; t < LOADS; ++t) r.w[t] = load_raw((const E*) w + at[t] + 32 * c);
            },
            [&](const Reg& r) {
                RowPair::put(lx, r.x, lane);
#pragma unroll
                for (int t = 0; t < LOADS; ++t)
                    *(lds_ptr<f32x4>) (lw + (lane + 64 * t) / PER * S::kRowPitch + col) = r.w[t];
            },
            [&](int) { multiply(); });
    }
#pragma unroll 1
    for (int c = whole + wave; c < (K + 31) / 32; c += S::kWaves) {  // the last columns; all where quads are not aligned
        f32x4 v[2];
        x.load_some(v, 32 * c, K - 32 * c - 4 * (lane % 8));
        RowPair::put(lx, v, lane);
        const int k = 32 * c + lane % 32;
        for (int r = lane / 32; r < 16 * RT; r += 2)
            lw[r * S::kRowPitch + lane % 32] = k < K ? ((const E*) w)[(int64_t) min(r, rank - 1) * K + k] : E(0);
        wave_lds_order();
        multiply();
        wave_lds_order();
    }
}
// The waves' sums added up in wave order, times s, as a matrix of rows in LDS: u[row][rank], 0 past the last rank up to whole
// steps (what a clamped rank left there is not used).  Returns whether all are finite, the same in every wave
template <int T, int RT>
__device__ __forceinline__ bool sum_waves(const f32x4 (&acc)[RT], float s, int rank, f32x4* lds, float* u, int wave, int lane) {
    using S = Shape<T, RT>;
    __syncthreads();  // the pieces and u are used up
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) lds[(wave * RT + rt) * 64 + lane] = acc[rt];
    __syncthreads();
    bool finite = true;
    for (int q = wave * 64 + lane; q < S::kStep * 4; q += S::kWaves * 64) {  // ranks 16 (q / 64) + 4 (q / 16 % 4) .. of row q % 16
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
        const int r = 16 * (q >> 6) + 4 * ((q >> 4) & 3);
        if (r < rank) {
            t = lds[q];
#pragma unroll
            for (int w = 1; w < S::kWaves; ++w) t += lds[w * RT * 64 + q];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                t[c] = r + c < rank ? t[c] * s : 0.f;
                finite &= fabsf(t[c]) < INFINITY;
            }
        }
        *(f32x4*) (u + (q & 15) * S::kUPitch + r) = t;
    }
    return !__syncthreads_or(!finite);
}
// u of a tile: A x, summed and scaled.  Where the parts of x leave anything but numbers the fp32 instructions
// are asked, which keep infinities apart from NaN
template <int T, int RT, bool VEC>
__device__ __forceinline__ void tile_u(float* u, const void* w, float s, int rank, const RowPair& x, int K, char* lds,
                                       char* own, int wave, int lane, int turn) {
    constexpr bool kSplit = T == TSX_BF16;
    {
        f32x4 acc[RT] = {};
        contract_rows<T, RT, VEC, kSplit>(acc, w, rank, x, K, own, wave, lane, turn);
        if (sum_waves<T, RT>(acc, s, rank, (f32x4*) lds, u, wave, lane) || !kSplit) return;
    }
    if constexpr (kSplit) {
        f32x4 acc[RT] = {};
        contract_rows<T, RT, VEC, false>(acc, w, rank, x, K, own, wave, lane, turn);
        sum_waves<T, RT>(acc, s, rank, (f32x4*) lds, u, wave, lane);
    }
}
// u as an operand: row i, ranks 32 s + 8 g ..
template <int T, int RT> struct UOperand {
    static constexpr int kSteps = (RT + 1) / 2;
    Oct<TSX_F32> f[T == TSX_BF16 ? 1 : kSteps];
    Parts q[T == TSX_BF16 ? kSteps : 1];
    __device__ __forceinline__ UOperand(const float* u, int i, int g) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const Oct<TSX_F32> o = lds_oct<TSX_F32>(u + i * Shape<T, RT>::kUPitch + 32 * s + 8 * g);
            if constexpr (T == TSX_BF16) q[s] = split(o);
            else f[s] = o;
        }
    }
};
// the 16 x 16 product of u and columns whose ranks get(s) gives as operands: row 4 g + r of column i in d[r]
template <int T, int RT, typename Get>
__device__ __forceinline__ f32x4 expand(const UOperand<T, RT>& o, const float* u, int i, int g, const Get& get) {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
    auto in_fp32 = [&](const Oct<TSX_F32>& f, int s) {
        const Oct<T> w = get(s);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = mfma(f.at(e), w.at(e), d);
    };
    if constexpr (T == TSX_BF16) {
#pragma unroll
        for (int s = 0; s < o.kSteps; ++s) {
            const Oct<T> w = get(s);
#pragma unroll
            for (int t = 2; t >= 0; --t) d = mfma_bf16(o.q[s].w[t], w.w, d);
        }
        bool finite = true;
#pragma unroll
        for (int r = 0; r < 4; ++r) finite &= fabsf(d[r]) < INFINITY;
        if (__all(finite)) return d;
        d = f32x4{0.f, 0.f, 0.f, 0.f};  // as in tile_u
#pragma unroll
        for (int s = 0; s < o.kSteps; ++s) in_fp32(lds_oct<TSX_F32>(u + i * Shape<T, RT>::kUPitch + 32 * s + 8 * g), s);
    } else {
#pragma unroll
        for (int s = 0; s < o.kSteps; ++s) in_fp32(o.f[s], s);
    }
    return d;
}

// the rows 4 g + r of a tile as lanes store them, -1 for none
struct OutRows {
    int64_t row[4];
    __device__ __forceinline__ OutRows(int64_t of_lane, int g) {
#pragma unroll
        for (int r = 0; r < 4; ++r) row[r] = __shfl(of_lane, 4 * g + r, 64);
    }
    __device__ __forceinline__ void load(float (&v)[4], const float* p, int64_t ld, int col) const {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = row[r] >= 0 ? p[row[r] * ld + col] : 0.f;
    }
    __device__ __forceinline__ void store(float* p, int64_t ld, int col, const f32x4& d, const float (&v)[4]) const {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (row[r] >= 0) p[row[r] * ld + col] = d[r] + v[r];
    }
};

template <int T, int RT, bool VEC>
__global__ void __launch_bounds__((64 * Shape<T, RT>::kWaves))
__attribute__((amdgpu_waves_per_eu(RT <= (T == TSX_F32 ? 2 : 4) ? 4 : 1)))
adapters_kernel(AdArgs p) {
    using S = Shape<T, RT>;
    using E = elem_t<T>;
    constexpr int WAVES = S::kWaves;
    extern __shared__ int s_count[];
    __shared__ __attribute__((aligned(16))) char lds[S::kLds];
    __shared__ __attribute__((aligned(16))) float u[16 * S::kUPitch];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = blockIdx.y * p.cols, c1 = min(c0 + p.cols, p.n_out);
#pragma unroll 1
    for (int round = 0;; ++round) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // nothing that hangs on it is kept from one round for the next, in registers
        const int lane = tid & 63, i = lane & 15, g = lane >> 4;
        Tile t;
        if (!find_tile<WAVES>(t, p.ids, p.rows, p.n, p.regroup, p.extra, round, s_count, tid)) return;
        if (t.cur < 0 && p.base == p.y) continue;  // in place: rows without an adapter stay
        char* own = lds + wave * S::kOwn;
        E* lw = (E*) own;
        const bool some = t.cur >= 0;
        if (some) {
            const int64_t first = __shfl(t.row, 0, 64);  // (every lane takes part)
            const int64_t at = t.row >= 0 ? t.row : first;
            tile_u<T, RT, VEC>(u, matrix_at<T>(p.a, t.cur * p.a_stride), p.scale ? p.scale[t.cur] : 1.f, p.rank,
                               RowPair(p.x, at, p.ld_x, lane), p.n_in, lds, own, wave, lane, (int) blockIdx.x * 5);
        }
        const UOperand<T, RT> uo(u, i, g);
        const OutRows rows(t.row, g);
        const E* b = some ? (const E*) matrix_at<T>(p.b, t.cur * p.b_stride) : nullptr;
        // the block's columns 16 at a time: the wave's run of them, each column's ranks a row of LDS
        constexpr int LOADS = 16 * 16 * RT / 4 / 64, UN = RT <= 2 ? 4 : RT <= 4 ? 2 : 1;
        using Four = four_t<T>;
        struct Reg {
            float old[4];
            Four w[VEC ? LOADS : 1];
        };
        float old[4];
        int from[LOADS], to[LOADS];
        if (VEC) {
#pragma unroll
            for (int l = 0; l < LOADS; ++l) {
                from[l] = min(4 * (lane + 64 * l), 16 * p.rank - 4);
                to[l] = from[l] / p.rank * S::kOutPitch + from[l] % p.rank;
            }
        }
        if (some && p.rank < S::kStep)  // the ranks past the last, up to whole steps
            for (int q = lane; q < 16 * (S::kStep - p.rank); q += 64)
                lw[q / (S::kStep - p.rank) * S::kOutPitch + p.rank + q % (S::kStep - p.rank)] = E(0);
        const int tiles = (c1 - c0 + 15) / 16, run = (tiles + WAVES - 1) / WAVES;
        in_turn<UN, Reg>(
            min(tiles, (wave + 1) * run), wave * run, UN,
            [&](Reg& r, int c) {
                const int m = c0 + 16 * c;
                if (p.base) rows.load(r.old, p.base, p.ld_base, min(m + i, c1 - 1));
                if (VEC && some) {
                    const E* h = b + (int64_t) m * p.rank;
                    const int64_t most = (int64_t) (p.n_out - m) * p.rank - 4;  // (a column past the last holds anything)
#pragma unroll
                    for (int l = 0; l < LOADS; ++l) r.w[l] = *(const Four*) (h + std::min<int64_t>(from[l], most));
                }
            },
            [&](const Reg& r) {
#pragma unroll
                for (int k = 0; k < 4; ++k) old[k] = p.base ? r.old[k] : 0.f;
                if (VEC && some) {
#pragma unroll
                    for (int l = 0; l < LOADS; ++l) *(lds_ptr<Four>) (lw + to[l]) = r.w[l];
                }
            },
            [&](int c) {
                const int m = c0 + 16 * c;
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
                if (some) {
                    if (!VEC) {
                        for (int q = lane; q < 16 * p.rank; q += 64) {
                            const int k = q / p.rank, r = q % p.rank;
                            lw[k * S::kOutPitch + r] = m + k < c1 ? b[(int64_t) (m + k) * p.rank + r] : E(0);
                        }
                        wave_lds_order();
                    }
                    d = expand<T, RT>(uo, u, i, g, [&](int s) { return lds_oct<T>(lw + i * S::kOutPitch + 32 * s + 8 * g); });
                }
                if (m + i < c1) rows.store(p.y, p.ld_y, m + i, d, old);
            });
    }
}

template <int T, int RT> void launch_vec(bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    const size_t count = k.extra ? (size_t) (k.n + 1) * 4 : 0;
    if (vec) adapters_kernel<T, RT, true><<<grid, 64 * Shape<T, RT>::kWaves, count, st>>>(k);
    else adapters_kernel<T, RT, false><<<grid, 64 * Shape<T, RT>::kWaves, count, st>>>(k);
}
template <int T> void launch_rank(bool vec, const AdArgs& k, dim3 grid, hipStream_t st) {
    if (k.rank <= 16) launch_vec<T, 1>(vec, k, grid, st);
    else if (k.rank <= 32) launch_vec<T, 2>(vec, k, grid, st);
    else if (k.rank <= 64) launch_vec<T, 4>(vec, k, grid, st);
    else if (k.rank <= 128) launch_vec<T, 8>(vec, k, grid, st);
    else launch_vec<T, 16>(vec, k, grid, st);
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
    TSX_REQUIRE(y != x, "tsx_moe_adapters: x is read by other blocks than the one that writes y");
    AdArgs k{};
    const Tiles t(rows, p->n, 320);
    fill(k, p, ids, rows, t);
    k.x = x, k.ld_x = ld_x, k.base = base, k.ld_base = ld_base, k.y = y, k.ld_y = ld_y;
    const bool vec = matrix_quads(p) && quads(x, ld_x, 4);
    k.cols = columns_per_block((rows + 15) / 16, p->n_out, 128);
    TSX_REQUIRE(grid_fits(t.blocks(), 512), "tsx_moe_adapters: too many rows");
    const dim3 grid((unsigned) t.blocks(), (unsigned) ((p->n_out + k.cols - 1) / k.cols));
    const hipStream_t st = (hipStream_t) stream;
    if (p->type == TSX_F32) launch_rank<TSX_F32>(vec, k, grid, st);
    else if (p->type == TSX_F16) launch_rank<TSX_F16>(vec, k, grid, st);
    else launch_rank<TSX_BF16>(vec, k, grid, st);
    return launch_status("tsx_moe_adapters");
}

}  // extern "C"
