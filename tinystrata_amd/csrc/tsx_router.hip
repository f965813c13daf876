// tsx_router.hip - routing by the rules of several model families on gfx950, and its gradient: tsx_moe_route,
// tsx_moe_route_backward, tsx_moe_combine_backward.
//
// Routing.  Scores s_e = softmax over the experts, or sigmoid(l_e); an expert whose logit is -inf or NaN has none and is
// never picked.  Choice values c_e = s_e + bias_e, or the logits themselves without a bias (both scores grow with the
// logit, and a logit is not rounded).  With groups, the topk_group groups of largest value (the largest c, or the sum of
// the two largest s + bias) keep their experts.  The k largest c are picked, ties to the lower id.
//
// The order of the experts is that of exact arithmetic on the logits and biases given: two scores can lie nearer to each
// other than their fp32 roundings (about one token in a thousand of a 16384 x 256 batch picks otherwise), so c is formed in
// 64 bits where a bias or a sum enters it.  gfx950 issues 64-bit adds, products and maxima at the rate of 32-bit ones, so
// this costs the polynomial of the exponential and no slower instructions.  The weights are in fp32.
//
// One fp64 key per expert holds c and, in its low 9 bits, the id (43 bits of c stay: two c that agree in them differ by less
// than 2^-43 of their size), so that a maximum carries its id along and no two keys are equal.  A token belongs to L lanes;
// each lane sorts its keys with a network, and log2 L exchanges merge the lanes' K largest: max(a[i], b[K - 1 - i]) leaves
// the K largest of two sorted lists as a bitonic sequence, which log2 K stages sort.  No rounds of argmax, no ballots: the
// chains are short and the stages' maxima independent.
#include "tsx_common.hpp"
#include "tsx_device.hpp"

#include <cmath>

namespace tsx {
namespace {

constexpr int kMaxRouteK = 16, kMaxGroups = 64;

struct RouteArgs {
    const void* logits;
    int64_t ld;
    const float* bias;
    int32_t* ids;
    float* wts;
    int32_t* prow;
    int32_t* counts;
    float scale, floor;
    int type, sigmoid, norm, vec, need64;
    int n_tok, n_expert, k, n_group, topk_group, group_top, group_size, lg_shift;
};

// logit e of a row, and four of them from e on (row + e aligned to four elements)
__device__ __forceinline__ float logit_at(const void* row, int type, int64_t e) {
    if (type == TSX_F32) return ((const float*) row)[e];
    const uint16_t h = ((const uint16_t*) row)[e];
    return type == TSX_F16 ? h2f(h) : __builtin_bit_cast(float, (uint32_t) h << 16);
}
__device__ __forceinline__ void logits4_at(const void* row, int type, int64_t e, float (&o)[4]) {
    if (type == TSX_F32) {
        const float4 v = *(const float4*) ((const float*) row + e);
        o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
        return;
    }
    const uint2 w = *(const uint2*) ((const uint16_t*) row + e);
    const uint32_t h[4] = {w.x & 0xFFFFu, w.x >> 16, w.y & 0xFFFFu, w.y >> 16};
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = type == TSX_F16 ? h2f((uint16_t) h[c]) : __builtin_bit_cast(float, h[c] << 16);
}
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {  // to nearest, ties to even; NaN stays NaN
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    if (__builtin_isnan(f)) return (uint16_t) ((u >> 16) | 0x40u);
    return (uint16_t) ((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
// a logit that takes part, or -inf
__device__ __forceinline__ float live_logit(float l) { return l > -INFINITY ? l : -INFINITY; }

// e^x in 64 bits, |x| clamped to 708: x = n ln 2 + r, |r| <= ln 2 / 2, Taylor's polynomial of degree 12 in r (the next term
// is below 2e-16) times 2^n
__device__ __forceinline__ double exp64(double x) {
    x = __builtin_fmin(__builtin_fmax(x, -708.0), 708.0);
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(-n, 0.6931471805599453, x);
    r = __builtin_fma(-n, 2.3190468138462996e-17, r);
    double p = 1.0 / 479001600.0;
    constexpr double f[12] = {1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                              1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
    for (int i = 0; i < 12; ++i) p = __builtin_fma(p, r, f[i]);
    return __builtin_ldexp(p, (int) n);
}
// 1 / d, d in [1, 1e308): the hardware's estimate and two Newton steps
__device__ __forceinline__ double rcp64(double d) {
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}

// c with the low bits of its mantissa replaced so that among equal c the lower id is the larger key
template <int BITS>
__device__ __forceinline__ double pack_key(double c, uint32_t id) {
    constexpr uint64_t mask = (1ull << BITS) - 1;
    c = __builtin_fmin(c, 1.79769313486231e308) + 0.0;  // +inf would become a NaN; -0 and 0 are equal
    const uint64_t u = __builtin_bit_cast(uint64_t, c);
    const uint64_t low = (u >> 63) ? id : mask - id;
    return __builtin_bit_cast(double, (u & ~mask) | low);
}
template <int BITS>
__device__ __forceinline__ int key_id(double key) {
    constexpr uint64_t mask = (1ull << BITS) - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, key);
    return (int) ((u >> 63) ? (u & mask) : mask - (u & mask));
}
constexpr int kIdBits = 9, kGroupBits = 6;
static_assert((1 << kIdBits) >= kMaxExperts && (1 << kGroupBits) >= kMaxGroups, "ids fit the keys");

// the value of the lane M apart in the exchange order 1, 2, 4, .. : from 4 on any lane of the other half will do, since the
// lanes of a half hold the same values by then
template <int M>
__device__ __forceinline__ int swap32(int v) {
    if constexpr (M == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);
    if constexpr (M == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);
    if constexpr (M == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);
    if constexpr (M == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);
    return __shfl_xor(v, M, 64);
}
template <int M>
__device__ __forceinline__ double swap64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t) swap32<M>((int) (uint32_t) u), hi = (uint32_t) swap32<M>((int) (uint32_t) (u >> 32));
    return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
template <int M>
__device__ __forceinline__ float swapf(float v) {
    return __builtin_bit_cast(float, swap32<M>(__builtin_bit_cast(int, v)));
}
// op over a token's L lanes, every lane ending with the same bits
template <int L, int M = 1, typename Op>
__device__ __forceinline__ float token_reduce(float v, Op op) {
    if constexpr (M < L) return token_reduce<L, 2 * M>(op(v, swapf<M>(v)), op);
    return v;
}
template <int L, int M = 1>
__device__ __forceinline__ double token_sum(double v) {
    if constexpr (M < L) return token_sum<L, 2 * M>(v + swap64<M>(v));
    return v;
}

__device__ __forceinline__ void sort_pair(double& a, double& b) {  // the larger into a
    const double hi = __builtin_fmax(a, b), lo = __builtin_fmin(a, b);
    a = hi;
    b = lo;
}
// v[0..N) largest first: the odd-even merge sorting network
template <int N>
__device__ __forceinline__ void sort_keys(double* v) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) sort_pair(v[i + j], v[i + j + q]);
}
// a = the K largest of two lists of K sorted largest first, sorted
template <int K>
__device__ __forceinline__ void merge_top(double (&a)[K], const double (&b)[K]) {
#pragma unroll
    for (int i = 0; i < K; ++i) a[i] = __builtin_fmax(a[i], b[K - 1 - i]);
#pragma unroll
    for (int q = K / 2; q >= 1; q /= 2)
#pragma unroll
        for (int i = 0; i < K; ++i)
            if ((i & q) == 0) sort_pair(a[i], a[i + q]);
}
template <int L, int K, int M = 1>
__device__ __forceinline__ void merge_lanes(double (&a)[K]) {
    if constexpr (M < L) {
        double b[K];
#pragma unroll
        for (int i = 0; i < K; ++i) b[i] = swap64<M>(a[i]);
        merge_top<K>(a, b);
        merge_lanes<L, K, 2 * M>(a);
    }
}
// the two largest values of a group, over the lanes that hold it (1 << lg of them)
template <int L, int M = 1>
__device__ __forceinline__ void merge_two(double& m1, double& m2, int lanes) {
    if constexpr (M < L) {
        if (M < lanes) {  // uniform
            const double o1 = swap64<M>(m1), o2 = swap64<M>(m2);
            m2 = __builtin_fmax(__builtin_fmin(m1, o1), __builtin_fmax(m2, o2));
            m1 = __builtin_fmax(m1, o1);
            merge_two<L, 2 * M>(m1, m2, lanes);
        }
    }
}

// A token's L lanes, L >> lg_shift.. : lane = group * Lg + i with Lg = 1 << lg_shift lanes per group (one group: Lg = L);
// the lane holds the four experts from 4 (i + Lg q) of its group on, q < V / 4.
template <int L, int V, int K>
__global__ void __launch_bounds__(256) route_kernel(RouteArgs a) {
    extern __shared__ int s_count[];
    const int lane = threadIdx.x & 63, sub = lane & (L - 1);
    if (a.counts) {
        for (int e = threadIdx.x; e < a.n_expert; e += 256) s_count[e] = 0;
        __syncthreads();
    }
    const int per_block = 4 * (64 / L);
    // every lane stays for the exchanges; a group of lanes past the last token repeats it and stores nothing
    for (int t0 = blockIdx.x * per_block; t0 < a.n_tok; t0 += gridDim.x * per_block) {
        const int tt = t0 + (int) threadIdx.x / L, t = min(tt, a.n_tok - 1);
        const int g = sub >> a.lg_shift, lg = 1 << a.lg_shift, i = sub & (lg - 1);
        const int size = g < a.n_group ? a.group_size : 0, e0 = g * a.group_size;
        const void* row = (const char*) a.logits + (int64_t) t * a.ld * (a.type == TSX_F32 ? 4 : 2);
        float l[V];
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const int pos = 4 * (i + lg * q);
            float o[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (a.vec) {
                if (pos < size) logits4_at(row, a.type, e0 + pos, o);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (pos + c < size) o[c] = logit_at(row, a.type, e0 + pos + c);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) l[4 * q + c] = live_logit(o[c]);
        }
        float m = 0.f, sum = 1.f;
        if (!a.sigmoid) {
            m = -INFINITY;
#pragma unroll
            for (int v = 0; v < V; ++v) m = __builtin_fmaxf(m, l[v]);
            m = token_reduce<L>(m, OpMax());
        }
        // a softmax over a logit of +inf has no values, and one over nothing none either
        const bool any = a.sigmoid || (m > -INFINITY && m < INFINITY);
        double key[V];
        if (a.need64) {
            double c[V];
            double total = 0.0;
            if (a.sigmoid) {
#pragma unroll
                for (int v = 0; v < V; ++v) c[v] = rcp64(1.0 + exp64(-(double) l[v]));
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    c[v] = l[v] > -INFINITY ? exp64((double) l[v] - (double) m) : 0.0;
                    total += c[v];
                }
                total = token_sum<L>(total);
                sum = (float) total;
                const double r = any ? 1.0 / total : 0.0;
#pragma unroll
                for (int v = 0; v < V; ++v) c[v] *= r;
            }
            if (a.bias) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int pos = 4 * (i + lg * (v / 4)) + v % 4;
                    if (pos < size) c[v] += (double) a.bias[e0 + pos];
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = any && l[v] > -INFINITY && c[v] > -INFINITY ? c[v] : -INFINITY;
        } else {
            if (!a.sigmoid) {
                sum = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v) sum += expf(l[v] - m);  // -inf and no other: NaN, unused
                sum = token_reduce<L>(sum, OpAdd());
            }
#pragma unroll
            for (int v = 0; v < V; ++v) key[v] = any ? (double) l[v] : -INFINITY;
        }
        if (a.n_group > 1) {
            double m1 = -INFINITY, m2 = -INFINITY;
            // without a bias the largest logit has the largest score; sums need the scores, and need64 brought them
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m2 = __builtin_fmax(m2, __builtin_fmin(m1, key[v]));
                m1 = __builtin_fmax(m1, key[v]);
            }
            merge_two<L>(m1, m2, lg);
            double gv = m1;
            if (a.group_top == 2 && m2 > -INFINITY) gv += m2;
            const double mine = gv > -INFINITY ? pack_key<kGroupBits>(gv, (uint32_t) g & 63u) : -INFINITY;
            int better = 0;  // groups before this one
            for (int o = 0; o < a.n_group; ++o) better += __shfl(mine, o << a.lg_shift, L) > mine;
            if (better >= a.topk_group) {
#pragma unroll
                for (int v = 0; v < V; ++v) key[v] = -INFINITY;
            }
            if (a.need64 && !a.bias) {  // the experts' own order without a bias is that of the logits
#pragma unroll
                for (int v = 0; v < V; ++v) key[v] = key[v] > -INFINITY ? (double) l[v] : -INFINITY;
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = e0 + 4 * (i + lg * (v / 4)) + v % 4;
            key[v] = key[v] > -INFINITY ? pack_key<kIdBits>(key[v], (uint32_t) e) : -INFINITY;
        }
        double top[K];
        if constexpr (V <= K) {
            sort_keys<V>(key);
#pragma unroll
            for (int v = 0; v < K; ++v) top[v] = v < V ? key[v < V ? v : 0] : -INFINITY;
        } else {
            static_assert(V == 2 * K, "a lane's keys sort as one list or two");
            sort_keys<K>(key);
            sort_keys<K>(key + K);
            double second[K];
#pragma unroll
            for (int v = 0; v < K; ++v) top[v] = key[v], second[v] = key[K + v];
            merge_top<K>(top, second);
        }
        merge_lanes<L, K>(top);
        // lane j of the token takes pick j
        double mine = top[0];
#pragma unroll
        for (int j = 1; j < K; ++j) mine = sub == j ? top[j] : mine;
        const bool picked = sub < a.k && mine > -INFINITY;
        const int id = picked ? key_id<kIdBits>(mine) : -1;
        float s = 0.f;
        if (picked) {
            const float lj = logit_at(row, a.type, id);
            s = a.sigmoid ? 1.0f / (1.0f + expf(-lj)) : expf(lj - m) / sum;
        }
        float w = s * a.scale;
        if (a.norm) w *= 1.0f / __builtin_fmaxf(token_reduce<L>(s, OpAdd()), a.floor);
        if (tt < a.n_tok && sub < a.k) {
            const int64_t ent = (int64_t) tt * a.k + sub;
            a.ids[ent] = id;
            a.wts[ent] = w;
            if (a.prow) a.prow[ent] = id < 0 ? -1 : (int32_t) ent;
            if (a.counts && id >= 0) atomicAdd(&s_count[id], 1);
        }
    }
    if (a.counts) {
        __syncthreads();
        for (int e = threadIdx.x; e < a.n_expert; e += 256)
            if (const int c = s_count[e]) atomicAdd(&a.counts[e], c);  // whole numbers: any order gives the same
    }
}

struct RouteBackArgs {
    const void* logits;
    int64_t ld, ld_d;
    const int32_t* ids;
    const float* dwts;
    void* dlogits;
    float scale, floor;
    int type, sigmoid, norm, vec_in, vec_out;
    int n_tok, n_expert, k;
};

// w_j = scale s_j / max(S, floor), S the sum of the picks' scores:
//   ds_j = scale / S (dw_j - sum_i dw_i s_i / S) above the floor, scale / floor dw_j below it, scale dw_j without norm;
//   sigmoid: dl_e = ds_e s_e (1 - s_e) of the picks, 0 elsewhere;  softmax: dl_e = p_e ds_e - p_e sum_j ds_j p_j.
// Sixteen lanes a token, lane j its pick j; the picks' terms meet the row in LDS (an expert named twice gets both), and the
// row leaves whole.  Bound by the rows' bytes.
template <int V>
__global__ void __launch_bounds__(256) route_back_kernel(RouteBackArgs a) {
    extern __shared__ float s_row[];
    const int sub = threadIdx.x & 15, tt = blockIdx.x * 16 + (int) threadIdx.x / 16, t = min(tt, a.n_tok - 1);
    const int e_pad = (a.n_expert + 3) & ~3;
    float* mine = s_row + (threadIdx.x / 16) * e_pad;
    const void* row = (const char*) a.logits + (int64_t) t * a.ld * (a.type == TSX_F32 ? 4 : 2);
    int id = -1;
    float dw = 0.f, lj = 0.f;
    if (sub < a.k) {
        id = a.ids[(int64_t) t * a.k + sub];
        dw = a.dwts[(int64_t) t * a.k + sub];
        if (id < 0 || id >= a.n_expert) id = -1;
    }
    if (id >= 0) lj = logit_at(row, a.type, id);
    if (!(lj > -INFINITY)) id = -1;
    if (id < 0) dw = 0.f;
    float p[V];  // the softmax's values
    float m = 0.f, sum = 1.f;
    if (!a.sigmoid) {
        m = -INFINITY;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const int e = 4 * (sub + 16 * q);
            float o[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (a.vec_in) {
                if (e < a.n_expert) logits4_at(row, a.type, e, o);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (e + c < a.n_expert) o[c] = logit_at(row, a.type, e + c);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                p[4 * q + c] = live_logit(o[c]);
                m = __builtin_fmaxf(m, p[4 * q + c]);
            }
        }
        m = token_reduce<16>(m, OpMax());
        const bool any = m > -INFINITY && m < INFINITY;
        if (!any) id = -1, dw = 0.f;
        sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            p[v] = any ? expf(p[v] - m) : 0.f;
            sum += p[v];
        }
        sum = any ? token_reduce<16>(sum, OpAdd()) : 1.f;
    }
    // s_j, and for a sigmoid s_j (1 - s_j) without the difference: e / (1 + e)^2, e = exp(-|l|)
    float s = 0.f, slope = 0.f;
    if (id >= 0) {
        if (a.sigmoid) {
            const float e = expf(-fabsf(lj)), r = 1.0f / (1.0f + e);
            s = lj >= 0.f ? r : e * r;
            slope = e * r * r;
        } else {
            s = expf(lj - m) / sum;
        }
    }
    float ds = a.scale * dw;
    if (a.norm) {
        const float S = token_reduce<16>(s, OpAdd()), r = 1.0f / __builtin_fmaxf(S, a.floor);
        const float mean = token_reduce<16>(dw * s, OpAdd()) * r;
        ds = a.scale * r * (S > a.floor ? dw - mean : dw);
    }
    const float term = id < 0 ? 0.f : a.sigmoid ? ds * slope : ds * s;
    const float dot = a.sigmoid ? 0.f : token_reduce<16>(term, OpAdd());
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        const int e = 4 * (sub + 16 * q);
        if (e < a.n_expert) *(float4*) (mine + e) = float4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
    if (id >= 0) atomicAdd(mine + id, term);
    __syncthreads();
    if (tt >= a.n_tok) return;
    const float back = a.sigmoid ? 0.f : dot / sum;
    char* out = (char*) a.dlogits + (int64_t) tt * a.ld_d * (a.type == TSX_F32 ? 4 : 2);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        const int e = 4 * (sub + 16 * q);
        if (e >= a.n_expert) continue;
        const float4 r = *(const float4*) (mine + e);
        float d[4] = {r.x, r.y, r.z, r.w};
        if (!a.sigmoid) {
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c] -= p[4 * q + c] * back;
        }
        if (a.type == TSX_F32) {
            float* o = (float*) out + e;
            if (a.vec_out) {
                *(float4*) o = float4{d[0], d[1], d[2], d[3]};
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (e + c < a.n_expert) o[c] = d[c];
            }
            continue;
        }
        uint32_t h[4];  // the logits' type: one rounding
#pragma unroll
        for (int c = 0; c < 4; ++c) h[c] = a.type == TSX_F16 ? f2h(d[c]) : f32_to_bf16(d[c]);
        uint16_t* o = (uint16_t*) out + e;
        if (a.vec_out) {
            *(uint2*) o = uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (e + c < a.n_expert) o[c] = (uint16_t) h[c];
        }
    }
}

// The combine's gradient, one wave per token and part row (and one for the token's shared row): the row's weight gradient is
// its dot product with dy[t], and its own gradient w dy[t].  Every part row is read once and its gradient written once; dy[t]
// is read by the token's k waves, after the first from the caches.  Bound by the rows' bytes.
template <bool VEC>
__global__ void __launch_bounds__(256) combine_back_kernel(const float* __restrict__ dy, const float* __restrict__ parts,
                                                           const int32_t* __restrict__ prow, const float* __restrict__ wts,
                                                           int k, const float* __restrict__ shared,
                                                           const float* __restrict__ sgate, int sg_stride, int n, int64_t n_work,
                                                           int slots, float* __restrict__ dwts, float* __restrict__ dparts,
                                                           float* __restrict__ dshared, float* __restrict__ dsgate) {
    const int lane = threadIdx.x & 63;
    const int64_t work = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (work >= n_work) return;
    const int64_t t = work / slots;
    const int j = (int) (work - t * slots);
    const float* d = dy + t * n;
    const float* p;
    float* o;
    float w, slope = 0.f;
    if (j < k) {
        const int64_t row = prow ? prow[t * k + j] : t * k + j;
        if (row < 0) {  // an entry without a row
            if (lane == 0 && dwts) dwts[t * k + j] = 0.f;
            return;
        }
        p = parts + row * n;
        o = dparts ? dparts + row * n : nullptr;
        w = wts[t * k + j];
        if (!dwts) p = nullptr;
        if (!p && !o) return;
    } else {
        p = dsgate ? shared + t * n : nullptr;
        o = dshared ? dshared + t * n : nullptr;
        const float g = sgate[t * sg_stride], e = expf(-fabsf(g)), r = 1.0f / (1.0f + e);
        w = g >= 0.f ? r : e * r;
        slope = e * r * r;
    }
    float dot = 0.f;
    if (VEC) {
        for (int i = 4 * lane; i < n; i += 256) {
            const float4 v = *(const float4*) (d + i);
            if (p) {
                const float4 q = *(const float4*) (p + i);
                dot = __builtin_fmaf(v.x, q.x, dot);
                dot = __builtin_fmaf(v.y, q.y, dot);
                dot = __builtin_fmaf(v.z, q.z, dot);
                dot = __builtin_fmaf(v.w, q.w, dot);
            }
            if (o) *(float4*) (o + i) = float4{w * v.x, w * v.y, w * v.z, w * v.w};
        }
    } else {
        for (int i = lane; i < n; i += 64) {
            const float v = d[i];
            if (p) dot = __builtin_fmaf(v, p[i], dot);
            if (o) o[i] = w * v;
        }
    }
    if (!p) return;
    dot = tree_sum<64>(dot);
    if (lane == 0) {
        if (j < k) dwts[t * k + j] = dot;
        else dsgate[t] = slope * dot;
    }
}

int check_router(const char* what, const tsx_router* r) {
    TSX_REQUIRE(r, "%s: no router", what);
    if (r->type != TSX_F32 && r->type != TSX_F16 && r->type != TSX_BF16) {
        set_error("%s: logits of type %d (fp32, fp16 or bf16)", what, r->type);
        return TSX_ERR_UNSUPPORTED;
    }
    if (r->n_expert < 1 || r->n_expert > kMaxExperts || r->k < 1 || r->k > kMaxRouteK || r->k > r->n_expert) {
        set_error("%s: %d experts / top-%d not supported (1..512 experts, k 1..16)", what, r->n_expert, r->k);
        return TSX_ERR_UNSUPPORTED;
    }
    const int G = r->n_group;
    if (G < 1 || G > kMaxGroups || r->n_expert % G != 0 || r->topk_group < 1 || r->topk_group > G ||
        (r->group_top != 1 && r->group_top != 2) || (G > 1 && r->group_top > r->n_expert / G) ||
        r->k > r->topk_group * (r->n_expert / G)) {
        set_error("%s: %d groups, %d kept, by their %d largest, for top-%d of %d experts not supported (1..64 groups of equal "
                  "size, by 1 or 2 of their experts, those kept holding k)",
                  what, G, r->topk_group, r->group_top, r->k, r->n_expert);
        return TSX_ERR_UNSUPPORTED;
    }
    TSX_REQUIRE(r->score == TSX_SCORE_SOFTMAX || r->score == TSX_SCORE_SIGMOID, "%s: score %d", what, r->score);
    TSX_REQUIRE(std::isfinite(r->scale) && std::isfinite(r->floor) && r->floor > 0.f,
                "%s: scale finite, floor finite and above 0", what);
    TSX_REQUIRE(aligned(r->bias, 4), "%s: bias 4-byte aligned", what);
    return TSX_OK;
}
inline size_t elem_size(int type) { return type == TSX_F32 ? 4 : 2; }
inline int pow2_at_least(int v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

template <int L, int V>
void launch_route(const RouteArgs& a, hipStream_t st) {
    const int per_block = 4 * (64 / L);
    unsigned blocks = (unsigned) ((a.n_tok + per_block - 1) / per_block);
    size_t lds = 0;
    if (a.counts) {
        // a block adds its counts once per expert at its end: no more blocks than fill the card
        blocks = std::min(blocks, 1024u);
        lds = (size_t) a.n_expert * 4;
    }
    if (a.k <= 8) route_kernel<L, V, 8><<<blocks, 256, lds, st>>>(a);
    else route_kernel<L, V, 16><<<blocks, 256, lds, st>>>(a);
}

}  // namespace
}  // namespace tsx

using namespace tsx;

extern "C" {

TSX_API int tsx_moe_route(const tsx_router* r, const void* logits, int64_t ld, int32_t* ids, float* weights, int32_t* prow,
                          int32_t* counts, int n_tok, void* stream) {
    if (const int rc = check_router("tsx_moe_route", r)) return rc;
    TSX_REQUIRE(n_tok >= 0 && ld >= r->n_expert, "tsx_moe_route: n_tok >= 0, ld at least the experts");
    if (n_tok == 0) return TSX_OK;
    TSX_REQUIRE(logits && ids && weights && aligned(logits, elem_size(r->type)) && aligned(ids, 4) && aligned(weights, 4) &&
                    aligned(prow, 4) && aligned(counts, 4),
                "tsx_moe_route: logits, ids, weights (and prow, counts) aligned to their types");
    TSX_REQUIRE((int64_t) n_tok * r->k <= INT32_MAX, "tsx_moe_route: more than 2^31 - 1 entries");
    RouteArgs a{};
    a.logits = logits, a.ld = ld, a.bias = r->bias, a.ids = ids, a.wts = weights, a.prow = prow, a.counts = counts;
    a.scale = r->scale, a.floor = r->floor;
    a.type = r->type, a.sigmoid = r->score == TSX_SCORE_SIGMOID, a.norm = r->norm != 0;
    a.n_tok = n_tok, a.n_expert = r->n_expert, a.k = r->k, a.n_group = r->n_group, a.topk_group = r->topk_group;
    a.group_top = r->group_top, a.group_size = r->n_expert / r->n_group;
    a.need64 = r->bias != nullptr || (r->n_group > 1 && r->group_top == 2);
    a.vec = a.group_size % 4 == 0 && ld % 4 == 0 && aligned(logits, 4 * elem_size(r->type));
    // 16 lanes per token where each then holds at most 16 experts (four tokens share a wave's instructions), else 64
    const int gp = pow2_at_least(r->n_group), quads = (a.group_size + 3) / 4;
    auto quads_per_lane = [&](int L) { return gp <= L ? (quads + L / gp - 1) / (L / gp) : 1 << 20; };
    const int L = quads_per_lane(16) <= 4 ? 16 : 64, q = quads_per_lane(L);
    for (int lanes = L / gp; lanes > 1; lanes /= 2) ++a.lg_shift;
    const hipStream_t st = (hipStream_t) stream;
    if (L == 16) {
        if (q <= 1) launch_route<16, 4>(a, st);
        else if (q <= 2) launch_route<16, 8>(a, st);
        else launch_route<16, 16>(a, st);
    } else {
        if (q <= 1) launch_route<64, 4>(a, st);
        else if (q <= 2) launch_route<64, 8>(a, st);
        else launch_route<64, 16>(a, st);
    }
    return launch_status("tsx_moe_route");
}

TSX_API int tsx_moe_route_backward(const tsx_router* r, const void* logits, int64_t ld, const int32_t* ids,
                                   const float* dweights, void* dlogits, int64_t ld_d, int n_tok, void* stream) {
    if (const int rc = check_router("tsx_moe_route_backward", r)) return rc;
    TSX_REQUIRE(n_tok >= 0 && ld >= r->n_expert && ld_d >= r->n_expert,
                "tsx_moe_route_backward: n_tok >= 0, ld and ld_d at least the experts");
    if (n_tok == 0) return TSX_OK;
    TSX_REQUIRE(logits && ids && dweights && dlogits && aligned(logits, elem_size(r->type)) &&
                    aligned(dlogits, elem_size(r->type)) && aligned(ids, 4) && aligned(dweights, 4),
                "tsx_moe_route_backward: logits, ids, dweights, dlogits aligned to their types");
    RouteBackArgs a{};
    a.logits = logits, a.ld = ld, a.ld_d = ld_d, a.ids = ids, a.dwts = dweights, a.dlogits = dlogits;
    a.scale = r->scale, a.floor = r->floor;
    a.type = r->type, a.sigmoid = r->score == TSX_SCORE_SIGMOID, a.norm = r->norm != 0;
    a.n_tok = n_tok, a.n_expert = r->n_expert, a.k = r->k;
    const size_t quad = 4 * elem_size(r->type);
    a.vec_in = r->n_expert % 4 == 0 && ld % 4 == 0 && aligned(logits, quad);
    a.vec_out = r->n_expert % 4 == 0 && ld_d % 4 == 0 && aligned(dlogits, quad);
    const unsigned blocks = (unsigned) (((int64_t) n_tok + 15) / 16);
    const size_t lds = (size_t) 16 * ((r->n_expert + 3) & ~3) * 4;
    const hipStream_t st = (hipStream_t) stream;
    if (r->n_expert <= 64) route_back_kernel<4><<<blocks, 256, lds, st>>>(a);
    else if (r->n_expert <= 128) route_back_kernel<8><<<blocks, 256, lds, st>>>(a);
    else if (r->n_expert <= 256) route_back_kernel<16><<<blocks, 256, lds, st>>>(a);
    else route_back_kernel<32><<<blocks, 256, lds, st>>>(a);
    return launch_status("tsx_moe_route_backward");
}

TSX_API int tsx_moe_combine_backward(const float* dy, const float* parts, const int32_t* prow, const float* wts, int k,
                                     const float* shared, const float* sgate, int sg_stride, int n, int n_tok,
                                     float* dwts, float* dparts, float* dshared, float* dsgate, void* stream) {
    TSX_REQUIRE(k >= 1 && n >= 1 && n_tok >= 0, "tsx_moe_combine_backward: k >= 1, n >= 1, n_tok >= 0");
    if (n_tok == 0) return TSX_OK;
    TSX_REQUIRE(dy && parts && wts && (!shared || sgate),
                "tsx_moe_combine_backward: dy, parts, wts (and sgate with shared)");
    TSX_REQUIRE(shared || (!dshared && !dsgate), "tsx_moe_combine_backward: dshared and dsgate go with shared");
    TSX_REQUIRE(aligned(dy, 4) && aligned(parts, 4) && aligned(prow, 4) && aligned(wts, 4) && aligned(shared, 4) &&
                    aligned(sgate, 4) && aligned(dwts, 4) && aligned(dparts, 4) && aligned(dshared, 4) && aligned(dsgate, 4),
                "tsx_moe_combine_backward: every buffer 4-byte aligned");
    if (!(dwts || dparts || dshared || dsgate)) return TSX_OK;
    const int slots = k + (dshared || dsgate ? 1 : 0);
    const int64_t n_work = (int64_t) n_tok * slots, blocks = (n_work + 3) / 4;
    TSX_REQUIRE(blocks <= INT32_MAX, "tsx_moe_combine_backward: too many rows");
    const hipStream_t st = (hipStream_t) stream;
    if (n % 4 == 0 && aligned(dy, 16) && aligned(parts, 16) && aligned(shared, 16) && aligned(dparts, 16) &&
        aligned(dshared, 16))
        combine_back_kernel<true><<<(unsigned) blocks, 256, 0, st>>>(dy, parts, prow, wts, k, shared, sgate, sg_stride, n,
                                                                     n_work, slots, dwts, dparts, dshared, dsgate);
    else
        combine_back_kernel<false><<<(unsigned) blocks, 256, 0, st>>>(dy, parts, prow, wts, k, shared, sgate, sg_stride, n,
                                                                      n_work, slots, dwts, dparts, dshared, dsgate);
    return launch_status("tsx_moe_combine_backward");
}

}  // extern "C"
