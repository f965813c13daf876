// tsx_router.hip - routing by the rules of several model families on gfx950, and its gradient: tsx_moe_route,
// tsx_moe_route_backward, tsx_moe_combine_backward.
//
// Routing.  Scores s_e = softmax over the experts, or sigmoid(l_e); an expert whose logit is -inf or NaN has none and is
// never picked.  Choice values c_e = s_e + bias_e, or the logits themselves without a bias (both scores grow with the
// logit, and a logit is not rounded).  With groups, the topk_group groups of largest value (the largest c, or the sum of
// the two largest s + bias) keep their experts.  The k largest c are picked, ties to the lower id.
//
// The order of the experts is that of exact arithmetic on the logits and biases given: two scores can lie nearer to each
// other than their fp32 roundings (about one token in a thousand of a 16384 x 256 batch picks otherwise).  The choice is made on
// fp32 values of known error, and made again in 64 bits where two values that decide it lie within that error (route_kernel).
// The weights are in fp32.
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
    int type, sigmoid, norm, vec, vec_bias, need64;
    int n_tok, n_expert, k, n_group, topk_group, group_top, group_size, shift;
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

// c with the low bits of its mantissa replaced so that among equal c the lower id is the larger key.  c = -inf stands for
// none: its key lies below kNone, and every other one above (a c that fp32 values make is far from the ends of the range).
constexpr double kNone = -1e308;
template <int BITS>
__device__ __forceinline__ double pack_key(double c, uint32_t id) {
    constexpr uint32_t mask = (1u << BITS) - 1;
    // an infinity would become a NaN; -0 and 0 are equal
    c = __builtin_fmax(__builtin_fmin(c, 1.79769313486231e308), -1.79769313486231e308) + 0.0;
    const uint64_t u = __builtin_bit_cast(uint64_t, c);
    const uint32_t low = (mask - id) ^ ((uint32_t) ((int32_t) (u >> 32) >> 31) & mask);
    return __builtin_bit_cast(double, (u & ~(uint64_t) mask) | low);
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
__device__ __forceinline__ int token_count(int v) {
    if constexpr (M < L) return token_count<L, 2 * M>(v + swap32<M>(v));
    return v;
}
template <int L, int M = 1>
__device__ __forceinline__ double token_sum(double v) {
    if constexpr (M < L) return token_sum<L, 2 * M>(v + swap64<M>(v));
    return v;
}

template <int L, int M = 1>
__device__ __forceinline__ double token_min(double v) {
    if constexpr (M < L) return token_min<L, 2 * M>(__builtin_fmin(v, swap64<M>(v)));
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

// How a token's experts lie on L lanes: lane = group * lanes + i with `lanes` = 1 << shift of them per group (one group: all
// L); the lane holds the four experts from 4 (i + lanes q) of its group on, q < V / 4.
struct Place {
    int i, lanes, size, e0;
    __device__ __forceinline__ Place(const RouteArgs& a, int sub, int shift) {
        const int g = sub >> shift;
        lanes = 1 << shift;
        i = sub & (lanes - 1);
        size = g < a.n_group ? a.group_size : 0;
        e0 = g * a.group_size;
    }
    __device__ __forceinline__ int pos(int v) const { return 4 * (i + lanes * (v / 4)) + v % 4; }
};
// the lane's logits (-inf for one that takes no part), and biases; in quads without a condition, all in flight together
template <int V>
__device__ __forceinline__ void fetch_logits(const RouteArgs& a, const void* row, const Place& p, float (&l)[V]) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        const int pos = p.pos(4 * q);
        float o[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (a.vec) {
            logits4_at(row, a.type, pos < p.size ? p.e0 + pos : 0, o);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (pos + c < p.size) o[c] = logit_at(row, a.type, p.e0 + pos + c);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) l[4 * q + c] = pos + c < p.size ? live_logit(o[c]) : -INFINITY;
    }
}
template <int V>
__device__ __forceinline__ void fetch_bias(const RouteArgs& a, const Place& p, float (&b)[V]) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        const int pos = p.pos(4 * q);
        float4 o = {0.f, 0.f, 0.f, 0.f};
        if (a.vec_bias) {
            o = *(const float4*) (a.bias + (pos < p.size ? p.e0 + pos : 0));
        } else {
            if (pos < p.size) o.x = a.bias[p.e0 + pos];
            if (pos + 1 < p.size) o.y = a.bias[p.e0 + pos + 1];
            if (pos + 2 < p.size) o.z = a.bias[p.e0 + pos + 2];
            if (pos + 3 < p.size) o.w = a.bias[p.e0 + pos + 3];
        }
        b[4 * q] = o.x, b[4 * q + 1] = o.y, b[4 * q + 2] = o.z, b[4 * q + 3] = o.w;
    }
}
// a group's value on every lane of it, with the group's number in its low bits, and how many groups come before it
template <int L, int V>
__device__ __forceinline__ double group_rank(const RouteArgs& a, const double (&key)[V], int sub, int shift, int& before) {
    double m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        m2 = __builtin_fmax(m2, __builtin_fmin(m1, key[v]));
        m1 = __builtin_fmax(m1, key[v]);
    }
    merge_two<L>(m1, m2, 1 << shift);
    if (a.group_top == 2 && m2 > -INFINITY) m1 += m2;
    const double mine = pack_key<kGroupBits>(m1, (uint32_t) (sub >> shift) & 63u);
    before = 0;
    for (int o = 0; o < a.n_group; ++o) before += __shfl(mine, o << shift, L) > mine;
    return mine;
}

// the wave's largest value, in every lane: within the rows of 16 by exchanges, then the four rows' read out
__device__ __forceinline__ double wave_max64(double v) {
    v = -token_min<16>(-v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    auto row = [&](int l) {
        const uint32_t lo = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) u, l);
        const uint32_t hi = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (u >> 32), l);
        return __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
    };
    return __builtin_fmax(__builtin_fmax(row(0), row(16)), __builtin_fmax(row(32), row(48)));
}

// One token's picks in 64 bits by a whole wave: lane r returns pick r, -1 for none.  Expert e = lane + 64 i; `keys` are
// kMaxExperts values of LDS, the wave's own, for the sums over groups.  The rare way (every wave of a batch waits for the one
// that takes it, so its latency counts: 4 us): k rounds of the largest key below the last one.
__device__ __forceinline__ int pick_precise(const RouteArgs& a, const void* row, int lane, double* keys) {
    constexpr int V = kMaxExperts / 64;
    const int E = a.n_expert;
    float l[V];
    float m = a.sigmoid ? 0.f : -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = lane + 64 * i < E ? live_logit(logit_at(row, a.type, lane + 64 * i)) : -INFINITY;
    if (!a.sigmoid) {
#pragma unroll
        for (int i = 0; i < V; ++i) m = __builtin_fmaxf(m, l[i]);
        m = token_reduce<64>(m, OpMax());
    }
    const bool any = m > -INFINITY && m < INFINITY;
    double key[V], total = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        key[i] = -1.0;  // takes no part
        if (64 * i < E) {
            double s = exp64(a.sigmoid ? -(double) l[i] : (double) l[i] - (double) m);
            if (a.sigmoid) s = rcp64(1.0 + s);
            if (any && l[i] > -INFINITY) {
                key[i] = s;
                total += s;
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // one after the other: side by side they would take the register file
    }
    const double r = a.sigmoid ? 1.0 : 1.0 / token_sum<64>(total);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        const double c = __builtin_fma(key[i], r, a.bias && e < E ? (double) a.bias[e] : 0.0);
        key[i] = key[i] >= 0.0 && c > -INFINITY ? c : -INFINITY;  // (a bias may be NaN)
    }
    uint64_t kept = ~0ull;
    if (a.n_group > 1) {  // lane g: group g
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (lane + 64 * i < E) keys[lane + 64 * i] = key[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        double m1 = -INFINITY, m2 = -INFINITY;
        const int e0 = min(lane, a.n_group - 1) * a.group_size;
#pragma unroll 4
        for (int j = 0; j < a.group_size; ++j) {
            const double c = keys[e0 + j];
            m2 = __builtin_fmax(m2, __builtin_fmin(m1, c));
            m1 = __builtin_fmax(m1, c);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (a.group_top == 2 && m2 > -INFINITY) m1 += m2;
        const double mine = pack_key<kGroupBits>(m1, (uint32_t) lane);
        int before = 0;
        for (int o = 0; o < a.n_group; ++o) before += __shfl(mine, o, 64) > mine;
        kept = __ballot(lane < a.n_group && before < a.topk_group);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        double c = key[i];
        if (a.n_group > 1 && !(kept >> (e / a.group_size) & 1)) c = -INFINITY;
        if (!a.bias && c > -INFINITY) c = (double) l[i];  // the experts' own order is that of the logits
        key[i] = pack_key<kIdBits>(c, (uint32_t) e);
    }
    double last = INFINITY;
    int id = -1;
    for (int j = 0; j < a.k; ++j) {
        double best = -INFINITY;  // nothing below the last one
#pragma unroll
        for (int i = 0; i < V; ++i) best = key[i] < last ? __builtin_fmax(best, key[i]) : best;
        last = wave_max64(best);
        if (lane == j && last > kNone) id = key_id<kIdBits>(last);
    }
    return id;
}

// Choice values that need the scores are formed in fp32, from the hardware's exponential and reciprocal, and the selection is
// made on them; only where two values that decide it lie within those roundings of each other is it made again in 64 bits: on
// the few values near the last pick for a sigmoid, by pick_precise for a softmax and for the choice of groups.
// `slack` bounds how far a value in fp32 is from the exact one.  A sigmoid: the exponential is off by 1.5 |l| + 2 units of
// 2^-24, which s (1 - s) takes to less than 1, the sum with 1 and the reciprocal by 3; the sum with the bias by half a step of
// at most 1 + |bias|: 5 + |bias| units in all.  A softmax: (2.5 |l - m| + 30) units of its size, |l - m| below 104 where it is
// not 0, and half a step for the sum: less than 2^-15 of |c| + |bias|.  Equal logits with equal biases have equal values in
// any precision and need no second look.
//
// Measured (us, sigmoid scores, bias, 8 groups by their two largest, top-8 of 256): 16384 tokens in 64 bits throughout 35.
// Sixteen lanes a token or 64: one token 7.3 or 5.0, 2048 (no groups) 4.5 or 4.3, 4096 4.5 or 5.7, 16384 7.6 or 15.1; of 64
// experts 2.6 or 3.4 at one token already.  With values that leave doubt among them: 2048 tokens 8.2, 16384 18.1 (12.0 and 21.7
// when pick_precise took every one); counts add 2.
template <int L, int V, int K, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) route_kernel(RouteArgs a) {
    extern __shared__ int s_count[];
    __shared__ double s_keys[WAVES][kMaxExperts];
    const int lane = threadIdx.x & 63, sub = lane & (L - 1);
    if (a.counts) {
        for (int e = threadIdx.x; e < a.n_expert; e += 64 * WAVES) s_count[e] = 0;
        __syncthreads();
    }
    constexpr int per_block = WAVES * (64 / L);
    const Place p(a, sub, a.shift);
    // every lane stays for the exchanges; a group of lanes past the last token repeats it and stores nothing
    const int64_t t0 = (int64_t) blockIdx.x * per_block;
    const int64_t tt = t0 + (int) threadIdx.x / L, t = tt < a.n_tok ? tt : a.n_tok - 1;
    const void* row = (const char*) a.logits + t * a.ld * (a.type == TSX_F32 ? 4 : 2);
    float c[V];  // the choice values
    fetch_logits<V>(a, row, p, c);
    float m = 0.f, sum = 1.f, most_bias = 0.f;
    constexpr float kLog2e = 1.44269504f;
    if (!a.sigmoid) {
        m = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; ++v) m = __builtin_fmaxf(m, c[v]);
        m = token_reduce<L>(m, OpMax());
        sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) sum += __builtin_amdgcn_exp2f((c[v] - m) * kLog2e);  // (of -inf: 0)
        sum = token_reduce<L>(sum, OpAdd());
    }
    // a softmax over a logit of +inf has no values, and one over nothing none either
    const bool any = a.sigmoid || (m > -INFINITY && m < INFINITY);
    if (a.need64) {
        float b[V] = {};
        if (a.bias) fetch_bias<V>(a, p, b);
        const float r = __builtin_amdgcn_rcpf(sum);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-c[v] * kLog2e))
                                      : __builtin_amdgcn_exp2f((c[v] - m) * kLog2e) * r;
            const float sb = s + b[v];
            c[v] = any && c[v] > -INFINITY && sb > -INFINITY ? sb : -INFINITY;
            if (fabsf(b[v]) < INFINITY) most_bias = __builtin_fmaxf(most_bias, fabsf(b[v]));
        }
        most_bias = token_reduce<L>(most_bias, OpMax());
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = any ? c[v] : -INFINITY;
    }
    auto slack = [&](double x) -> double {
        return a.sigmoid ? (6.0 + (double) most_bias) * 0x1p-24 : (__builtin_fabs(x) + (double) most_bias) * 0x1p-15;
    };
    bool open = false, kept = true;  // open: the values in fp32 do not decide
    double key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = (double) c[v];
    if (a.n_group > 1) {
        int before;
        const double mine = group_rank<L, V>(a, key, sub, a.shift, before);
        kept = before < a.topk_group;
        if (a.need64) {  // the least group kept and the best one dropped
            const double least = token_min<L>(kept ? mine : (double) INFINITY);
            const double best = -token_min<L>(kept ? (double) INFINITY : -mine);
            open = best > kNone && least - best <= 2.0 * (slack(least) + slack(best));
            if (!a.bias) {  // the experts' own order without a bias is that of the logits
                float l[V];
                fetch_logits<V>(a, row, p, l);
#pragma unroll
                for (int v = 0; v < V; ++v) key[v] = c[v] > -INFINITY ? (double) l[v] : -INFINITY;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = pack_key<kIdBits>(kept ? key[v] : -INFINITY, (uint32_t) (p.e0 + p.pos(v)));
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
    double mine = top[0], next = -INFINITY, last = top[0];
#pragma unroll
    for (int j = 1; j < K; ++j) {
        mine = sub == j ? top[j] : mine;
        next = sub == j - 1 ? top[j] : next;
        last = j == a.k - 1 ? top[j] : last;
    }
    bool picked = sub < a.k && mine > kNone;
    int id = picked ? key_id<kIdBits>(mine) : -1;
    if (a.bias) {
        // the order of neighbours among the picks, and the last pick against what is left: more values than picks that lie above
        // it less its slack
        bool near = sub + 1 < a.k && next > kNone && mine - next <= 2.0 * slack(mine);
        const float cl = (float) last, edge = cl - 2.f * (float) slack(last);  // the id's bits round away
        const int el = key_id<kIdBits>(last);
        int above = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) above += c[v] >= edge;
        near |= last > kNone && token_count<L>(kept ? above : 0) > a.k;
        if (__any(near)) {
            bool doubt = false;
            if (sub + 1 < a.k && next > kNone && mine - next <= 2.0 * slack(mine)) {
                const int e = key_id<kIdBits>(next);
                doubt |= !(logit_at(row, a.type, id) == logit_at(row, a.type, e) && a.bias[id] == a.bias[e]);
            }
            if (kept && last > kNone) {
                const float ll = logit_at(row, a.type, el), bl = a.bias[el];
                float l[V], b[V];
                fetch_logits<V>(a, row, p, l);
                fetch_bias<V>(a, p, b);
#pragma unroll
                for (int v = 0; v < V; ++v)
                    doubt |= c[v] >= edge && (c[v] < cl || (c[v] == cl && p.e0 + p.pos(v) > el)) &&
                             !(l[v] == ll && b[v] == bl);
            }
            if (!a.sigmoid) {
                open |= doubt;
            } else if (__any(doubt)) {
                // A sigmoid needs no sum over the experts: the values that reach the last pick less its slack, which hold
                // every true pick, are formed in 64 bits (one or two a lane, as a rule) and merged again
                uint32_t again = 0;
#pragma unroll
                for (int v = 0; v < V; ++v) again |= kept && c[v] > -INFINITY && c[v] >= edge ? 1u << v : 0u;
#pragma unroll
                for (int j = 0; j < K; ++j) top[j] = -INFINITY;
#pragma unroll 1
                while (__any(again != 0)) {
                    double x = -INFINITY;
                    if (again) {
                        const int e = p.e0 + p.pos(__builtin_ctz(again));
                        const double s = rcp64(1.0 + exp64(-(double) logit_at(row, a.type, e)));
                        x = pack_key<kIdBits>(s + (double) a.bias[e], (uint32_t) e);
                        again &= again - 1;
                    }
#pragma unroll
                    for (int j = 0; j < K; ++j) sort_pair(top[j], x);
                }
                merge_lanes<L, K>(top);
                mine = top[0];
#pragma unroll
                for (int j = 1; j < K; ++j) mine = sub == j ? top[j] : mine;
                picked = sub < a.k && mine > kNone;
                id = picked ? key_id<kIdBits>(mine) : -1;
            }
        }
    }
    if (const uint64_t again = __ballot(open)) {
#pragma unroll 1
        for (int o = 0; o < 64; o += L) {  // the wave's tokens with an open choice, one at a time
            if (((again >> o) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) == 0) continue;
            const int64_t to = t0 + (int) (threadIdx.x & ~63u) / L + o / L;
            const void* r = (const char*) a.logits + (to < a.n_tok ? to : a.n_tok - 1) * a.ld * (a.type == TSX_F32 ? 4 : 2);
            int own = lane;
            asm volatile("" : "+v"(own));  // nothing of it is computed ahead of the loop, in registers of every wave
            const int got = __shfl(pick_precise(a, r, own, s_keys[threadIdx.x >> 6]), sub, 64);
            if ((lane & ~(L - 1)) == o) {
                id = sub < a.k ? got : -1;
                picked = id >= 0;
            }
        }
    }
    float s = 0.f;
    if (picked) {
        const float lj = logit_at(row, a.type, id);
        s = a.sigmoid ? 1.0f / (1.0f + expf(-lj)) : expf(lj - m) / sum;
    }
    float w = s * a.scale;
    if (a.norm) w *= 1.0f / __builtin_fmaxf(token_reduce<L>(s, OpAdd()), a.floor);
    if (tt < a.n_tok && sub < a.k) {
        const int64_t ent = tt * a.k + sub;
        a.ids[ent] = id;
        a.wts[ent] = w;
        if (a.prow) a.prow[ent] = id < 0 ? -1 : (int32_t) ent;
        if (a.counts && id >= 0) atomicAdd(&s_count[id], 1);
    }
    if (a.counts) {
        __syncthreads();
        for (int e = threadIdx.x; e < a.n_expert; e += 64 * WAVES)
            if (const int n = s_count[e]) atomicAdd(&a.counts[e], n);  // whole numbers: any order gives the same
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

template <int L, int V, int K, int WAVES>
void launch_waves(const RouteArgs& a, hipStream_t st) {
    constexpr int per_block = WAVES * (64 / L);
    const unsigned blocks = (unsigned) (((int64_t) a.n_tok + per_block - 1) / per_block);
    route_kernel<L, V, K, WAVES><<<blocks, 64 * WAVES, a.counts ? (size_t) a.n_expert * 4 : 0, st>>>(a);
}
template <int L, int V>
void launch_route(const RouteArgs& a, hipStream_t st) {
    // with counts a block adds its own once per expert at its end: large blocks make these additions few
    if (a.k <= 8) a.counts ? launch_waves<L, V, 8, 8>(a, st) : launch_waves<L, V, 8, 4>(a, st);
    else a.counts ? launch_waves<L, V, 16, 8>(a, st) : launch_waves<L, V, 16, 4>(a, st);
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
    TSX_REQUIRE(grid_fits(n_tok, 64), "tsx_moe_route: more than 2^26 - 1 tokens");
    RouteArgs a{};
    a.logits = logits, a.ld = ld, a.bias = r->bias, a.ids = ids, a.wts = weights, a.prow = prow, a.counts = counts;
    a.scale = r->scale, a.floor = r->floor;
    a.type = r->type, a.sigmoid = r->score == TSX_SCORE_SIGMOID, a.norm = r->norm != 0;
    a.n_tok = n_tok, a.n_expert = r->n_expert, a.k = r->k, a.n_group = r->n_group, a.topk_group = r->topk_group;
    a.group_top = r->group_top, a.group_size = r->n_expert / r->n_group;
    a.need64 = r->bias != nullptr || (r->n_group > 1 && r->group_top == 2);
    a.vec_bias = a.group_size % 4 == 0 && aligned(r->bias, 16);
    a.vec = a.group_size % 4 == 0 && ld % 4 == 0 && aligned(logits, 4 * elem_size(r->type));
    // 16 lanes per token where each then holds at most 16 experts (four tokens share a wave's instructions), but 64 while the
    // tokens leave the card room and a lane of 16 would hold more than 8 (the shorter chains are then what counts)
    const int gp = pow2_at_least(r->n_group), quads = (a.group_size + 3) / 4;
    auto quads_per_lane = [&](int L) { return gp <= L ? (quads + L / gp - 1) / (L / gp) : 1 << 20; };
    const int q16 = quads_per_lane(16), L = q16 <= (n_tok <= 2048 ? 2 : 4) ? 16 : 64, q = quads_per_lane(L);
    for (int lanes = L / gp; lanes > 1; lanes /= 2) ++a.shift;
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
    TSX_REQUIRE(grid_fits(blocks, 256), "tsx_moe_route_backward: more than 2^28 - 16 tokens");
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
    TSX_REQUIRE(grid_fits(blocks, 256), "tsx_moe_combine_backward: too many rows");
    TSX_REQUIRE(dparts != dy && dshared != dy,
                "tsx_moe_combine_backward: dy is read by every entry of its token, not overwritten");
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
