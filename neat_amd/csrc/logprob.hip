// Log probability of a given token per row of logits, the row's entropy, its most probable alternatives, and the gradient.
//
// With x the logits of a row, f the scale, m = max x, d_j = f (x_j - m), s = sum exp d_j, p_j = exp(d_j) / s:
//   logp_t = d_t - log s        H = log s - sum(exp(d_j) d_j) / s      (both parts of H are >= 0: nothing cancels)
//   d(a logp_t + b H) / dx_j = f (a (delta_jt - p_j) - b p_j (d_j - log s + H))
// One reading of the row gives all of it: a workgroup holds its row in registers (up to 32 fp32 or 64 bf16 values a lane, 64 fp32 for gradients of rows above 32 768), so
// that neither the alternatives nor the gradient read it again.  Rows longer than a workgroup's registers are cut, the pieces'
// (m, s, sum) and lists are joined by a second launch, and the gradient is a pass of its own.
//
// What a mask leaves out is -inf: probability 0, no share in H, gradient 0.  A row with nothing left has logp = -inf, H = 0,
// alternatives of -inf and no gradient.  NaN (or +inf) makes the row's results NaN; it is never an alternative itself.
//
// Alternatives: the k-th largest of 64 group maxima bounds the k-th largest value from below; the few values that reach it are
// collected and ranked by counting (value, then lower index): no sort, and no atomic that matters to the result.  Where many
// reach it (a row of few different values, or mostly masked), 64-bit keys (value, index) that never tie take its place: the
// k-th largest of 256 to 1 024 groups' keys leaves at most k groups' elements, for which there is room.
//
// Bound by HBM where there are rows for all CUs: 4 928 x 49 408 bf16 with gradient 183 us (974 MB, 5.3 TB/s; the vector ALU is
// nine tenths busy there, and run back to back it takes 204 us), 2 000 x 25 014 fp32 with 10 alternatives 41 us (200 MB, 4.8 TB/s;
// the ranking of one row runs under the loads of another).  bf16 rows with alternatives are bound by the vector ALU (10 of them: rows
// of 49 408 4.4 TB/s, of 16 385 3.8), short ones by what is paid once a row (of 1 000 2.6).  One row of 49 408 with 5 alternatives:
// 8 us, half of it the exponentials of one CU.  Cutting it over 13 CUs makes the sums 1 us faster and the joining launch takes 1 us
// with them, so rows are cut only where they do not fit.
#include "wave.h"

namespace neat {

constexpr int LP_NV = 8;                     // 16-B vectors a lane holds
constexpr int LP_MAX_K = 32;
constexpr int LP_MAX_SPLIT = 64;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr float LP_LOWEST = -160.f;          // exp2 of it is zero: keeps 0 * -inf out of the sums
constexpr float LP_MAX_SCALE = 0x1p100f;     // and 0 * inf out of the gradient, whose factors reach 160 scale x weight

struct LpArgs {
    const void* z;                           // [R, V], row pitch ld
    const int64_t* target;                   // [R] or null
    const float *a, *b;                      // gradient weights of logp and H, [R] or null
    float *logp, *ent, *stats;               // [R], [R], [3, R] = max, sum, entropy (any may be null)
    float* top;                              // [R, k] log probabilities
    int32_t* idx;                            // [R, k]
    void* dz;                                // [R, V], row pitch ldz
    float* part;                             // [R, S, 4] when the rows are cut
    uint64_t* keys;                          // [R, S, k]
    long ld, ldz;
    int R, V, k, S, chunk;
    int row0;                                // first row of this launch
    float scale;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// rows may start at any element: loads and stores of 16 B need the element's own alignment only
template <typename T> struct LpIo;
template <> struct LpIo<float> {
    static constexpr int VEC = 4;
    static constexpr uint32_t NEG = 0xff800000u;
    typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float get(u32x4 r, int j) { return __uint_as_float(r[j]); }
    static __device__ __forceinline__ void put(u32x4& r, int j, float x) { r[j] = __float_as_uint(x); }
    static __device__ __forceinline__ u32x4 pack(const float (&o)[4]) {
        return u32x4{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])};
    }
    static __device__ __forceinline__ float one(const void* p, long i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store1(void* p, long i, float x) { static_cast<float*>(p)[i] = x; }
};
template <> struct LpIo<bf16_t> {
    static constexpr int VEC = 8;
    static constexpr uint32_t NEG = 0xff80ff80u;
    typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
    static __device__ __forceinline__ float get(u32x4 r, int j) {
        return __uint_as_float(j & 1 ? r[j >> 1] & 0xffff0000u : r[j >> 1] << 16);
    }
    static __device__ __forceinline__ void put(u32x4& r, int j, float x) {
        const uint32_t h = __float_as_uint(x) >> 16;           // x is a bf16 number
        r[j >> 1] = j & 1 ? (r[j >> 1] & 0xffffu) | h << 16 : (r[j >> 1] & 0xffff0000u) | h;
    }
    static __device__ __forceinline__ u32x4 pack(const float (&o)[8]) {
        return u32x4{pack2bf(o[0], o[1]), pack2bf(o[2], o[3]), pack2bf(o[4], o[5]), pack2bf(o[6], o[7])};
    }
    static __device__ __forceinline__ float one(const void* p, long i) { return bf2f(static_cast<const bf16_t*>(p)[i]); }
    static __device__ __forceinline__ void store1(void* p, long i, float x) { static_cast<bf16_t*>(p)[i] = f2bf(x); }
};
// ONCE: past the caches, for logits that are not read again (a forward pass alone leaves them for its backward pass); so is the
// gradient written, which no call here reads (4 928 x 49 408 bf16, both: 204 -> 191 us)
template <bool ONCE, typename T>
__device__ __forceinline__ u32x4 lp_load(const T* p, long i) {
    const auto* q = reinterpret_cast<const typename LpIo<T>::vec*>(p + i);
    return ONCE ? __builtin_nontemporal_load(q) : *q;
}
template <typename T>
__device__ __forceinline__ void lp_store(T* p, long i, u32x4 v) {
    __builtin_nontemporal_store((typename LpIo<T>::vec)v, reinterpret_cast<typename LpIo<T>::vec*>(p + i));
}

// value order as an unsigned number, -0 as +0, NaN as -inf
__device__ __forceinline__ uint32_t lp_order(float x) {
    x = x == x ? x + 0.f : -INFINITY;
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_from_order(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// an element's key: value, then the smaller index as the larger one.  No element's key is 0.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t i) { return (uint64_t)lp_order(x) << 32 | (0xffffffffu - i); }
__device__ __forceinline__ float lp_value(uint64_t key) { return lp_from_order((uint32_t)(key >> 32)); }
__device__ __forceinline__ int32_t lp_index(uint64_t key) { return (int32_t)(0xffffffffu - (uint32_t)key); }
__device__ __forceinline__ uint64_t lp_shfl_xor(uint64_t v, int m) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), m) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, m);
}

struct LpSums { float m, s, t; };            // max; sum 2^d; sum 2^d d, d in units of log 2 relative to m

// joins the sums that lanes 0 .. n-1 hold (the other lanes hold the empty sum); m = -inf stands for nothing but masks
__device__ __forceinline__ LpSums lp_join(LpSums v, float c) {
    const float M = wave_max_f(v.m), M0 = M == -INFINITY ? 0.f : M;
    const float shift = v.m == -INFINITY ? 0.f : fmaxf((v.m - M0) * c, LP_LOWEST);
    const float w = v.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((v.m - M0) * c);
    return LpSums{M, wave_sum_f(v.s * w), wave_sum_f(w * __builtin_fmaf(v.s, shift, v.t))};
}

struct LpRow { float m0, logs, ent; };
__device__ __forceinline__ LpRow lp_row(const LpSums& v) {
    const float logs = logf(v.s);
    return LpRow{v.m == -INFINITY ? 0.f : v.m, logs, v.s == 0.f ? 0.f : logs - v.t / v.s * LN2};
}
__device__ __forceinline__ float lp_logp(float x, const LpRow& r, float s, float scale) {
    return s == 0.f ? -INFINITY : (x - r.m0) * scale - r.logs;
}

// what one lane writes of a row's numbers
template <typename T>
__device__ __forceinline__ void lp_write_row(const LpArgs& g, int row, const LpSums& v, const LpRow& r) {
    if (g.logp) {
        const int64_t t = g.target[row];
        g.logp[row] = t < 0 ? 0.f
                    : t >= g.V ? NAN : lp_logp(LpIo<T>::one(g.z, (long)row * g.ld + t), r, v.s, g.scale);
    }
    if (g.ent) g.ent[row] = r.ent;
    if (g.stats) {
        g.stats[row] = r.m0;
        g.stats[(long)g.R + row] = v.s;
        g.stats[2L * g.R + row] = r.ent;
    }
}

// The gradient of a row at x is 2^(c (x - m0)) (k0 + k1 c (x - m0)), and `add` more at its target.
struct LpGrad { float m0, k0, k1, add; long t; };
__device__ __forceinline__ LpGrad lp_grad(const LpArgs& g, int row, float m0, float s, float ent) {
    const int64_t t = g.target ? g.target[row] : -1;
    float a = g.a && t >= 0 ? g.a[row] : 0.f;
    const float b = g.b ? g.b[row] : 0.f;
    if (t >= g.V) a = NAN;                   // a target that no row has shows in the whole row
    const float inv = s == 0.f ? 0.f : g.scale / s;
    if (s == 0.f && a == a) a = 0.f;         // nothing left of the row: nothing to change
    return LpGrad{m0, s == 0.f ? a : -inv * (a + b * (ent - logf(s))), -inv * b * LN2, g.scale * a, t};
}
template <typename T>
__device__ __forceinline__ u32x4 lp_grad_vec(u32x4 raw, const LpGrad& q, float c, long first) {
    float o[LpIo<T>::VEC];
#pragma unroll
    for (int j = 0; j < LpIo<T>::VEC; ++j) {
        const float d = (LpIo<T>::get(raw, j) - q.m0) * c;
        o[j] = __builtin_amdgcn_exp2f(d) * __builtin_fmaf(fmaxf(d, LP_LOWEST), q.k1, q.k0);
    }
    const long at = q.t - first;
    if (at >= 0 && at < LpIo<T>::VEC) {
#pragma unroll
        for (int j = 0; j < LpIo<T>::VEC; ++j) o[j] += at == j ? q.add : 0.f;
    }
    return LpIo<T>::pack(o);
}

enum { LP_SUMS = 0, LP_TOP = 1, LP_GRAD = 2 };

// groups of the exact bound: parts of a lane's vectors
template <int THREADS> struct LpGroups { static constexpr int PARTS = THREADS < 256 ? 256 / THREADS : 1; };
constexpr int LP_FEW = 256;                  // candidates of the first bound that are ranked; more go by keys

// the k largest of the `total` keys in `cand`, in order
template <int THREADS>
__device__ __forceinline__ void lp_rank(const LpArgs& g, const uint64_t* cand, int total, int row, int piece, const LpRow& r,
                                        float s) {
    const int k = g.k;
    for (int i = threadIdx.x; i < total; i += THREADS) {
        const uint64_t own = cand[i];
        int rank = 0, q = 0;
        for (; q + 8 <= total; q += 8) {     // eight at a time: their loads wait together
            uint64_t other[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) other[j] = cand[q + j];
#pragma unroll
            for (int j = 0; j < 8; ++j) rank += other[j] > own ? 1 : 0;
        }
        for (; q < total; ++q) rank += cand[q] > own ? 1 : 0;
        if (rank < k) {
            if (g.part) {
                g.keys[((long)row * g.S + piece) * k + rank] = own;
            } else {
                g.idx[(long)row * k + rank] = lp_index(own);
                g.top[(long)row * k + rank] = lp_logp(lp_value(own), r, s, g.scale);
            }
        }
    }
    if (g.part)
        for (int i = total + threadIdx.x; i < k; i += THREADS) g.keys[((long)row * g.S + piece) * k + i] = 0;
}

// raw: this lane's elements; lane_m: the largest of them; least: a bound that at least k elements reach; *count is 0
template <typename T, int THREADS>
__device__ __forceinline__ void lp_alternatives(const LpArgs& g, const T* z, const u32x4 (&raw)[LP_NV], int row, int piece, int lo,
                                                int n, float lane_m, float least, int* count, const LpRow& r, float s) {
    constexpr int VEC = LpIo<T>::VEC;
    extern __shared__ __attribute__((aligned(16))) uint64_t cand[];
    const int tid = threadIdx.x, first = __builtin_amdgcn_readfirstlane(tid);
    // NaN counts as -inf, which is why the comparisons are turned round
    if (!(lane_m < least)) {
#pragma unroll
        for (int i = 0; i < LP_NV; ++i) {
            if ((first + i * THREADS) * VEC >= n) break;
            const int e = (tid + i * THREADS) * VEC;
            uint32_t hit = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) hit |= !(LpIo<T>::get(raw[i], j) < least) ? 1u << j : 0u;
            if (e < n) {
                for (; hit; hit &= hit - 1) {
                    const int at_j = __builtin_ctz(hit);
                    float x = 0.f;           // eight ways to choose from take over 64 registers: asked from the cache again
                    if constexpr (VEC == 4) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) x = j == at_j ? LpIo<T>::get(raw[i], j) : x;
                    } else if (e + at_j < n) {
                        x = LpIo<T>::one(z, e + at_j);
                    }
                    if (e + at_j < n) {
                        const int at = atomicAdd(count, 1);
                        if (at < LP_FEW) cand[at] = lp_key(x, lo + e + at_j);
                    }
                }
            }
        }
    }
    __syncthreads();
    const int total = *count;
    if (total <= LP_FEW) {
        lp_rank<THREADS>(g, cand, total, row, piece, r, s);
        return;
    }
    // many values reach the bound: the same once more with keys that never tie, from memory (the row is in the caches).  A group
    // is a lane's vectors, or a part of them where there are few lanes: the fewer elements it has, the less LDS its candidates
    // need (64 lanes with whole lanes for groups: 16 KiB at k = 32, and only nine workgroups fit a CU)
    constexpr int PARTS = LpGroups<THREADS>::PARTS, GROUPS = THREADS * PARTS, PER = LP_NV / PARTS;
    __shared__ uint64_t group[GROUPS];
    __shared__ uint64_t bound;
    __syncthreads();
    uint64_t mine[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        mine[p] = 0;
        for (int i = p * PER; i < (p + 1) * PER; ++i) {
            const int first = (tid + i * THREADS) * VEC, last = min(first + VEC, n);
            for (int e = first; e < last; ++e) {
                const uint64_t key = lp_key(LpIo<T>::one(z, e), lo + e);
                mine[p] = key > mine[p] ? key : mine[p];
            }
        }
        group[tid * PARTS + p] = mine[p];
    }
    if (tid == 0) {
        bound = 0;
        *count = 0;
    }
    __syncthreads();
    int rank[PARTS] = {};
    for (int q = 0; q < GROUPS; ++q) {
        const uint64_t other = group[q];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) rank[p] += other > mine[p] ? 1 : 0;
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
        if (rank[p] == g.k - 1 && mine[p] != 0) bound = mine[p];             // fewer groups than k: everything is a candidate
    __syncthreads();
    const uint64_t floor_key = bound;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if (mine[p] == 0 || mine[p] < floor_key) continue;
        for (int i = p * PER; i < (p + 1) * PER; ++i) {
            const int first = (tid + i * THREADS) * VEC, last = min(first + VEC, n);
            for (int e = first; e < last; ++e) {
                const uint64_t key = lp_key(LpIo<T>::one(z, e), lo + e);
                if (key >= floor_key) cand[atomicAdd(count, 1)] = key;
            }
        }
    }
    __syncthreads();
    lp_rank<THREADS>(g, cand, *count, row, piece, r, s);
}

// One workgroup, one row (or one piece of it).  At most 64 registers, so that eight waves share a SIMD and some load while others
// compute (bf16 rows of 16 385 with 10 alternatives 3.1 TB/s with five waves, 3.4 with eight; of 1 000 2.3 and 2.4).
template <typename T, int THREADS, int MODE, int NV = LP_NV>
__global__ __launch_bounds__(THREADS, NV > LP_NV ? 4 : 8) void logprob_kernel(LpArgs g) {
    constexpr int VEC = LpIo<T>::VEC, WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = g.row0 + blockIdx.x / g.S, piece = blockIdx.x % g.S;
    const int lo = piece * g.chunk, n = min(g.chunk, g.V - lo);
    const T* z = static_cast<const T*>(g.z) + (long)row * g.ld + lo;
    const float c = g.scale * LOG2E;
    const int first = __builtin_amdgcn_readfirstlane(tid);     // a wave skips the vectors behind the row's end (187 -> 183 us)

    u32x4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = (tid + i * THREADS) * VEC;
        raw[i] = u32x4{LpIo<T>::NEG, LpIo<T>::NEG, LpIo<T>::NEG, LpIo<T>::NEG};
        if (e + VEC <= n) {
            raw[i] = lp_load<MODE == LP_GRAD>(z, e);
        } else if (e < n) {                  // the row's end: one lane, the rest of its vector stays masked
#pragma unroll
            for (int j = 0; j < VEC - 1; ++j)
                if (e + j < n) LpIo<T>::put(raw[i], j, LpIo<T>::one(z, e + j));
        }
    }
    float lane_m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if ((first + i * THREADS) * VEC < n) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) lane_m = fmaxf(lane_m, LpIo<T>::get(raw[i], j));
        }
    }
    const float row_m = row_max(lane_m);     // of 16 lanes
    const float m = fmaxf(fmaxf(lane_f(row_m, 0), lane_f(row_m, 16)), fmaxf(lane_f(row_m, 32), lane_f(row_m, 48)));
    const float m0 = m == -INFINITY ? 0.f : m;
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if ((first + i * THREADS) * VEC < n) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = (LpIo<T>::get(raw[i], j) - m0) * c, e = __builtin_amdgcn_exp2f(d);
                s += e;
                t = __builtin_fmaf(e, fmaxf(d, LP_LOWEST), t);
            }
        }
    }
    LpSums v{m, wave_sum_f(s), wave_sum_f(t)};

    // what the first wave finds out for all: the row's sums, and the least value of a candidate
    __shared__ float red[3][WAVES], group[64], joined[4];
    __shared__ int count;
    constexpr int GL = THREADS / 64;         // lanes of the 64 groups: 1, 2, 4, 8 or a row of 16
    float group_m = lane_m;
    if constexpr (GL >= 2) group_m = fmaxf(group_m, dpp_f<DPP_XOR1>(group_m));
    if constexpr (GL >= 4) group_m = fmaxf(group_m, dpp_f<DPP_XOR2>(group_m));
    if constexpr (GL >= 8) group_m = fmaxf(group_m, dpp_f<DPP_HALF_MIRROR>(group_m));
    if constexpr (GL == 16) group_m = row_m;
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            red[0][wave] = v.m;
            red[1][wave] = v.s;
            red[2][wave] = v.t;
        }
        if (MODE == LP_TOP && tid % GL == 0) group[tid / GL] = group_m;
        __syncthreads();
    }
    if (wave == 0) {
        if constexpr (WAVES > 1) {
            v = LpSums{-INFINITY, 0.f, 0.f};
            if (lane < WAVES) v = LpSums{red[0][lane], red[1][lane], red[2][lane]};
            v = lp_join(v, c);
        }
        float least = 0.f;
        if constexpr (MODE == LP_TOP) {      // the k-th largest of 64, bit by bit: the largest number that k of them reach.  bf16
            // numbers have nothing in the low half, which lp_order turns round below zero
            const uint32_t own = lp_order(WAVES > 1 ? group[lane] : group_m);
            uint32_t kth = 0;
#pragma unroll
            for (int bit = 31; bit >= (VEC == 8 ? 16 : 0); --bit) {
                const uint32_t probe = kth | 1u << bit;
                if ((int)__popcll(__ballot(own >= probe)) >= g.k) kth = probe;
            }
            if (VEC == 8 && !(kth & 0x80000000u)) kth |= 0xffffu;
            least = lp_from_order(kth);
            if (lane == 0) count = 0;
        }
        if (lane == 0) {
            joined[0] = v.m;
            joined[1] = v.s;
            joined[2] = v.t;
            joined[3] = least;
        }
    }
    if constexpr (WAVES > 1 || MODE == LP_TOP) {
        __syncthreads();
        v = LpSums{joined[0], joined[1], joined[2]};
    }
    const LpRow r = lp_row(v);
    if (tid == 0) {
        if (g.part) {
            float* p = g.part + ((long)row * g.S + piece) * 4;
            p[0] = v.m;
            p[1] = v.s;
            p[2] = v.t;
        } else {
            lp_write_row<T>(g, row, v, r);
        }
    }
    if constexpr (MODE == LP_TOP) lp_alternatives<T, THREADS>(g, z, raw, row, piece, lo, n, lane_m, joined[3], &count, r, v.s);
    if constexpr (MODE == LP_GRAD) {
        const LpGrad q = lp_grad(g, row, r.m0, v.s, r.ent);
        T* dz = static_cast<T*>(g.dz) + (long)row * g.ldz;
        if (WAVES > 1) __syncthreads();      // dz may be the logits: lane 0 has read the target's before anything is written
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (tid + i * THREADS) * VEC;
            if (e < n) {
                const u32x4 o = lp_grad_vec<T>(raw[i], q, c, e);
                if (e + VEC <= n) {
                    lp_store<T>(dz, e, o);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC - 1; ++j)
                        if (e + j < n) LpIo<T>::store1(dz, e + j, LpIo<T>::get(o, j));
                }
            }
        }
    }
}

// Joins the pieces of a row: one workgroup, one row.  The lists are in order, so the k-th largest of all is at least every
// list's k-th and, S ceil(k / S) keys being at least k, the least of the lists' ceil(k / S)-th: only keys that reach both are
// ranked (one of them after the other, a wave's maximum each, took 0.4 us a key).
constexpr int LPJ_THREADS = 256;
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void logprob_join_kernel(LpArgs g) {
    __shared__ float joined[3];
    __shared__ uint64_t bound;
    __shared__ int count;
    extern __shared__ __attribute__((aligned(16))) uint64_t cand[];
    const int row = g.row0 + blockIdx.x, lane = threadIdx.x & 63;
    const float c = g.scale * LOG2E;
    const uint64_t* keys = g.keys + (long)row * g.S * g.k;
    if (threadIdx.x < 64) {
        LpSums v{-INFINITY, 0.f, 0.f};
        if (lane < g.S) {
            const float* p = g.part + ((long)row * g.S + lane) * 4;
            v = LpSums{p[0], p[1], p[2]};
        }
        v = lp_join(v, c);
        if (lane == 0) lp_write_row<T>(g, row, v, lp_row(v));
        if (THREADS > 64) {
            uint64_t last = 0, early = ~0ull;
            if (lane < g.S) {
                last = keys[(long)lane * g.k + g.k - 1];
                early = keys[(long)lane * g.k + (g.k + g.S - 1) / g.S - 1];
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const uint64_t a = lp_shfl_xor(last, o), b = lp_shfl_xor(early, o);
                last = a > last ? a : last;
                early = b < early ? b : early;
            }
            if (lane == 0) {
                joined[0] = v.m;
                joined[1] = v.s;
                joined[2] = v.t;
                bound = last > early ? last : early;
                count = 0;
            }
        }
    }
    if (THREADS == 64) return;
    __syncthreads();
    const uint64_t least = bound > 0 ? bound : 1;               // 0: a list shorter than k has no key there
    for (int i = threadIdx.x; i < g.S * g.k; i += THREADS) {
        const uint64_t key = keys[i];
        if (key >= least) cand[atomicAdd(&count, 1)] = key;
    }
    __syncthreads();
    const LpSums v{joined[0], joined[1], joined[2]};
    const LpRow r = lp_row(v);
    g.part = nullptr;                                           // ranked into the results
    lp_rank<THREADS>(g, cand, count, row, 0, r, v.s);
}

// The gradient from a forward pass's numbers: every lane reads and writes its own elements, so that dz may be the logits.
constexpr int LPB_THREADS = 256, LPB_NV = 4;
template <typename T>
__global__ __launch_bounds__(LPB_THREADS) void logprob_bwd_kernel(LpArgs g) {
    constexpr int VEC = LpIo<T>::VEC;
    const int row = g.row0 + blockIdx.x / g.S, piece = blockIdx.x % g.S;
    const long base = (long)piece * (LPB_THREADS * LPB_NV * VEC);
    const float c = g.scale * LOG2E;
    const T* z = static_cast<const T*>(g.z) + (long)row * g.ld;
    T* dz = static_cast<T*>(g.dz) + (long)row * g.ldz;
    const LpGrad q = lp_grad(g, row, g.stats[row], g.stats[(long)g.R + row], g.stats[2L * g.R + row]);
    u32x4 raw[LPB_NV];
#pragma unroll
    for (int i = 0; i < LPB_NV; ++i) {
        const long e = base + (long)(threadIdx.x + i * LPB_THREADS) * VEC;
        raw[i] = u32x4{0, 0, 0, 0};
        if (e + VEC <= g.V) {
            raw[i] = lp_load<false>(z, e);
        } else if (e < g.V) {
#pragma unroll
            for (int j = 0; j < VEC - 1; ++j)
                if (e + j < g.V) LpIo<T>::put(raw[i], j, LpIo<T>::one(z, e + j));
        }
    }
#pragma unroll
    for (int i = 0; i < LPB_NV; ++i) {
        const long e = base + (long)(threadIdx.x + i * LPB_THREADS) * VEC;
        if (e < g.V) {
            const u32x4 o = lp_grad_vec<T>(raw[i], q, c, e);
            if (e + VEC <= g.V) {
                lp_store<T>(dz, e, o);
            } else {
#pragma unroll
                for (int j = 0; j < VEC - 1; ++j)
                    if (e + j < g.V) LpIo<T>::store1(dz, e + j, LpIo<T>::get(o, j));
            }
        }
    }
}

// how a row is laid over workgroups: lanes per workgroup, pieces per row and their length
struct LpPlan { int threads, S, chunk, nv; };
static LpPlan lp_plan(int vec, int V, bool grad = false) {
    LpPlan p;
    int lane = LP_NV * vec;
    // a gradient's second reading costs more than a CU with one workgroup loses (400 MB of fp32 rows of 49 408: 3.8 TB/s cut and
    // read twice, 5.4 so): fp32 rows that need it get twice the registers
    if (grad && vec == 4 && V > 1024 * lane && V <= 2 * 1024 * lane) lane *= 2;
    p.nv = lane / vec;
    p.threads = 64;                          // the fewest lanes that hold the row
    while (p.threads < 1024 && V > p.threads * lane) p.threads *= 2;
    const long cap = (long)p.threads * lane;
    p.S = cdiv(V, cap);
    p.chunk = p.S == 1 ? V : (cdiv(V, p.S) + vec - 1) / vec * vec;
    p.S = cdiv(V, p.chunk);
    return p;
}
// candidates of k groups of the exact bound, or of the first one
static size_t lp_cand_bytes(const LpPlan& p, int vec, int k) {
    const int parts = p.threads < 256 ? 256 / p.threads : 1, held = cdiv(p.chunk, (long)p.threads * vec);
    const size_t b = (size_t)k * (held < LP_NV / parts ? held : LP_NV / parts) * vec * 8;
    return b > LP_FEW * 8 ? b : LP_FEW * 8;
}
static long lp_part_bytes(long R, const LpPlan& p) { return p.S == 1 ? 0 : (R * p.S * 16 + 255) / 256 * 256; }

// launches over at most 2^31 work items each
template <typename F>
static int lp_rows(LpArgs& g, int per_row, int threads, const char* what, F&& launch) {
    const long most = (1L << 31) / ((long)per_row * threads);
    for (long r = 0; r < g.R; r += most) {
        g.row0 = (int)r;
        launch(dim3((unsigned)((g.R - r < most ? g.R - r : most) * per_row)));
        NEAT_LAUNCH_CHECK(what);
    }
    return NEAT_OK;
}
template <typename T, int MODE>
static int lp_launch(LpArgs& g, const LpPlan& p, size_t lds, const char* what, hipStream_t s) {
    return lp_rows(g, g.S, p.threads, what, [&](dim3 grid) {
        if (p.threads == 64) hipLaunchKernelGGL((logprob_kernel<T, 64, MODE>), grid, dim3(64), lds, s, g);
        else if (p.threads == 128) hipLaunchKernelGGL((logprob_kernel<T, 128, MODE>), grid, dim3(128), lds, s, g);
        else if (p.threads == 256) hipLaunchKernelGGL((logprob_kernel<T, 256, MODE>), grid, dim3(256), lds, s, g);
        else if (p.threads == 512) hipLaunchKernelGGL((logprob_kernel<T, 512, MODE>), grid, dim3(512), lds, s, g);
        else if constexpr (MODE == LP_GRAD && sizeof(T) == 4) {
            if (p.nv > LP_NV) hipLaunchKernelGGL((logprob_kernel<T, 1024, MODE, 2 * LP_NV>), grid, dim3(1024), lds, s, g);
            else hipLaunchKernelGGL((logprob_kernel<T, 1024, MODE>), grid, dim3(1024), lds, s, g);
        }
        else hipLaunchKernelGGL((logprob_kernel<T, 1024, MODE>), grid, dim3(1024), lds, s, g);
    });
}
template <typename T>
static int lp_forward(LpArgs& g, const LpPlan& p, hipStream_t s) {
    const char* what = "neat_token_logprobs";
    int rc = g.k > 0 ? lp_launch<T, LP_TOP>(g, p, lp_cand_bytes(p, LpIo<T>::VEC, g.k), what, s)
                     : lp_launch<T, LP_SUMS>(g, p, 0, what, s);
    if (rc || g.S == 1) return rc;
    return lp_rows(g, 1, LPJ_THREADS, what, [&](dim3 grid) {
        if (g.k == 0) hipLaunchKernelGGL((logprob_join_kernel<T, 64>), grid, dim3(64), 0, s, g);
        else hipLaunchKernelGGL((logprob_join_kernel<T, LPJ_THREADS>), grid, dim3(LPJ_THREADS), (size_t)g.S * g.k * 8, s, g);
    });
}
template <typename T>
static int lp_backward(LpArgs g, hipStream_t s) {
    g.S = cdiv(g.V, (long)LPB_THREADS * LPB_NV * LpIo<T>::VEC);
    return lp_rows(g, g.S, LPB_THREADS, "neat_token_logprobs_bwd", [&](dim3 grid) {
        hipLaunchKernelGGL(logprob_bwd_kernel<T>, grid, dim3(LPB_THREADS), 0, s, g);
    });
}

static int lp_check(const char* who, const void* z, long ld, int dtype, int R, int V, float scale) {
    NEAT_REQUIRE(z || R == 0, NEAT_ERR_ARG, "%s: null pointer", who);
    NEAT_REQUIRE(dtype == NEAT_F32 || dtype == NEAT_BF16, NEAT_ERR_ARG, "%s: dtype=%d", who, dtype);
    const int vec = dtype == NEAT_F32 ? 4 : 8;
    NEAT_REQUIRE(R >= 0 && V >= 1 && (R <= 1 || ld >= V), NEAT_ERR_SHAPE, "%s: R=%d V=%d row pitch=%ld", who, R, V, ld);
    NEAT_REQUIRE(V <= LP_MAX_SPLIT * 1024 * LP_NV * vec, NEAT_ERR_SHAPE, "%s: V=%d is above %d", who, V,
                 LP_MAX_SPLIT * 1024 * LP_NV * vec);
    NEAT_REQUIRE(((uintptr_t)z & (dtype == NEAT_F32 ? 3 : 1)) == 0, NEAT_ERR_ARG, "%s: logits are not aligned to their elements", who);
    NEAT_REQUIRE(scale > 0.f && scale <= LP_MAX_SCALE, NEAT_ERR_ARG, "%s: scale=%g must be positive, and 2^100 at most", who, (double)scale);
    return NEAT_OK;
}

// whether two sets of R rows of w bytes share a byte, pitches pa and pb >= w (host)
static bool lp_rows_meet(uintptr_t a, long pa, uintptr_t b, long pb, long R, long w) {
    if (R <= 0 || (long)(b - a) >= (R - 1) * pa + w || (long)(a - b) >= (R - 1) * pb + w) return false;
    if (R == 1) return true;
    if (pa == pb) {                          // columns of one buffer, say: b's rows lie q rows and d bytes behind a's
        const long off = (long)(b - a), q = off >= 0 ? off / pa : -((-off + pa - 1) / pa), d = off - q * pa;
        return (d < w && -R < q && q < R) || (d + w > pa && -R < q + 1 && q + 1 < R);
    }
    for (long i = 0, j = 0; i < R && j < R;) {
        const uintptr_t x = a + (uintptr_t)(i * pa), y = b + (uintptr_t)(j * pb);
        if (x < y + (uintptr_t)w && y < x + (uintptr_t)w) return true;
        if (x < y) ++i; else ++j;
    }
    return false;
}
// the gradient lies over the logits element by element, or apart from them
static int lp_check_out(const char* who, const void* z, long ld, const void* dz, long ldz, int dtype, int R, int V) {
    const long t = dtype == NEAT_F32 ? 4 : 2;
    const bool same = z == dz && (ld == ldz || R <= 1);
    NEAT_REQUIRE(same || !lp_rows_meet((uintptr_t)z, ld * t, (uintptr_t)dz, ldz * t, R, V * t), NEAT_ERR_ARG,
                 "%s: the gradient overlaps the logits (it may be the logits themselves)", who);
    return NEAT_OK;
}

}  // namespace neat

using namespace neat;

extern "C" long neat_token_logprobs_ws_bytes(int dtype, int R, int V, int k) {
    if (R <= 0 || V <= 0 || k < 0 || k > LP_MAX_K) return 0;
    const LpPlan p = lp_plan(dtype == NEAT_F32 ? 4 : 8, V);
    return p.S == 1 ? 0 : lp_part_bytes(R, p) + (long)R * p.S * k * 8;
}

extern "C" int neat_token_logprobs(const void* logits, long ld, int dtype, const int64_t* target, float scale, int k, float* logp,
                                   float* entropy, float* stats, float* top_logp, int32_t* top_idx, int R, int V, void* ws,
                                   void* stream) {
    if (int rc = lp_check("neat_token_logprobs", logits, ld, dtype, R, V, scale)) return rc;
    NEAT_REQUIRE(!logp || target || R == 0, NEAT_ERR_ARG, "neat_token_logprobs: logp needs targets");
    NEAT_REQUIRE(k >= 0 && k <= LP_MAX_K && k <= V, NEAT_ERR_SHAPE, "neat_token_logprobs: k=%d (at most %d, and V=%d)", k,
                 LP_MAX_K, V);
    NEAT_REQUIRE(k == 0 || R == 0 || (top_logp && top_idx), NEAT_ERR_ARG, "neat_token_logprobs: null pointer (alternatives)");
    if (R == 0) return NEAT_OK;
    const LpPlan p = lp_plan(dtype == NEAT_F32 ? 4 : 8, V);
    NEAT_REQUIRE(p.S == 1 || (ws && ((uintptr_t)ws & 15) == 0), NEAT_ERR_ARG,
                 "neat_token_logprobs: rows of %d need a 16-byte aligned workspace", V);
    LpArgs g{};
    g.z = logits; g.ld = ld; g.target = target; g.scale = scale; g.k = k; g.logp = logp; g.ent = entropy; g.stats = stats;
    g.top = top_logp; g.idx = top_idx; g.R = R; g.V = V; g.S = p.S; g.chunk = p.chunk;
    if (p.S > 1) {
        g.part = static_cast<float*>(ws);
        g.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + lp_part_bytes(R, p));
    }
    hipStream_t s = (hipStream_t)stream;
    return dtype == NEAT_F32 ? lp_forward<float>(g, p, s) : lp_forward<bf16_t>(g, p, s);
}

extern "C" int neat_token_logprobs_bwd(const void* logits, long ld, int dtype, const int64_t* target, const float* stats,
                                       const float* dlogp, const float* dentropy, float scale, void* dlogits, long ld_out, int R,
                                       int V, void* stream) {
    if (int rc = lp_check("neat_token_logprobs_bwd", logits, ld, dtype, R, V, scale)) return rc;
    if (R == 0) return NEAT_OK;
    NEAT_REQUIRE(stats && dlogits, NEAT_ERR_ARG, "neat_token_logprobs_bwd: null pointer");
    NEAT_REQUIRE(!dlogp || target, NEAT_ERR_ARG, "neat_token_logprobs_bwd: dlogp needs targets");
    NEAT_REQUIRE(R <= 1 || ld_out >= V, NEAT_ERR_SHAPE, "neat_token_logprobs_bwd: output row pitch %ld below V=%d", ld_out, V);
    NEAT_REQUIRE(((uintptr_t)dlogits & (dtype == NEAT_F32 ? 3 : 1)) == 0, NEAT_ERR_ARG,
                 "neat_token_logprobs_bwd: gradient is not aligned to its elements");
    if (int rc = lp_check_out("neat_token_logprobs_bwd", logits, ld, dlogits, ld_out, dtype, R, V)) return rc;
    LpArgs g{};
    g.z = logits; g.ld = ld; g.target = target; g.stats = const_cast<float*>(stats); g.a = dlogp; g.b = dentropy; g.scale = scale;
    g.dz = dlogits; g.ldz = ld_out; g.R = R; g.V = V;
    hipStream_t s = (hipStream_t)stream;
    return dtype == NEAT_F32 ? lp_backward<float>(g, s) : lp_backward<bf16_t>(g, s);
}

extern "C" int neat_token_logprobs_fwd_bwd(const void* logits, long ld, int dtype, const int64_t* target, const float* dlogp,
                                           const float* dentropy, float scale, float* logp, float* entropy, float* stats,
                                           void* dlogits, long ld_out, int R, int V, void* ws, void* stream) {
    if (int rc = lp_check("neat_token_logprobs_fwd_bwd", logits, ld, dtype, R, V, scale)) return rc;
    if (R == 0) return NEAT_OK;
    NEAT_REQUIRE(dlogits && (target || (!logp && !dlogp)), NEAT_ERR_ARG, "neat_token_logprobs_fwd_bwd: null pointer");
    NEAT_REQUIRE(R <= 1 || ld_out >= V, NEAT_ERR_SHAPE, "neat_token_logprobs_fwd_bwd: output row pitch %ld below V=%d", ld_out, V);
    NEAT_REQUIRE(((uintptr_t)dlogits & (dtype == NEAT_F32 ? 3 : 1)) == 0, NEAT_ERR_ARG,
                 "neat_token_logprobs_fwd_bwd: gradient is not aligned to its elements");
    if (int rc = lp_check_out("neat_token_logprobs_fwd_bwd", logits, ld, dlogits, ld_out, dtype, R, V)) return rc;
    const LpPlan p = lp_plan(dtype == NEAT_F32 ? 4 : 8, V, true);
    if (p.S > 1) {                            // longer than a workgroup's registers: two passes
        NEAT_REQUIRE(stats, NEAT_ERR_ARG, "neat_token_logprobs_fwd_bwd: rows of %d need stats", V);
        if (int rc = neat_token_logprobs(logits, ld, dtype, target, scale, 0, logp, entropy, stats, nullptr, nullptr, R, V, ws,
                                         stream)) return rc;
        return neat_token_logprobs_bwd(logits, ld, dtype, target, stats, dlogp, dentropy, scale, dlogits, ld_out, R, V, stream);
    }
    LpArgs g{};
    g.z = logits; g.ld = ld; g.target = target; g.a = dlogp; g.b = dentropy; g.scale = scale; g.logp = logp; g.ent = entropy;
    g.stats = stats; g.dz = dlogits; g.ldz = ld_out; g.R = R; g.V = V; g.S = 1; g.chunk = V;
    hipStream_t s = (hipStream_t)stream;
    const char* what = "neat_token_logprobs_fwd_bwd";
    return dtype == NEAT_F32 ? lp_launch<float, LP_GRAD>(g, p, 0, what, s) : lp_launch<bf16_t, LP_GRAD>(g, p, 0, what, s);
}
