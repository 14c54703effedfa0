// The norms before and after a block, fused with its gate and residual scale, forward and backward.
//
//   n = N_post(h)  (or h);   x' = x + n * scale[c] * gate[g(row), c];   y = N_pre(x')
//   N(u) = uh * w + b,  uh = (u - mean u) / sqrt(var u + eps)  (LayerNorm)  or  u / sqrt(mean u^2 + eps)  (RMS)
// h is a block's output (attention, MLP), x the residual stream it joins, y what the next block reads: the junction of towers
// with LayerScale, with norms behind the blocks, or with gates that depend on the sequence.
// Backward, e = d/dx':
//   e = dres + N_pre'(dy);   dx = e;   dn = e * scale * gate;   dh = N_post'(dn)
//   dw_pre = sum dy xh, db_pre = sum dy, dw_post = sum dn hh, db_post = sum dn, dgate[g] = scale * sum_{rows of g} e n,
//   dscale = sum_g gate[g] * sum_{rows of g} e n
//   N'(d) = r (z - mean z - uh mean(z uh)), z = d w (RMS: without mean z)
//
// Both directions read every input once and write every output once: 8 + 2t bytes an element forward, 12 + 3t backward (t = 2
// for bf16, 4 for fp32).  A team of 1 to 8 waves holds a row (up to five 16-B chunks a lane) in registers and takes a contiguous
// run of rows, balanced to one row whatever the groups' lengths.  Column sums stay in registers over the run.  A group's sum is
// left behind at each group's end in slot team + group: runs and groups advance together, so no two (team, group) pairs share a
// slot, and a second launch adds each group's slots, and the column sums, in a fixed order: no atomics, equal bits on every run.
//
// Bound by HBM: 78 848 x 512 (bf16 branch, a gate per 77 rows) forward 90 us (484 MB, 5.4 TB/s), backward 140 us (727 MB, 5.2)
// and 9 us for the sums; 50 000 x 1 280 forward 146 us (768 MB, 5.3).  What is left of 14 851 x 768 in ragged groups (31 + 50 + 10
// us) is the second launch and the teams' partial sums, a tenth of the traffic there.  One row: 3.1 us, a launch's latency.
#include <initializer_list>

#include "wave.h"

namespace neat {

constexpr int RN_MAX_COLS = 4096;
constexpr int RN_MAX_GROUPS = 1 << 30;                    // team + group and the search's probes stay within an int
constexpr int RN_FWD_WAVES = 4, RN_BWD_WAVES = 4;         // waves of a workgroup whose teams are single waves
constexpr int RN_SUMS = 5;                                // column sums: pre_w, pre_b, post_w, post_b, scale

struct RnArgs {
    const float* x;                                       // [rows, cols]; the backward pass's x' stands here
    const void* h;
    const float *pre_w, *pre_b, *post_w, *post_b, *scale, *gate;
    const int32_t* cu;                                    // [groups + 1] or null: groups of rows / groups rows
    float* x_out;
    void* y;
    float* stats;                                         // [4, rows]: mean, 1/deviation of h; of x'
    const void* dy;
    const float* dres;
    float* dx;
    void* dh;
    float* part;                                          // [workgroups, RN_SUMS, cols]
    float* slots;                                         // [teams + groups, cols]
    int rows, cols, groups, teams;
    int rms, zero_rest;
    float eps;
};

// What comes in is read once here and next touched a whole block later: loaded past the caches, as is dx written (together 270 ->
// 244 us for 78 848 x 512 in both directions).  x_out and y are read again at once by what follows: they stay.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x4 rn_once(const float* p, long i) {
    return __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p) + i);
}
template <typename T> struct RnIo;
template <> struct RnIo<float> {
    typedef f32x4 raw;
    static __device__ __forceinline__ raw fetch(const void* p, long i) { return rn_once(static_cast<const float*>(p), i); }
    static __device__ __forceinline__ f32x4 open(raw w) { return w; }
    static __device__ __forceinline__ f32x4 load(const void* p, long i) { return reinterpret_cast<const f32x4*>(p)[i]; }
    static __device__ __forceinline__ void store(void* p, long i, f32x4 v) { reinterpret_cast<f32x4*>(p)[i] = v; }
};
template <> struct RnIo<bf16_t> {
    typedef u32x2 raw;
    static __device__ __forceinline__ raw fetch(const void* p, long i) {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p) + i);
    }
    static __device__ __forceinline__ f32x4 open(raw w) {
        return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u)};
    }
    static __device__ __forceinline__ void store(void* p, long i, f32x4 v) {
        reinterpret_cast<uint2*>(p)[i] = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
    }
};

// a / b of whole numbers, 0 <= a < 2^52: the double quotient cannot reach the next whole number (1 / b is far above its rounding),
// and takes a tenth of the instructions of a 64-bit division
__device__ __forceinline__ long rn_div(long a, long b) { return (long)((double)a / (double)b); }

// rows of one team: [lo, hi) of the rows that belong to a group (all, without cu)
struct RnRun { long lo, hi, used; };
__device__ __forceinline__ long rn_used(const RnArgs& a) {
    if (!a.cu) return a.rows;
    const int u = a.cu[a.groups];
    return u < 0 ? 0 : u > a.rows ? a.rows : u;
}
__device__ __forceinline__ RnRun rn_run(const RnArgs& a, int team) {
    const long used = rn_used(a);
    return RnRun{rn_div(used * team, a.teams), rn_div(used * (team + 1), a.teams), used};
}
// first row behind group g; the last group ends with the rows
__device__ __forceinline__ long rn_group_end(const RnArgs& a, int g, long used) {
    if (g >= a.groups - 1) return used;
    const long e = a.cu ? (long)a.cu[g + 1] : (long)(a.rows / a.groups) * (g + 1);
    return e < used ? e : used;
}
// the group of a row: the first one that ends behind it, by the lanes of a wave together (two rounds for 4 096 groups)
__device__ __forceinline__ int rn_group(const RnArgs& a, long row, long used) {
    if (!a.cu) return (int)rn_div(row, a.rows / a.groups);
    int lo = 0, n = a.groups;                              // it is one of lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 63) >> 6, last = lo + n - 1;
        const int probe = min(lo + (int)(threadIdx.x & 63) * step + step - 1, last);
        const uint64_t behind = __ballot(rn_group_end(a, probe, used) > row);
        const int first = behind ? __builtin_ctzll(behind) : 63;
        lo = min(lo + first * step, last);
        n = min(step, last - lo + 1);
    }
    return lo;
}

// sums over a team; teams of several waves meet in LDS, two places in turn, so that one barrier a sum is enough
template <int WPR>
struct RnTeam {
    float (*red)[2][8];
    int turn;
    __device__ __forceinline__ void sum2(float& p, float& q) {
        p = row_sum(p);
        q = row_sum(q);
        p = (lane_f(p, 0) + lane_f(p, 16)) + (lane_f(p, 32) + lane_f(p, 48));
        q = (lane_f(q, 0) + lane_f(q, 16)) + (lane_f(q, 32) + lane_f(q, 48));
        if constexpr (WPR > 1) {
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) {
                red[turn][0][wave] = p;
                red[turn][1][wave] = q;
            }
            __syncthreads();
            p = q = 0.f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) {
                p += red[turn][0][w];
                q += red[turn][1][w];
            }
            turn ^= 1;
        }
    }
    __device__ __forceinline__ float sum(float p) {
        float q = 0.f;
        sum2(p, q);
        return p;
    }
};

#define RN_EACH(i, c) \
    _Pragma("unroll") for (int i = 0; i < NCH; ++i) \
        if (const int c = lane + 64 * WPR * i; c < nch)

// uh in place of u; (mean, 1/deviation) of the row
template <int WPR, int NCH>
__device__ __forceinline__ float2 rn_unit(f32x4 (&u)[NCH], int lane, int nch, float inv, float eps, int rms, RnTeam<WPR>& team) {
    float mu = 0.f;
    if (!rms) {
        float s = 0.f;
        RN_EACH(i, c) s += (u[i][0] + u[i][1]) + (u[i][2] + u[i][3]);
        mu = team.sum(s) * inv;
    }
    float q = 0.f;
    RN_EACH(i, c) {
        u[i] -= mu;
        q += (u[i][0] * u[i][0] + u[i][1] * u[i][1]) + (u[i][2] * u[i][2] + u[i][3] * u[i][3]);
    }
    const float r = rsqrtf(team.sum(q) * inv + eps);
    RN_EACH(i, c) u[i] *= r;
    return make_float2(mu, r);
}

// weights in LDS, one copy a workgroup: they are read once a row from there, and the registers they would fill hold rows in
// flight.  Zeros (ones) stand for what is not given.
template <int THREADS>
__device__ __forceinline__ void rn_stage(f32x4* dst, const float* src, float otherwise, int nch) {
    for (int c = threadIdx.x; c < nch; c += THREADS)
        dst[c] = src ? RnIo<float>::load(src, c) : f32x4{otherwise, otherwise, otherwise, otherwise};
}

// the factor of a row's branch: scale times its group's gate
template <int WPR, int NCH>
__device__ __forceinline__ void rn_factor(f32x4 (&f)[NCH], const RnArgs& a, int g, int lane, int nch) {
    RN_EACH(i, c) {
        f[i] = RnIo<float>::load(a.gate, (long)g * nch + c);
        if (a.scale) f[i] *= RnIo<float>::load(a.scale, c);
    }
}
__device__ __forceinline__ int rn_next_group(const RnArgs& a, int g, long row, long used) {
    do ++g; while (rn_group_end(a, g, used) <= row && g < a.groups - 1);
    return g;
}

// Waves a SIMD that the forward kernel's registers are kept to (wide: fp32 activations).  Teams of four waves want a few more: 3 to 9
// registers a lane are in scratch with two chunks (1 284 to 2 048 columns, 5.3 to 5.8 TB/s) and with four in bf16 with both norms
// (above 3 072 columns, 5.0 TB/s)
constexpr int rn_fwd_waves(int nch, bool wide) { return nch == 1 ? 7 : nch == 2 ? 6 : nch <= 4 - wide ? 4 : 3; }

template <typename T, int WPR, int NCH, bool POST>
__global__ __launch_bounds__(WPR == 1 ? 64 * RN_FWD_WAVES : 64 * WPR, rn_fwd_waves(NCH, sizeof(T) == 4)) void res_norm_fwd_kernel(RnArgs a) {
    constexpr int THREADS = WPR == 1 ? 64 * RN_FWD_WAVES : 64 * WPR;
    __shared__ float red[2][2][8];
    extern __shared__ __attribute__((aligned(16))) f32x4 lds[];               // pre_w, pre_b, post_w, post_b: [4][cols]
    RnTeam<WPR> sums{red, 0};
    const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int team = WPR == 1 ? blockIdx.x * RN_FWD_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    const int nch = a.cols >> 2;
    const float inv = 1.f / (float)a.cols;
    const RnRun run = rn_run(a, team);
    const f32x4 one = {1.f, 1.f, 1.f, 1.f}, none = {0.f, 0.f, 0.f, 0.f};
    f32x4 x[NCH], f[NCH];
    typename RnIo<T>::raw hn[NCH];
    if (run.lo < run.hi) {                                // the first row is under way while the weights are staged
        RN_EACH(i, c) {
            x[i] = rn_once(a.x, run.lo * nch + c);
            hn[i] = RnIo<T>::fetch(a.h, run.lo * nch + c);
        }
    }
    rn_stage<THREADS>(lds, a.pre_w, 1.f, nch);
    rn_stage<THREADS>(lds + nch, a.pre_b, 0.f, nch);
    if constexpr (POST) {
        rn_stage<THREADS>(lds + 2 * nch, a.post_w, 1.f, nch);
        rn_stage<THREADS>(lds + 3 * nch, a.post_b, 0.f, nch);
    }
    RN_EACH(i, c) f[i] = a.scale ? RnIo<float>::load(a.scale, c) : one;
    __syncthreads();
    int g = -1;
    long end = a.gate ? run.lo : run.used;
    for (long row = run.lo; row < run.hi; ++row) {
        const long base = row * nch;
        f32x4 h[NCH], xn[NCH];
        RN_EACH(i, c) h[i] = RnIo<T>::open(hn[i]);
        if (row + 1 < run.hi) {                           // the next row, while this one is worked on
            RN_EACH(i, c) {
                xn[i] = rn_once(a.x, base + nch + c);
                hn[i] = RnIo<T>::fetch(a.h, base + nch + c);
            }
        }
        if (row >= end) {
            g = g < 0 ? rn_group(a, row, run.used) : rn_next_group(a, g, row, run.used);
            end = rn_group_end(a, g, run.used);
            rn_factor<WPR, NCH>(f, a, g, lane, nch);
        }
        float2 s1 = make_float2(0.f, 1.f);
        if constexpr (POST) {
            s1 = rn_unit<WPR, NCH>(h, lane, nch, inv, a.eps, a.rms, sums);
            RN_EACH(i, c) h[i] = h[i] * lds[2 * nch + c] + lds[3 * nch + c];
        }
        RN_EACH(i, c) {
            x[i] += h[i] * f[i];
            RnIo<float>::store(a.x_out, base + c, x[i]);
        }
        const float2 s2 = rn_unit<WPR, NCH>(x, lane, nch, inv, a.eps, a.rms, sums);
        RN_EACH(i, c) RnIo<T>::store(a.y, base + c, x[i] * lds[c] + lds[nch + c]);
        if (a.stats && lane == 0) {
            a.stats[row] = s1.x;
            a.stats[(long)a.rows + row] = s1.y;
            a.stats[2L * a.rows + row] = s2.x;
            a.stats[3L * a.rows + row] = s2.y;
        }
        RN_EACH(i, c) x[i] = xn[i];
    }
    if (a.zero_rest) {                                    // rows behind the last group, in outputs that nobody has filled
        for (long row = run.used + team; row < a.rows; row += a.teams) {
            RN_EACH(i, c) {
                if (a.zero_rest & 1) RnIo<float>::store(a.x_out, row * nch + c, none);
                if (a.zero_rest & 2) RnIo<T>::store(a.y, row * nch + c, none);
            }
        }
    }
}

// Waves a SIMD that the backward kernel's registers are kept to: two rows in flight a wave and fewer waves are faster than one
// row and one wave more (14 851 x 768: 91 against 96 us in both directions).
constexpr int rn_bwd_waves(int nch) { return nch == 1 ? 4 : nch == 2 ? 3 : 2; }
template <typename T, int WPR, int NCH, bool POST>
__global__ __launch_bounds__(WPR == 1 ? 64 * RN_BWD_WAVES : 64 * WPR, rn_bwd_waves(NCH)) void res_norm_bwd_kernel(RnArgs a) {
    constexpr int TEAMS = WPR == 1 ? RN_BWD_WAVES : 1, THREADS = 64 * WPR * TEAMS;
    __shared__ float red[2][2][8];
    // pre_w, post_w, post_b: [3][cols]; behind them a team's sum of gate times group sums [TEAMS][cols]; at the end the sums
    extern __shared__ __attribute__((aligned(16))) f32x4 lds[];
    RnTeam<WPR> sums{red, 0};
    const int wave = WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int team = blockIdx.x * TEAMS + wave;
    const int nch = a.cols >> 2;
    const float inv = 1.f / (float)a.cols;
    const RnRun run = rn_run(a, team);
    const f32x4 one = {1.f, 1.f, 1.f, 1.f}, none = {0.f, 0.f, 0.f, 0.f};
    const bool scaled = a.scale || a.gate;
    f32x4* gated = lds + (3 + wave) * nch;
    rn_stage<THREADS>(lds, a.pre_w, 1.f, nch);
    if constexpr (POST) {
        rn_stage<THREADS>(lds + nch, a.post_w, 1.f, nch);
        rn_stage<THREADS>(lds + 2 * nch, a.post_b, 0.f, nch);
    }
    f32x4 f[NCH];
    f32x4 sum[4][NCH], own[NCH];                          // own: sum of e n over the current group (all rows, without a gate)
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        own[i] = none;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k][i] = none;
    }
    RN_EACH(i, c) {
        f[i] = a.scale ? RnIo<float>::load(a.scale, c) : one;
        if (a.gate) gated[c] = none;
    }
    __syncthreads();
    struct {
        typename RnIo<T>::raw d[NCH], h[NCH];
        f32x4 x[NCH], e[NCH];
        float stat[4];
    } next;
    const auto fetch = [&](long row) {
        const long base = row * nch;
        RN_EACH(i, c) {
            next.d[i] = RnIo<T>::fetch(a.dy, base + c);
            next.x[i] = rn_once(a.x, base + c);
            next.e[i] = a.dres ? rn_once(a.dres, base + c) : none;
            next.h[i] = RnIo<T>::fetch(a.h, base + c);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) next.stat[k] = a.stats[(long)k * a.rows + row];
    };
    if (run.lo < run.hi) fetch(run.lo);
    int g = -1;
    long end = a.gate ? run.lo : run.used;
    for (long row = run.lo; row < run.hi; ++row) {
        const long base = row * nch;
        f32x4 d[NCH], x[NCH], e[NCH], h[NCH];
        RN_EACH(i, c) {
            d[i] = RnIo<T>::open(next.d[i]);
            x[i] = next.x[i];
            e[i] = next.e[i];
            h[i] = RnIo<T>::open(next.h[i]);
        }
        const float mu1 = next.stat[0], r1 = next.stat[1], mu2 = next.stat[2], r2 = next.stat[3];
        if (row + 1 < run.hi) fetch(row + 1);             // the next row, while this one is worked on
        if (row >= end) {
            if (g >= 0) {
                RN_EACH(i, c) {
                    RnIo<float>::store(a.slots, (long)(team + g) * nch + c, own[i]);
                    gated[c] += own[i] * RnIo<float>::load(a.gate, (long)g * nch + c);
                    own[i] = none;
                }
            }
            g = g < 0 ? rn_group(a, row, run.used) : rn_next_group(a, g, row, run.used);
            end = rn_group_end(a, g, run.used);
            rn_factor<WPR, NCH>(f, a, g, lane, nch);
        }
        float p = 0.f, q = 0.f;
        RN_EACH(i, c) {
            x[i] = (x[i] - mu2) * r2;
            sum[0][i] += d[i] * x[i];
            sum[1][i] += d[i];
            d[i] *= lds[c];
            p += (d[i][0] + d[i][1]) + (d[i][2] + d[i][3]);
            q += (d[i][0] * x[i][0] + d[i][1] * x[i][1]) + (d[i][2] * x[i][2] + d[i][3] * x[i][3]);
        }
        sums.sum2(p, q);
        p = a.rms ? 0.f : p * inv;
        q *= inv;
        RN_EACH(i, c) {
            e[i] += (d[i] - p - x[i] * q) * r2;
            __builtin_nontemporal_store(e[i], reinterpret_cast<f32x4*>(a.dx) + base + c);
        }
        if constexpr (POST) {
            p = q = 0.f;
            RN_EACH(i, c) {
                const f32x4 w1 = lds[nch + c];
                h[i] = (h[i] - mu1) * r1;
                if (scaled) own[i] += e[i] * (h[i] * w1 + lds[2 * nch + c]);
                e[i] *= f[i];
                sum[2][i] += e[i] * h[i];
                sum[3][i] += e[i];
                e[i] *= w1;
                p += (e[i][0] + e[i][1]) + (e[i][2] + e[i][3]);
                q += (e[i][0] * h[i][0] + e[i][1] * h[i][1]) + (e[i][2] * h[i][2] + e[i][3] * h[i][3]);
            }
            sums.sum2(p, q);
            p = a.rms ? 0.f : p * inv;
            q *= inv;
            RN_EACH(i, c) RnIo<T>::store(a.dh, base + c, (e[i] - p - h[i] * q) * r1);
        } else {
            RN_EACH(i, c) {
                if (scaled) own[i] += e[i] * h[i];
                RnIo<T>::store(a.dh, base + c, e[i] * f[i]);
            }
        }
    }
    if (a.gate) {
        if (g >= 0) {
            RN_EACH(i, c) {
                RnIo<float>::store(a.slots, (long)(team + g) * nch + c, own[i]);
                own[i] = gated[c] + own[i] * RnIo<float>::load(a.gate, (long)g * nch + c);
            }
        }
    }
    if (a.zero_rest) {
        for (long row = run.used + team; row < a.rows; row += a.teams) {
            RN_EACH(i, c) {
                if (a.zero_rest & 1) RnIo<float>::store(a.dx, row * nch + c, none);
                if (a.zero_rest & 2) RnIo<T>::store(a.dh, row * nch + c, none);
            }
        }
    }
    // the workgroup's column sums, one kind after the other
    float* part = a.part + (long)blockIdx.x * RN_SUMS * a.cols;
    if constexpr (TEAMS == 1) {
#pragma unroll
        for (int k = 0; k < RN_SUMS; ++k) RN_EACH(i, c) RnIo<float>::store(part, (long)k * nch + c, k < 4 ? sum[k & 3][i] : own[i]);
    } else {
#pragma unroll
        for (int k = 0; k < RN_SUMS; ++k) {
            __syncthreads();
            RN_EACH(i, c) lds[wave * nch + c] = k < 4 ? sum[k & 3][i] : own[i];
            __syncthreads();
            for (int c = threadIdx.x; c < nch; c += THREADS) {
                f32x4 s = lds[c];
#pragma unroll
                for (int w = 1; w < TEAMS; ++w) s += lds[w * nch + c];
                RnIo<float>::store(part, (long)k * nch + c, s);
            }
        }
    }
}

// Second launch of the backward pass: column sums over workgroups, and each group's slots.  64 columns x 16 slices.
constexpr int RNF_SLICES = 16;
constexpr int RNF_LONG = 128;                             // slots that one slice adds up alone
struct RnOut { float* col[RN_SUMS]; float* gate; };
__global__ __launch_bounds__(64 * RNF_SLICES) void res_norm_finalize_kernel(RnArgs a, RnOut o, int blocks, int col_blocks,
                                                                           int gate_rows) {
    __shared__ float red[RNF_SLICES][64];
    const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
    const int cb = cdiv_dev(a.cols, 64);
    if ((int)blockIdx.x < col_blocks) {
        const int k = blockIdx.x / cb, c = (blockIdx.x % cb) * 64 + lane;
        if (!o.col[k]) return;
        float s = 0.f;
        if (c < a.cols)
#pragma unroll 8
            for (int b = slice; b < blocks; b += RNF_SLICES) s += a.part[((long)b * RN_SUMS + k) * a.cols + c];
        red[slice][lane] = s;
        __syncthreads();
        if (slice == 0 && c < a.cols) {
            s = 0.f;
#pragma unroll
            for (int i = 0; i < RNF_SLICES; ++i) s += red[i][lane];
            o.col[k][c] = s;
        }
        return;
    }
    // gate_rows == 1: 16 slices of one group's slots; else one group a slice, and all slices together, one after the other, the
    // groups that are long beside their neighbours (one sequence of 13 831 rows among 1 020 of one has 1 907 slots: one by one they
    // are off by as many roundings, and the backward pass of 768 bf16 columns takes 278 us instead of 91)
    __shared__ long first[RNF_SLICES], count[RNF_SLICES];
    const int rest = blockIdx.x - col_blocks;
    const int c = (rest % cb) * 64 + lane;
    const int g = (rest / cb) * gate_rows + (gate_rows == 1 ? 0 : slice);
    const long used = rn_used(a);
    // the teams from the one with a group's first row to the one with its last; with fewer rows than teams most have none, and the
    // rows' own teams are gone through
    const bool few = used < a.teams;
    long w0 = 0, n = 0;                                   // few: the first row
    if (g < a.groups) {
        const long lo = g == 0 ? 0 : rn_group_end(a, g - 1, used), hi = rn_group_end(a, g, used);
        if (lo >= 0 && hi > lo) {
            w0 = few ? lo : rn_div((lo + 1) * a.teams - 1, used);
            n = few ? hi - lo : rn_div(hi * a.teams - 1, used) - w0 + 1;
        }
    }
    const auto add = [&](int group, long at, long n, long j, int step) {
        float s = 0.f;
#pragma unroll 4
        for (; j < n; j += step) {
            const long w = few ? rn_div((at + j + 1) * a.teams - 1, used) : at + j;
            s += a.slots[(w + group) * a.cols + c];
        }
        return s;
    };
    const auto join = [&] {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < RNF_SLICES; ++i) s += red[i][lane];
        return s;
    };
    float s = 0.f;
    if (gate_rows == 1) {
        red[slice][lane] = c < a.cols ? add(g, w0, n, slice, RNF_SLICES) : 0.f;
        __syncthreads();
        if (slice != 0) return;
        s = join();
    } else {
        if (lane == 0) {
            first[slice] = w0;
            count[slice] = n;
        }
        if (n <= RNF_LONG && c < a.cols) s = add(g, w0, n, 0, 1);
        __syncthreads();
        // which of them are long: the same for the whole workgroup, and mostly none
        for (uint64_t some = __ballot(lane < RNF_SLICES && count[lane & (RNF_SLICES - 1)] > RNF_LONG); some; some &= some - 1) {
            const int q = __builtin_ctzll(some);
            red[slice][lane] = c < a.cols ? add(g - slice + q, first[q], count[q], slice, RNF_SLICES) : 0.f;
            __syncthreads();
            if (slice == q) s = join();
            __syncthreads();
        }
    }
    if (g < a.groups && c < a.cols) o.gate[(long)g * a.cols + c] = a.scale ? s * a.scale[c] : s;
}

// Waves of a team.  Forward a lane holds up to five chunks of x and h, backward three beside five sums of them: with four the
// registers spill (30 M elements backward, TB/s with four / three chunks: 1 024 columns 1.8 / 4.7, 2 048 1.6 / 4.9).
// fp32 activations take twice the registers in flight: two chunks (20 M elements backward at 768 columns 3.9 TB/s with three).
static int rn_bwd_wave_cols(bool wide) { return wide ? 512 : 768; }
static int rn_fwd_wpr(int cols) { return cols <= 1280 ? 1 : 4; }
static int rn_bwd_wpr(int cols, bool wide) {
    const int w = rn_bwd_wave_cols(wide);
    return cols <= w ? 1 : cols <= 2 * w ? 2 : cols <= 4 * w ? 4 : 8;
}
// Where all workgroups can run at once (by registers and LDS; forward every one has four waves) with at most four rows a team, as
// few rows as that takes.  6 M bf16 elements at 768 columns with both norms 4.3 / 5.0 / 3.9 TB/s with one / two / four, 11 M 4.4 /
// 4.8 / 5.0, 12 M at 1 024 columns 4.5 / 4.9 / 4.8 and 5.2 with the three that the rule takes.
// Beyond that two: more leave the chip's last workgroups uneven, one loads the weights for every row.  40 M at 512 / 1 024 columns
// 4.8 / 5.2 TB/s with one, 5.3 / 5.1 with two, 5.0 / 4.8 with four; 50 000 x 1 280 with one norm 147 / 146 / 156 us.
// A workgroup that is one team and stages two norms' weights wants more rows for them: 40 M at 1 664 / 2 560 / 4 096 columns 4.8 /
// 4.4 / 4.2 TB/s with two, 4.9 / 4.6 / 4.6 with four, 4.8 / 4.4 / 4.3 with six; 4 M at 4 096 2.5 with one, 3.1 with two.
// At most 2^18 workgroups: rows times teams stay below the 2^52 that the row runs' quotients are exact for.
static int rn_fwd_blocks(int rows, int cols, bool wide, bool post) {
    const int wpr = rn_fwd_wpr(cols), all = cdiv(rows, wpr == 1 ? RN_FWD_WAVES : 1);
    const int waves = rn_fwd_waves(cdiv(cols / 4, 64 * wpr), wide), by_lds = 160 * 1024 / ((post ? 16 : 8) * cols + 64);
    const int few = cdiv(all, 256 * (by_lds < waves ? by_lds : waves));
    const bool staged = wpr > 1 && post;
    const int run = few > 4 ? (staged ? 4 : 2) : few == 1 && staged && all > 512 ? 2 : few, b = cdiv(all, run);
    return b < 1 << 18 ? b : 1 << 18;
}
// Backward every workgroup leaves sums behind: as many as run at once, whole ones on each of the 256 CUs, and two rows a team.  40 M
// bf16 elements with both norms at 768 / 4 096 columns 4.5 / 4.3 TB/s with half as many, 5.1 / 4.9 so, 5.0 / 4.6 with twice as many
// (4.1 at 4 096 with one and a half a CU; 20 M fp32 at 128 columns 3.3 with five workgroups a CU of which four run, 4.4 with four).
static int rn_bwd_blocks(int rows, int cols, bool wide) {
    const int wpr = rn_bwd_wpr(cols, wide), per = wpr == 1 ? RN_BWD_WAVES : 1;
    const int most = 256 * (4 * rn_bwd_waves(cdiv(cols / 4, 64 * wpr)) / (wpr * per)), b = cdiv(rows, per * 2);
    return b < 1 ? 1 : b > most ? most : b;
}

// dynamic LDS that any launch may have beside the static, and the most that is asked for (4 rows of 4 096 columns)
constexpr size_t RN_PLAIN_LDS = 60 * 1024;
constexpr int RN_MOST_LDS = 64 * 1024;
template <typename T, bool POST> struct RnForward {
    template <int WPR, int NCH> static int go(const RnArgs& a, int blocks, hipStream_t s) {
        const size_t lds = (size_t)(POST ? 4 : 2) * a.cols * 4;
        if (lds > RN_PLAIN_LDS) {
            static unsigned long long done = 0;
            if (int rc = ensure_dynamic_lds((const void*)res_norm_fwd_kernel<T, WPR, NCH, POST>, RN_MOST_LDS, &done, "neat_res_norm_fwd"))
                return rc;
        }
        hipLaunchKernelGGL((res_norm_fwd_kernel<T, WPR, NCH, POST>), dim3(blocks),
                           dim3(WPR == 1 ? 64 * RN_FWD_WAVES : 64 * WPR), lds, s, a);
        NEAT_LAUNCH_CHECK("neat_res_norm_fwd");
        return NEAT_OK;
    }
    static int pick(const RnArgs& a, int blocks, hipStream_t s) {
        const int wpr = rn_fwd_wpr(a.cols);
        const int nch = cdiv(a.cols / 4, 64 * wpr);
        if (wpr == 1) {
            switch (nch) {
                case 1: return go<1, 1>(a, blocks, s);
                case 2: return go<1, 2>(a, blocks, s);
                case 3: return go<1, 3>(a, blocks, s);
                case 4: return go<1, 4>(a, blocks, s);
                default: return go<1, 5>(a, blocks, s);
            }
        }
        return nch == 2 ? go<4, 2>(a, blocks, s) : nch == 3 ? go<4, 3>(a, blocks, s) : go<4, 4>(a, blocks, s);
    }
};
template <typename T, bool POST> struct RnBackward {
    template <int WPR, int NCH> static int go(const RnArgs& a, int blocks, hipStream_t s) {
        const int teams = WPR == 1 ? RN_BWD_WAVES : 1, rows = 3 + (a.gate ? teams : 0);     // at least `teams`, for the sums
        const size_t lds = (size_t)(rows > teams ? rows : teams) * a.cols * 4;
        if (lds > RN_PLAIN_LDS) {
            static unsigned long long done = 0;
            if (int rc = ensure_dynamic_lds((const void*)res_norm_bwd_kernel<T, WPR, NCH, POST>, RN_MOST_LDS, &done, "neat_res_norm_bwd"))
                return rc;
        }
        hipLaunchKernelGGL((res_norm_bwd_kernel<T, WPR, NCH, POST>), dim3(blocks),
                           dim3(WPR == 1 ? 64 * RN_BWD_WAVES : 64 * WPR), lds, s, a);
        NEAT_LAUNCH_CHECK("neat_res_norm_bwd");
        return NEAT_OK;
    }
    static int pick(const RnArgs& a, int blocks, hipStream_t s) {
        const int wpr = rn_bwd_wpr(a.cols, sizeof(T) == 4), nch = cdiv(a.cols / 4, 64 * wpr);
        if constexpr (sizeof(T) == 2) {
            if (nch == 3) return wpr == 1 ? go<1, 3>(a, blocks, s) : wpr == 2 ? go<2, 3>(a, blocks, s) : go<4, 3>(a, blocks, s);
        }
        if (nch == 1) return go<1, 1>(a, blocks, s);
        return wpr == 1 ? go<1, 2>(a, blocks, s) : wpr == 2 ? go<2, 2>(a, blocks, s) : wpr == 4 ? go<4, 2>(a, blocks, s) : go<8, 2>(a, blocks, s);
    }
};
template <template <typename, bool> class Launch>
static int rn_pick(int dtype, const RnArgs& a, int blocks, hipStream_t s) {
    if (dtype == NEAT_F32) return a.post_w ? Launch<float, true>::pick(a, blocks, s) : Launch<float, false>::pick(a, blocks, s);
    return a.post_w ? Launch<bf16_t, true>::pick(a, blocks, s) : Launch<bf16_t, false>::pick(a, blocks, s);
}

static bool rn_aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
static int rn_check(const char* who, const RnArgs& a, int dtype, int kind) {
    NEAT_REQUIRE(dtype == NEAT_F32 || dtype == NEAT_BF16, NEAT_ERR_ARG, "%s: dtype=%d", who, dtype);
    NEAT_REQUIRE(kind == NEAT_NORM_LAYER || kind == NEAT_NORM_RMS, NEAT_ERR_ARG, "%s: kind=%d", who, kind);
    NEAT_REQUIRE(a.rows >= 0 && a.cols > 0 && a.cols % 4 == 0 && a.cols <= RN_MAX_COLS, NEAT_ERR_SHAPE,
                 "%s: rows=%d cols=%d unsupported (cols %% 4 == 0, <= %d)", who, a.rows, a.cols, RN_MAX_COLS);
    NEAT_REQUIRE(a.groups <= RN_MAX_GROUPS, NEAT_ERR_SHAPE, "%s: groups=%d is too large", who, a.groups);
    NEAT_REQUIRE(a.groups >= 0 && (a.gate == nullptr) == (a.groups == 0), NEAT_ERR_ARG, "%s: groups=%d need a gate each", who, a.groups);
    NEAT_REQUIRE(!a.cu || a.gate, NEAT_ERR_ARG, "%s: cu without a gate", who);
    NEAT_REQUIRE(!a.gate || a.cu || a.rows % a.groups == 0, NEAT_ERR_SHAPE, "%s: rows=%d do not divide into %d groups", who,
                 a.rows, a.groups);
    NEAT_REQUIRE(!a.post_b || a.post_w, NEAT_ERR_ARG, "%s: post_b without post_w", who);
    for (const void* p : {(const void*)a.x, (const void*)a.pre_w, (const void*)a.pre_b, (const void*)a.post_w,
                          (const void*)a.post_b, (const void*)a.scale, (const void*)a.gate, (const void*)a.x_out,
                          (const void*)a.dres, (const void*)a.dx, (const void*)a.part})
        NEAT_REQUIRE(rn_aligned(p, 16), NEAT_ERR_ARG, "%s: a float32 array is not 16-byte aligned", who);
    for (const void* p : {a.h, (const void*)a.y, a.dy, (const void*)a.dh})
        NEAT_REQUIRE(rn_aligned(p, dtype == NEAT_F32 ? 16 : 8), NEAT_ERR_ARG, "%s: an activation is not aligned to four elements", who);
    return NEAT_OK;
}

// A byte range of an argument; row_elem: the element's size where it is [rows, cols] (such arrays may lie over each other exactly: a
// row is read before anything is written in its place), else 0.
struct RnSpan { const void* p; long bytes; int row_elem; };
static bool rn_meet(const RnSpan& a, const RnSpan& b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
static int rn_apart(const char* who, std::initializer_list<RnSpan> outs, std::initializer_list<RnSpan> ins) {
    for (const RnSpan* o = outs.begin(); o != outs.end(); ++o) {
        for (const RnSpan* q = o + 1; q != outs.end(); ++q)
            NEAT_REQUIRE(!rn_meet(*o, *q), NEAT_ERR_ARG, "%s: two outputs overlap", who);
        for (const RnSpan& i : ins)
            NEAT_REQUIRE(!rn_meet(*o, i) || (o->p == i.p && o->row_elem && o->row_elem == i.row_elem), NEAT_ERR_ARG,
                         "%s: an output overlaps an input (it may lie over an activation of its element size exactly)", who);
    }
    return NEAT_OK;
}

}  // namespace neat

using namespace neat;

extern "C" int neat_res_norm_fwd(const float* x, const void* h, int dtype, int kind, const float* pre_w, const float* pre_b,
                                 const float* post_w, const float* post_b, const float* scale, const float* gate, int groups,
                                 const int32_t* cu, float* x_out, void* y, float* stats, int zero_rest, int rows, int cols,
                                 float eps, void* stream) {
    RnArgs a{};
    a.x = x; a.h = h; a.pre_w = pre_w; a.pre_b = pre_b; a.post_w = post_w; a.post_b = post_b; a.scale = scale; a.gate = gate;
    a.groups = groups; a.cu = cu; a.x_out = x_out; a.y = y; a.stats = stats; a.zero_rest = zero_rest; a.rows = rows; a.cols = cols;
    a.rms = kind == NEAT_NORM_RMS; a.eps = eps;
    if (int rc = rn_check("neat_res_norm_fwd", a, dtype, kind)) return rc;
    if (rows == 0) return NEAT_OK;
    NEAT_REQUIRE(x && h && pre_w && x_out && y, NEAT_ERR_ARG, "neat_res_norm_fwd: null pointer");
    const int t = dtype == NEAT_F32 ? 4 : 2;
    const long n = (long)rows * cols, w = 4L * cols;
    if (int rc = rn_apart("neat_res_norm_fwd", {{x_out, 4 * n, 4}, {y, t * n, t}, {stats, 16L * rows, 0}},
                          {{x, 4 * n, 4}, {h, t * n, t}, {pre_w, w, 0}, {pre_b, w, 0}, {post_w, w, 0}, {post_b, w, 0}, {scale, w, 0},
                           {gate, w * groups, 0}, {cu, 4L * groups + 4, 0}})) return rc;
    const int blocks = rn_fwd_blocks(rows, cols, dtype == NEAT_F32, post_w != nullptr);
    a.teams = blocks * (rn_fwd_wpr(cols) == 1 ? RN_FWD_WAVES : 1);
    return rn_pick<RnForward>(dtype, a, blocks, (hipStream_t)stream);
}

extern "C" long neat_res_norm_ws_floats(int dtype, int rows, int cols, int groups) {
    if (rows < 0 || cols <= 0 || cols > RN_MAX_COLS || groups < 0) return 0;
    const bool wide = dtype == NEAT_F32;
    const long blocks = rn_bwd_blocks(rows, cols, wide), teams = blocks * (rn_bwd_wpr(cols, wide) == 1 ? RN_BWD_WAVES : 1);
    return blocks * RN_SUMS * cols + (groups ? (teams + groups) * cols : 0);
}

extern "C" int neat_res_norm_bwd(const void* dy, const float* dres, const void* h, const float* x_out, const float* stats, int dtype,
                                 int kind, const float* pre_w, const float* post_w, const float* post_b, const float* scale,
                                 const float* gate, int groups, const int32_t* cu, float* dx, void* dh, float* dpre_w,
                                 float* dpre_b, float* dpost_w, float* dpost_b, float* dscale, float* dgate, float* ws,
                                 int zero_rest, int rows, int cols, void* stream) {
    RnArgs a{};
    a.dy = dy; a.dres = dres; a.h = h; a.x = x_out; a.stats = const_cast<float*>(stats); a.pre_w = pre_w; a.post_w = post_w;
    a.post_b = post_b; a.scale = scale; a.gate = gate; a.groups = groups; a.cu = cu; a.dx = dx; a.dh = dh; a.part = ws;
    a.zero_rest = zero_rest; a.rows = rows; a.cols = cols; a.rms = kind == NEAT_NORM_RMS;
    if (int rc = rn_check("neat_res_norm_bwd", a, dtype, kind)) return rc;
    NEAT_REQUIRE((dy && h && x_out && stats && dx && dh) || rows == 0, NEAT_ERR_ARG, "neat_res_norm_bwd: null pointer");
    NEAT_REQUIRE(pre_w && ws, NEAT_ERR_ARG, "neat_res_norm_bwd: null pointer");
    NEAT_REQUIRE((!dpost_w && !dpost_b) || post_w, NEAT_ERR_ARG, "neat_res_norm_bwd: gradients of a norm that is not there");
    NEAT_REQUIRE((!dscale || scale) && (!dgate || gate), NEAT_ERR_ARG, "neat_res_norm_bwd: gradients of a scale or gate that is not there");
    const int t = dtype == NEAT_F32 ? 4 : 2;
    const long n = (long)rows * cols, w = 4L * cols, ws_bytes = 4 * neat_res_norm_ws_floats(dtype, rows, cols, groups);
    const RnSpan sc = {scale, w, 0}, gt = {gate, w * groups, 0}, at = {cu, 4L * groups + 4, 0};
    const RnSpan o1 = {dx, 4 * n, 4}, o2 = {dh, t * n, t}, o3 = {ws, ws_bytes, 0};
    if (int rc = rn_apart("neat_res_norm_bwd", {o1, o2, o3},
                          {{dy, t * n, t}, {dres, 4 * n, 4}, {h, t * n, t}, {x_out, 4 * n, 4}, {stats, 16L * rows, 0}, {pre_w, w, 0},
                           {post_w, w, 0}, {post_b, w, 0}, sc, gt, at})) return rc;
    // the sums are written by the second launch, which reads these
    if (int rc = rn_apart("neat_res_norm_bwd", {{dpre_w, w, 0}, {dpre_b, w, 0}, {dpost_w, w, 0}, {dpost_b, w, 0}, {dscale, w, 0},
                          {dgate, w * groups, 0}}, {o1, o2, o3, sc, at})) return rc;
    const bool wide = dtype == NEAT_F32;
    const int blocks = rn_bwd_blocks(rows, cols, wide);
    a.teams = blocks * (rn_bwd_wpr(cols, wide) == 1 ? RN_BWD_WAVES : 1);
    a.slots = gate ? ws + (long)blocks * RN_SUMS * cols : nullptr;
    const int cb = cdiv(cols, 64);
    // few groups with many slots each: 16 slices a group; many groups: one slice each
    const int gate_rows = groups > 0 && a.teams / groups >= 8 ? 1 : RNF_SLICES;
    const long col_blocks = RN_SUMS * cb, gate_blocks = dgate ? (long)cb * cdiv(groups, gate_rows) : 0;
    NEAT_REQUIRE((col_blocks + gate_blocks) * 64 * RNF_SLICES < 1L << 32, NEAT_ERR_SHAPE,
                 "neat_res_norm_bwd: a gate of groups=%d x cols=%d is too large for its gradient", groups, cols);
    hipStream_t s = (hipStream_t)stream;
    if (int rc = rn_pick<RnBackward>(dtype, a, blocks, s)) return rc;
    const RnOut o{{dpre_w, dpre_b, dpost_w, dpost_b, dscale}, dgate};
    hipLaunchKernelGGL(res_norm_finalize_kernel, dim3((unsigned)(col_blocks + gate_blocks)), dim3(64 * RNF_SLICES), 0, s, a, o, blocks,
                       (int)col_blocks, gate_rows);
    NEAT_LAUNCH_CHECK("neat_res_norm_bwd (sums)");
    return NEAT_OK;
}
