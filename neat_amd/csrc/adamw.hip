// AdamW over many tensors at once, moments in 32 or in 8 bits.
//
// Same rule as neat_adamw_flat (torch.optim.AdamW, reference main_TTA.py:271), for tensors that stay where they are:
//   p *= 1 - lr wd;  m += (g - m)(1 - b1);  v = v b2 + g g (1 - b2);  p -= lr/bc1 * m / (sqrt(v)/sqrt(bc2) + eps)
// The moments of all tensors lie in two caller-owned arrays, cut into blocks of 256 elements of ONE tensor.
//
// 8 bits: a block of m is 256 e4m3 numbers and one power of two, a block of v the same for sqrt(v).  The root halves v's range of
// exponents, so that both moments lose gradients below 2^-18 of the block's largest only.  A power of two makes scaling exact:
// the one rounding is e4m3's (half a step, 2^-4 of the value).  It is chosen so that the block's largest lies in (224, 448] times
// it, 448 being e4m3's largest.  A root above zero never becomes zero (it is held at the smallest code): a second moment lost
// beside a first moment that is not would blow the next step up.  The step itself uses the moments before they are rounded.
//
// Mapping: a wave takes four blocks, a row of 16 lanes each, four times four contiguous elements a lane: whole 256-B runs of
// fp32 per row and load, one reduction for four blocks, and all loads of a unit in flight together.  Tensor addresses travel as
// kernel arguments (96 tensors a launch): no table in device memory, so no copy to order behind other work and none to keep alive.
//
// Bound by HBM: 37.7 M fp32 parameters in 144 tensors 183 us (1 059 MB, 5.8 TB/s); in bf16 with 8-bit moments 80 us (381 MB, 4.7
// TB/s).  Small tensors are bound by the host: 6 us of 15 for 48 x 512.
#include <math.h>

#include "common.h"

namespace neat {

constexpr int AW_BLOCK = 256;       // elements per block of moments = 16 lanes x 16
constexpr int AW_WAVES = 4;
constexpr int AW_UNIT = 4;          // blocks a wave takes, one for each row of 16 lanes
constexpr long AW_MOST = 1L << 26;  // units of a launch: 2^32 work items are the limit
constexpr int AW_TENSORS = 96;      // 96 x 40 B of kernel arguments beside the launch's own ~80 B; 4 096 B is the limit

struct AwTensor {
    void* p;
    const void* g;
    long n;
    uint32_t unit0;                 // its first unit in the launch
    uint32_t state_block;           // its first block in the moment arrays
    float step_size, inv_sqrt_bc2;
};

struct AwLaunch {
    void *m, *v;
    float *ms, *vs;
    uint32_t count, units;
    double omb1_64, b2_64, omb2_64; // 1 - beta1, beta2, 1 - beta2 as the caller has them
    float decay, omb1, b2, omb2, eps;
    AwTensor t[AW_TENSORS];
};
static_assert(sizeof(AwLaunch) <= 4096, "kernel arguments");

// Everything is touched once a step: loaded and stored past the caches (37.7 M fp32 parameters 210 -> 191 us).  Gradients are
// often views of a communication bucket that start at any element: loads of four elements need the element's own alignment
// only (global memory takes unaligned wide accesses).
template <typename T> struct AwIo;
template <> struct AwIo<float> {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ f32x4 load(const void* p, long i) {
        return __builtin_nontemporal_load(reinterpret_cast<const vec*>(static_cast<const float*>(p) + i));
    }
    static __device__ __forceinline__ void store(void* p, long i, f32x4 x) {
        __builtin_nontemporal_store((vec)x, reinterpret_cast<vec*>(static_cast<float*>(p) + i));
    }
    static __device__ __forceinline__ float load1(const void* p, long i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store1(void* p, long i, float x) { static_cast<float*>(p)[i] = x; }
};
template <> struct AwIo<bf16_t> {
    typedef uint32_t vec __attribute__((ext_vector_type(2), aligned(2)));
    static __device__ __forceinline__ f32x4 load(const void* p, long i) {
        const vec w = __builtin_nontemporal_load(reinterpret_cast<const vec*>(static_cast<const bf16_t*>(p) + i));
        return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u)};
    }
    static __device__ __forceinline__ void store(void* p, long i, f32x4 x) {
        vec w = {pack2bf(x[0], x[1]), pack2bf(x[2], x[3])};
        __builtin_nontemporal_store(w, reinterpret_cast<vec*>(static_cast<bf16_t*>(p) + i));
    }
    static __device__ __forceinline__ float load1(const void* p, long i) { return bf2f(static_cast<const bf16_t*>(p)[i]); }
    static __device__ __forceinline__ void store1(void* p, long i, float x) { static_cast<bf16_t*>(p)[i] = f2bf(x); }
};

// Largest x <= 448 x 2^e fixes e; both as bits, x >= 0 and normal or zero (a block of zeros takes the smallest power).
// For a first moment |m|: one more where the mantissa is above 448 / 256 = 1.75.
__device__ __forceinline__ int aw_exponent(uint32_t u) {
    const int e = (int)(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
// The same for a root, from the second moment itself: sqrt(v) <= 448 x 2^e  <=>  v <= 448^2 x 4^e, 448^2 = 1.53125 x 2^17
// (a rounded root lies on the same side: the float behind 448^2 x 4^e has a root above 448 x 2^e by more than half a step).
__device__ __forceinline__ int aw_root_exponent(uint32_t u) {
    const int e = ((int)(u >> 23) - 143 + ((u & 0x7fffffu) > 0x440000u ? 1 : 0)) >> 1;
    return u == 0u ? -126 : e;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// largest of a row of 16 lanes, on the vector ALU alone
__device__ __forceinline__ uint32_t aw_row_max(uint32_t v) {
    uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);       // lane ^ 1
    v = o > v ? o : v;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);                // lane ^ 2
    v = o > v ? o : v;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true);               // half a row mirrored
    v = o > v ? o : v;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true);               // the row mirrored
    return o > v ? o : v;
}

// four numbers to e4m3, nearest even
__device__ __forceinline__ uint32_t to_e4m3(f32x4 q) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}
__device__ __forceinline__ f32x4 from_e4m3(uint32_t w) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f32x4{a[0], a[1], b[0], b[1]};
}

// A wave's moments as they are held, between its loads and its stores: four groups of four elements a lane.
template <bool SMALL> struct AwHeld;
template <> struct AwHeld<false> { f32x4 m[4], v[4]; };
template <> struct AwHeld<true> { uint32_t m[4], v[4]; float ms, vs; };

// the scales of a row's new moments, and the moments as multiples of them
__device__ __forceinline__ void aw_encode(AwHeld<true>& h, f32x4 (&m)[4], f32x4 (&v)[4], f32x4 (&r)[4], const f32x4 (&g)[4],
                                          const AwLaunch& a) {
    constexpr uint32_t INF = 0x7f800000u, TINY = 0x00800000u;
    uint32_t mm = 0, vm = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {                   // as bits: what is not finite is larger than all that is
            const uint32_t um = __float_as_uint(m[k][j]) & 0x7fffffffu, uv = __float_as_uint(v[k][j]) & 0x7fffffffu;
            mm = um > mm ? um : mm;
            vm = uv > vm ? uv : vm;
        }
    mm = aw_row_max(mm);
    vm = aw_row_max(vm);
    if (__any(mm >= INF || vm >= INF)) {                // what is not finite does not set the scale of its neighbours
        asm volatile("");                               // rare: to be branched around, not computed along
        mm = vm = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t um = __float_as_uint(m[k][j]) & 0x7fffffffu, uv = __float_as_uint(v[k][j]) & 0x7fffffffu;
                mm = um > mm && um < INF ? um : mm;
                vm = uv > vm && uv < INF ? uv : vm;
                if (um >= INF) m[k][j] = NAN;
                if (uv >= INF) r[k][j] = INFINITY;      // no e4m3 number: becomes NaN
            }
        mm = aw_row_max(mm);
        vm = aw_row_max(vm);
    }
    const int me = aw_exponent(mm);
    int re = aw_root_exponent(vm);
    if (__any(vm != 0u && vm < TINY)) re = vm < TINY ? aw_exponent(__float_as_uint(sqrtf(__uint_as_float(vm)))) : re;
    const float mi = pow2i(-me), ri = pow2i(-re);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[k][j] *= mi;
            // above zero: at least the smallest code.  The median of three is that maximum where the root is above zero
            // (times 2^100 it is far above every code) and zero where it is zero
            const float q = r[k][j] * ri, up = r[k][j] * 0x1p100f;
            r[k][j] = __builtin_amdgcn_fmed3f(q, up, 0x1p-9f);
        }
    // A normal first moment is off by one rounding of itself and three of what is added to the old one: by 7 x 2^-24 of the larger of
    // old and new at most.  Where that leaves two codes, the sign of its distance from their middle decides, which 64 bits give
    // exactly (short numbers, and one product and sum in one rounding): the codes are the exact moments' on every step, not 32
    // bits', which put moments of short gradients in the middle (bf16: 1 to 4 in 100).  An old moment is taken for 1 024 units of the
    // new codes at most, so that never more than one middle is in reach: beyond that a block has cancelled, and the 32-bit moment
    // with it
    const float mr = h.ms * mi;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f32x4 was = from_e4m3(h.m[k]) * mr;
        f32x4 off;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            off[j] = 0x1.8p-21f * __builtin_amdgcn_fmed3f(__builtin_fabsf(m[k][j]), __builtin_fabsf(was[j]), 1024.f);
        uint32_t code = to_e4m3(m[k] - off);
        const uint32_t above = to_e4m3(m[k] + off);
        if (__any(code != above)) {
            asm volatile("");                           // to be branched around, not computed along
            const f32x4 lo = from_e4m3(code), hi = from_e4m3(above);
#pragma unroll
            for (int j = 0; j < 4; ++j) {               // in units of the new codes; one code: both ends of the median are it
                const float mid = 0.5f * (lo[j] + hi[j]);
                const double old = (double)was[j], grad = (double)(g[k][j] * mi);
                const float side = (float)__builtin_fma(grad - old, a.omb1_64, old - (double)mid);
                m[k][j] = __builtin_amdgcn_fmed3f(lo[j], hi[j], __builtin_fmaf(side, 0x1p100f, mid));
            }
            code = to_e4m3(m[k]);
        }
        h.m[k] = code;
    }
    // A normal second moment's root is off by 2^-22 of itself at most (the square of a held root is exact; four roundings of the
    // sum, halved, and the hardware's root).  Where that leaves two codes, squares in 64 bits decide between them: the codes are
    // the exact roots'
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t code = to_e4m3(r[k] * (1.f - 0x1p-21f));
        const uint32_t above = to_e4m3(r[k] * (1.f + 0x1p-21f));
        if (__any(code != above)) {
            asm volatile("");
            const f32x4 lo = from_e4m3(code), hi = from_e4m3(above), was = from_e4m3(h.v[k]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double mid = 0.5 * ((double)lo[j] + (double)hi[j]) * (double)pow2i(re), root = (double)(was[j] * h.vs);
                const double side = __builtin_fma(root * root, a.b2_64, (double)g[k][j] * (double)g[k][j] * a.omb2_64) - mid * mid;
                if (lo[j] < hi[j]) r[k][j] = side > 0.0 ? hi[j] : side < 0.0 ? lo[j] : 0.5f * (lo[j] + hi[j]);
            }
            code = to_e4m3(r[k]);
        }
        h.v[k] = code;
    }
    h.ms = pow2i(me);
    h.vs = pow2i(re);
}

// put: stores p, which then needs no registers while the moments are rounded (168 otherwise, three waves a SIMD, and 88 us where
// 80 are measured)
template <bool SMALL, typename F>
__device__ __forceinline__ void aw_step(AwHeld<SMALL>& h, f32x4 (&p)[4], const f32x4 (&g)[4], const AwLaunch& a,
                                        const AwTensor& t, F&& put) {
    f32x4 m[4], v[4], r[4];
    bool odd = false;                                   // a moment that is subnormal or infinite
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (SMALL) {
            m[k] = from_e4m3(h.m[k]);
            v[k] = from_e4m3(h.v[k]);
        } else {
            m[k] = h.m[k];
            v[k] = h.v[k];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (SMALL) {
                m[k][j] *= h.ms;
                const float root = v[k][j] * h.vs;
                v[k][j] = root * root;
            }
            m[k][j] = m[k][j] + (g[k][j] - m[k][j]) * a.omb1;
            v[k][j] = v[k][j] * a.b2 + g[k][j] * g[k][j] * a.omb2;
            // root and reciprocal of the hardware (one unit in the last place each): the step they scale is added to a
            // parameter that is larger by orders of magnitude
            r[k][j] = __builtin_amdgcn_sqrtf(v[k][j]);
            odd |= __builtin_amdgcn_classf(v[k][j], 0x280);
        }
    }
    if (__any(odd)) {                                   // the hardware's root takes a subnormal for zero
        asm volatile("");
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) r[k][j] = sqrtf(v[k][j]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float u = m[k][j] * __builtin_amdgcn_rcpf(__builtin_fmaf(r[k][j], t.inv_sqrt_bc2, a.eps));
            p[k][j] = __builtin_fmaf(-t.step_size, u, p[k][j] * a.decay);
        }
    }
    put();
    if constexpr (SMALL) {
        aw_encode(h, m, v, r, g, a);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h.m[k] = m[k];
            h.v[k] = v[k];
        }
    }
}

// sb: the row's block of moments; at: the lane's first element in it
template <bool SMALL>
__device__ __forceinline__ void aw_load(AwHeld<SMALL>& h, const AwLaunch& a, long sb, int at) {
    const long i = (sb * AW_BLOCK + at) >> 2;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (SMALL) {
            h.m[k] = __builtin_nontemporal_load(static_cast<const uint32_t*>(a.m) + i + 16 * k);
            h.v[k] = __builtin_nontemporal_load(static_cast<const uint32_t*>(a.v) + i + 16 * k);
        } else {
            h.m[k] = __builtin_nontemporal_load(static_cast<const f32x4*>(a.m) + i + 16 * k);
            h.v[k] = __builtin_nontemporal_load(static_cast<const f32x4*>(a.v) + i + 16 * k);
        }
    }
    if constexpr (SMALL) {
        h.ms = a.ms[sb];
        h.vs = a.vs[sb];
    }
}
template <bool SMALL>
__device__ __forceinline__ void aw_store(const AwHeld<SMALL>& h, const AwLaunch& a, long sb, int at) {
    const long i = (sb * AW_BLOCK + at) >> 2;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (SMALL) {
            __builtin_nontemporal_store(h.m[k], static_cast<uint32_t*>(a.m) + i + 16 * k);
            __builtin_nontemporal_store(h.v[k], static_cast<uint32_t*>(a.v) + i + 16 * k);
        } else {
            __builtin_nontemporal_store(h.m[k], static_cast<f32x4*>(a.m) + i + 16 * k);
            __builtin_nontemporal_store(h.v[k], static_cast<f32x4*>(a.v) + i + 16 * k);
        }
    }
    if constexpr (SMALL) {
        if (at == 0) {
            a.ms[sb] = h.ms;
            a.vs[sb] = h.vs;
        }
    }
}

// 128 registers for 8-bit moments: four waves a SIMD
template <typename T, bool SMALL>
__global__ __launch_bounds__(64 * AW_WAVES, SMALL ? 4 : 1) void adamw_multi_kernel(AwLaunch a) {
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * AW_WAVES + (threadIdx.x >> 6));
    if (unit >= a.units) return;
    uint32_t lo = 0, hi = a.count;                      // the tensor of this unit: the last one with unit0 <= unit
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (a.t[mid].unit0 <= unit) lo = mid; else hi = mid;
    }
    const AwTensor& t = a.t[lo];
    const long b0 = (long)(unit - t.unit0) * AW_UNIT, n = t.n;
    const int row = (threadIdx.x & 63) >> 4, at = (threadIdx.x & 15) * 4;
    const long b = b0 + row, i = b * AW_BLOCK + at;
    f32x4 p[4], g[4];
    AwHeld<SMALL> h;
    if ((b0 + AW_UNIT) * AW_BLOCK <= n) {               // a whole unit: all its loads go out before the first is needed
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            g[k] = AwIo<T>::load(t.g, i + 64 * k);
            p[k] = AwIo<T>::load(t.p, i + 64 * k);
        }
        aw_load<SMALL>(h, a, t.state_block + b, at);
        aw_step<SMALL>(h, p, g, a, t, [&] {
#pragma unroll
            for (int k = 0; k < 4; ++k) AwIo<T>::store(t.p, i + 64 * k, p[k]);
        });
        aw_store<SMALL>(h, a, t.state_block + b, at);
        return;
    }
    // the end of a tensor: nothing is read behind it, and zeros there keep the padding of its last block zero
    const bool mine = b * AW_BLOCK < n;
    if (mine) {
        aw_load<SMALL>(h, a, t.state_block + b, at);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) h.m[k] = h.v[k] = {};
        if constexpr (SMALL) h.ms = h.vs = 1.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const long x = i + 64 * k;
        p[k] = g[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (x + 4 <= n) {
            p[k] = AwIo<T>::load(t.p, x);
            g[k] = AwIo<T>::load(t.g, x);
        } else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (x + j < n) {
                    p[k][j] = AwIo<T>::load1(t.p, x + j);
                    g[k][j] = AwIo<T>::load1(t.g, x + j);
                }
        }
    }
    aw_step<SMALL>(h, p, g, a, t, [&] {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long x = i + 64 * k;
            if (x + 4 <= n) {
                AwIo<T>::store(t.p, x, p[k]);
            } else {
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (x + j < n) AwIo<T>::store1(t.p, x + j, p[k][j]);
            }
        }
    });
    if (mine) aw_store<SMALL>(h, a, t.state_block + b, at);
}

}  // namespace neat

using namespace neat;

extern "C" int neat_adamw_multi(int count, void* const* p, const void* const* g, const int64_t* n, const int64_t* state_block,
                                const int32_t* step, int dtype, void* m, void* v, float* m_scale, float* v_scale,
                                int state_bits, double lr, double beta1, double beta2, double eps, double wd, void* stream) {
    NEAT_REQUIRE(count >= 0, NEAT_ERR_SHAPE, "neat_adamw_multi: count=%d", count);
    if (count == 0) return NEAT_OK;
    NEAT_REQUIRE(p && g && n && state_block && step && m && v, NEAT_ERR_ARG, "neat_adamw_multi: null pointer");
    NEAT_REQUIRE(dtype == NEAT_F32 || dtype == NEAT_BF16, NEAT_ERR_ARG, "neat_adamw_multi: dtype=%d", dtype);
    NEAT_REQUIRE(state_bits == 32 || state_bits == 8, NEAT_ERR_ARG, "neat_adamw_multi: state_bits=%d (32 or 8)", state_bits);
    NEAT_REQUIRE(state_bits == 32 || (m_scale && v_scale), NEAT_ERR_ARG, "neat_adamw_multi: 8-bit moments need their scales");
    NEAT_REQUIRE(((uintptr_t)m & 15) == 0 && ((uintptr_t)v & 15) == 0, NEAT_ERR_ARG,
                 "neat_adamw_multi: moments must be 16-byte aligned");
    const uintptr_t mis = dtype == NEAT_F32 ? 3 : 1;
    for (int i = 0; i < count; ++i) {                   // everything is checked before anything is launched
        NEAT_REQUIRE(n[i] >= 0 && state_block[i] >= 0, NEAT_ERR_SHAPE, "neat_adamw_multi: tensor %d: n=%ld state_block=%ld", i,
                     (long)n[i], (long)state_block[i]);
        NEAT_REQUIRE(n[i] < AW_MOST * AW_UNIT * AW_BLOCK && state_block[i] < (1L << 32) - AW_MOST * AW_UNIT, NEAT_ERR_SHAPE,
                     "neat_adamw_multi: tensor %d too large", i);
        NEAT_REQUIRE(step[i] >= 1, NEAT_ERR_SHAPE, "neat_adamw_multi: tensor %d: step=%d", i, step[i]);
        NEAT_REQUIRE(n[i] == 0 || (p[i] && g[i]), NEAT_ERR_ARG, "neat_adamw_multi: tensor %d: null pointer", i);
        NEAT_REQUIRE((((uintptr_t)p[i] | (uintptr_t)g[i]) & mis) == 0, NEAT_ERR_ARG,
                     "neat_adamw_multi: tensor %d is not aligned to its elements", i);
    }
    AwLaunch a;
    a.m = m; a.v = v; a.ms = m_scale; a.vs = v_scale;
    a.decay = (float)(1.0 - lr * wd);
    a.omb1 = (float)(1.0 - beta1);
    a.omb1_64 = 1.0 - beta1;
    a.b2_64 = beta2;
    a.omb2_64 = 1.0 - beta2;
    a.b2 = (float)beta2;
    a.omb2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    int i = 0, known = 0;
    float step_size = 0.f, inv_sqrt_bc2 = 1.f;
    while (i < count) {
        a.count = 0;
        long units = 0;
        for (; i < count && a.count < AW_TENSORS; ++i) {
            if (n[i] == 0) continue;
            const long nu = (n[i] + AW_BLOCK * AW_UNIT - 1) / (AW_BLOCK * AW_UNIT);
            if (units + nu > AW_MOST) break;           // one tensor alone always fits
            if (step[i] != known) {                     // mostly one step count for all: two pow per launch
                known = step[i];
                step_size = (float)(lr / (1.0 - pow(beta1, known)));
                inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, known)));
            }
            a.t[a.count++] = AwTensor{p[i], g[i], (long)n[i], (uint32_t)units, (uint32_t)state_block[i], step_size, inv_sqrt_bc2};
            units += nu;
        }
        if (a.count == 0) break;
        a.units = (uint32_t)units;
        const dim3 grid(cdiv(units, AW_WAVES)), block(64 * AW_WAVES);
        hipStream_t s = (hipStream_t)stream;
        if (dtype == NEAT_F32) {
            if (state_bits == 8) hipLaunchKernelGGL((adamw_multi_kernel<float, true>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((adamw_multi_kernel<float, false>), grid, block, 0, s, a);
        } else {
            if (state_bits == 8) hipLaunchKernelGGL((adamw_multi_kernel<bf16_t, true>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((adamw_multi_kernel<bf16_t, false>), grid, block, 0, s, a);
        }
        NEAT_LAUNCH_CHECK("neat_adamw_multi");
    }
    return NEAT_OK;
}
