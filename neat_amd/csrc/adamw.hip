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
// Mapping: four contiguous elements a lane (16 B of fp32), a block of 256 elements per wave instruction, four blocks a wave.  Tensor addresses travel as kernel arguments (96 tensors a launch): no table in device memory, so no copy to order
// behind other work and none to keep alive.
#include <math.h>

#include "common.h"

namespace neat {

constexpr int AW_BLOCK = 256;       // elements per block of moments = 64 lanes x 4
constexpr int AW_WAVES = 4;
constexpr int AW_UNIT = 4;          // blocks a wave takes, their loads in flight together
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
    double omb1_64;                 // 1 - beta1 as the caller has it
    float decay, omb1, b2, omb2, eps;
    AwTensor t[AW_TENSORS];
};
static_assert(sizeof(AwLaunch) <= 4096, "kernel arguments");

// gradients are often views of a communication bucket that start at any element: loads of four elements need the element's own
// alignment only (global memory takes unaligned wide accesses)
template <typename T> struct AwIo;
template <> struct AwIo<float> {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ f32x4 load(const void* p, long i) {
        return *reinterpret_cast<const vec*>(static_cast<const float*>(p) + i);
    }
    static __device__ __forceinline__ void store(void* p, long i, f32x4 x) {
        *reinterpret_cast<vec*>(static_cast<float*>(p) + i) = x;
    }
    static __device__ __forceinline__ float load1(const void* p, long i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void store1(void* p, long i, float x) { static_cast<float*>(p)[i] = x; }
};
template <> struct AwIo<bf16_t> {
    typedef uint32_t vec __attribute__((ext_vector_type(2), aligned(2)));
    static __device__ __forceinline__ f32x4 load(const void* p, long i) {
        const vec w = *reinterpret_cast<const vec*>(static_cast<const bf16_t*>(p) + i);
        return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u)};
    }
    static __device__ __forceinline__ void store(void* p, long i, f32x4 x) {
        vec w = {pack2bf(x[0], x[1]), pack2bf(x[2], x[3])};
        *reinterpret_cast<vec*>(static_cast<bf16_t*>(p) + i) = w;
    }
    static __device__ __forceinline__ float load1(const void* p, long i) { return bf2f(static_cast<const bf16_t*>(p)[i]); }
    static __device__ __forceinline__ void store1(void* p, long i, float x) { static_cast<bf16_t*>(p)[i] = f2bf(x); }
};

// 2^e with the largest finite |x| of a block in (224, 448] x 2^e; 2^-126 for a block of zeros
__device__ __forceinline__ int aw_exponent(float largest) {
    const uint32_t u = __float_as_uint(largest);
    const int e = (int)(u >> 23) - 126 - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);   // mantissa above 1.75: one more
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// four numbers to e4m3, nearest even; what is not finite becomes NaN
__device__ __forceinline__ uint32_t to_e4m3(f32x4 q) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (!(fabsf(q[j]) < INFINITY)) q[j] = NAN;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}
__device__ __forceinline__ f32x4 from_e4m3(uint32_t w) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f32x4{a[0], a[1], b[0], b[1]};
}

// largest of a wave, on the vector ALU alone: four steps inside rows of 16 lanes, then across the rows
__device__ __forceinline__ float aw_wave_max(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xf, 0xf, true)));     // lane ^ 1
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xf, 0xf, true)));     // lane ^ 2
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xf, 0xf, true)));    // half row mirrored
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xf, 0xf, true)));    // row mirrored
    const float a = fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0)),
                          __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16)));
    const float b = fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32)),
                          __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 48)));
    return fmaxf(a, b);
}

// One block of 256 elements between its loads and its stores.  g, p in, p out; m, v as they are held, in and out.
template <bool SMALL> struct AwHeld;
template <> struct AwHeld<false> { f32x4 m, v; };
template <> struct AwHeld<true> { uint32_t m, v; float ms, vs; };

template <bool SMALL>
__device__ __forceinline__ void aw_load(AwHeld<SMALL>& h, const AwLaunch& a, long sb, int lane) {
    if constexpr (SMALL) {
        h.m = static_cast<const uint32_t*>(a.m)[sb * 64 + lane];
        h.v = static_cast<const uint32_t*>(a.v)[sb * 64 + lane];
        h.ms = a.ms[sb];
        h.vs = a.vs[sb];
    } else {
        h.m = static_cast<const f32x4*>(a.m)[sb * 64 + lane];
        h.v = static_cast<const f32x4*>(a.v)[sb * 64 + lane];
    }
}

template <bool SMALL>
__device__ __forceinline__ void aw_step(AwHeld<SMALL>& h, f32x4& p, f32x4 g, const AwLaunch& a, const AwTensor& t) {
    f32x4 m, v, r;
    double tie[4];
    if constexpr (SMALL) {
        m = from_e4m3(h.m);
        v = from_e4m3(h.v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] *= h.ms;
            const float root = v[j] * h.vs;
            v[j] = root * root;
        }
    } else {
        m = h.m;
        v = h.v;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float d = g[j] - m[j], add = d * a.omb1;
        if constexpr (SMALL) tie[j] = m[j] == 0.f ? __builtin_fma((double)d, a.omb1_64, -(double)add) : 0.0;
        m[j] = m[j] + add;
        v[j] = v[j] * a.b2 + g[j] * g[j] * a.omb2;
        // root and reciprocal of the hardware (one unit in the last place each): the step they scale is added to a parameter
        // that is larger by orders of magnitude
        r[j] = __builtin_amdgcn_sqrtf(v[j]);
        p[j] = p[j] * a.decay - t.step_size * (m[j] * __builtin_amdgcn_rcpf(r[j] * t.inv_sqrt_bc2 + a.eps));
    }
    if constexpr (SMALL) {
        float mm = 0.f, vm = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {                   // what is not finite does not set the scale of its neighbours
            const float am = fabsf(m[j]);
            mm = fmaxf(mm, am < INFINITY ? am : 0.f);
            vm = fmaxf(vm, v[j] < INFINITY ? v[j] : 0.f);
        }
        // the block's largest root is rounded exactly: it decides the power of two
        const int me = aw_exponent(aw_wave_max(mm)), re = aw_exponent(sqrtf(aw_wave_max(vm)));
        const float mi = pow2i(-me), ri = pow2i(-re);
        f32x4 mq, rq;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mq[j] = m[j] * mi;
            // a moment that starts from zero is one product, and products of short gradients often land halfway between two
            // codes only by their own rounding: what was rounded off (found in 64 bits) decides then
            const uint32_t u = __float_as_uint(mq[j]);
            if ((tie[j] > 0.0 || tie[j] < 0.0) && mq[j] != 0.f && (u & 0x7ffffu) == 0) mq[j] = __uint_as_float((tie[j] > 0.0) == (mq[j] > 0.f) ? u + 1 : u - 1);
            rq[j] = r[j] * ri;
            if (v[j] > 0.f) rq[j] = fmaxf(rq[j], 0x1p-9f);
        }
        h.m = to_e4m3(mq);
        h.v = to_e4m3(rq);
        h.ms = pow2i(me);
        h.vs = pow2i(re);
    } else {
        h.m = m;
        h.v = v;
    }
}

template <bool SMALL>
__device__ __forceinline__ void aw_store(const AwHeld<SMALL>& h, const AwLaunch& a, long sb, int lane) {
    if constexpr (SMALL) {
        static_cast<uint32_t*>(a.m)[sb * 64 + lane] = h.m;
        static_cast<uint32_t*>(a.v)[sb * 64 + lane] = h.v;
        if (lane == 0) {
            a.ms[sb] = h.ms;
            a.vs[sb] = h.vs;
        }
    } else {
        static_cast<f32x4*>(a.m)[sb * 64 + lane] = h.m;
        static_cast<f32x4*>(a.v)[sb * 64 + lane] = h.v;
    }
}

template <typename T, bool SMALL>
__global__ __launch_bounds__(64 * AW_WAVES) void adamw_multi_kernel(AwLaunch a) {
    const int lane = threadIdx.x & 63;
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * AW_WAVES + (threadIdx.x >> 6));
    if (unit >= a.units) return;
    uint32_t lo = 0, hi = a.count;                      // the tensor of this unit: the last one with unit0 <= unit
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (a.t[mid].unit0 <= unit) lo = mid; else hi = mid;
    }
    const AwTensor& t = a.t[lo];
    const long b0 = (long)(unit - t.unit0) * AW_UNIT, n = t.n;
    const long sb0 = (long)t.state_block + b0, i0 = b0 * AW_BLOCK + lane * 4;
    if ((b0 + AW_UNIT) * AW_BLOCK <= n) {               // a whole unit: all its loads go out before the first is needed
        f32x4 p[AW_UNIT], g[AW_UNIT];
        AwHeld<SMALL> h[AW_UNIT];
#pragma unroll
        for (int k = 0; k < AW_UNIT; ++k) {
            g[k] = AwIo<T>::load(t.g, i0 + k * AW_BLOCK);
            p[k] = AwIo<T>::load(t.p, i0 + k * AW_BLOCK);
            aw_load<SMALL>(h[k], a, sb0 + k, lane);
        }
#pragma unroll
        for (int k = 0; k < AW_UNIT; ++k) {
            aw_step<SMALL>(h[k], p[k], g[k], a, t);
            AwIo<T>::store(t.p, i0 + k * AW_BLOCK, p[k]);
            aw_store<SMALL>(h[k], a, sb0 + k, lane);
        }
        return;
    }
    for (int k = 0; k < AW_UNIT && (b0 + k) * AW_BLOCK < n; ++k) {
        const long i = i0 + k * AW_BLOCK, left = n - i;
        f32x4 p = {0.f, 0.f, 0.f, 0.f}, g = p;          // behind the tensor: nothing, so that the padding stays zero
        AwHeld<SMALL> h;
        aw_load<SMALL>(h, a, sb0 + k, lane);
        if (left >= 4) {
            p = AwIo<T>::load(t.p, i);
            g = AwIo<T>::load(t.g, i);
        } else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (j < left) {
                    p[j] = AwIo<T>::load1(t.p, i + j);
                    g[j] = AwIo<T>::load1(t.g, i + j);
                }
        }
        aw_step<SMALL>(h, p, g, a, t);
        if (left >= 4) {
            AwIo<T>::store(t.p, i, p);
        } else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (j < left) AwIo<T>::store1(t.p, i + j, p[j]);
        }
        aw_store<SMALL>(h, a, sb0 + k, lane);
    }
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
        NEAT_REQUIRE(n[i] < (1L << 38) && state_block[i] < (1L << 32) - (1L << 30), NEAT_ERR_SHAPE,
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
            if (units + nu > (1L << 31)) break;
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
