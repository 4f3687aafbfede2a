// step_kernel.hpp -- gfx950 kernels of the optimizer step: the global norm of
// many gradient tensors, and AdamW on many tensors at once with 32- or 8-bit
// states.  Formulas: include/xccl_rocm_step.h.
//
// Both stream: nothing is read twice and nothing but registers lies between
// load and store.  The unit of work is a chunk, STEP_CHUNK consecutive
// elements of one tensor, found through the plan's chunk table; a wave takes
// tiles of 256 elements, 4 consecutive ones per lane, so that a 32-bit array
// moves as one 16-byte access per lane and an 8-bit block (256 elements of a
// tensor) is exactly one tile: its maximum is a reduction within the wave.
// Vector accesses are emitted whatever the alignment (the device runs in
// unaligned access mode); the last tile of a tensor goes element by element
// where a lane's four are not all there.
#pragma once

#include "step_plan.h"

#include <hip/hip_runtime.h>

namespace xccl_rocm {

constexpr uint32_t kStepThreads = 256;
constexpr uint32_t kStepWaves   = kStepThreads / 64;
constexpr uint32_t kStepTile    = 256; // elements a wave takes at once
constexpr uint32_t kStepTiles   = STEP_CHUNK / kStepTile;
static_assert(kStepTile == XCCL_ROCM_STEP_BLOCK, "a tile is a block of the 8-bit states");

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The entries' pointers come out of memory; without the address space the
// compiler would have to use flat accesses for them.
#define STEP_GLOBAL __attribute__((address_space(1)))

// ---- four consecutive elements, as 32-bit numbers -------------------------

template <typename T> struct Four {
    typedef T V __attribute__((ext_vector_type(4)));
    typedef V VU __attribute__((aligned(sizeof(T)))); // wherever an element may lie
    static __device__ __forceinline__ f32x4 load(const char *p, uint64_t e)
    {
        return __builtin_convertvector((V)__builtin_nontemporal_load((const STEP_GLOBAL VU *)((const T *)p + e)), f32x4);
    }
    static __device__ __forceinline__ void store(char *p, uint64_t e, f32x4 x)
    {
        __builtin_nontemporal_store((VU)__builtin_convertvector(x, V), (STEP_GLOBAL VU *)((T *)p + e));
    }
};

// `count` of a lane's four elements exist (uniformly 4 but for a tensor's last tile).
template <typename T>
__device__ __forceinline__ f32x4 load4(const char *p, uint64_t e, uint32_t count)
{
    if (count == 4) {
        return Four<T>::load(p, e);
    }
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t k = 0; k < 3; ++k) {
        if (k < count) {
            x[k] = (float)((const STEP_GLOBAL T *)p)[e + k];
        }
    }
    return x;
}

template <typename T>
__device__ __forceinline__ void store4(char *p, uint64_t e, uint32_t count, f32x4 x)
{
    if (count == 4) {
        Four<T>::store(p, e, x);
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 3; ++k) {
        if (k < count) {
            ((STEP_GLOBAL T *)p)[e + k] = (T)x[k];
        }
    }
}

__device__ __forceinline__ uint32_t load_codes(const char *p, uint64_t e, uint32_t count)
{
    typedef uint32_t U __attribute__((aligned(1)));
    if (count == 4) {
        return __builtin_nontemporal_load((const STEP_GLOBAL U *)(p + e));
    }
    uint32_t x = 0;
#pragma unroll
    for (uint32_t k = 0; k < 3; ++k) {
        if (k < count) {
            x |= (uint32_t)((const STEP_GLOBAL uint8_t *)p)[e + k] << (8 * k);
        }
    }
    return x;
}

__device__ __forceinline__ void store_codes(char *p, uint64_t e, uint32_t count, uint32_t x)
{
    typedef uint32_t U __attribute__((aligned(1)));
    if (count == 4) {
        __builtin_nontemporal_store(x, (STEP_GLOBAL U *)(p + e));
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 3; ++k) {
        if (k < count) {
            ((STEP_GLOBAL uint8_t *)p)[e + k] = (uint8_t)(x >> (8 * k));
        }
    }
}

// Elements of the lane's four that exist, for the tile whose first element is e0.
__device__ __forceinline__ uint32_t lane_count(uint64_t size, uint64_t e)
{
    return e >= size ? 0u : (size - e < 4 ? (uint32_t)(size - e) : 4u);
}

// a = grad + peer{0}; a = peer{j} + a: reduce_multi's order, in 32 bits whatever the gradient's type.
template <typename G>
__device__ __forceinline__ f32x4 fold4(const char *grad, const char *peers, uint32_t n_peers, size_t stride, uint64_t e,
                                       uint32_t count)
{
    f32x4 a = load4<G>(grad, e, count);
    for (uint32_t j = 0; j < n_peers; ++j) {
        a = load4<G>(peers + j * stride, e, count) + a;
    }
    return a;
}

// ---- the norm ---------------------------------------------------------------

struct NormArgs {
    const step_entry_t *entries;
    const step_chunk_t *chunks;
    step_partial_t     *partials;
    uint32_t           *arrivals;
    double             *stats;
    size_t              peer_stride;
    uint32_t            n_chunks;
    uint32_t            n_peers;
    uint32_t            grid;
    uint32_t            writes_fold;
};

__device__ __forceinline__ double wave_sum(double x)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        x += __shfl_xor(x, d);
    }
    return x;
}

// Sum over the workgroup, in thread 0.
__device__ __forceinline__ double group_sum(double x, double *lds)
{
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    x = 0;
    for (uint32_t w = 0; w < kStepWaves; ++w) {
        x += lds[w];
    }
    __syncthreads();
    return x;
}

// Which chunks a workgroup takes and the order of every sum depend on the plan
// alone, so equal gradients give equal results.  The squares are summed in 64
// bits: a 32-bit square would overflow from 1.8e19 and vanish below 1e-23.
// The last workgroup to arrive adds the partial results up.
template <typename G>
__global__ void __launch_bounds__(kStepThreads) grad_norm_kernel(const NormArgs a)
{
    __shared__ double lds[kStepWaves];
    __shared__ bool   last;
    const uint32_t    lane = threadIdx.x & 63;
    const uint32_t    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    double            sum  = 0;
    uint32_t          bad  = 0;

    for (uint32_t c = blockIdx.x; c < a.n_chunks; c += a.grid) {
        const step_chunk_t chunk = a.chunks[c];
        const step_entry_t t     = a.entries[chunk.entry];
        const uint64_t     first = (uint64_t)chunk.index * STEP_CHUNK;
        for (uint32_t i = wave; i < kStepTiles; i += kStepWaves) {
            const uint64_t tile = first + i * kStepTile;
            if (tile >= t.size) {
                break;
            }
            const uint64_t e     = tile + lane * 4;
            const uint32_t count = lane_count(t.size, e);
            f32x4          x     = fold4<G>(t.grad, t.peers, a.n_peers, a.peer_stride, e, count);
            if (a.n_peers != 0) {
                // rounded to the gradient's type, written or not: the norm does not depend on whether it is
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = (float)(G)x[k];
                }
                if (a.writes_fold) {
                    store4<G>(t.folded, e, count, x);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double d = (double)x[k];
                sum = __builtin_fma(d, d, sum);
                bad += !__builtin_isfinite(x[k]);
            }
        }
    }
    sum             = group_sum(sum, lds);
    double bad_sum = group_sum((double)bad, lds);
    if (a.grid > 1) {
        if (threadIdx.x == 0) {
            // written through to memory, and there before this workgroup counts itself in
            __hip_atomic_store(&a.partials[blockIdx.x].sum, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            __hip_atomic_store(&a.partials[blockIdx.x].bad, bad_sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            last = atomicInc(a.arrivals, a.grid - 1) == a.grid - 1; // wraps to 0: ready for the next launch
        }
        __syncthreads();
        if (!last) {
            return;
        }
        sum     = 0;
        bad_sum = 0;
        for (uint32_t b = threadIdx.x; b < a.grid; b += kStepThreads) {
            sum += __hip_atomic_load(&a.partials[b].sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            bad_sum += __hip_atomic_load(&a.partials[b].bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
        sum     = group_sum(sum, lds);
        bad_sum = group_sum(bad_sum, lds);
    }
    if (threadIdx.x == 0) {
        a.stats[0] = sum;
        a.stats[1] = bad_sum;
    }
}

// ---- AdamW ------------------------------------------------------------------

struct AdamwKernelArgs {
    const step_entry_t           *entries;
    const step_chunk_t           *chunks;
    const double                 *stats;
    const xccl_rocm_step_clock_t *clock;
    size_t                        peer_stride;
    uint32_t                      n_peers;
    uint32_t                      use_folded;
    uint32_t                      copy; // 0 none, 1 FLOAT16, 2 BFLOAT16
    float                         b1, omb1, b2, omb2, eps;
    double                        beta1, beta2, lr, grad_scale, max_norm;
    uint64_t                      step;
};

// What depends on step number, rate and norm; 64 bits, because 1 - beta^t loses its digits in 32 for small t.
struct StepScalars {
    double lr;
    float  g;      // factor of the folded gradient
    float  size;   // lr / (1 - beta1^t)
    float  inv_c2; // 1 / sqrt(1 - beta2^t)
};

__host__ __device__ inline double power(double base, uint64_t n)
{
    double x = 1;
    for (; n != 0; n >>= 1) {
        if (n & 1) {
            x *= base;
        }
        base *= base;
    }
    return x;
}

__device__ __forceinline__ StepScalars step_scalars(const AdamwKernelArgs &a)
{
    const uint64_t t  = a.clock ? a.clock->steps + 1 : a.step;
    const double   lr = a.clock ? a.clock->lr : a.lr;
    double         k  = a.grad_scale;
    if (a.max_norm > 0) {
        const double clip = a.max_norm / (sqrt(a.stats[0]) * a.grad_scale + 1e-6);
        k *= clip < 1 ? clip : 1;
    }
    StepScalars s;
    s.lr     = lr;
    s.g      = (float)k;
    s.size   = (float)(lr / (1 - power(a.beta1, t)));
    s.inv_c2 = (float)(1 / sqrt(1 - power(a.beta2, t)));
    return s;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t y = __shfl_xor(x, d);
        x = y > x ? y : x;
    }
    return x;
}

// Four e4m3 codes of x, and the power of two they are to be multiplied with.
// Magnitudes order as their bits do; adding 0x1fffff carries into the exponent
// iff the mantissa is above 1.75, i.e. iff 448 of 2^(exponent - 8) is too small.
// Positive: what is above zero stays above zero.
template <bool Positive>
__device__ __forceinline__ uint32_t quantize(f32x4 x, float &scale)
{
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float    xk = x[k]; // (a bit cast of the vector's element itself takes element 0)
        const uint32_t b  = __builtin_bit_cast(uint32_t, xk) & 0x7fffffffu;
        most = b > most ? b : most;
    }
    most = wave_max(most);
    const int   up  = (int)((most + 0x1fffffu) >> 23) - 8;
    const int   e   = up < 1 ? 1 : up;
    const float inv = __builtin_bit_cast(float, (254 - e) << 23);
    scale = __builtin_bit_cast(float, e << 23);
    f32x4 y;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        y[k] = x[k] * inv;
        if (Positive) {
            y[k] = x[k] > 0 && y[k] < 0x1p-9f ? 0x1p-9f : y[k];
        }
    }
    int code = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], code, true);
}

__device__ __forceinline__ f32x4 dequantize(uint32_t codes, float scale)
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return f32x4{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}

template <typename P, typename G, bool Eight>
__global__ void __launch_bounds__(kStepThreads) adamw_kernel(const AdamwKernelArgs a)
{
    if (a.stats != nullptr && a.stats[1] != 0) {
        return; // a gradient that is not finite: the whole step is skipped
    }
    const StepScalars  s     = step_scalars(a);
    const step_chunk_t chunk = a.chunks[blockIdx.x];
    const step_entry_t t     = a.entries[chunk.entry];
    const uint64_t     first = (uint64_t)chunk.index * STEP_CHUNK;
    const uint32_t     lane  = threadIdx.x & 63;
    const uint32_t     wave  = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float        keep  = (float)(1 - s.lr * t.decay);
    const char        *grad  = a.use_folded ? t.folded : t.grad;

    for (uint32_t i = wave; i < kStepTiles; i += kStepWaves) {
        const uint64_t tile = first + i * kStepTile;
        if (tile >= t.size) {
            break;
        }
        const uint64_t e     = tile + lane * 4;
        const uint32_t count = lane_count(t.size, e);
        const f32x4    g     = fold4<G>(grad, t.peers, a.n_peers, a.peer_stride, e, count) * s.g;
        f32x4          p     = load4<P>(t.param, e, count);
        f32x4          m, v, r;
        if (Eight) {
            m = dequantize(load_codes(t.avg, e, count), ((STEP_GLOBAL float *)t.avg_scale)[tile / kStepTile]);
            r = dequantize(load_codes(t.sq, e, count), ((STEP_GLOBAL float *)t.sq_scale)[tile / kStepTile]);
            v = r * r;
        } else {
            m = load4<float>(t.avg, e, count);
            v = load4<float>(t.sq, e, count);
        }
        m = m * a.b1 + g * a.omb1;
        v = v * a.b2 + (g * a.omb2) * g;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            r[k] = sqrtf(v[k]);
            p[k] = p[k] * keep - s.size * (m[k] / (r[k] * s.inv_c2 + a.eps));
        }
        store4<P>(t.param, e, count, p);
        if (a.copy == 1) {
            store4<_Float16>(t.copy, e, count, p);
        } else if (a.copy == 2) {
            store4<__bf16>(t.copy, e, count, p);
        }
        if (Eight) {
            float m_scale, r_scale;
            store_codes(t.avg, e, count, quantize<false>(m, m_scale));
            store_codes(t.sq, e, count, quantize<true>(r, r_scale));
            if (lane == 0) {
                ((STEP_GLOBAL float *)t.avg_scale)[tile / kStepTile] = m_scale;
                ((STEP_GLOBAL float *)t.sq_scale)[tile / kStepTile]  = r_scale;
            }
        } else {
            store4<float>(t.avg, e, count, m);
            store4<float>(t.sq, e, count, v);
        }
    }
}

// Behind the step, which reads the number: counts it, unless it was skipped.
__global__ void clock_kernel(xccl_rocm_step_clock_t *clock, const double *stats)
{
    if (stats == nullptr || stats[1] == 0) {
        clock->steps += 1;
    }
}

} // namespace xccl_rocm
