// step_kernel.hpp -- gfx950 kernels of the optimizer step: the global norm of
// many gradient tensors, and AdamW on many tensors at once with 32- or 8-bit
// states.  Formulas: include/xccl_rocm_step.h.
//
// Both stream: nothing is read twice and nothing but registers lies between
// load and store.  Elements are found through the plan's table of chunks,
// STEP_CHUNK consecutive elements of one tensor each.  Accesses are buffer
// instructions as in reduce_kernel.hpp: the base sits in scalar registers, the
// alignment may be any (the device runs in unaligned access mode), what lies
// beyond the descriptor's length is read as zero and not written.  That length
// is honoured per 32-bit word, so the last elements of a tensor of 8- or 16-bit
// values go one by one.
#pragma once

#include "step_plan.h"

#include <hip/hip_runtime.h>

// Pointers that come out of memory are generic to the compiler; this says that
// they are not, where a plain access goes through one.
#define STEP_GLOBAL __attribute__((address_space(1)))

namespace xccl_rocm {

typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4s __attribute__((ext_vector_type(4)));

// Cache policy: loads nt; stores written through (sc0 sc1) or nt.  With 32-bit
// gradients writing through is faster, with 16-bit ones nt is.  Measured, step,
// written through / nt, us: 32-bit gradients, 32-bit states 256 Mi 1111 / 1147, 3
// peers 32 Mi 216 / 223, 8-bit states 256 Mi 650 / 663; 16-bit gradients, 32-bit
// states 64 Mi 300 / 292, 8-bit states 64 Mi 177 / 175, 1 peer 24 Mi 53 / 52.
constexpr int kStepAuxLoad = 0x02;
template <typename G> constexpr int kStepAuxStore = sizeof(G) == 4 ? 0x11 : 0x02;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t step_rsrc(const char *base, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)bytes, 0x00027000);
}

// ---- four consecutive elements, as 32-bit numbers -------------------------

template <typename T, int Bytes = sizeof(T)> struct Four;

template <typename T> struct Four<T, 4> {
    static __device__ __forceinline__ f32x4 load(__amdgpu_buffer_rsrc_t r, uint32_t off)
    {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, kStepAuxLoad));
    }
    template <int Aux> static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t off, f32x4 x)
    {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4s, x), r, (int)off, 0, Aux);
    }
};

template <typename T> struct Four<T, 2> {
    typedef T V __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4 load(__amdgpu_buffer_rsrc_t r, uint32_t off)
    {
        return __builtin_convertvector(
            __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, kStepAuxLoad)), f32x4);
    }
    template <int Aux> static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t off, f32x4 x)
    {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, __builtin_convertvector(x, V)), r, (int)off, 0, Aux);
    }
};

// One element.
template <typename T> __device__ __forceinline__ float load_one(__amdgpu_buffer_rsrc_t r, uint32_t off)
{
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, kStepAuxLoad));
    } else {
        return (float)__builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, kStepAuxLoad));
    }
}

template <typename T, int Aux> __device__ __forceinline__ void store_one(__amdgpu_buffer_rsrc_t r, uint32_t off, float x)
{
    if constexpr (sizeof(T) == 4) {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, (int)off, 0, Aux);
    } else {
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (T)x), r, (int)off, 0, Aux);
    }
}

// Up to 256 consecutive elements of a tensor, 4 to a lane.  Full: all 256.
struct Span {
    uint64_t first;
    uint32_t left;
};

// Tile `i` of a tensor: its elements in [256 i - shift, 256 (i + 1) - shift).
__device__ __forceinline__ Span tile_span(const step_entry_t &t, uint64_t i)
{
    const int64_t from = (int64_t)(i * 256) - t.shift;
    const int64_t to   = from + 256 < (int64_t)t.size ? from + 256 : (int64_t)t.size;
    Span          s;
    s.first = from < 0 ? 0 : (uint64_t)from;
    s.left  = to > (int64_t)s.first ? (uint32_t)(to - (int64_t)s.first) : 0;
    return s;
}

template <typename T, bool Full>
__device__ __forceinline__ f32x4 load4(const char *p, const Span &s, uint32_t lane)
{
    const __amdgpu_buffer_rsrc_t r   = step_rsrc(p + s.first * sizeof(T), s.left * (uint32_t)sizeof(T));
    const uint32_t               off = lane * 4 * (uint32_t)sizeof(T);
    if (Full || sizeof(T) == 4) {
        return Four<T>::load(r, off);
    }
    f32x4 x;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        x[k] = load_one<T>(r, off + k * (uint32_t)sizeof(T));
    }
    return x;
}

template <typename T, bool Full, int Aux>
__device__ __forceinline__ void store4(char *p, const Span &s, uint32_t lane, f32x4 x)
{
    const __amdgpu_buffer_rsrc_t r   = step_rsrc(p + s.first * sizeof(T), s.left * (uint32_t)sizeof(T));
    const uint32_t               off = lane * 4 * (uint32_t)sizeof(T);
    if (Full || sizeof(T) == 4) {
        Four<T>::template store<Aux>(r, off, x);
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        store_one<T, Aux>(r, off + k * (uint32_t)sizeof(T), x[k]);
    }
}

template <bool Full> __device__ __forceinline__ uint32_t load_codes(const char *p, const Span &s, uint32_t lane)
{
    const __amdgpu_buffer_rsrc_t r = step_rsrc(p + s.first, s.left);
    if (Full) {
        return __builtin_amdgcn_raw_buffer_load_b32(r, (int)lane * 4, 0, kStepAuxLoad);
    }
    uint32_t x = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        x |= (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)(lane * 4 + k), 0, kStepAuxLoad) << (8 * k);
    }
    return x;
}

template <bool Full, int Aux>
__device__ __forceinline__ void store_codes(char *p, const Span &s, uint32_t lane, uint32_t x)
{
    const __amdgpu_buffer_rsrc_t r = step_rsrc(p + s.first, s.left);
    if (Full) {
        __builtin_amdgcn_raw_buffer_store_b32(x, r, (int)lane * 4, 0, Aux);
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)(x >> (8 * k)), r, (int)(lane * 4 + k), 0, Aux);
    }
}

// a = grad + peer{0}; a = peer{j} + a: reduce_multi's order, in 32 bits whatever
// the gradient's type, N tiles at once.  The vectors are walked one by one, and a
// wave has one of the peers' in flight at a time: with 32-bit elements a round of
// the loop begins or ends with a wait for all loads, with 16-bit ones, which are
// converted where they are requested, every request is waited for at once.  Other
// waves have to cover that.  The last 32-bit vector is requested by begin and
// added by end, so that what the caller requests in between goes out with it; with
// 16-bit elements the caller's requests come behind the whole fold.
template <typename G, bool Full, bool Peers, int N> struct Fold {
    f32x4 sum[N], more[Peers ? N : 1];

    static __device__ __forceinline__ void request(f32x4 *to, const char *p, const Span *s, uint32_t lane)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            to[i] = load4<G, Full>(p, s[i], lane);
        }
    }

    __device__ __forceinline__ void add(const f32x4 *x)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sum[i] = x[i] + sum[i];
        }
    }

    __device__ __forceinline__ void begin(const char *grad, const char *peers, uint32_t n_peers, size_t stride,
                                          const Span *s, uint32_t lane)
    {
        request(sum, grad, s, lane);
        if constexpr (Peers) {
            request(more, peers, s, lane);
            for (uint32_t j = 1; j < n_peers; ++j) {
                f32x4 next[N];
                peers += stride;
                request(next, peers, s, lane);
                __builtin_amdgcn_sched_barrier(0);
                add(more);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    more[i] = next[i];
                }
            }
        }
    }

    __device__ __forceinline__ void end()
    {
        if constexpr (Peers) {
            add(more);
        }
    }
};

// ---- the norm ---------------------------------------------------------------

constexpr uint32_t kNormWaves = STEP_NORM_WAVES;

struct NormArgs {
    const step_entry_t *entries;
    const step_chunk_t *chunks;
    const step_piece_t *pieces;
    step_partial_t     *partials;
    uint32_t           *arrivals;
    double             *stats;
    size_t              peer_stride;
    uint32_t            n_chunks;
    uint32_t            n_peers;
    uint32_t            grid;
    uint32_t            writes_fold;
};

// What a thread, a wave, a workgroup has found.
struct NormTotal {
    double   sum;
    uint64_t bad;

    // Over the workgroup, in every thread.
    __device__ __forceinline__ void gather(NormTotal *lds)
    {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            sum += __shfl_xor(sum, d);
            bad += __shfl_xor(bad, d);
        }
        if ((threadIdx.x & 63) == 0) {
            lds[threadIdx.x >> 6] = *this;
        }
        __syncthreads();
        sum = lds[0].sum;
        bad = lds[0].bad;
#pragma unroll
        for (uint32_t w = 1; w < kNormWaves; ++w) {
            sum += lds[w].sum;
            bad += lds[w].bad;
        }
        __syncthreads();
    }
};

// What the threads have found -> stats.  The last workgroup to arrive adds the
// partial results up, in an order that does not depend on who that is.
__device__ __forceinline__ void norm_finish(const NormArgs &a, NormTotal t)
{
    __shared__ NormTotal lds[kNormWaves];
    __shared__ bool      last;
    t.gather(lds);
    if (a.grid > 1) {
        if (threadIdx.x == 0) {
            // written through to memory, and there before this workgroup counts itself in
            __hip_atomic_store(&a.partials[blockIdx.x].sum, t.sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            __hip_atomic_store(&a.partials[blockIdx.x].bad, t.bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            // in two levels: arrivals on one counter take their turn, 12 ns each
            const uint32_t shards = a.grid < STEP_ARRIVAL_SHARDS ? a.grid : STEP_ARRIVAL_SHARDS;
            const uint32_t shard  = blockIdx.x % shards;
            const uint32_t total  = a.grid / shards + (shard < a.grid % shards ? 1u : 0u);
            bool           end    = atomicInc(a.arrivals + (1 + shard) * STEP_ARRIVAL_STRIDE, total - 1) == total - 1;
            if (end) { // (atomicInc wraps to 0 at its bound: ready for the next launch)
                end = atomicInc(a.arrivals, shards - 1) == shards - 1;
            }
            last = end;
        }
        __syncthreads();
        if (!last) {
            return;
        }
        t = {0, 0};
        for (uint32_t b = threadIdx.x; b < a.grid; b += kNormWaves * 64) {
            t.sum += __hip_atomic_load(&a.partials[b].sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            t.bad += __hip_atomic_load(&a.partials[b].bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
        t.gather(lds);
    }
    if (threadIdx.x == 0) {
        a.stats[0] = t.sum;
        a.stats[1] = (double)t.bad;
    }
}

// Squares are summed in 64 bits: in 32 they would overflow from 1.8e19 and
// vanish below 1e-23.  Two chains of additions, one for each half of the lane's elements.
struct NormSum {
    double even = 0, odd = 0;
    __device__ __forceinline__ void add(float x, bool is_odd)
    {
        const double d = (double)x;
        double      &s = is_odd ? odd : even;
        s              = __builtin_fma(d, d, s);
    }
};

// The elements of one chunk: 16 bytes per lane and load.
template <typename G> struct NormChunk {
    static constexpr int Loads = STEP_CHUNK * sizeof(G) / 1024;
    u32x4s               x[Loads];
    uint16_t             last; // 16-bit types: the odd element behind the whole words

    __device__ __forceinline__ void load(const char *base, uint32_t left)
    {
        const uint32_t               bytes = left * (uint32_t)sizeof(G);
        const uint32_t               lane  = threadIdx.x & 63;
        const __amdgpu_buffer_rsrc_t r     = step_rsrc(base, bytes & ~3u);
#pragma unroll
        for (int i = 0; i < Loads; ++i) {
            x[i] = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(i * 1024 + lane * 16), 0, kStepAuxLoad);
        }
        if constexpr (sizeof(G) == 2) {
            last = __builtin_amdgcn_raw_buffer_load_b16(step_rsrc(base + (bytes & ~3u), bytes & 3u), (int)lane * 2, 0, kStepAuxLoad);
        }
    }

    __device__ __forceinline__ uint32_t bad() const
    {
        typedef G V __attribute__((ext_vector_type(16 / sizeof(G))));
        uint32_t  n = 0;
#pragma unroll
        for (int i = 0; i < Loads; ++i) {
            const V v = __builtin_bit_cast(V, x[i]);
#pragma unroll
            for (uint32_t k = 0; k < 16 / sizeof(G); ++k) {
                n += !__builtin_isfinite((float)v[k]);
            }
        }
        if constexpr (sizeof(G) == 2) {
            n += !__builtin_isfinite((float)__builtin_bit_cast(G, last));
        }
        return n;
    }

    __device__ __forceinline__ void sum(NormSum &s) const
    {
        typedef G V __attribute__((ext_vector_type(16 / sizeof(G))));
#pragma unroll
        for (int i = 0; i < Loads; ++i) {
            const V v = __builtin_bit_cast(V, x[i]);
#pragma unroll
            for (uint32_t k = 0; k < 16 / sizeof(G); ++k) {
                s.add((float)v[k], k & 1);
            }
        }
        if constexpr (sizeof(G) == 2) {
            s.add((float)__builtin_bit_cast(G, last), false);
        }
    }
};

// The piece of chunk c, or of the last chunk; a wave whose chunk lies behind that
// masks its elements when it uses them, not here, where that would wait for them.
__device__ __forceinline__ step_piece_t norm_piece(const NormArgs &a, uint32_t c)
{
    const auto   at = (const __attribute__((address_space(4))) step_piece_t *)a.pieces + (c < a.n_chunks ? c : a.n_chunks - 1);
    step_piece_t p;
    p.grad = at->grad;
    p.left = at->left;
    return p;
}

__device__ __forceinline__ uint32_t norm_left(const NormArgs &a, const step_piece_t &p, uint32_t c)
{
    return (uint32_t)p.left & (uint32_t)(((uint64_t)c - a.n_chunks) >> 32); // all ones up to the last chunk: no branch
}

// One vector per tensor.  Which chunks a wave takes and the order of every sum
// depend on the plan alone, so equal gradients give equal results.  A wave
// requests 4 KiB before it sums up the last 4 KiB, and has read where they lie
// a round before that.  The scheduling barriers keep it so: left alone, the
// compiler puts the requests behind the sums.
template <typename G>
__global__ void __launch_bounds__(kNormWaves * 64) grad_norm_kernel(const NormArgs a)
{
    constexpr uint32_t K    = STEP_NORM_BYTES / (STEP_CHUNK * sizeof(G)); // chunks at once
    const uint32_t     wave = blockIdx.x * kNormWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t     step = a.grid * kNormWaves * K;
    NormSum            s;
    if (a.n_chunks != 0) {
        NormChunk<G> x[K], y[K];
        step_piece_t piece[K];
        uint32_t     c = wave * K; // what x holds; piece is `step` further
        auto request = [&](NormChunk<G>(&to)[K], uint32_t at) {
#pragma unroll
            for (uint32_t k = 0; k < K; ++k) {
                to[k].load(piece[k].grad, norm_left(a, piece[k], at + k));
            }
#pragma unroll
            for (uint32_t k = 0; k < K; ++k) {
                piece[k] = norm_piece(a, at + step + k);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto sum = [&](const NormChunk<G>(&of)[K]) {
#pragma unroll
            for (uint32_t k = 0; k < K; ++k) {
                of[k].sum(s);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) {
            piece[k] = norm_piece(a, c + k);
        }
        request(x, c);
        while (c < a.n_chunks) {
            request(y, c + step);
            sum(x);
            request(x, c + 2 * step);
            sum(y);
            c += 2 * step;
        }
    }
    // 64 bits hold the sum of any number of 32-bit squares: it is finite unless an element is not.  Only then
    // are those counted, in a second pass of the wave over its chunks, which spares the first a third of its work.
    NormTotal t = {s.even + s.odd, 0};
    if (__any(!__builtin_isfinite(t.sum))) {
        for (uint32_t c = wave * K; c < a.n_chunks; c += step) {
            for (uint32_t k = 0; k < K; ++k) {
                const step_piece_t piece = norm_piece(a, c + k);
                NormChunk<G>       x;
                x.load(piece.grad, norm_left(a, piece, c + k));
                t.bad += x.bad();
            }
        }
    }
    norm_finish(a, t);
}

// With peers' vectors: a wave folds N tiles at a time, and writes the fold if
// there is a place for it.
constexpr int      kFoldTiles    = STEP_FOLD_TILES;
constexpr uint32_t kFoldPerChunk = STEP_CHUNK / 256 / kFoldTiles;

template <typename G, bool Full, int N>
__device__ __forceinline__ void fold_tiles(const NormArgs &a, const step_entry_t &t, const Span *span, NormSum &s,
                                           uint32_t &bad)
{
    const uint32_t         lane = threadIdx.x & 63;
    Fold<G, Full, true, N> fold;
    fold.begin(t.grad, t.peers, a.n_peers, a.peer_stride, span, lane);
    fold.end();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        f32x4 x = fold.sum[i];
        // The step reads what is written, so the norm is that of the rounded values; what is written nowhere stays as it
        // is in 32 bits, which is what a step that folds the vectors itself works with.
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = a.writes_fold ? (float)(G)x[k] : x[k];
            s.add(x[k], k & 1);
            bad += !__builtin_isfinite(x[k]);
        }
        if (a.writes_fold) {
            store4<G, Full, kStepAuxStore<G>>(t.folded, span[i], lane, x);
        }
    }
}

// Measured, 3 peers, 16 Mi elements, 32 bits, the fold written (335 MB): tiles at
// once 1 / 2 / 4 with 512 workgroups 98 / 65 / 65 us, 1024: 64 / 57 / 60, 2048:
// 59 / 59 / 59, 4096: 61 / 60 / 60.
template <typename G>
__global__ void __launch_bounds__(kNormWaves * 64) fold_norm_kernel(const NormArgs a)
{
    constexpr int  N    = kFoldTiles;
    const uint32_t wave = blockIdx.x * kNormWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    NormSum        s;
    uint32_t       bad = 0;
    for (uint32_t u = wave; u < a.n_chunks * kFoldPerChunk; u += a.grid * kNormWaves) {
        const step_chunk_t chunk = a.chunks[u / kFoldPerChunk];
        const step_entry_t t     = a.entries[chunk.entry];
        const uint64_t     first = (uint64_t)chunk.index * (STEP_CHUNK / 256) + u % kFoldPerChunk * N;
        Span               span[N];
        uint32_t           have = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            span[i] = tile_span(t, first + i);
            have += span[i].left;
        }
        if (have == 256 * N) {
            fold_tiles<G, true, N>(a, t, span, s, bad);
        } else {
            for (int i = 0; i < N; ++i) {
                const Span one = tile_span(t, first + i);
                fold_tiles<G, false, 1>(a, t, &one, s, bad);
            }
        }
    }
    norm_finish(a, {s.even + s.odd, bad});
}

// ---- AdamW ------------------------------------------------------------------

// A workgroup is one wave and takes one tile: 256 consecutive elements of a
// tensor, 4 to a lane.  A 32-bit array moves as one 16-byte access per lane, and
// an 8-bit block is exactly one tile: its maximum is a reduction within the wave.
constexpr uint32_t kStepTile  = 256;
constexpr uint32_t kStepTiles = STEP_CHUNK / kStepTile;
static_assert(kStepTile == XCCL_ROCM_STEP_BLOCK, "a tile is a block of the 8-bit states");

struct AdamwKernelArgs {
    const step_entry_t   *entries;
    const step_chunk_t   *chunks;
    const step_scalars_t *from;    // device: read instead of `s` if not NULL
    const double         *stats;   // device, or NULL
    step_scalars_t        s;
    double                zero[2]; // read instead of *stats if there is none
    double                grad_scale, max_norm;
    uint32_t              clip;    // work the factor out here: there is a norm, and no clock
    size_t                peer_stride;
    uint32_t              n_peers;
    uint32_t              use_folded;
    uint32_t              copy; // 0 none, 1 FLOAT16, 2 BFLOAT16
    float                 b1, omb1, b2, omb2, eps;
};

// base^n; the relative error grows with n, to n 2^-53, where base^n itself vanishes.
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

// 64 bits, because 1 - beta^t loses its digits in 32 for small t.
__host__ __device__ inline void step_rate(step_scalars_t &s, double beta1, double beta2, double lr, uint64_t t)
{
    s.lr     = lr;
    s.size   = (float)(lr / (1 - power(beta1, t)));
    s.inv_c2 = (float)(1 / sqrt(1 - power(beta2, t)));
}

// Whether the whole step is skipped, by the bits of its stats: an element was
// not finite, or the sum of squares is no such sum (negative, infinite, NaN).
__device__ __forceinline__ bool step_skips(uint64_t sum, uint64_t bad)
{
    return (bad << 1) != 0 || (sum >> 52) >= 0x7ff;
}

// Ahead of a step that has a clock: reads it for the step, and counts the step
// unless it is going to be skipped.  All loads go out at once, the stats from a
// place that holds zeros if there are none.
struct ClockArgs {
    xccl_rocm_step_clock_t *clock;
    const double           *stats;
    step_scalars_t         *to;
    double                  beta1, beta2, grad_scale, max_norm;
};

// The factor of the folded gradient.
__device__ __forceinline__ float step_factor(double sum, double grad_scale, double max_norm)
{
    const double k = max_norm / (sqrt(sum) * grad_scale + 1e-6);
    return (float)(max_norm > 0 && k < 1 ? grad_scale * k : grad_scale);
}

__global__ void step_clock_kernel(const ClockArgs a)
{
    const double   lr  = a.clock->lr;
    const uint64_t t   = a.clock->steps + 1;
    const uint64_t sum = __builtin_bit_cast(uint64_t, a.stats[0]), bad = __builtin_bit_cast(uint64_t, a.stats[1]);
    step_scalars_t s;
    step_rate(s, a.beta1, a.beta2, lr, t);
    s.g   = step_factor(__builtin_bit_cast(double, sum), a.grad_scale, a.max_norm);
    *a.to = s;
    if (!step_skips(sum, bad)) {
        a.clock->steps = t;
    }
}

// Maximum over the wave, in a scalar register: within rows of 16 lanes (shifts
// by 1, 2, 4, 8), then from row to row; lane 63 ends up with all of it.
template <int Ctrl, int Rows> __device__ __forceinline__ uint32_t max_step(uint32_t x)
{
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, Ctrl, Rows, 0xf, false);
    return y > x ? y : x;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x)
{
    x = max_step<0x111, 0xf>(x);
    x = max_step<0x112, 0xf>(x);
    x = max_step<0x114, 0xf>(x);
    x = max_step<0x118, 0xf>(x);
    x = max_step<0x142, 0xa>(x); // row 0's last lane to row 1, row 2's to row 3
    x = max_step<0x143, 0xc>(x); // row 1's last lane to rows 2 and 3
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// The square root, within one unit of the last place, or (Nearest) correctly
// rounded: the hardware's is off by one unit at most, and which of the three is
// nearest tells the sign of what the product with a neighbour leaves of x
// (Tuckerman's test).  The remainders are multiples of the product of two units
// of the last place, which from x = 2^-102 up is at least the smallest number
// there is, so that none is lost.  Below that, and for subnormal x, which the
// hardware takes for 0, the root of 2^64 x is taken, exactly 2^32 times as
// large.  0 and infinity stay what they are.
template <bool Nearest> __device__ __forceinline__ float square_root(float x)
{
    const bool  small = x < 0x1p-96f;
    const float y     = small ? x * 0x1p64f : x;
    float       r     = __builtin_amdgcn_sqrtf(y);
    if constexpr (Nearest) {
        const float    s     = r;
        const uint32_t bits  = __builtin_bit_cast(uint32_t, s);
        const float    below = __builtin_bit_cast(float, bits - 1), above = __builtin_bit_cast(float, bits + 1);
        r = __builtin_fmaf(-below, s, y) <= 0 ? below : s;
        r = __builtin_fmaf(-above, s, y) > 0 ? above : r;
    }
    return small ? r * 0x1p-32f : r;
}

// The power of two that a block's values are divided by for their e4m3 codes.
// Magnitudes order as their bits do; adding 0x1fffff carries into the exponent
// iff the mantissa is above 1.75, i.e. iff 448 of 2^(exponent - 8) is too small.
__device__ __forceinline__ float block_scale(f32x4 x)
{
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float    xk = x[k]; // (a bit cast of the vector's element itself takes element 0)
        const uint32_t b  = __builtin_bit_cast(uint32_t, xk) & 0x7fffffffu;
        most = b > most ? b : most;
    }
    const int e = (int)((wave_max(most) + 0x1fffffu) >> 23) - 8;
    return __builtin_bit_cast(float, (e < 1 ? 1 : e) << 23);
}

// Codes of four values.  The instruction divides by the scale's power of two.
__device__ __forceinline__ uint32_t quantize(f32x4 x, float scale)
{
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 c = {0, 0};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, x[0], x[1], scale, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, x[2], x[3], scale, true);
    return __builtin_bit_cast(uint32_t, c);
}

// And back, by a product, so that a scale which some other code wrote need not be a power of two.
__device__ __forceinline__ f32x4 dequantize(uint32_t codes, float scale)
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return f32x4{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}

// r = sqrt(v), but nothing above zero below the smallest code.  As integers, which leaves a NaN what it is.
__device__ __forceinline__ f32x4 above_zero(f32x4 r, f32x4 v, float scale)
{
    const uint32_t least = __builtin_bit_cast(uint32_t, scale * 0x1p-9f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float    rk = r[k];
        const uint32_t b  = __builtin_bit_cast(uint32_t, rk), l = v[k] > 0 ? least : 0u;
        r[k] = __builtin_bit_cast(float, b > l ? b : l);
    }
    return r;
}

template <typename P, typename G, bool Eight, bool Peers, bool Full>
__device__ __forceinline__ void adamw_tile(const AdamwKernelArgs &a, const step_scalars_t &s, const step_entry_t &t,
                                           const Span &span)
{
    const uint32_t          lane  = threadIdx.x;
    const uint64_t          block = span.first / kStepTile;
    f32x4                   m, v, r;
    uint32_t                m_codes, r_codes;
    float                   m_scale, r_scale;
    Fold<G, Full, Peers, 1> fold;
    fold.begin(a.use_folded ? t.folded : t.grad, t.peers, a.n_peers, a.peer_stride, &span, lane);
    f32x4 p = load4<P, Full>(t.param, span, lane);
    if constexpr (Eight) {
        m_codes = load_codes<Full>(t.avg, span, lane);
        r_codes = load_codes<Full>(t.sq, span, lane);
        m_scale = ((const STEP_GLOBAL float *)t.avg_scale)[block];
        r_scale = ((const STEP_GLOBAL float *)t.sq_scale)[block];
    } else {
        m = load4<float, Full>(t.avg, span, lane);
        v = load4<float, Full>(t.sq, span, lane);
    }
    const float keep   = (float)(1 - s.lr * t.decay);
    float       factor = s.g;
    if (a.clip) {
        factor = step_factor(*(const __attribute__((address_space(4))) double *)a.stats, a.grad_scale, a.max_norm);
    }
    fold.end();
    const f32x4 g = fold.sum[0] * factor;
    if constexpr (Eight) {
        m = dequantize(m_codes, m_scale);
        r = dequantize(r_codes, r_scale);
        v = r * r;
    }
    m = m * a.b1 + g * a.omb1;
    v = v * a.b2 + (g * a.omb2) * g;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float vk = v[k];
        // One unit of the last place of the root and of the hardware's reciprocal are two roundings of the many that the
        // parameter sees.  The root that is stored as a code is the nearest one: a block's scale hangs on it.
        r[k] = square_root<Eight>(vk);
        const float u = m[k] * __builtin_amdgcn_rcpf(__builtin_fmaf(r[k], s.inv_c2, a.eps));
        p[k]          = __builtin_fmaf(-s.size, u, p[k] * keep);
    }
    store4<P, Full, kStepAuxStore<G>>(t.param, span, lane, p);
    if (a.copy == 1) {
        store4<_Float16, Full, kStepAuxStore<G>>(t.copy, span, lane, p);
    } else if (a.copy == 2) {
        store4<__bf16, Full, kStepAuxStore<G>>(t.copy, span, lane, p);
    }
    if constexpr (Eight) {
        m_scale = block_scale(m);
        r_scale = block_scale(r);
        store_codes<Full, kStepAuxStore<G>>(t.avg, span, lane, quantize(m, m_scale));
        store_codes<Full, kStepAuxStore<G>>(t.sq, span, lane, quantize(above_zero(r, v, r_scale), r_scale));
        if (lane == 0) {
            ((STEP_GLOBAL float *)t.avg_scale)[block] = m_scale;
            ((STEP_GLOBAL float *)t.sq_scale)[block]  = r_scale;
        }
    } else {
        store4<float, Full, kStepAuxStore<G>>(t.avg, span, lane, m);
        store4<float, Full, kStepAuxStore<G>>(t.sq, span, lane, v);
    }
}

template <typename P, typename G, bool Eight, bool Peers>
__global__ void __launch_bounds__(64) adamw_kernel(const AdamwKernelArgs a)
{
    // All of it lies in memory that is constant meanwhile: a choice of addresses, and no branch in front of the loads.
    typedef const __attribute__((address_space(4))) char *Constant;
    const Constant args = (Constant)__builtin_amdgcn_kernarg_segment_ptr();
    const auto     from  = (const __attribute__((address_space(4))) step_scalars_t *)(
        a.from != nullptr ? (Constant)a.from : args + offsetof(AdamwKernelArgs, s));
    const auto     stats = (const __attribute__((address_space(4))) uint64_t *)(
        a.stats != nullptr ? (Constant)a.stats : args + offsetof(AdamwKernelArgs, zero));
    const bool     skip  = step_skips(stats[0], stats[1]);
    step_scalars_t s;
    s.lr     = from->lr;
    s.size   = from->size;
    s.inv_c2 = from->inv_c2;
    s.g      = from->g;
    const step_chunk_t chunk = a.chunks[blockIdx.x / kStepTiles];
    const step_entry_t t     = a.entries[chunk.entry];
    Span               span  = tile_span(t, (uint64_t)chunk.index * kStepTiles + blockIdx.x % kStepTiles);
    if (skip) {
        span.left = 0; // nothing is read or written
    }
    if (span.left == kStepTile) {
        adamw_tile<P, G, Eight, Peers, true>(a, s, t, span);
    } else if (span.left != 0) {
        adamw_tile<P, G, Eight, Peers, false>(a, s, t, span);
    }
}

} // namespace xccl_rocm
