// Optimiser step over many tensors at once: AdamW with fp32 or 8-bit moments, the global gradient norm and clipping by it, and the
// conversion between fp32 and 8-bit moments.
//
// A call takes n tensors of any sizes. k_opt_table copies their addresses out of the kernel arguments into a table in the workspace (64 B
// a tensor, up to 99 of them a launch (164 gradients), so that every later kernel is ONE launch whatever n is), advances the step counts and works out what
// is the same for a whole tensor. Then one launch per storage kind (type of the parameters x bits of the moments) has a workgroup for each
// tile of 2048 consecutive elements of a tensor; no tile spans two tensors. A wave owns blocks of 256 consecutive elements, which are also
// the blocks that share a scale of the 8-bit moments: the maximum never leaves the wave. Calls of few small tensors skip the table,
// and clipping of tensors of one type does; a clipped step writes it in the norm's launch if its tensors are of one kind and fit the arguments.
//
// AdamW, t = count + 1, g' = g * factor (factor = clip / loss scale):
//   m = b1 m + (1 - b1) g'        v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) * m / (sqrt(v) * (1 - b2^t)^-1/2 + eps)
// in fp32 with every operation rounded by itself (this file is compiled without contraction), so that the 8-bit codes do not depend on how a
// compiler fuses; 1 - b^t, lr / (1 - b1^t) and the factor are worked out in fp64 and rounded once. Parameters and gradients in 16 bits are
// read to fp32 and the new parameter is rounded once, to nearest even.
//
// 8-bit moments: m and r = sqrt(v) as e4m3 codes with one fp32 scale = max |.| / 448 a block. r instead of v because e4m3 spans 2^17.8 and
// v's range is the square of the gradients'. m is rounded to nearest even (it changes by 10 % a step, codes are 6 - 12 % apart); r changes
// by about 0.05 % a step and would never leave its code under rounding to nearest, so it is rounded up with the probability of its distance
// from the code below: the expected value of the stored r is r (that of r^2 is larger by the rounding's variance: a stationary v settles 5 - 6 %
// too large at b2 = 0.999, r 1.3 %). The 16 random bits an element come from its index in the tensor and
// t alone (opt_mix), so a step is reproducible. An r that is not zero is not stored as zero: m / (0 + eps) would be a step of any size.
//
// Bound: HBM. Every input is read once and every output written once, 28 B an element with fp32 moments and 16.06 B with 8-bit ones (fp32
// parameters). Measured (k_adamw alone, fp32 parameters): 295.5 M elements 1.46 ms = 5.7 TB/s and 0.76 ms = 6.3 TB/s (a large copy on the
// same card: 4.7 - 5.0, a large in-place product 5.9 TB/s); 19.0 M elements 78 us = 6.8 TB/s and 52 us = 5.8 TB/s (part of it stays in the
// 256 MB cache between steps).
#include "common.h"
#include <math.h>
#include <stddef.h>
#include <string.h>

static constexpr int OPT_WG = 256;               // threads of a workgroup: 4 waves
static constexpr int OPT_BLOCK = 256;            // elements of a wave's block = elements that share a scale
// Rounds of four blocks in a tile. 2 for the step and the moments' conversion: 8 loads a lane in flight; 1 was 4 % faster for fp32 moments of 295 M
// elements and 8 % slower for 8-bit ones and for the norm, 4 was 5 - 10 % slower at 13 - 19 M. Clipping alone moves fewer bytes a tile: 4 (150
// tensors of 23.6 M: 36 us of GPU time without the scaling, 42 with 2).
static constexpr int OPT_NB = 2, OPT_CLIP_NB = 4;
// One workgroup a tile up to this many (a grid is limited to 2^32 threads). 2048 workgroups that walk over the tiles instead were 15 - 20 % slower.
static constexpr int OPT_GRID = 1 << 20;
static constexpr int OPT_PARTIALS = 2048;        // workgroups (and fp64 partial sums) of the norm per storage kind (1024: 1 - 2 % slower)
// A norm of up to OPT_INLINE_TILES tiles is cut into at most OPT_INLINE partial sums, which every workgroup behind it adds up by itself: one launch
// less, 3 us of host time and 1 - 3 us of GPU time (an AdamW step of 10 tensors of 8000 elements with clipping 20.7 / 10.6 -> 17.8 / 9.3 us of host / GPU
// time, and 15.4 / 7.6 with the table written by k_opt_sumsq_own). With more tiles so few workgroups take longer than the launch, and more partial sums are too many to add up everywhere.
static constexpr int OPT_INLINE = 256, OPT_INLINE_TILES = 1024;
static constexpr int OPT_NORM_WG = 1024;         // threads of the workgroup that adds them up
// The kernels for few small tensors (16 waves a tensor) take one type, as many tensors as the kernel arguments hold, none above OPT_FEW elements: at 8000
// elements a tensor 11.1 / 5.7 us of host / GPU time with them and 13.5 / 6.3 without (10 tensors), at 16000 10.8 / 8.0 and 13.7 / 6.1: a replayed graph
// would lose.
static constexpr int OPT_FEW = 8192, OPT_FEW_WG = 1024;
// A norm in ONE workgroup, elements a tensor and in all. Clipping alone saves the second launch, 3 us of host time (60 tensors of 1000 elements 12.6 / 6.7 us
// of host / GPU time, 15.6 / 5.7 over many workgroups). A clipped step has two launches either way: 10 tensors of 1000 elements 6.8 us of GPU time, 7.6
// over many workgroups, 60 of them 10.2 and 8.3.
struct OptFewNorm { int most; int64_t total; };
static constexpr OptFewNorm OPT_FEW_CLIP = {4096, 65536}, OPT_FEW_STEP = {2048, 16384};

struct OptEntry {                                // one tensor in the workspace's table
    void* p; const void* g; void* m; void* v; float* ms; float* rs;
    int64_t numel;
    uint64_t pad;
};
static_assert(sizeof(OptEntry) == 64, "four 16-byte stores");
struct OptCoef { float size, unbias, decay; uint32_t t; };
struct OptHead { float factor; int32_t skip; int32_t pad[14]; };

// A tensor in the kernel arguments: its PTRS addresses (48 bits each; 1: grad, 4: param, grad, moments, 6: and the scales), numel below 2^40, slot.
template <int PTRS> struct OptArg { uint32_t lo[PTRS]; uint16_t hi[PTRS]; uint32_t numel_lo, numel_hi_slot; float wd; uint32_t tile0; };
template <int PTRS> struct OptTableArgs {
    static constexpr int MOST = PTRS == 1 ? 164 : PTRS == 4 ? 99 : 76;     // tensors a launch: what OPT_ARGS holds besides a kernel's other arguments
    OptHead* head; OptEntry* entry; OptCoef* coef; uint32_t* tile0; int32_t* steps;
    const float* lr_ptr; const float* found_inf; const float* grad_scale;
    double lr, log2_b1, log2_b2;
    int32_t n, first;                                    // tensors of this launch; first: it also writes the head
    OptArg<PTRS> a[MOST];
};
// Bytes of a kernel's arguments in their order. All kernels here keep to 4 KB, the size that kernel arguments can be relied on to have.
static constexpr size_t OPT_ARGS = 4096;
template <typename... T> constexpr size_t opt_args_bytes() {
    size_t n = 0;
    ((n = (n + alignof(T) - 1) / alignof(T) * alignof(T) + sizeof(T)), ...);
    return n;
}

// After 16-byte stores, with all arithmetic before them (a sched_barrier): nothing may overwrite a store's data registers in its next slots
// (tools/scan_store_hazard.py).
__device__ __forceinline__ void opt_stored() {
    asm volatile("s_nop 0");
    __builtin_amdgcn_sched_barrier(0);
}

template <int PTRS> __device__ __forceinline__ OptEntry opt_entry(const OptArg<PTRS>& a) {
    uint64_t at[6] = {0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < PTRS; ++k) at[PTRS == 1 ? 1 : k] = a.lo[k] | (uint64_t)a.hi[k] << 32;
    return {(void*)at[0], (const void*)at[1], (void*)at[2], (void*)at[3], (float*)at[4], (float*)at[5],
            (int64_t)(a.numel_lo | (uint64_t)(a.numel_hi_slot & 0xffu) << 32), 0};
}
template <int PTRS> __device__ __forceinline__ OptCoef opt_coef(const OptTableArgs<PTRS>& A, float wd, int32_t t) {
    const double lr = A.lr_ptr ? (double)*A.lr_ptr : A.lr;
    OptCoef c;
    c.size = (float)(lr / (1.0 - exp2((double)t * A.log2_b1)));
    c.unbias = (float)(1.0 / sqrt(1.0 - exp2((double)t * A.log2_b2)));
    c.decay = (float)(1.0 - lr * (double)wd);
    c.t = (uint32_t)t;
    return c;
}
template <int PTRS> __device__ __forceinline__ bool opt_skip(const OptTableArgs<PTRS>& A) { return A.found_inf && *A.found_inf != 0.0f; }
template <int PTRS> __device__ __forceinline__ float opt_factor(const OptTableArgs<PTRS>& A) { return A.grad_scale ? (float)(1.0 / (double)*A.grad_scale) : 1.0f; }

template <int PTRS> __device__ __forceinline__ void opt_write_table(const OptTableArgs<PTRS>& A, int i) {
    const bool skip = opt_skip(A);
    if (A.first && i == 0) {
        A.head->skip = skip;
        A.head->factor = opt_factor(A);          // (the norm's kernel writes it again)
    }
    if (i >= A.n) return;
    const OptArg<PTRS>& a = A.a[i];
    const OptEntry e = opt_entry(a);
    u32x4 v[4];
    __builtin_memcpy(v, &e, sizeof(v));
    u32x4* to = (u32x4*)(A.entry + i);
    A.tile0[i] = a.tile0;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) to[k] = v[k];
    opt_stored();
    if (!A.steps) return;
    const uint32_t slot = a.numel_hi_slot >> 8;
    const int32_t t = A.steps[slot] + 1;
    if (!skip) A.steps[slot] = t;
    A.coef[i] = opt_coef(A, a.wd, t);
    opt_stored();
}
template <int PTRS>
__global__ __launch_bounds__(192) void k_opt_table(const OptTableArgs<PTRS> A) {
    static_assert(opt_args_bytes<OptTableArgs<PTRS>>() <= OPT_ARGS && OptTableArgs<PTRS>::MOST <= 192, "arguments; a thread a tensor");
    opt_write_table(A, threadIdx.x);
}

// The table is written by an earlier kernel and constant in this one: read it through the scalar cache, so that what is uniform for a
// workgroup stays in scalar registers (the compiler cannot see that the kernel's own stores do not touch it).
template <typename T> __device__ __forceinline__ T opt_uniform(const T* p) {
    const auto* w = (const __attribute__((address_space(4))) uint32_t*)(uintptr_t)p;
    uint32_t v[sizeof(T) / 4];
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 4; ++i) v[i] = w[i];
    T x;
    __builtin_memcpy(&x, v, sizeof(T));
    return x;
}

// Where a kernel finds its tensors: in the workspace's table, or (no more tensors than the arguments hold) in its own arguments.
struct OptMem {
    const OptEntry* e; const uint32_t* t0; int n;
    __device__ __forceinline__ uint32_t lane_tile0(int i) const { return t0[i]; }
    __device__ __forceinline__ uint32_t tile0(int i) const { return opt_uniform(t0 + i); }
    __device__ __forceinline__ OptEntry entry(int i) const { return opt_uniform(e + i); }
};
template <int PTRS> struct OptOwn {
    const OptTableArgs<PTRS>& A; int n;
    __device__ __forceinline__ uint32_t lane_tile0(int i) const { return A.a[i].tile0; }
    __device__ __forceinline__ uint32_t tile0(int i) const { return A.a[i].tile0; }
    __device__ __forceinline__ OptEntry entry(int i) const { return opt_entry(A.a[i]); }
};

// index of the tensor whose tiles contain `tile`: the last one with tile0 <= tile (tile0 does not decrease). 256 tensors a round, one latency.
template <typename S> __device__ __forceinline__ int opt_find(const S& src, uint32_t tile) {
    const int n = src.n, lane = threadIdx.x & 63;
    int found = 0;
    for (int b = 0; b < n; b += 256) {
        uint32_t t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = b + 64 * k + lane < n ? src.lane_tile0(b + 64 * k + lane) : 0xffffffffu;
        int c = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) c += __popcll(__ballot(t[k] <= tile));
        found += c;
        if (c < 256) break;
    }
    return __builtin_amdgcn_readfirstlane(found - 1);
}

// whether four elements of g (and p) of `size` bytes each are aligned vectors, and m and v are aligned to `state` bytes (0: not used)
__device__ __forceinline__ bool opt_vectors(const OptEntry& e, int size, bool params, int state) {
    uintptr_t a = (uintptr_t)e.g & (4 * size - 1);
    if (params) a |= (uintptr_t)e.p & (4 * size - 1);
    if (state) a |= ((uintptr_t)e.m | (uintptr_t)e.v) & (state - 1);
    return a == 0;
}

// The walk of a workgroup over the tiles blockIdx.x, blockIdx.x + gridDim.x, ... (one tile alone where the grid covers them): at any time the
// chip works on neighbouring addresses. The tensor is looked up again only when the walk leaves it.
template <int NB, typename S> struct OptWalk {
    static constexpr int TILE = NB * 4 * OPT_BLOCK;
    const S src; uint32_t tiles, step, tile, start, end;
    int i;
    OptEntry cur;
    __device__ OptWalk(const S& s, uint32_t tiles_, uint32_t wgs = gridDim.x) : src(s), tiles(tiles_), step(wgs), tile(blockIdx.x), end(0), i(-1) {}
    __device__ __forceinline__ void next() { tile += step; }
    __device__ __forceinline__ bool enter() {    // true if the tile is another tensor's than the last one
        if (tile < end) return false;
        i = opt_find(src, tile);
        cur = src.entry(i);
        start = src.tile0(i);
        end = i + 1 < src.n ? src.tile0(i + 1) : tiles;
        return true;
    }
    // A tile is NB rounds of four blocks, one a wave. First element of this wave's first block (its others follow 4 * OPT_BLOCK apart), and how
    // many elements of the tensor there are from it on (<= 0: none).
    __device__ __forceinline__ int64_t base() const { return (int64_t)(tile - start) * TILE + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * OPT_BLOCK; }
    __device__ __forceinline__ int left() const {
        const int64_t r = cur.numel - base();
        return r < TILE ? (int)r : TILE;                  // (a tile is not empty: r > -TILE)
    }
};

// ---- four elements a lane. FULL (a whole block of an aligned tensor): one vector a lane, elements 4 lane + 0..3; else element by element,
// lane + 64 k while that is below rem, zeros behind. The addresses come out of the table, so the compiler is told that they are global.
template <typename T> using OptPtr = __attribute__((address_space(1))) T*;
template <typename T> __device__ __forceinline__ OptPtr<T> opt_at(const void* p, int64_t i) { return (OptPtr<T>)(uintptr_t)p + i; }
// STREAM: nontemporal. What a step reads and writes once would only push the rest out of the caches: with plain accesses the step of 295 M
// parameters takes 1.57 ms instead of 1.46 (nontemporal loads alone 1.585, stores alone 1.57), a clipped one with 8-bit moments 1.11 instead of 0.96, reading
// the 8-bit moments 0.514 instead of 0.503 (stores alone: 0.491).
template <typename T> struct OptVec4;
template <> struct OptVec4<float> { typedef f32x4 type; };
template <> struct OptVec4<bf16_t> { typedef bf16_t type __attribute__((ext_vector_type(4))); };
template <> struct OptVec4<f16_t> { typedef f16_t type __attribute__((ext_vector_type(4))); };

template <bool FULL, bool STREAM, typename T> __device__ __forceinline__ void opt_load(OptPtr<T> p, int lane, int rem, float* x) {
    if constexpr (FULL) {
        typename OptVec4<T>::type v;
        if constexpr (STREAM) v = __builtin_nontemporal_load((OptPtr<typename OptVec4<T>::type>)p + lane);
        else v = ((OptPtr<typename OptVec4<T>::type>)p)[lane];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = Elem<T>::ld(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = lane + 64 * k < rem ? Elem<T>::ld(p[lane + 64 * k]) : 0.0f;
    }
}
template <bool FULL, bool STREAM, typename T> __device__ __forceinline__ void opt_store(OptPtr<T> p, int lane, int rem, const float* x) {
    if constexpr (FULL) {
        typename OptVec4<T>::type v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = Elem<T>::st(x[k]);
        if constexpr (STREAM) __builtin_nontemporal_store(v, (OptPtr<typename OptVec4<T>::type>)p + lane);
        else ((OptPtr<typename OptVec4<T>::type>)p)[lane] = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane + 64 * k < rem) p[lane + 64 * k] = Elem<T>::st(x[k]);
    }
}
template <bool FULL> __device__ __forceinline__ uint32_t opt_load_codes(OptPtr<uint8_t> p, int lane, int rem) {
    if constexpr (FULL) return __builtin_nontemporal_load((OptPtr<uint32_t>)p + lane);
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) c |= (lane + 64 * k < rem ? (uint32_t)p[lane + 64 * k] : 0u) << (8 * k);
    return c;
}
template <bool FULL> __device__ __forceinline__ void opt_store_codes(OptPtr<uint8_t> p, int lane, int rem, uint32_t c) {
    if constexpr (FULL) { __builtin_nontemporal_store(c, (OptPtr<uint32_t>)p + lane); return; }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < rem) p[lane + 64 * k] = (uint8_t)(c >> (8 * k));
}

// ---- the 8-bit format
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {          // DPP: rows of 16, then across the rows; the result is in lane 63
#define OPT_MAX(ctrl, rows) { const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, true); x = o > x ? o : x; }
    OPT_MAX(0x111, 0xf) OPT_MAX(0x112, 0xf) OPT_MAX(0x114, 0xf) OPT_MAX(0x118, 0xf) OPT_MAX(0x142, 0xa) OPT_MAX(0x143, 0xc)
#undef OPT_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// scale of a block from its values: max |x| / 448, 0 where that is below 2^-110 (1 / scale stays finite). Magnitudes are compared as
// integers, so a NaN (an inf) is the largest and makes the scale NaN (inf): the block then reads back as NaN. ROOT: no signs.
template <bool ROOT> __device__ __forceinline__ float opt_scale(const float* x) {
    uint32_t a = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) a = max(a, ROOT ? __float_as_uint(x[k]) : __float_as_uint(x[k]) & 0x7fffffffu);
    const float s = __uint_as_float(wave_max_u32(a)) * (float)(1.0 / 448.0);
    return s < 0x1p-110f ? 0.0f : s;
}
__device__ __forceinline__ void opt_decode(uint32_t c, float s, float* x) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    x[0] = lo[0] * s; x[1] = lo[1] * s; x[2] = hi[0] * s; x[3] = hi[1] * s;
}
// Square root and quotient of the 8-bit step, which with the IEEE sequences kept its vector units busy for 73 % (19.0 M elements) to 94 % (295 M) of
// the time with 85 instructions an element; now 64, 57 % and 77 %. 19 and 13 issue slots for those sequences, 12 and 8 for these: 60.5 -> 57.7 us at
// 19.0 M, no change at 295 M. With 16-bit parameters (10 B an element) the vector units are the bound of large calls: 66 (fp16) and 72 (bf16) instructions an
// element, busy all the time at 60 M elements (122 and 121 us, 5.0 TB/s); at 6.2 M (17 us) 43 % of it, in 1.7 rounds of workgroups.
// One residual step behind the hardware's reciprocal (root): correctly rounded but for about one value in 2^22.
__device__ __forceinline__ float opt_root(float v) {
    const float y = __builtin_amdgcn_rsqf(v), s = v * y;
    return fmaf(fmaf(-s, s, v), 0.5f * y, s);
}
// Roots of four numbers >= 0. Below 2^-96 the residual falls out of the normal range, and below 2^-126 so does v itself: those are scaled by
// 2^64 first, behind a branch that ordinary second moments never take (one test for the four: v - 1 as an integer sends 0 to the top).
__device__ __forceinline__ void opt_roots(const float* v, float* r) {
    constexpr uint32_t SMALL = (127 - 96) << 23;
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float x = opt_root(v[k]);
        r[k] = __builtin_amdgcn_classf(v[k], 0x100) ? x : v[k];          // 0, inf and NaN are their own roots
        least = min(least, __float_as_uint(v[k]) - 1);
    }
    if (least < SMALL - 1) {
#pragma unroll 1
        for (int k = 0; k < 4; ++k)
            if (__float_as_uint(v[k]) - 1 < SMALL - 1) r[k] = opt_root(v[k] * 0x1p64f) * 0x1p-32f;
    }
}
__device__ __forceinline__ float opt_quotient(float m, float d) {       // d is not a denormal: roots are 0 or above 2^-75, eps is 0 or normal, scales 0 or above 2^-110
    const float y = __builtin_amdgcn_rcpf(d), q = m * y;
    return __builtin_amdgcn_div_fixupf(fmaf(fmaf(-d, q, m), y, q), d, m);
}

// 1 / scale, 0 for a block of zeros (whose codes are then 0)
__device__ __forceinline__ float opt_inverse(float s) { return s == 0.0f ? 0.0f : opt_quotient(1.0f, s); }
__device__ __forceinline__ uint32_t opt_encode(const float* x, float s, bool root) {      // to nearest even
    const float inv = opt_inverse(s);
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        y[k] = x[k] * inv;
        if (root && x[k] > 0.0f) y[k] = y[k] < 0x1p-9f ? 0x1p-9f : y[k];
    }
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
}
// 32 well mixed bits for elements 2 * pair and 2 * pair + 1 at step t. The factors are the fractional bits of the golden ratio (made odd),
// of sqrt 2 and of sqrt 3; flipping any input bit flips every output bit with probability 0.5 +- 0.004.
__device__ __forceinline__ uint32_t opt_mix(uint32_t pair, uint32_t t) {
    uint32_t x = pair + t * 0x9E3779B1u;
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}
// code of x / s >= 0, rounded up with the probability (in 16 bits) of its distance from the code below. Times 2^-120 the exponent field of an
// fp32 number is e4m3's, denormals among them: adding 20 random bits below the code and cutting them off is the rounding.
template <bool FULL> __device__ __forceinline__ uint32_t opt_encode_root(const float* x, float s, int64_t index, uint32_t t) {
    const float inv = opt_inverse(s);
    uint32_t c = 0, bits = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = FULL ? index + k : index + 64 * k;
        if (!FULL || !(k & 1)) bits = opt_mix((uint32_t)(i >> 1), t);
        const uint32_t u = ((FULL ? k : (int)i) & 1 ? bits >> 16 : bits & 0xffffu) * 16 + 8;
        const uint32_t q = (__float_as_uint(x[k] * inv * 0x1p-120f) + u) >> 20;
        const uint32_t least = min(__float_as_uint(x[k]), 1u);           // x > 0 is not stored as 0
        c |= min(max(q, least), 0x7eu) << (8 * k);
    }
    return c;
}

// Runs f over the blocks of the walk's tiles: f(OptWhole<U>, base, 256) on U whole blocks of an aligned tensor (4 * OPT_BLOCK apart), f(OptPart, base,
// rem) on one block of rem elements. `enter` is called when the walk comes to another tensor and tells whether that is aligned.
template <int U> struct OptWhole { static constexpr bool FULL = true; static constexpr int N = U; };
struct OptPart { static constexpr bool FULL = false; static constexpr int N = 1; };
template <int NB, int U, typename W, typename E, typename F> __device__ __forceinline__ void opt_blocks(W& w, E enter, F f) {
    static_assert(NB % U == 0, "whole steps");
    bool aligned = false;
    for (; w.tile < w.tiles; w.next()) {
        if (w.enter()) aligned = enter();
        int64_t base = w.base();
        int left = w.left();
        if (aligned && left >= (NB - 1) * 4 * OPT_BLOCK + OPT_BLOCK) {
#pragma unroll 1
            for (int u = 0; u < NB; u += U) f(OptWhole<U>(), base + u * 4 * OPT_BLOCK, OPT_BLOCK);
            continue;
        }
        for (; left > 0; left -= 4 * OPT_BLOCK, base += 4 * OPT_BLOCK) {
            if (aligned && left >= OPT_BLOCK) f(OptWhole<1>(), base, OPT_BLOCK);
            else f(OptPart(), base, left < OPT_BLOCK ? left : OPT_BLOCK);
        }
    }
}

// norm of the unscaled gradients from the sum of squares, and the factor they are multiplied with: min(1, max_norm / (norm + 1e-6)) / loss scale
__device__ __forceinline__ float opt_norm_of(double sum, const float* grad_scale) { return (float)(sqrt(sum) / (grad_scale ? (double)*grad_scale : 1.0)); }
__device__ __forceinline__ float opt_clip(float norm, const float* grad_scale, double max_norm) {
    const double clip = max_norm / ((double)norm + 1e-6), scale = grad_scale ? (double)*grad_scale : 1.0;
    return (float)((1.0 / scale) * (clip > 1.0 ? 1.0 : clip));           // (a NaN norm gives a NaN factor)
}

// The partial sums of a norm. Up to OPT_INLINE of them are added up by every workgroup that needs the factor (all in one order, so all get the same),
// and the first one writes the norm; more are added up by k_opt_norm before (count 0 here, the factor is in the head).
struct OptSums { const double* partial; int count; const float* grad_scale; double max_norm; float* norm; };
__device__ __forceinline__ float opt_own_factor(const OptSums& N) {
    __shared__ double part[OPT_INLINE / 64];
    __shared__ float all;
    if (threadIdx.x < OPT_INLINE) {
        const double s = wave_sum_f64((int)threadIdx.x < N.count ? N.partial[threadIdx.x] : 0.0);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int k = 0; k < OPT_INLINE / 64; ++k) sum += part[k];
        const float norm = opt_norm_of(sum, N.grad_scale);
        all = opt_clip(norm, N.grad_scale, N.max_norm);
        if (blockIdx.x == 0 && N.norm) *N.norm = norm;
    }
    __syncthreads();
    return all;
}

struct OptHyper { float b1, omb1, b2, omb2, eps; };

template <typename T, int BITS, bool FULL, int U>
__device__ __forceinline__ void adamw_block(const OptEntry& e, int64_t base, int rem, const OptCoef& c, const OptHyper& H, float factor, int lane) {
    float p[U][4], g[U][4], m[U][4], v[U][4];
    uint32_t cm[U], cv[U];
    float sm[U], sr[U];
    const int64_t block = base / OPT_BLOCK;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = base + u * 4 * OPT_BLOCK;
        opt_load<FULL, true>(opt_at<T>(e.g, at), lane, rem, g[u]);
        if constexpr (BITS == 8) {
            cm[u] = opt_load_codes<FULL>(opt_at<uint8_t>(e.m, at), lane, rem);
            cv[u] = opt_load_codes<FULL>(opt_at<uint8_t>(e.v, at), lane, rem);
            sm[u] = *opt_at<float>(e.ms, block + 4 * u);
            sr[u] = *opt_at<float>(e.rs, block + 4 * u);
        } else {
            opt_load<FULL, true>(opt_at<float>(e.m, at), lane, rem, m[u]);
            opt_load<FULL, true>(opt_at<float>(e.v, at), lane, rem, v[u]);
        }
        opt_load<FULL, true>(opt_at<T>(e.p, at), lane, rem, p[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = base + u * 4 * OPT_BLOCK;
        float r[4];
        if constexpr (BITS == 8) {
            opt_decode(cm[u], sm[u], m[u]);
            opt_decode(cv[u], sr[u], v[u]);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[u][k] = v[u][k] * v[u][k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            g[u][k] = g[u][k] * factor;
            m[u][k] = m[u][k] * H.b1 + g[u][k] * H.omb1;
            v[u][k] = v[u][k] * H.b2 + (g[u][k] * g[u][k]) * H.omb2;
            if constexpr (BITS != 8) r[k] = sqrtf(v[u][k]);
        }
        if constexpr (BITS == 8) opt_roots(v[u], r);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float den = r[k] * c.unbias + H.eps;
            p[u][k] = p[u][k] * c.decay - (BITS == 8 ? opt_quotient(m[u][k], den) : m[u][k] / den) * c.size;
        }
        if constexpr (BITS == 8) {
            if constexpr (!FULL) {               // lanes past the end do not count in the maxima (a factor that is not finite would be in them)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (lane + 64 * k >= rem) m[u][k] = r[k] = 0.0f;
            }
            const float nm = opt_scale<false>(m[u]), nr = opt_scale<true>(r);
            cm[u] = opt_encode(m[u], nm, false);
            cv[u] = opt_encode_root<FULL>(r, nr, at + (FULL ? 4 * lane : lane), c.t);
            sm[u] = nm; sr[u] = nr;
        }
        __builtin_amdgcn_sched_barrier(0);
        opt_store<FULL, true>(opt_at<T>(e.p, at), lane, rem, p[u]);
        if constexpr (BITS == 8) {
            opt_store_codes<FULL>(opt_at<uint8_t>(e.m, at), lane, rem, cm[u]);
            opt_store_codes<FULL>(opt_at<uint8_t>(e.v, at), lane, rem, cv[u]);
            if (lane == 0) { *opt_at<float>(e.ms, block + 4 * u) = sm[u]; *opt_at<float>(e.rs, block + 4 * u) = sr[u]; }
        } else {
            opt_store<FULL, true>(opt_at<float>(e.m, at), lane, rem, m[u]);
            opt_store<FULL, true>(opt_at<float>(e.v, at), lane, rem, v[u]);
        }
        opt_stored();
    }
}

template <typename T, int BITS>
__global__ __launch_bounds__(OPT_WG) void k_adamw(const OptHead* head, OptMem src, const OptCoef* coef, uint32_t tiles, OptHyper H, OptSums N) {
    const float factor = N.count ? opt_own_factor(N) : opt_uniform(&head->factor);
    if (opt_uniform(&head->skip)) return;
    const int lane = threadIdx.x & 63;
    OptCoef c = {};
    OptWalk<OPT_NB, OptMem> w(src, tiles);
    opt_blocks<OPT_NB, OPT_NB>(w, [&] { c = opt_uniform(coef + w.i); return opt_vectors(w.cur, sizeof(T), true, BITS == 8 ? 4 : 16); },
                              [&](auto kind, int64_t base, int rem) { adamw_block<T, BITS, kind.FULL, kind.N>(w.cur, base, rem, c, H, factor, lane); });
}

// ---- global gradient norm: squares summed in fp64 (no overflow, and fp64 multiply-add runs at the rate of fp32 here), a fixed order
template <bool FULL, int U, typename T> __device__ __forceinline__ double opt_sumsq(const OptEntry& e, int64_t base, int rem, int lane, double s) {
    float g[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) opt_load<FULL, false>(opt_at<T>(e.g, base + u * 4 * OPT_BLOCK), lane, rem, g[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) s = fma((double)g[u][k], (double)g[u][k], s);
    return s;
}
template <typename T, int NB, typename S> __device__ __forceinline__ void opt_sumsq_walk(const S& src, uint32_t tiles, uint32_t wgs, double* partial) {
    __shared__ double part[OPT_WG / 64];
    const int lane = threadIdx.x & 63;
    double s = 0.0;
    OptWalk<NB, S> w(src, tiles, wgs);
    opt_blocks<NB, NB>(w, [&] { return opt_vectors(w.cur, sizeof(T), false, 0); },
                       [&](auto kind, int64_t base, int rem) { s = opt_sumsq<kind.FULL, kind.N, T>(w.cur, base, rem, lane, s); });
    s = wave_sum_f64(s);
    if (lane == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}
template <typename T, int NB>
__global__ __launch_bounds__(OPT_WG) void k_opt_sumsq(OptMem src, uint32_t tiles, double* partial) { opt_sumsq_walk<T, NB>(src, tiles, gridDim.x, partial); }
// The same with the tensors in the kernel arguments. A step (PTRS > 1) needs the table in the kernel behind: a workgroup of its own, the last, writes it.
template <typename T, int NB, int PTRS>
__global__ __launch_bounds__(OPT_WG) void k_opt_sumsq_own(const OptTableArgs<PTRS> A, uint32_t tiles, double* partial) {
    static_assert(opt_args_bytes<OptTableArgs<PTRS>, uint32_t, double*>() <= OPT_ARGS && OptTableArgs<PTRS>::MOST <= (PTRS > 1 ? OPT_WG : 1 << 30), "arguments; a thread a tensor");
    const uint32_t wgs = gridDim.x - (PTRS > 1);
    if (PTRS > 1 && blockIdx.x == wgs) opt_write_table(A, threadIdx.x);
    else opt_sumsq_walk<T, NB>(OptOwn<PTRS>{A, A.n}, tiles, wgs, partial);
}

// The norm (count < 0: given at norm_at) and the factor. One workgroup, a launch of its own: 4 us. Finishing in the last workgroup of k_opt_sumsq
// instead (a ticket) was no faster: 1024 tickets on one address take 6 us, and with 256 larger workgroups the sums themselves take 3 us more.
__global__ __launch_bounds__(OPT_NORM_WG) void k_opt_norm(const double* partial, int count, const float* grad_scale, double max_norm, float* norm_at, OptHead* head) {
    __shared__ double part[OPT_NORM_WG / 64];
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += OPT_NORM_WG) s += partial[i];
    s = wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int k = 0; k < OPT_NORM_WG / 64; ++k) sum += part[k];
        const float norm = count < 0 ? *norm_at : opt_norm_of(sum, grad_scale);
        head->factor = opt_clip(norm, grad_scale, max_norm);
        if (norm_at && count >= 0) *norm_at = norm;
    }
}

template <bool FULL, int U, typename T> __device__ __forceinline__ void opt_scale_block(const OptEntry& e, int64_t base, int rem, int lane, float factor) {
    float g[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) opt_load<FULL, false>(opt_at<T>(e.g, base + u * 4 * OPT_BLOCK), lane, rem, g[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) g[u][k] = g[u][k] * factor;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) opt_store<FULL, false>(opt_at<T>(e.g, base + u * 4 * OPT_BLOCK), lane, rem, g[u]);
    opt_stored();
}
template <typename T, typename S> __device__ __forceinline__ void opt_scale_walk(const S& src, uint32_t tiles, const OptHead* head, const OptSums& N) {
    const float factor = N.count ? opt_own_factor(N) : opt_uniform(&head->factor);
    if (factor == 1.0f) return;                  // nothing to clip: x * 1 is x for every x
    const int lane = threadIdx.x & 63;
    OptWalk<OPT_CLIP_NB, S> w(src, tiles);
    opt_blocks<OPT_CLIP_NB, 2>(w, [&] { return opt_vectors(w.cur, sizeof(T), false, 0); },
                               [&](auto kind, int64_t base, int rem) { opt_scale_block<kind.FULL, kind.N, T>(w.cur, base, rem, lane, factor); });
}
template <typename T>
__global__ __launch_bounds__(OPT_WG) void k_opt_scale(OptMem src, uint32_t tiles, const OptHead* head, OptSums N) { opt_scale_walk<T>(src, tiles, head, N); }
template <typename T>
__global__ __launch_bounds__(OPT_WG) void k_opt_scale_own(const OptTableArgs<1> A, uint32_t tiles, OptSums N) {
    static_assert(opt_args_bytes<OptTableArgs<1>, uint32_t, OptSums>() <= OPT_ARGS, "arguments");
    opt_scale_walk<T>(OptOwn<1>{A, A.n}, tiles, A.head, N);
}

// ---- fp32 moments (p: exp_avg, g: exp_avg_sq) <-> 8-bit moments
template <bool FULL, bool WRITE> __device__ __forceinline__ void opt_state8_block(const OptEntry& e, int64_t base, int rem, int lane) {
    const int64_t block = base / OPT_BLOCK;
    float m[4], v[4];
    if constexpr (WRITE) {
        opt_load<FULL, true>(opt_at<float>(e.p, base), lane, rem, m);
        opt_load<FULL, true>(opt_at<float>(e.g, base), lane, rem, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = sqrtf(v[k]);
        const float sm = opt_scale<false>(m), sr = opt_scale<true>(v);
        opt_store_codes<FULL>(opt_at<uint8_t>(e.m, base), lane, rem, opt_encode(m, sm, false));
        opt_store_codes<FULL>(opt_at<uint8_t>(e.v, base), lane, rem, opt_encode(v, sr, true));
        if (lane == 0) { *opt_at<float>(e.ms, block) = sm; *opt_at<float>(e.rs, block) = sr; }
    } else {
        const uint32_t cm = opt_load_codes<FULL>(opt_at<uint8_t>(e.m, base), lane, rem);
        const uint32_t cv = opt_load_codes<FULL>(opt_at<uint8_t>(e.v, base), lane, rem);
        opt_decode(cm, *opt_at<float>(e.ms, block), m);
        opt_decode(cv, *opt_at<float>(e.rs, block), v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = v[k] * v[k];
        __builtin_amdgcn_sched_barrier(0);
        opt_store<FULL, true>(opt_at<float>(e.p, base), lane, rem, m);
        opt_store<FULL, true>(opt_at<float>(e.g, base), lane, rem, v);
        opt_stored();
    }
}
template <bool WRITE>
__global__ __launch_bounds__(OPT_WG) void k_opt_state8(OptMem src, uint32_t tiles) {
    const int lane = threadIdx.x & 63;
    OptWalk<OPT_NB, OptMem> w(src, tiles);
    opt_blocks<OPT_NB, 1>(w, [&] { return opt_vectors(w.cur, 4, true, 4); },
                          [&](auto kind, int64_t base, int rem) { opt_state8_block<kind.FULL, WRITE>(w.cur, base, rem, lane); });
}

// ---- few small tensors: no table. The tensors are read from the kernel arguments by the kernel that works on them, one workgroup a tensor, which
// also advances its count: one launch instead of two (clipping alone one instead of two; a clipped step two either way). A launch costs 4 us of
// host time and 2 - 4 us of GPU time, which is what such a call consists of.
template <typename T, int BITS>
__global__ __launch_bounds__(OPT_FEW_WG) void k_adamw_few(const OptTableArgs<BITS == 8 ? 6 : 4> A, OptHyper H, int clipped) {
    static_assert(opt_args_bytes<OptTableArgs<BITS == 8 ? 6 : 4>, OptHyper, int>() <= OPT_ARGS, "arguments");
    if (opt_skip(A)) return;
    const OptEntry e = opt_entry(A.a[blockIdx.x]);
    const uint32_t slot = A.a[blockIdx.x].numel_hi_slot >> 8;
    const int32_t t = A.steps[slot] + 1;
    const OptCoef c = opt_coef(A, A.a[blockIdx.x].wd, t);
    const float factor = clipped ? A.head->factor : opt_factor(A);
    __syncthreads();                             // every wave has read the count
    if (threadIdx.x == 0) A.steps[slot] = t;
    const bool vec = opt_vectors(e, sizeof(T), true, BITS == 8 ? 4 : 16);
    const int lane = threadIdx.x & 63, n = (int)e.numel;
    for (int base = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * OPT_BLOCK; base < n; base += OPT_FEW_WG / 64 * OPT_BLOCK) {
        if (vec && n - base >= OPT_BLOCK) adamw_block<T, BITS, true, 1>(e, base, OPT_BLOCK, c, H, factor, lane);
        else adamw_block<T, BITS, false, 1>(e, base, min(n - base, OPT_BLOCK), c, H, factor, lane);
    }
}

// The norm of all tensors of the call by one workgroup, a wave a tensor; SCALE: and the gradients multiplied by the factor.
template <typename T, bool SCALE, int PTRS>
__global__ __launch_bounds__(OPT_FEW_WG) void k_opt_norm_few(const OptTableArgs<PTRS> A, double max_norm, float* norm_at) {
    static_assert(opt_args_bytes<OptTableArgs<PTRS>, double, float*>() <= OPT_ARGS, "arguments");
    __shared__ double part[OPT_FEW_WG / 64];
    __shared__ float all;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    double s = 0.0;
    for (int i = wave; i < A.n; i += OPT_FEW_WG / 64) {
        const OptEntry e = opt_entry(A.a[i]);
        const bool vec = opt_vectors(e, sizeof(T), false, 0);
        const int n = (int)e.numel;
        for (int base = 0; base < n; base += OPT_BLOCK) {
            if (vec && n - base >= OPT_BLOCK) s = opt_sumsq<true, 1, T>(e, base, OPT_BLOCK, lane, s);
            else s = opt_sumsq<false, 1, T>(e, base, min(n - base, OPT_BLOCK), lane, s);
        }
    }
    s = wave_sum_f64(s);
    if (lane == 0) part[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int k = 0; k < OPT_FEW_WG / 64; ++k) sum += part[k];
        const float norm = opt_norm_of(sum, A.grad_scale);
        all = opt_clip(norm, A.grad_scale, max_norm);
        if (!SCALE) A.head->factor = all;
        if (norm_at) *norm_at = norm;
    }
    if constexpr (SCALE) {
        if (max_norm < 0.0) return;              // the norm alone
        __syncthreads();
        const float factor = all;
        if (factor == 1.0f) return;
        for (int i = wave; i < A.n; i += OPT_FEW_WG / 64) {
            const OptEntry e = opt_entry(A.a[i]);
            const bool vec = opt_vectors(e, sizeof(T), false, 0);
            const int n = (int)e.numel;
            for (int base = 0; base < n; base += OPT_BLOCK) {
                if (vec && n - base >= OPT_BLOCK) opt_scale_block<true, 1, T>(e, base, OPT_BLOCK, lane, factor);
                else opt_scale_block<false, 1, T>(e, base, min(n - base, OPT_BLOCK), lane, factor);
            }
        }
    }
}
template <bool WRITE>
__global__ __launch_bounds__(OPT_FEW_WG) void k_opt_state8_few(const OptTableArgs<6> A) {
    const OptEntry e = opt_entry(A.a[blockIdx.x]);
    const bool vec = opt_vectors(e, 4, true, 4);
    const int lane = threadIdx.x & 63, n = (int)e.numel;
    for (int base = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * OPT_BLOCK; base < n; base += OPT_FEW_WG / 64 * OPT_BLOCK) {
        if (vec && n - base >= OPT_BLOCK) opt_state8_block<true, WRITE>(e, base, OPT_BLOCK, lane);
        else opt_state8_block<false, WRITE>(e, base, min(n - base, OPT_BLOCK), lane);
    }
}

// ---- host side
// kinds of a launch: parameter type x bits of the moments
static inline int opt_kind(const NndetOptTensor& t) { return t.dtype + (t.state_bits == 8 ? 3 : 0); }

static size_t opt_bytes(int64_t n) {
    return sizeof(OptHead) + 6 * OPT_PARTIALS * sizeof(double) + (size_t)n * (sizeof(OptEntry) + sizeof(OptCoef) + sizeof(uint32_t));
}
extern "C" size_t nndet_opt_workspace_bytes(int32_t n) { return n < 0 ? 0 : opt_bytes(n); }

struct OptPlan {                                 // the tensors of a call in the order of their kinds, as they lie in the table
    OptHead* head; double* partial; OptEntry* entry; OptCoef* coef; uint32_t* tile0;
    int first[7];                                // entries of kind k: first[k] .. first[k + 1]
    int64_t tiles[6];
};

struct OptScalars { int32_t* steps; const float *lr_ptr, *found_inf, *grad_scale; double lr, b1, b2; };

template <int PTRS> static void opt_scalars(const OptScalars& S, OptHead* head, OptTableArgs<PTRS>& A) {
    memset(&A, 0, offsetof(OptTableArgs<PTRS>, a));
    A.head = head; A.steps = S.steps; A.lr_ptr = S.lr_ptr; A.found_inf = S.found_inf; A.grad_scale = S.grad_scale;
    A.lr = S.lr; A.log2_b1 = log2(S.b1); A.log2_b2 = log2(S.b2);
}
template <int PTRS> static void opt_arg(const NndetOptTensor& t, uint32_t tile0, OptArg<PTRS>& a) {
    const uint64_t p[6] = {(uint64_t)t.param, (uint64_t)t.grad, (uint64_t)t.exp_avg, (uint64_t)t.exp_avg_sq, (uint64_t)t.exp_avg_scale, (uint64_t)t.root_scale};
    for (int q = 0; q < PTRS; ++q) {
        const uint64_t at = p[PTRS == 1 ? 1 : q];
        a.lo[q] = (uint32_t)at; a.hi[q] = (uint16_t)(at >> 32);
    }
    a.numel_lo = (uint32_t)t.numel; a.numel_hi_slot = (uint32_t)(t.numel >> 32) | (uint32_t)t.slot << 8;
    a.wd = (float)t.weight_decay;
    a.tile0 = tile0;
}

// k_opt_table for the tensors of kinds k0 .. k0 + 2 (PTRS as their moments need); `head`: the first launch also writes the head.
template <int PTRS>
static int opt_table(const NndetOptTensor* t, int32_t n, const OptScalars& S, int nb, int k0, bool head, OptPlan& P, hipStream_t st) {
    OptTableArgs<PTRS> A;
    opt_scalars(S, P.head, A);
    A.first = head;
    int at = P.first[k0];
    for (int k = k0; k < k0 + 3; ++k) {
        P.first[k] = at;
        int64_t tiles = 0;
        for (int i = 0; i <= n; ++i) {
            if (i < n && (opt_kind(t[i]) != k || (t[i].numel == 0 && !S.steps))) continue;
            if (i < n) {
                opt_arg(t[i], (uint32_t)tiles, A.a[A.n++]);
                tiles += ceil_div64(t[i].numel, nb * 4 * OPT_BLOCK);
                ++at;
            }
            const bool end = i == n && k == k0 + 2;
            if (A.n == OptTableArgs<PTRS>::MOST || (end && (A.n || A.first))) {
                A.entry = P.entry + at - A.n; A.coef = P.coef + at - A.n; A.tile0 = P.tile0 + at - A.n;
                k_opt_table<PTRS><<<1, 192, 0, st>>>(A);
                LAUNCH_CHECK();
                A.n = 0; A.first = 0;
            }
        }
        P.tiles[k] = tiles;
    }
    P.first[k0 + 3] = at;
    return 0;
}

// Checks the tensors (all of them, before anything is launched) and lays the workspace out. `need`: bit 0 param, 1 grad, 2 moments (scales with 8 bits).
static int opt_check(const NndetOptTensor* t, int32_t n, int need, void* ws, size_t ws_bytes, OptPlan& P) {
    if (n < 0 || (n > 0 && !t) || n >= (1 << 24)) return NNDET_EINVAL;
    if (!ws || ((uintptr_t)ws & 15)) return NNDET_EINVAL;
    if (ws_bytes < opt_bytes(n)) return NNDET_EWORKSPACE;
    P.head = (OptHead*)ws;
    P.partial = (double*)(P.head + 1);
    P.entry = (OptEntry*)(P.partial + 6 * OPT_PARTIALS);
    P.coef = (OptCoef*)(P.entry + n);
    P.tile0 = (uint32_t*)(P.coef + n);
    int64_t tiles = 0;
    for (int i = 0; i < n; ++i) {
        if (t[i].dtype < 0 || t[i].dtype > 2 || (t[i].state_bits != 32 && t[i].state_bits != 8)) return NNDET_EINVAL;
        if (t[i].numel < 0 || t[i].numel >= (int64_t)1 << 40 || t[i].slot < 0 || t[i].slot >= (1 << 24)) return NNDET_EINVAL;
        const uint64_t any = (uint64_t)t[i].param | (uint64_t)t[i].grad | (uint64_t)t[i].exp_avg | (uint64_t)t[i].exp_avg_sq | (uint64_t)t[i].exp_avg_scale | (uint64_t)t[i].root_scale;
        tiles += ceil_div64(t[i].numel, 4 * OPT_BLOCK);
        if (any >> 48 || tiles >= ((int64_t)1 << 32) - OPT_GRID) return NNDET_EINVAL;      // (a walk steps past the last tile)
        if (t[i].numel == 0) continue;
        if (((need & 1) && !t[i].param) || ((need & 2) && !t[i].grad) || ((need & 4) && (!t[i].exp_avg || !t[i].exp_avg_sq))) return NNDET_EINVAL;
        if ((need & 4) && t[i].state_bits == 8 && (!t[i].exp_avg_scale || !t[i].root_scale)) return NNDET_EINVAL;
    }
    return 0;
}

// Writes the table.
static int opt_begin(const NndetOptTensor* t, int32_t n, const OptScalars& S, int nb, OptPlan& P, hipStream_t st, bool grads_alone = false) {
    bool any8 = false, any32 = n == 0;
    for (int i = 0; i < n; ++i) (t[i].state_bits == 8 ? any8 : any32) = true;
    P.first[0] = 0;
    int rc = 0;
    if (any32) rc = grads_alone ? opt_table<1>(t, n, S, nb, 0, true, P, st) : opt_table<4>(t, n, S, nb, 0, true, P, st);
    else for (int k = 0; k < 4; ++k) { P.first[k] = 0; if (k < 3) P.tiles[k] = 0; }
    if (rc) return rc;
    if (any8) return opt_table<6>(t, n, S, nb, 3, !any32, P, st);
    for (int k = 3; k < 7; ++k) { P.first[k] = P.first[3]; if (k < 6) P.tiles[k] = 0; }
    return 0;
}

// The arguments of the few-tensor kernels, if the call is one for them: one kind, no more tensors than the arguments hold, none above `most`
// elements, `total` elements at most in all. Returns the kind, or -1 if it is not.
template <int PTRS>
static int opt_few(const NndetOptTensor* t, int32_t n, int64_t most, int64_t total, const OptScalars& S, OptPlan& P, OptTableArgs<PTRS>& A) {
    if (n < 1 || n > OptTableArgs<PTRS>::MOST || (PTRS == 6) != (t[0].state_bits == 8)) return -1;
    const int kind = opt_kind(t[0]);
    for (int i = 0; i < n; ++i) {
        total -= t[i].numel;
        if (opt_kind(t[i]) != kind || t[i].numel > most || total < 0) return -1;
    }
    opt_scalars(S, P.head, A);
    A.n = n;
    for (int i = 0; i < n; ++i) opt_arg(t[i], 0, A.a[i]);
    return kind;
}

static inline unsigned opt_grid(int64_t tiles, int most) { return (unsigned)(tiles < most ? tiles : most); }

static OptMem opt_mem(const OptPlan& P, int k) { return {P.entry + P.first[k], P.tile0 + P.first[k], P.first[k + 1] - P.first[k]}; }

// The norm's launches. own: all tensors, of one type, with PTRS addresses each (0: none; above 1 the table is written on the way). N: what the kernels behind them need
// (N.count 0: the factor is in the head).
template <int NB, int PTRS>
static int opt_norm(const OptPlan& P, const OptTableArgs<PTRS ? PTRS : 1>* own, const float* grad_scale, double max_norm, float* norm, bool given, OptSums& N, hipStream_t st) {
    int64_t tiles = 0;
    int kinds = 0, count = 0;
    for (int k = 0; k < 6; ++k) tiles += P.tiles[k], kinds += P.tiles[k] != 0;
    N = {P.partial, 0, grad_scale, max_norm, norm};
    const bool finish = given || !kinds || max_norm < 0.0 || tiles > OPT_INLINE_TILES;
    for (int k = 0; k < 6 && !given; ++k) {
        if (!P.tiles[k]) continue;
        const unsigned g = opt_grid(P.tiles[k], finish ? OPT_PARTIALS : OPT_INLINE / kinds);
#define OPT_OWN(T) (k_opt_sumsq_own<T, NB, PTRS><<<g + (PTRS > 1), OPT_WG, 0, st>>>(*own, (uint32_t)P.tiles[k], P.partial))
#define OPT_CALL(T) (k_opt_sumsq<T, NB><<<g, OPT_WG, 0, st>>>(opt_mem(P, k), (uint32_t)P.tiles[k], P.partial + count))
        if constexpr (PTRS != 0)
            if (own) NNDET_DISPATCH_DTYPE(k % 3, OPT_OWN);
        if constexpr (PTRS < 2)
            if (!own) NNDET_DISPATCH_DTYPE(k % 3, OPT_CALL);
#undef OPT_OWN
#undef OPT_CALL
        LAUNCH_CHECK();
        count += (int)g;
    }
    if (!finish) {
        N.count = count;
        return 0;
    }
    k_opt_norm<<<1, OPT_NORM_WG, 0, st>>>(P.partial, given ? -1 : count, grad_scale, max_norm, norm, P.head);
    LAUNCH_CHECK();
    return 0;
}

// The plan of a call whose tensors are of one kind and in A; false if they are not (or are all empty).
template <int PTRS>
static bool opt_own(const NndetOptTensor* t, int32_t n, const OptScalars& S, int nb, OptPlan& P, OptTableArgs<PTRS>& A) {
    const int kind = opt_few(t, n, INT64_MAX, INT64_MAX, S, P, A);
    if (kind < 0) return false;
    int64_t tiles = 0;
    for (int i = 0; i < n; ++i) {
        A.a[i].tile0 = (uint32_t)tiles;
        tiles += ceil_div64(t[i].numel, nb * 4 * OPT_BLOCK);
    }
    for (int k = 0; k < 7; ++k) P.first[k] = k <= kind ? 0 : n;
    for (int k = 0; k < 6; ++k) P.tiles[k] = k == kind ? tiles : 0;
    return tiles != 0;
}

// The norm of a step, with the table: one launch if the tensors fit the kernel arguments.
template <int PTRS>
static int adamw_norm(const NndetOptTensor* t, int32_t n, const NndetAdamw* a, const OptScalars& S, OptPlan& P, OptSums& N, hipStream_t st, bool* done) {
    OptTableArgs<PTRS> A;
    *done = opt_own(t, n, S, OPT_NB, P, A);
    if (!*done) return 0;
    A.entry = P.entry; A.coef = P.coef; A.tile0 = P.tile0;
    A.first = 1;
    return opt_norm<OPT_NB, PTRS>(P, &A, a->grad_scale, a->max_norm, a->norm, false, N, st);
}

// An AdamW step of few tensors: true if it was one (its return code in rc).
template <int BITS>
static bool adamw_few(const NndetOptTensor* t, int32_t n, const NndetAdamw* a, const OptScalars& S, const OptHyper& H, OptPlan& P, hipStream_t st, int* rc) {
    OptTableArgs<BITS == 8 ? 6 : 4> A;
    const bool clip = a->max_norm >= 0.0;
    if (clip && a->norm_given) return false;
    const int k = opt_few(t, n, clip ? OPT_FEW_STEP.most : OPT_FEW, clip ? OPT_FEW_STEP.total : INT64_MAX, S, P, A);
    if (k < 0) return false;
#define OPT_NORM(T) (k_opt_norm_few<T, false><<<1, OPT_FEW_WG, 0, st>>>(A, a->max_norm, a->norm))
#define OPT_CALL(T) (k_adamw_few<T, BITS><<<n, OPT_FEW_WG, 0, st>>>(A, H, clip))
    if (clip) NNDET_DISPATCH_DTYPE(k % 3, OPT_NORM);
    NNDET_DISPATCH_DTYPE(k % 3, OPT_CALL);
#undef OPT_NORM
#undef OPT_CALL
    *rc = (int)hipGetLastError();
    return true;
}

extern "C" int nndet_adamw_step(const NndetOptTensor* tensors, int32_t n, const NndetAdamw* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!a || !a->steps || !(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0) || !(a->eps == 0.0 || a->eps >= 0x1p-126)) return NNDET_EINVAL;
    if (a->max_norm != a->max_norm || (a->norm_given && (!a->norm || a->max_norm < 0.0))) return NNDET_EINVAL;
    // the norm is written while other workgroups read the scalars
    if (a->norm && !a->norm_given && (a->norm == a->grad_scale || a->norm == a->lr_device || a->norm == a->found_inf)) return NNDET_EINVAL;
    hipStream_t st = as_stream(stream);
    const OptScalars S = {a->steps, a->lr_device, a->found_inf, a->grad_scale, a->lr, a->beta1, a->beta2};
    const OptHyper H = {(float)a->beta1, (float)(1.0 - a->beta1), (float)a->beta2, (float)(1.0 - a->beta2), (float)a->eps};
    OptPlan P;
    int rc = opt_check(tensors, n, 7, workspace, workspace_bytes, P);
    if (rc || adamw_few<32>(tensors, n, a, S, H, P, st, &rc) || adamw_few<8>(tensors, n, a, S, H, P, st, &rc)) return rc;
    OptSums N = {};
    bool own = false;
    if (a->max_norm >= 0.0 && !a->norm_given) {
        rc = adamw_norm<4>(tensors, n, a, S, P, N, st, &own);
        if (!rc && !own) rc = adamw_norm<6>(tensors, n, a, S, P, N, st, &own);
        if (rc) return rc;
    }
    if (!own) {
        rc = opt_begin(tensors, n, S, OPT_NB, P, st);
        if (!rc && a->max_norm >= 0.0) rc = opt_norm<OPT_NB, 0>(P, nullptr, a->grad_scale, a->max_norm, a->norm, a->norm_given != 0, N, st);
        if (rc) return rc;
    }
    for (int k = 0; k < 6; ++k) {
        if (!P.tiles[k]) continue;
        const unsigned g = opt_grid(P.tiles[k], OPT_GRID);
        const OptCoef* c = P.coef + P.first[k];
#define OPT_CALL8(T) (k_adamw<T, 8><<<g, OPT_WG, 0, st>>>(P.head, opt_mem(P, k), c, (uint32_t)P.tiles[k], H, N))
#define OPT_CALL32(T) (k_adamw<T, 32><<<g, OPT_WG, 0, st>>>(P.head, opt_mem(P, k), c, (uint32_t)P.tiles[k], H, N))
        if (k >= 3) NNDET_DISPATCH_DTYPE(k % 3, OPT_CALL8);
        else NNDET_DISPATCH_DTYPE(k % 3, OPT_CALL32);
#undef OPT_CALL8
#undef OPT_CALL32
        LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int nndet_grad_clip(const NndetOptTensor* tensors, int32_t n, double max_norm, const float* grad_scale, float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (max_norm != max_norm || !norm_out || (grad_scale && max_norm >= 0.0)) return NNDET_EINVAL;
    hipStream_t st = as_stream(stream);
    const OptScalars S = {nullptr, nullptr, nullptr, nullptr, 0.0, 0.0, 0.0};
    OptPlan P;
    int rc = opt_check(tensors, n, 2, workspace, workspace_bytes, P);
    if (rc) return rc;
    for (int i = 0; i < n; ++i)
        if (tensors[i].state_bits != 32) return NNDET_EINVAL;
    OptTableArgs<1> A;
    const int few = opt_few(tensors, n, OPT_FEW_CLIP.most, OPT_FEW_CLIP.total, {nullptr, nullptr, nullptr, grad_scale, 0.0, 0.0, 0.0}, P, A);
    if (few >= 0) {
#define OPT_CALL(T) (k_opt_norm_few<T, true><<<1, OPT_FEW_WG, 0, st>>>(A, max_norm, norm_out))
        NNDET_DISPATCH_DTYPE(few % 3, OPT_CALL);
#undef OPT_CALL
        LAUNCH_CHECK();
        return 0;
    }
    // Tensors of one type that fit the kernel arguments need no table (10 tensors of 8000 elements 18.5 / 8.8 -> 13.5 / 5.3 us of host / GPU time together
    // with the norm's finish in the scaling kernel).
    const bool own = opt_own(tensors, n, S, OPT_CLIP_NB, P, A);
    if (!own && (rc = opt_begin(tensors, n, S, OPT_CLIP_NB, P, st, true))) return rc;
    OptSums N;
    rc = opt_norm<OPT_CLIP_NB, 1>(P, own ? &A : nullptr, grad_scale, max_norm, norm_out, false, N, st);
    if (rc || max_norm < 0.0) return rc;         // the norm alone
    for (int k = 0; k < 3; ++k) {
        if (!P.tiles[k]) continue;
        const unsigned g = opt_grid(P.tiles[k], OPT_GRID);
#define OPT_OWN(T) (k_opt_scale_own<T><<<g, OPT_WG, 0, st>>>(A, (uint32_t)P.tiles[k], N))
#define OPT_CALL(T) (k_opt_scale<T><<<g, OPT_WG, 0, st>>>(opt_mem(P, k), (uint32_t)P.tiles[k], P.head, N))
        if (own) NNDET_DISPATCH_DTYPE(k % 3, OPT_OWN);
        else NNDET_DISPATCH_DTYPE(k % 3, OPT_CALL);
#undef OPT_OWN
#undef OPT_CALL
        LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int nndet_adam_state8(const NndetOptTensor* tensors, int32_t n, int32_t write, void* workspace, size_t workspace_bytes, void* stream) {
    for (int i = 0; tensors && i < n; ++i)
        if (tensors[i].dtype != NNDET_F32 || tensors[i].state_bits != 8) return NNDET_EINVAL;
    hipStream_t st = as_stream(stream);
    const OptScalars S = {nullptr, nullptr, nullptr, nullptr, 0.0, 0.0, 0.0};
    OptPlan P;
    int rc = opt_check(tensors, n, 7, workspace, workspace_bytes, P);
    if (rc) return rc;
    OptTableArgs<6> A;
    const int few = opt_few(tensors, n, OPT_FEW, INT64_MAX, S, P, A);
    if (few >= 0) {
        if (write) k_opt_state8_few<true><<<n, OPT_FEW_WG, 0, st>>>(A);
        else k_opt_state8_few<false><<<n, OPT_FEW_WG, 0, st>>>(A);
        LAUNCH_CHECK();
        return 0;
    }
    rc = opt_begin(tensors, n, S, OPT_NB, P, st);
    if (rc) return rc;
    const int k = NNDET_F32 + 3;
    if (!P.tiles[k]) return 0;
    const unsigned g = opt_grid(P.tiles[k], OPT_GRID);
    if (write) k_opt_state8<true><<<g, OPT_WG, 0, st>>>(opt_mem(P, k), (uint32_t)P.tiles[k]);
    else k_opt_state8<false><<<g, OPT_WG, 0, st>>>(opt_mem(P, k), (uint32_t)P.tiles[k]);
    LAUNCH_CHECK();
    return 0;
}
