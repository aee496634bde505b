// Optimiser step over many tensors at once: AdamW with fp32 or 8-bit moments, the global gradient norm and clipping by it, and the
// conversion between fp32 and 8-bit moments.
//
// A call takes n tensors of any sizes. k_opt_table copies their addresses out of the kernel arguments into a table in the workspace (64 B
// a tensor, OPT_ARGS of them a launch, so that every later kernel is ONE launch whatever n is), advances the step counts and works out what
// is the same for a whole tensor. Then one launch per storage kind walks over tiles of 1024 consecutive elements of a tensor; no tile spans
// two tensors. A wave owns 256 consecutive elements of its tile, which is also the block that shares a scale of the 8-bit moments: the
// block maximum never leaves the wave.
//
// AdamW, t = count + 1, g' = g * factor (factor = clip / loss scale):
//   m = b1 m + (1 - b1) g'        v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) * m / (sqrt(v) * (1 - b2^t)^-1/2 + eps)
// in fp32 with every operation rounded by itself (this file is compiled without contraction; division and square root are the IEEE ones),
// so that the 8-bit codes do not depend on how a compiler fuses; 1 - b^t, lr / (1 - b1^t) and the factor are worked out in fp64 and rounded
// once. Parameters and gradients in 16 bits are read to fp32 and the new parameter is rounded once, to nearest even.
//
// 8-bit moments: m and r = sqrt(v) as e4m3 codes with one fp32 scale = max |.| / 448 a block. r instead of v because e4m3 spans 2^17.8 and
// v's range is the square of the gradients'. m is rounded to nearest even (it changes by 10 % a step, codes are 6 - 12 % apart); r changes
// by about 0.05 % a step and would never leave its code under rounding to nearest, so it is rounded up with the probability of its distance
// from the code below: the expected value of the stored r is r. The 16 random bits an element come from its index in the tensor and
// t alone (opt_mix), so a step is reproducible. An r that is not zero is not stored as zero: m / (0 + eps) would be a step of any size.
#include "common.h"
#include <string.h>

static constexpr int OPT_WG = 256;               // threads of a workgroup: 4 waves
static constexpr int OPT_BLOCK = 256;            // elements of a wave's block = elements that share a scale
static constexpr int OPT_TILE = 1024;            // elements of a workgroup's tile
static constexpr int OPT_ARGS = 62;              // tensors per k_opt_table launch: 62 * 64 B + 88 B of scalars stay below 4 KB of arguments
static constexpr int OPT_PARTIALS = 1024;        // workgroups (and fp64 partial sums) of the norm per storage type
static constexpr int OPT_GRID = 2048;            // workgroups of a walk over the tiles: 8 for each of the 256 CUs

struct OptEntry {                                // one tensor in the workspace's table
    void* p; const void* g; void* m; void* v; float* ms; float* rs;
    int64_t numel;
    uint32_t tile0, pad;                         // first tile within its launch
};
struct OptCoef { float size, unbias, decay; uint32_t t; };
struct OptHead { float factor; int32_t skip; int32_t pad[14]; };

struct OptArg { void* p; const void* g; void* m; void* v; float* ms; float* rs; uint64_t numel_slot; float wd; uint32_t tile0; };
struct OptTableArgs {
    OptHead* head; OptEntry* entry; OptCoef* coef; int32_t* steps;
    const float* lr_ptr; const float* found_inf; const float* grad_scale;
    double lr, b1, b2;
    int32_t n, first;                            // entries of this launch; first: it also writes the head
    OptArg a[OPT_ARGS];
};
static_assert(sizeof(OptTableArgs) <= 4096, "kernel arguments are limited to 4 KB");

__global__ __launch_bounds__(64) void k_opt_table(const OptTableArgs A) {
    const int i = threadIdx.x;
    const bool skip = A.found_inf && *A.found_inf != 0.0f;
    if (A.first && i == 0) {
        A.head->skip = skip;
        A.head->factor = A.grad_scale ? (float)(1.0 / (double)*A.grad_scale) : 1.0f;   // (the norm's kernel writes it again)
    }
    if (i >= A.n) return;
    const OptArg& a = A.a[i];
    OptEntry e = {a.p, a.g, a.m, a.v, a.ms, a.rs, (int64_t)(a.numel_slot & ((1ull << 40) - 1)), a.tile0, 0};
    A.entry[i] = e;
    if (!A.steps) return;
    const uint32_t slot = (uint32_t)(a.numel_slot >> 40);
    const int32_t t = A.steps[slot] + 1;
    if (!skip) A.steps[slot] = t;
    const double lr = A.lr_ptr ? (double)*A.lr_ptr : A.lr;
    OptCoef c;
    c.size = (float)(lr / (1.0 - pow(A.b1, (double)t)));
    c.unbias = (float)(1.0 / sqrt(1.0 - pow(A.b2, (double)t)));
    c.decay = (float)(1.0 - lr * (double)a.wd);
    c.t = (uint32_t)t;
    A.coef[i] = c;
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

// index of the tensor whose tiles contain `tile`: the last entry with tile0 <= tile (entries are in order of tile0). One ballot per 64 tensors.
__device__ __forceinline__ int opt_find(const OptEntry* e, int n, uint32_t tile) {
    const int lane = threadIdx.x & 63;
    int found = 0;
    for (int b = 0; b < n; b += 64) {
        const bool le = b + lane < n && e[b + lane].tile0 <= tile;
        const int c = __popcll(__ballot(le));
        found += c;
        if (c < 64) break;
    }
    return __builtin_amdgcn_readfirstlane(found - 1);
}

// The walk of a workgroup over the tiles blockIdx.x, blockIdx.x + gridDim.x, ...: at any time the chip works on neighbouring addresses (few
// pages, few open DRAM rows). The tensor is looked up again only when the walk leaves it.
struct OptWalk {
    const OptEntry* e; int n; uint32_t tiles, tile, end;
    int i;
    OptEntry cur;
    __device__ OptWalk(const OptEntry* e_, int n_, uint32_t tiles_) : e(e_), n(n_), tiles(tiles_), tile(blockIdx.x), end(0), i(-1) {}
    __device__ __forceinline__ void next() { tile += gridDim.x; }
    __device__ __forceinline__ bool enter() {    // true if the tile is another tensor's than the last one
        if (tile < end) return false;
        i = opt_find(e, n, tile);
        cur = opt_uniform(e + i);
        end = i + 1 < n ? opt_uniform(&e[i + 1].tile0) : tiles;
        return true;
    }
    // this wave's block: its first element, and how many of its elements there are (<= 0: none)
    __device__ __forceinline__ int64_t base() const { return (int64_t)(tile - cur.tile0) * OPT_TILE + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * OPT_BLOCK; }
    __device__ __forceinline__ int rem() const {
        const int64_t r = cur.numel - base();
        return r < OPT_BLOCK ? (int)r : OPT_BLOCK;        // (a tile is not empty: r > -OPT_TILE)
    }
    // whether four elements of p (wp) and g (wg) are aligned vectors of T, and m and v are aligned to ms bytes (0: not used)
    template <typename T> __device__ __forceinline__ bool aligned(int wp, int wg, int ms) const {
        uintptr_t a = 0;
        if (wp) a |= (uintptr_t)cur.p & (4 * sizeof(T) - 1);
        if (wg) a |= (uintptr_t)cur.g & (4 * sizeof(T) - 1);
        if (ms) a |= ((uintptr_t)cur.m | (uintptr_t)cur.v) & (ms - 1);
        return a == 0;
    }
};

// ---- four elements a lane. FULL (a whole block of an aligned tensor): one vector a lane, elements 4 lane + 0..3; else element by element,
// lane + 64 k while that is below rem, zeros behind. The addresses come out of the table, so the compiler is told that they are global.
template <typename T> using OptPtr = __attribute__((address_space(1))) T*;
template <typename T> __device__ __forceinline__ OptPtr<T> opt_at(const void* p, int64_t i) { return (OptPtr<T>)(uintptr_t)p + i; }
template <typename T> struct OptVec4;
template <> struct OptVec4<float> { typedef f32x4 type; };
template <> struct OptVec4<bf16_t> { typedef bf16_t type __attribute__((ext_vector_type(4))); };
template <> struct OptVec4<f16_t> { typedef f16_t type __attribute__((ext_vector_type(4))); };

template <bool FULL, typename T> __device__ __forceinline__ void opt_load(OptPtr<T> p, int lane, int rem, float* x) {
    if constexpr (FULL) {
        const auto v = ((OptPtr<typename OptVec4<T>::type>)p)[lane];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = Elem<T>::ld(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = lane + 64 * k < rem ? Elem<T>::ld(p[lane + 64 * k]) : 0.0f;
    }
}
template <bool FULL, typename T> __device__ __forceinline__ void opt_store(OptPtr<T> p, int lane, int rem, const float* x) {
    if constexpr (FULL) {
        typename OptVec4<T>::type v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = Elem<T>::st(x[k]);
        ((OptPtr<typename OptVec4<T>::type>)p)[lane] = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane + 64 * k < rem) p[lane + 64 * k] = Elem<T>::st(x[k]);
    }
}
template <bool FULL> __device__ __forceinline__ uint32_t opt_load_codes(OptPtr<uint8_t> p, int lane, int rem) {
    if constexpr (FULL) return ((OptPtr<uint32_t>)p)[lane];
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) c |= (lane + 64 * k < rem ? (uint32_t)p[lane + 64 * k] : 0u) << (8 * k);
    return c;
}
template <bool FULL> __device__ __forceinline__ void opt_store_codes(OptPtr<uint8_t> p, int lane, int rem, uint32_t c) {
    if constexpr (FULL) { ((OptPtr<uint32_t>)p)[lane] = c; return; }
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
// integers, so a NaN (an inf) is the largest and makes the scale NaN (inf): the block then reads back as NaN.
__device__ __forceinline__ float opt_scale(const float* x) {
    uint32_t a = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) { const uint32_t b = __float_as_uint(x[k]) & 0x7fffffffu; a = b > a ? b : a; }
    const float s = __uint_as_float(wave_max_u32(a)) * (float)(1.0 / 448.0);
    return s < 0x1p-110f ? 0.0f : s;
}
__device__ __forceinline__ void opt_decode(uint32_t c, float s, float* x) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    x[0] = lo[0] * s; x[1] = lo[1] * s; x[2] = hi[0] * s; x[3] = hi[1] * s;
}
__device__ __forceinline__ uint32_t opt_encode(const float* x, float s, bool root) {      // to nearest even
    const float inv = 1.0f / s;
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        y[k] = s > 0.0f ? x[k] * inv : 0.0f;
        if (root && x[k] > 0.0f && s > 0.0f) y[k] = y[k] < 0x1p-9f ? 0x1p-9f : y[k];
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
    const float inv = 1.0f / s;
    uint32_t c = 0, bits = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = FULL ? index + k : index + 64 * k;
        if (!FULL || !(k & 1)) bits = opt_mix((uint32_t)(i >> 1), t);
        const uint32_t u = ((FULL ? k : (int)i) & 1 ? bits >> 16 : bits & 0xffffu) * 16 + 8;
        const float y = s > 0.0f ? x[k] * inv : 0.0f;
        uint32_t q = (__float_as_uint(y * 0x1p-120f) + u) >> 20;
        q = q > 0x7eu ? 0x7eu : q;
        if (q == 0 && x[k] > 0.0f && s > 0.0f) q = 1;
        c |= q << (8 * k);
    }
    return c;
}

struct OptHyper { float b1, omb1, b2, omb2, eps; };

template <typename T, int BITS, bool FULL>
__device__ __forceinline__ void adamw_block(const OptEntry& e, int64_t base, int rem, const OptCoef& c, const OptHyper& H, float factor, int lane) {
    float p[4], g[4], m[4], v[4], r[4];
    const int64_t block = base / OPT_BLOCK;
    opt_load<FULL>(opt_at<T>(e.g, base), lane, rem, g);
    if constexpr (BITS == 8) {
        const uint32_t cm = opt_load_codes<FULL>(opt_at<uint8_t>(e.m, base), lane, rem);
        const uint32_t cv = opt_load_codes<FULL>(opt_at<uint8_t>(e.v, base), lane, rem);
        const float sm = *opt_at<float>(e.ms, block), sr = *opt_at<float>(e.rs, block);
        opt_load<FULL>(opt_at<T>(e.p, base), lane, rem, p);
        opt_decode(cm, sm, m);
        opt_decode(cv, sr, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = v[k] * v[k];
    } else {
        opt_load<FULL>(opt_at<float>(e.m, base), lane, rem, m);
        opt_load<FULL>(opt_at<float>(e.v, base), lane, rem, v);
        opt_load<FULL>(opt_at<T>(e.p, base), lane, rem, p);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        g[k] = g[k] * factor;
        m[k] = m[k] * H.b1 + g[k] * H.omb1;
        v[k] = v[k] * H.b2 + (g[k] * g[k]) * H.omb2;
        r[k] = sqrtf(v[k]);
        p[k] = p[k] * c.decay - (m[k] / (r[k] * c.unbias + H.eps)) * c.size;
    }
    opt_store<FULL>(opt_at<T>(e.p, base), lane, rem, p);
    if constexpr (BITS == 8) {
        if constexpr (!FULL) {                   // lanes past the end do not count in the maxima (a factor that is not finite would be in them)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (lane + 64 * k >= rem) m[k] = r[k] = 0.0f;
        }
        const float sm = opt_scale(m), sr = opt_scale(r);
        opt_store_codes<FULL>(opt_at<uint8_t>(e.m, base), lane, rem, opt_encode(m, sm, false));
        opt_store_codes<FULL>(opt_at<uint8_t>(e.v, base), lane, rem, opt_encode_root<FULL>(r, sr, base + (FULL ? 4 * lane : lane), c.t));
        if (lane == 0) { *opt_at<float>(e.ms, block) = sm; *opt_at<float>(e.rs, block) = sr; }
    } else {
        opt_store<FULL>(opt_at<float>(e.m, base), lane, rem, m);
        opt_store<FULL>(opt_at<float>(e.v, base), lane, rem, v);
    }
}

template <typename T, int BITS>
__global__ __launch_bounds__(OPT_WG) void k_adamw(const OptHead* head, const OptEntry* entry, const OptCoef* coef, int n, uint32_t tiles, OptHyper H) {
    if (opt_uniform(&head->skip)) return;
    const float factor = opt_uniform(&head->factor);
    const int lane = threadIdx.x & 63;
    OptCoef c = {};
    for (OptWalk w(entry, n, tiles); w.tile < w.tiles; w.next()) {
        if (w.enter()) c = opt_uniform(coef + w.i);
        const int rem = w.rem();
        if (rem <= 0) continue;
        if (rem == OPT_BLOCK && w.aligned<T>(1, 1, BITS == 8 ? 4 : 16)) adamw_block<T, BITS, true>(w.cur, w.base(), rem, c, H, factor, lane);
        else adamw_block<T, BITS, false>(w.cur, w.base(), rem, c, H, factor, lane);
    }
}

// ---- global gradient norm: squares summed in fp64 (no overflow, and fp64 multiply-add runs at the rate of fp32 here), a fixed order
template <bool FULL, typename T> __device__ __forceinline__ double opt_sumsq(const OptEntry& e, int64_t base, int rem, int lane, double s) {
    float g[4];
    opt_load<FULL>(opt_at<T>(e.g, base), lane, rem, g);
#pragma unroll
    for (int k = 0; k < 4; ++k) s = fma((double)g[k], (double)g[k], s);
    return s;
}
template <typename T>
__global__ __launch_bounds__(OPT_WG) void k_opt_sumsq(const OptEntry* entry, int n, uint32_t tiles, double* partial) {
    __shared__ double part[OPT_WG / 64];
    const int lane = threadIdx.x & 63;
    double s = 0.0;
    for (OptWalk w(entry, n, tiles); w.tile < w.tiles; w.next()) {
        w.enter();
        const int rem = w.rem();
        if (rem <= 0) continue;
        if (rem == OPT_BLOCK && w.aligned<T>(0, 1, 0)) s = opt_sumsq<true, T>(w.cur, w.base(), rem, lane, s);
        else s = opt_sumsq<false, T>(w.cur, w.base(), rem, lane, s);
    }
    s = wave_sum_f64(s);
    if (lane == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// norm of the unscaled gradients (count < 0: given at norm_at) and the factor they are multiplied with: min(1, max_norm / (norm + 1e-6)) / loss scale. One workgroup.
__global__ __launch_bounds__(OPT_WG) void k_opt_norm(const double* partial, int count, const float* grad_scale, double max_norm, float* norm_at, OptHead* head) {
    __shared__ double part[OPT_WG / 64];
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += OPT_WG) s += partial[i];
    s = wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double scale = grad_scale ? (double)*grad_scale : 1.0;
        const float norm = count < 0 ? *norm_at : (float)(sqrt((part[0] + part[1]) + (part[2] + part[3])) / scale);
        const double clip = max_norm / ((double)norm + 1e-6);
        head->factor = (float)((1.0 / scale) * (clip > 1.0 ? 1.0 : clip));     // (a NaN norm gives a NaN factor)
        if (norm_at && count >= 0) *norm_at = norm;
    }
}

template <bool FULL, typename T> __device__ __forceinline__ void opt_scale_block(const OptEntry& e, int64_t base, int rem, int lane, float factor) {
    float g[4];
    opt_load<FULL>(opt_at<T>(e.g, base), lane, rem, g);
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = g[k] * factor;
    opt_store<FULL>(opt_at<T>(e.g, base), lane, rem, g);
}
template <typename T>
__global__ __launch_bounds__(OPT_WG) void k_opt_scale(const OptHead* head, const OptEntry* entry, int n, uint32_t tiles) {
    const float factor = opt_uniform(&head->factor);
    if (factor == 1.0f) return;                  // nothing to clip: x * 1 is x for every x
    const int lane = threadIdx.x & 63;
    for (OptWalk w(entry, n, tiles); w.tile < w.tiles; w.next()) {
        w.enter();
        const int rem = w.rem();
        if (rem <= 0) continue;
        if (rem == OPT_BLOCK && w.aligned<T>(0, 1, 0)) opt_scale_block<true, T>(w.cur, w.base(), rem, lane, factor);
        else opt_scale_block<false, T>(w.cur, w.base(), rem, lane, factor);
    }
}

// ---- fp32 moments (p: exp_avg, g: exp_avg_sq) <-> 8-bit moments
template <bool FULL, bool WRITE> __device__ __forceinline__ void opt_state8_block(const OptEntry& e, int64_t base, int rem, int lane) {
    const int64_t block = base / OPT_BLOCK;
    float m[4], v[4];
    if constexpr (WRITE) {
        opt_load<FULL>(opt_at<float>(e.p, base), lane, rem, m);
        opt_load<FULL>(opt_at<float>(e.g, base), lane, rem, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = sqrtf(v[k]);
        const float sm = opt_scale(m), sr = opt_scale(v);
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
        opt_store<FULL>(opt_at<float>(e.p, base), lane, rem, m);
        opt_store<FULL>(opt_at<float>(e.g, base), lane, rem, v);
    }
}
template <bool WRITE>
__global__ __launch_bounds__(OPT_WG) void k_opt_state8(const OptEntry* entry, int n, uint32_t tiles) {
    const int lane = threadIdx.x & 63;
    for (OptWalk w(entry, n, tiles); w.tile < w.tiles; w.next()) {
        w.enter();
        const int rem = w.rem();
        if (rem <= 0) continue;
        if (rem == OPT_BLOCK && w.aligned<float>(1, 1, 4)) opt_state8_block<true, WRITE>(w.cur, w.base(), rem, lane);
        else opt_state8_block<false, WRITE>(w.cur, w.base(), rem, lane);
    }
}

// ---- host side
// kinds of a launch: parameter type x bits of the moments
static inline int opt_kind(const NndetOptTensor& t) { return t.dtype * 2 + (t.state_bits == 8 ? 1 : 0); }

static size_t opt_bytes(int64_t n) {
    return sizeof(OptHead) + 3 * OPT_PARTIALS * sizeof(double) + (size_t)n * (sizeof(OptEntry) + sizeof(OptCoef));
}
extern "C" size_t nndet_opt_workspace_bytes(int32_t n) { return n < 0 ? 0 : opt_bytes(n); }

struct OptPlan {                                 // the tensors of a call in the order of their kinds, as they lie in the table
    OptHead* head; double* partial; OptEntry* entry; OptCoef* coef;
    int first[7];                                // entries of kind k: first[k] .. first[k + 1]
    int64_t tiles[6];
};

// Checks the tensors, lays the workspace out and launches k_opt_table. `need`: bit 0 param, 1 grad, 2 moments (scales with 8 bits).
static int opt_begin(const NndetOptTensor* t, int32_t n, int need, OptTableArgs& A, void* ws, size_t ws_bytes, OptPlan& P, hipStream_t st) {
    if (n < 0 || (n > 0 && !t) || n >= (1 << 24)) return NNDET_EINVAL;
    if (!ws || ((uintptr_t)ws & 15)) return NNDET_EINVAL;
    if (ws_bytes < opt_bytes(n)) return NNDET_EWORKSPACE;
    P.head = (OptHead*)ws;
    P.partial = (double*)(P.head + 1);
    P.entry = (OptEntry*)(P.partial + 3 * OPT_PARTIALS);
    P.coef = (OptCoef*)(P.entry + n);
    for (int i = 0; i < n; ++i) {
        if (t[i].dtype < 0 || t[i].dtype > 2 || (t[i].state_bits != 32 && t[i].state_bits != 8)) return NNDET_EINVAL;
        if (t[i].numel < 0 || t[i].numel >= (int64_t)1 << 40 || t[i].slot < 0 || t[i].slot >= (1 << 24)) return NNDET_EINVAL;
        if (t[i].numel == 0) continue;
        if (((need & 1) && !t[i].param) || ((need & 2) && !t[i].grad) || ((need & 4) && (!t[i].exp_avg || !t[i].exp_avg_sq))) return NNDET_EINVAL;
        if ((need & 4) && t[i].state_bits == 8 && (!t[i].exp_avg_scale || !t[i].root_scale)) return NNDET_EINVAL;
    }
    A.head = P.head; A.first = 1; A.n = 0;
    int at = 0;
    for (int k = 0; k < 6; ++k) {
        P.first[k] = at;
        int64_t tiles = 0;
        for (int i = 0; i < n; ++i) {
            if (opt_kind(t[i]) != k || (t[i].numel == 0 && !A.steps)) continue;
            OptArg& a = A.a[A.n++];
            a.p = t[i].param; a.g = t[i].grad; a.m = t[i].exp_avg; a.v = t[i].exp_avg_sq; a.ms = t[i].exp_avg_scale; a.rs = t[i].root_scale;
            a.numel_slot = (uint64_t)t[i].numel | ((uint64_t)t[i].slot << 40);
            a.wd = (float)t[i].weight_decay;
            a.tile0 = (uint32_t)tiles;
            tiles += ceil_div64(t[i].numel, OPT_TILE);
            if (tiles >= ((int64_t)1 << 32) - 65536) return NNDET_EINVAL;       // (a walk steps past the last tile)
            ++at;
            if (A.n == OPT_ARGS) {
                A.entry = P.entry + at - A.n; A.coef = P.coef + at - A.n;
                k_opt_table<<<1, 64, 0, st>>>(A);
                LAUNCH_CHECK();
                A.n = 0; A.first = 0;
            }
        }
        P.tiles[k] = tiles;
    }
    P.first[6] = at;
    if (A.n || A.first) {
        A.entry = P.entry + at - A.n; A.coef = P.coef + at - A.n;
        k_opt_table<<<1, 64, 0, st>>>(A);
        LAUNCH_CHECK();
    }
    return 0;
}

static inline unsigned opt_grid(int64_t tiles, int most) { return (unsigned)(tiles < most ? tiles : most); }

static int opt_norm(const OptPlan& P, const float* grad_scale, double max_norm, float* norm, bool given, hipStream_t st) {
    int count = 0;
    for (int k = 0; k < 6 && !given; ++k) {
        if (!P.tiles[k]) continue;
        const unsigned g = opt_grid(P.tiles[k], OPT_PARTIALS / 2);
        const OptEntry* e = P.entry + P.first[k];
        const int n = P.first[k + 1] - P.first[k];
#define OPT_CALL(T) (k_opt_sumsq<T><<<g, OPT_WG, 0, st>>>(e, n, (uint32_t)P.tiles[k], P.partial + count))
        NNDET_DISPATCH_DTYPE(k >> 1, OPT_CALL);
#undef OPT_CALL
        LAUNCH_CHECK();
        count += (int)g;
    }
    k_opt_norm<<<1, OPT_WG, 0, st>>>(P.partial, given ? -1 : count, grad_scale, max_norm, norm, P.head);
    LAUNCH_CHECK();
    return 0;
}

extern "C" int nndet_adamw_step(const NndetOptTensor* tensors, int32_t n, const NndetAdamw* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!a || !a->steps || !(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0) || !(a->eps >= 0.0)) return NNDET_EINVAL;
    if (a->max_norm != a->max_norm || (a->norm_given && (!a->norm || a->max_norm < 0.0))) return NNDET_EINVAL;
    hipStream_t st = as_stream(stream);
    OptTableArgs A;
    memset(&A, 0, sizeof(A));
    A.steps = a->steps; A.lr_ptr = a->lr_device; A.found_inf = a->found_inf; A.grad_scale = a->grad_scale;
    A.lr = a->lr; A.b1 = a->beta1; A.b2 = a->beta2;
    OptPlan P;
    int rc = opt_begin(tensors, n, 7, A, workspace, workspace_bytes, P, st);
    if (rc) return rc;
    if (a->max_norm >= 0.0) {
        rc = opt_norm(P, a->grad_scale, a->max_norm, a->norm, a->norm_given != 0, st);
        if (rc) return rc;
    }
    const OptHyper H = {(float)a->beta1, (float)(1.0 - a->beta1), (float)a->beta2, (float)(1.0 - a->beta2), (float)a->eps};
    for (int k = 0; k < 6; ++k) {
        if (!P.tiles[k]) continue;
        const unsigned g = opt_grid(P.tiles[k], OPT_GRID);
        const OptEntry* e = P.entry + P.first[k];
        const OptCoef* c = P.coef + P.first[k];
        const int m = P.first[k + 1] - P.first[k];
#define OPT_CALL8(T) (k_adamw<T, 8><<<g, OPT_WG, 0, st>>>(P.head, e, c, m, (uint32_t)P.tiles[k], H))
#define OPT_CALL32(T) (k_adamw<T, 32><<<g, OPT_WG, 0, st>>>(P.head, e, c, m, (uint32_t)P.tiles[k], H))
        if (k & 1) NNDET_DISPATCH_DTYPE(k >> 1, OPT_CALL8);
        else NNDET_DISPATCH_DTYPE(k >> 1, OPT_CALL32);
#undef OPT_CALL8
#undef OPT_CALL32
        LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int nndet_grad_clip(const NndetOptTensor* tensors, int32_t n, double max_norm, const float* grad_scale, float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (max_norm != max_norm || !norm_out || (grad_scale && max_norm >= 0.0)) return NNDET_EINVAL;
    hipStream_t st = as_stream(stream);
    OptTableArgs A;
    memset(&A, 0, sizeof(A));
    OptPlan P;
    int rc = opt_begin(tensors, n, 2, A, workspace, workspace_bytes, P, st);
    if (rc) return rc;
    rc = opt_norm(P, grad_scale, max_norm, norm_out, false, st);
    if (rc || max_norm < 0.0) return rc;         // the norm alone
    for (int k = 0; k < 6; ++k) {
        if (!P.tiles[k]) continue;
        const unsigned g = opt_grid(P.tiles[k], OPT_GRID);
        const OptEntry* e = P.entry + P.first[k];
        const int m = P.first[k + 1] - P.first[k];
#define OPT_CALL(T) (k_opt_scale<T><<<g, OPT_WG, 0, st>>>(P.head, e, m, (uint32_t)P.tiles[k]))
        NNDET_DISPATCH_DTYPE(k >> 1, OPT_CALL);
#undef OPT_CALL
        LAUNCH_CHECK();
    }
    return 0;
}

extern "C" int nndet_adam_state8(const NndetOptTensor* tensors, int32_t n, int32_t write, void* workspace, size_t workspace_bytes, void* stream) {
    for (int i = 0; tensors && i < n; ++i)
        if (tensors[i].dtype != NNDET_F32 || tensors[i].state_bits != 8) return NNDET_EINVAL;
    hipStream_t st = as_stream(stream);
    OptTableArgs A;
    memset(&A, 0, sizeof(A));
    OptPlan P;
    int rc = opt_begin(tensors, n, 7, A, workspace, workspace_bytes, P, st);
    if (rc) return rc;
    const int k = NNDET_F32 * 2 + 1;
    if (!P.tiles[k]) return 0;
    const unsigned g = opt_grid(P.tiles[k], OPT_GRID);
    const int m = P.first[k + 1] - P.first[k];
    if (write) k_opt_state8<true><<<g, OPT_WG, 0, st>>>(P.entry + P.first[k], m, (uint32_t)P.tiles[k]);
    else k_opt_state8<false><<<g, OPT_WG, 0, st>>>(P.entry + P.first[k], m, (uint32_t)P.tiles[k]);
    LAUNCH_CHECK();
    return 0;
}
