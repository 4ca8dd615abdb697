// Shared by the state-space layer's kernels (K12 norm, K13 convolution, K14 scan, K15 8-bit checkpoints): rows of fp32, bf16 or
// fp16 elements at any element alignment, computed on in fp32.
#pragma once
#include "dpk_common.h"

// gfx950 global accesses need no more than element alignment: a group of V elements is one access of V * sizeof(T) bytes
// wherever it starts (a row of 250 floats starts 8 bytes off a 16-byte boundary every other time).
template <int ALIGN, int W>
struct Words;
#define DPK_WORDS(ALIGN, W)                                                                     \
    template <>                                                                                 \
    struct Words<ALIGN, W> {                                                                    \
        typedef uint32_t type __attribute__((ext_vector_type(W), aligned(ALIGN)));              \
    };
DPK_WORDS(2, 2) DPK_WORDS(2, 4) DPK_WORDS(4, 4) DPK_WORDS(4, 8)
#undef DPK_WORDS

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }

template <typename T, int V>
__device__ __forceinline__ void load_full(const T* __restrict__ p, float (&f)[V]) {
    constexpr int W = V * (int)sizeof(T) / 4;
    union {
        typename Words<(int)sizeof(T), W>::type w;
        T e[V];
    } x;
    x.w = *reinterpret_cast<const typename Words<(int)sizeof(T), W>::type*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(x.e[i]);
}

// n of V elements; the others are 0
template <typename T, int V>
__device__ __forceinline__ void load_n(const T* __restrict__ p, int n, float (&f)[V]) {
    if (n >= V) {
        load_full<T, V>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}

// Results leave past the caches: what they would push out is the inputs that other workgroups are about to read (a convolution
// over 8 x 4096 x 1024 in bf16: 46 us with plain stores, 32 so; norm 317 -> 307, 8-bit round trip 195 -> 179).
template <typename T, int V>
__device__ __forceinline__ void store_n(T* __restrict__ p, int n, const float (&f)[V]) {
    if (n >= V) {
        constexpr int W = V * (int)sizeof(T) / 4;
        union {
            typename Words<(int)sizeof(T), W>::type w;
            T e[V];
        } x;
#pragma unroll
        for (int i = 0; i < V; ++i) x.e[i] = (T)f[i];
        __builtin_nontemporal_store(x.w, reinterpret_cast<typename Words<(int)sizeof(T), W>::type*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = (T)f[i];
    }
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// 1 / (1 + e^-x): the exponential overflows to inf for x << 0 and the reciprocal is then 0
__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_hw(-x * LOG2E)); }

// log(1 + e^x) and its derivative, the sigmoid.  e^x = 2^(x log2 e): the product's rounding error, times ln 2, is put back as a
// factor, so e keeps its relative accuracy for x << 0.  With w = fl(1 + e) the logarithm of w misses log(1 + e) by the rounding
// of w; the factor e / (w - 1) puts that back (w - 1 is exact).  Above 20 the result is x to the last bit of fp32.  Far below, where
// e^x is 0, the product's rounding error grows and is inf - inf from -2.4e38 on: it is held to 1, more than it ever is where it counts.
// (Holding x itself at -150 takes a register for the bound, which the scan's backward pass does not have: 932 us against 815 at
// 256 x 200 x 1024, N = 16, bf16.)
struct Softplus {
    float value, slope;
};
__device__ __forceinline__ Softplus softplus_f(float x) {
    constexpr float LOG2E_LOW = 1.9259629911266175e-8f;   // log2 e = LOG2E + LOG2E_LOW
    const float xc = x < 20.f ? x : 20.f;
    const float p = xc * LOG2E;
    const float low = __builtin_fmaf(xc, LOG2E, -p) + xc * LOG2E_LOW;
    const float e0 = exp2_hw(p);
    const float e = __builtin_fmaf(e0, __builtin_amdgcn_fmed3f(low * LN2, -1.f, 1.f), e0);
    const float w = 1.f + e;
    const float d = w - 1.f;
    const float l = d == 0.f ? e : __builtin_amdgcn_logf(w) * LN2 * e * __builtin_amdgcn_rcpf(d);
    Softplus r;
    r.value = x < 20.f ? l : x;   // a NaN fails the comparison and comes back as itself
    r.slope = x < 20.f ? e * __builtin_amdgcn_rcpf(w) : (x == x ? 1.f : x);
    return r;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// the least k >= -126 with amax <= 127 * 2^k, as the byte k + 127; 255 marks an amax that is inf or NaN
__device__ __forceinline__ int exponent_byte(float amax) {
    if (!(amax <= 3.4028234664e38f)) return 255;
    const uint32_t u = __float_as_uint(amax);
    const int k = (int)(u >> 23) - 126 - ((u & 0x7fffffu) > 0x7e0000u ? 6 : 7);   // 127 = 0.9921875 * 2^7
    return (k < -126 ? -126 : k) + 127;
}
__device__ __forceinline__ float exponent_value(int byte) {   // 2^k; 255 -> NaN
    return byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)byte << 23);
}
// 2^-k, exact: k is between -126 and 122
__device__ __forceinline__ float exponent_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
// v * 2^-k rounded to a whole number.  At the top scale 2^122 (byte 249) 64 * 2^122 would be past fp32's largest value: 63 is kept.
__device__ __forceinline__ int quantize8(float v, float inv, int byte) {
    const float top = byte == 249 ? 63.f : 127.f;
    return (int)__builtin_amdgcn_fmed3f(rintf(v * inv), -top, top);
}

// A launch counts its threads in 32 bits, and kernels count steps and channels in int with room for a tile past the end.
static inline bool dpk_launchable(int64_t blocks, int threads) {
    return blocks <= 0x7fffffffLL && blocks * threads <= 0xffffffffLL;
}
constexpr int MAX_DIM = 1 << 30;

#define DPK_DISPATCH_DTYPE(dtype, T, ...)                                   \
    switch (dtype) {                                                        \
        case DPK_F32: { using T = float; __VA_ARGS__ } break;               \
        case DPK_BF16: { using T = __bf16; __VA_ARGS__ } break;             \
        case DPK_F16: { using T = _Float16; __VA_ARGS__ } break;            \
        default: return DPK_EINVAL;                                         \
    }
