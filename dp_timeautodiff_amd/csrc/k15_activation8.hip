// K15 — activations held in 8 bits between forward and backward, and the fixed-order sum of partial rows that K12..K14
// use for parameter gradients.
//
// A block of 128 neighbours of a row shares one scale 2^k, k the least integer with max|v| <= 127 * 2^k; an element is kept as
// q = rint(v * 2^-k).  The scale being a power of two, v * 2^-k is exact, so q is the correctly rounded quotient, the error
// is at most 2^k / 2 <= max|v| / 127, and q * 2^k is exact in bf16 too.  (A scale of max/127 would halve the worst error but
// make q depend on the last bit of a division.)  Blocks that hold an inf or NaN restore as NaN: an overflow in the forward pass
// stays visible in the gradients.
// Both directions are HBM-bound: 4 + 1 + 1/128 bytes an fp32 element.
#include "ssm_common.h"

namespace {

constexpr int BLK = 128;

// 32 lanes hold one block, 4 elements each.
template <typename T>
__global__ void __launch_bounds__(256) compress_kernel(const T* __restrict__ X, int64_t ld_x, int8_t* __restrict__ Q,
                                                       uint8_t* __restrict__ E, int64_t rows, int C, int nb) {
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= rows * nb) return;
    const int64_t row = unit / nb;
    const int blk = (int)(unit - row * nb);
    const int lane = threadIdx.x & 31;
    const int c = blk * BLK + lane * 4;
    const int n = c < C ? (C - c < 4 ? C - c : 4) : 0;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (n > 0) load_n<T, 4>(X + row * ld_x + c, n, v);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = fabsf(v[i]);
        m = a <= m ? m : a;   // a NaN is taken, and stays
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const float o = __shfl_xor(m, off, 32);
        m = !(o <= m) ? o : m;
    }
    // (o <= m) is false for a NaN on either side: a lane that holds a NaN may have dropped it for a number above, so test once more
    const bool bad = !(v[0] - v[0] == 0.f) || !(v[1] - v[1] == 0.f) || !(v[2] - v[2] == 0.f) || !(v[3] - v[3] == 0.f);
    const uint64_t any = __ballot(bad);
    const bool half_bad = ((threadIdx.x & 32) ? (any >> 32) : (any & 0xffffffffull)) != 0;
    const int eb = half_bad ? 255 : exponent_byte(m);
    const float inv = half_bad ? 0.f : exponent_inverse(eb);
    if (n > 0) {
        int8_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = half_bad ? 0 : (int8_t)quantize8(v[i], inv, eb);
        int8_t* o = Q + row * C + c;
        if (n == 4) {
            typedef uint32_t u32b __attribute__((aligned(1)));
            *reinterpret_cast<u32b*>(o) = (uint32_t)(uint8_t)q[0] | (uint32_t)(uint8_t)q[1] << 8 |
                                          (uint32_t)(uint8_t)q[2] << 16 | (uint32_t)(uint8_t)q[3] << 24;
        } else {
            for (int i = 0; i < n; ++i) o[i] = q[i];
        }
    }
    if (lane == 0) E[row * nb + blk] = (uint8_t)eb;
}

template <typename T>
__global__ void __launch_bounds__(256) restore_kernel(const int8_t* __restrict__ Q, const uint8_t* __restrict__ E,
                                                      T* __restrict__ X, int64_t rows, int C, int nb) {
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= rows * nb) return;
    const int64_t row = unit / nb;
    const int blk = (int)(unit - row * nb);
    const int c = blk * BLK + (threadIdx.x & 31) * 4;
    const int n = c < C ? (C - c < 4 ? C - c : 4) : 0;
    if (n == 0) return;
    const float s = exponent_value(E[row * nb + blk]);
    const int8_t* q = Q + row * C + c;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (n == 4) {
        typedef uint32_t u32b __attribute__((aligned(1)));
        const uint32_t w = *reinterpret_cast<const u32b*>(q);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i)) * s;
    } else {
        for (int i = 0; i < n; ++i) v[i] = (float)q[i] * s;
    }
    store_n<T, 4>(X + row * C + c, n, v);
}

// out[g][c] (+)= scale * sum_r in[g][r][c], rows in a fixed order: slice s of 16 adds rows s, s + 16, ..., then the slices in order.
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ in, int R, int64_t P, int64_t in_stride,
                                                        float* __restrict__ out, int64_t out_stride, float scale,
                                                        int accumulate) {
    __shared__ float part[16][64];
    const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int slice = threadIdx.x >> 6;
    const float* base = in + (int64_t)blockIdx.y * R * in_stride;
    float s = 0.f;
    if (c < P) {
        int r = slice;
        for (; r + 48 < R; r += 64) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = base[(int64_t)(r + 16 * i) * in_stride + c];
            s += v[0]; s += v[1]; s += v[2]; s += v[3];
        }
        for (; r < R; r += 16) s += base[(int64_t)r * in_stride + c];
    }
    part[slice][threadIdx.x & 63] = s;
    __syncthreads();
    if (slice == 0 && c < P) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += part[i][threadIdx.x];
        float* o = out + (int64_t)blockIdx.y * out_stride + c;
        *o = accumulate ? *o + scale * t : scale * t;
    }
}

}  // namespace

extern "C" int dpk_compress_activation(const void* X, int64_t ld_x, int8_t* Q, uint8_t* E, int64_t rows, int C, int dtype,
                                       void* stream) {
    if (rows < 0 || C <= 0 || ld_x < 0) return DPK_EINVAL;
    if (rows == 0) return DPK_OK;
    if (!X || !Q || !E) return DPK_EINVAL;
    const int nb = (C + BLK - 1) / BLK;
    const int64_t grid = (rows * nb + 7) / 8;
    if (rows > (int64_t)1 << 40 || grid > 0x7fffffffLL) return DPK_ERANGE;
    DPK_DISPATCH_DTYPE(dtype, T, hipLaunchKernelGGL(compress_kernel<T>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,
                                                    (const T*)X, ld_x, Q, E, rows, C, nb);)
    return dpk_launch_status();
}

extern "C" int dpk_restore_activation(const int8_t* Q, const uint8_t* E, void* X, int64_t rows, int C, int dtype, void* stream) {
    if (rows < 0 || C <= 0) return DPK_EINVAL;
    if (rows == 0) return DPK_OK;
    if (!X || !Q || !E) return DPK_EINVAL;
    const int nb = (C + BLK - 1) / BLK;
    const int64_t grid = (rows * nb + 7) / 8;
    if (rows > (int64_t)1 << 40 || grid > 0x7fffffffLL) return DPK_ERANGE;
    DPK_DISPATCH_DTYPE(dtype, T, hipLaunchKernelGGL(restore_kernel<T>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, Q,
                                                    E, (T*)X, rows, C, nb);)
    return dpk_launch_status();
}

extern "C" int dpk_sum_rows(const float* in, int groups, int rows, int64_t P, int64_t in_stride, float* out, int64_t out_stride,
                            float scale, int accumulate, void* stream) {
    if (groups < 0 || rows < 0 || P <= 0 || in_stride < P || out_stride < P) return DPK_EINVAL;
    if (groups == 0) return DPK_OK;
    if (!out || (rows > 0 && !in)) return DPK_EINVAL;
    const int64_t gx = (P + 63) / 64;
    if (gx > 0x7fffffffLL || groups > 65535) return DPK_ERANGE;
    hipLaunchKernelGGL(sum_rows_kernel, dim3((unsigned)gx, (unsigned)groups), dim3(1024), 0, (hipStream_t)stream, in, rows, P,
                       in_stride, out, out_stride, scale, accumulate);
    return dpk_launch_status();
}
