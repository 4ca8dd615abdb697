// K15 — activations held in 8 bits between forward and backward, and the fixed-order sum of partial rows that K12..K14
// use for parameter gradients.
//
// A block of 128 neighbours of a row shares one scale 2^k, k the least integer with max|v| <= 127 * 2^k; an element is kept as
// q = rint(v * 2^-k).  The scale being a power of two, v * 2^-k is exact, so q is the correctly rounded quotient, the error
// is at most 2^k / 2 <= max|v| / 127, and q * 2^k is exact in bf16 too.  (A scale of max/127 would halve the worst error but
// make q depend on the last bit of a division.)  The error is larger than max|v| / 127 in two places: under the least scale, 2^-126,
// where it is up to 2^-127, and at k = 122, where q is held to 63 (64 * 2^122 is no fp32 number) and it is up to 2^122.  What rounds
// up to 2^16 (fp16 from 65024 on: q = 64, k = 10) is restored in fp16 as its largest value, 65504, and not as inf.  Blocks that hold
// an inf or NaN restore as NaN: an overflow in the forward pass stays visible in the gradients.
// Both directions are HBM-bound: 4 + 1 + 1/128 bytes an fp32 element.  Lanes take 16 bytes of the wide side each (32 lanes a block in
// fp32, 16 in 16 bits), so that every access of a wave is one run of memory, and a workgroup has four or two rounds of blocks
// under way.
#include "ssm_common.h"

namespace {

constexpr int BLK = 128;

// A workgroup's units (blocks of 128): BLK / LV lanes take one, LV elements each, ROUNDS of them in turn.
template <int LV_, int ROUNDS_>
struct Shape {
    static constexpr int LV = LV_, ROUNDS = ROUNDS_, LANES = BLK / LV, UNITS = 256 / LANES * ROUNDS;
};
template <typename T>
using ShapeOf = Shape<sizeof(T) == 4 ? 4 : 8, sizeof(T) == 4 ? 4 : 2>;

typedef uint32_t u32x2b __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32b __attribute__((aligned(1)));

// row and block of a unit; 64-bit division only where there are more than 2^32 units
template <typename S>
struct Unit {
    int64_t row;
    int blk, c, n;
    bool live;
    __device__ __forceinline__ Unit(int64_t unit, int64_t total, int C, int nb) {
        live = unit < total;
        if (!live) unit = 0;
        if (total <= 0xffffffffLL) {
            const uint32_t u = (uint32_t)unit, r = u / (uint32_t)nb;
            row = r;
            blk = (int)(u - r * (uint32_t)nb);
        } else {
            row = unit / nb;
            blk = (int)(unit - row * nb);
        }
        c = blk * BLK + (threadIdx.x & (S::LANES - 1)) * S::LV;
        n = live && c < C ? C - c : 0;
    }
};

template <typename T>
__global__ void __launch_bounds__(256) compress_kernel(const T* __restrict__ X, int64_t ld_x, int8_t* __restrict__ Q,
                                                       uint8_t* __restrict__ E, int64_t total, int C, int nb) {
    using S = ShapeOf<T>;
    constexpr int LV = S::LV, LANES = S::LANES, ROUNDS = S::ROUNDS, WORDS = LV / 4;
    float v[ROUNDS][LV];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const Unit<S> u((int64_t)blockIdx.x * S::UNITS + k * (256 / LANES) + threadIdx.x / LANES, total, C, nb);
        load_n<T, LV>(X + u.row * ld_x + u.c, u.n, v[k]);
    }
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const Unit<S> u((int64_t)blockIdx.x * S::UNITS + k * (256 / LANES) + threadIdx.x / LANES, total, C, nb);
        float m = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < LV; ++i) {
            m = fmaxf(m, fabsf(v[k][i]));
            bad |= !(v[k][i] - v[k][i] == 0.f);   // fmaxf drops a NaN
        }
#pragma unroll
        for (int off = LANES / 2; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const uint64_t group = ((1ull << LANES) - 1) << ((threadIdx.x & 63) / LANES * LANES);
        const bool any_bad = (__ballot(bad) & group) != 0;
        const int eb = any_bad ? 255 : exponent_byte(m);
        const float inv = any_bad ? 0.f : exponent_inverse(eb);
        if (u.n > 0) {
            uint32_t w[WORDS];
#pragma unroll
            for (int j = 0; j < WORDS; ++j) w[j] = 0u;
#pragma unroll
            for (int i = 0; i < LV; ++i) {
                const int q = any_bad ? 0 : quantize8(v[k][i], inv, eb);
                w[i / 4] |= (uint32_t)(uint8_t)q << (8 * (i % 4));
            }
            int8_t* o = Q + u.row * C + u.c;
            if (u.n >= LV) {
                if constexpr (LV == 8) {
                    const u32x2b p = {w[0], w[1]};
                    *reinterpret_cast<u32x2b*>(o) = p;
                } else {
                    *reinterpret_cast<u32b*>(o) = w[0];
                }
            } else {
#pragma unroll
                for (int i = 0; i < LV; ++i)
                    if (i < u.n) o[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
            }
            if ((threadIdx.x & (LANES - 1)) == 0) E[u.row * nb + u.blk] = (uint8_t)eb;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) restore_kernel(const int8_t* __restrict__ Q, const uint8_t* __restrict__ E,
                                                      T* __restrict__ X, int64_t total, int C, int nb) {
    using S = ShapeOf<T>;
    constexpr int LV = S::LV, LANES = S::LANES, ROUNDS = S::ROUNDS, WORDS = LV / 4;
    uint32_t w[ROUNDS][WORDS];
    int eb[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const Unit<S> u((int64_t)blockIdx.x * S::UNITS + k * (256 / LANES) + threadIdx.x / LANES, total, C, nb);
        const int8_t* q = Q + u.row * C + u.c;
        eb[k] = E[u.row * nb + u.blk];
#pragma unroll
        for (int j = 0; j < WORDS; ++j) w[k][j] = 0u;
        if (u.n >= LV) {
            if constexpr (LV == 8) {
                const u32x2b p = *reinterpret_cast<const u32x2b*>(q);
                w[k][0] = p[0];
                w[k][1] = p[1];
            } else {
                w[k][0] = *reinterpret_cast<const u32b*>(q);
            }
        } else {
#pragma unroll
            for (int i = 0; i < LV; ++i)
                if (i < u.n) w[k][i / 4] |= (uint32_t)(uint8_t)q[i] << (8 * (i % 4));
        }
    }
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const Unit<S> u((int64_t)blockIdx.x * S::UNITS + k * (256 / LANES) + threadIdx.x / LANES, total, C, nb);
        const float s = exponent_value(eb[k]);
        float v[LV];
#pragma unroll
        for (int i = 0; i < LV; ++i) {
            v[i] = (float)(int8_t)(w[k][i / 4] >> (8 * (i % 4))) * s;
            if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16))
                v[i] = fabsf(v[i]) == 65536.f ? __builtin_copysignf(65504.f, v[i]) : v[i];
        }
        if (u.n > 0) store_n<T, LV>(X + u.row * C + u.c, u.n, v);
    }
}

// out[g][c] (+)= scale * sum_r in[g][r][c], rows in a fixed order: slice s of 16 adds rows s, s + 16, ..., then the slices in order.
// The columns go to up to three destinations, one behind the other.
struct SumRows {
    const float* in;
    float* out[3];
    int64_t n[3], out_stride[3], in_stride, P;
    int R, accumulate;
    float scale;
};

// COLS columns and 1024 / COLS slices a workgroup: narrow results take few columns each, so that enough workgroups share a tall sum
// (1024 rows of 250: 3.6 us, 4.2 with 64 columns; of 4608: 8.0 with 64, 9.3 with 16, out of the Infinity Cache.  In a training step,
// behind the launch that writes those rows, they take 11).
template <int COLS>
__global__ void __launch_bounds__(1024) sum_rows_kernel(SumRows a) {
    constexpr int SLICES = 1024 / COLS;
    __shared__ float part[SLICES][COLS];
    int64_t c = (int64_t)blockIdx.x * COLS + threadIdx.x % COLS;
    const int slice = threadIdx.x / COLS;
    const float* base = a.in + (int64_t)blockIdx.y * a.R * a.in_stride;
    float s = 0.f;
    if (c < a.P) {
        int r = slice;
        for (; r + 3 * SLICES < a.R; r += 4 * SLICES) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = base[(int64_t)(r + SLICES * i) * a.in_stride + c];
            s += v[0]; s += v[1]; s += v[2]; s += v[3];
        }
        for (; r < a.R; r += SLICES) s += base[(int64_t)r * a.in_stride + c];
    }
    part[slice][threadIdx.x % COLS] = s;
    __syncthreads();
    if (slice == 0 && c < a.P) {
        float t = 0.f;
#pragma unroll 16
        for (int i = 0; i < SLICES; ++i) t += part[i][threadIdx.x];
        int k = 0;
        for (; k < 2 && c >= a.n[k]; ++k) c -= a.n[k];
        float* o = a.out[k] + (int64_t)blockIdx.y * a.out_stride[k] + c;
        *o = a.accumulate ? *o + a.scale * t : a.scale * t;
    }
}

}  // namespace

extern "C" int dpk_compress_activation(const void* X, int64_t ld_x, int8_t* Q, uint8_t* E, int64_t rows, int C, int dtype,
                                       void* stream) {
    if (rows < 0 || C <= 0 || ld_x < 0) return DPK_EINVAL;
    if (rows == 0) return DPK_OK;
    if (!X || !Q || !E) return DPK_EINVAL;
    if (C > MAX_DIM || rows > (int64_t)1 << 36) return DPK_ERANGE;
    const int nb = (C + BLK - 1) / BLK;
    const int64_t total = rows * nb, units = dtype == DPK_F32 ? ShapeOf<float>::UNITS : ShapeOf<__bf16>::UNITS, grid = (total + units - 1) / units;
    if (!dpk_launchable(grid, 256)) return DPK_ERANGE;
    DPK_DISPATCH_DTYPE(dtype, T, hipLaunchKernelGGL(compress_kernel<T>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,
                                                    (const T*)X, ld_x, Q, E, total, C, nb);)
    return dpk_launch_status();
}

extern "C" int dpk_restore_activation(const int8_t* Q, const uint8_t* E, void* X, int64_t rows, int C, int dtype, void* stream) {
    if (rows < 0 || C <= 0) return DPK_EINVAL;
    if (rows == 0) return DPK_OK;
    if (!X || !Q || !E) return DPK_EINVAL;
    if (C > MAX_DIM || rows > (int64_t)1 << 36) return DPK_ERANGE;
    const int nb = (C + BLK - 1) / BLK;
    const int64_t total = rows * nb, units = dtype == DPK_F32 ? ShapeOf<float>::UNITS : ShapeOf<__bf16>::UNITS, grid = (total + units - 1) / units;
    if (!dpk_launchable(grid, 256)) return DPK_ERANGE;
    DPK_DISPATCH_DTYPE(dtype, T, hipLaunchKernelGGL(restore_kernel<T>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, Q,
                                                    E, (T*)X, total, C, nb);)
    return dpk_launch_status();
}

extern "C" int dpk_sum_rows(const float* in, int groups, int rows, int64_t in_stride, float* const* out, const int64_t* n,
                            const int64_t* out_stride, float scale, int accumulate, void* stream) {
    if (groups < 0 || rows < 0 || in_stride < 0 || !out || !n || !out_stride) return DPK_EINVAL;
    SumRows a = {};
    for (int k = 0; k < 3; ++k) {
        if (n[k] < 0 || (n[k] > 0 && (!out[k] || out_stride[k] < n[k]))) return DPK_EINVAL;
        a.out[k] = out[k]; a.n[k] = n[k]; a.out_stride[k] = out_stride[k];
        a.P += n[k];
    }
    if (a.P <= 0 || in_stride < a.P) return DPK_EINVAL;
    if (groups == 0) return DPK_OK;
    if (rows > 0 && !in) return DPK_EINVAL;
    const bool narrow = a.P <= 2048 && rows > 64;
    const int64_t gx = narrow ? (a.P + 15) / 16 : (a.P + 63) / 64;
    if (!dpk_launchable(gx, 1024) || groups > 65535) return DPK_ERANGE;
    a.in = in; a.in_stride = in_stride; a.R = rows; a.accumulate = accumulate; a.scale = scale;
    const dim3 grid((unsigned)gx, (unsigned)groups);
    if (narrow)
        hipLaunchKernelGGL(sum_rows_kernel<16>, grid, dim3(1024), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(sum_rows_kernel<64>, grid, dim3(1024), 0, (hipStream_t)stream, a);
    return dpk_launch_status();
}
