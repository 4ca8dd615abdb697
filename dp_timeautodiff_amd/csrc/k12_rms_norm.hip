// K12 — RMS norm with the residual's addition, its backward pass and its (per-sample) weight gradient.
//
//   r = x + residual,  rstd = 1 / sqrt(mean_c r^2 + eps),  y = r * rstd * w
//   backward: g = dy * w, dr = rstd * (g - xhat * mean_c(g * xhat)) + dr_out with xhat = r * rstd; dx = dresidual = dr;
//   dw[c] = sum over a group's rows of dy * xhat (a group is one sample under DP-SGD, or all rows)
//
// HBM-bound: forward reads x and residual and writes y and r, backward reads r, dy, dr_out and writes dx; every element is touched
// once, in registers, and the sums over a row and over a group's rows are fp32.  In 16 bits backward reads x and residual in place
// of r: a weight gradient in fp32 from the rounded r would be off by up to half a step of r's type (1024 x 256 x 512 bf16: 260 us
// against 213, five arrays in place of four).  Four waves a SIMD are held to: 65536 x 1000 fp16 takes 210 us with three, 161 so.  LPR lanes hold one row, E elements each, as
// E / V accesses of 16 bytes; the norm is taken of the fp32 sum, before r is rounded to its type.
#include "ssm_common.h"

namespace {

constexpr int MAX_C = 16384;

template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
};

// sum over the LPR lanes of a row, in a fixed order; every lane gets it
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red, int parity) {
#pragma unroll
    for (int off = (LPR < 64 ? LPR : 64) / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (LPR > 64) {
        constexpr int NW = LPR / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) red[parity * 16 + w] = v;
        __syncthreads();   // two halves of `red` in turn: a wave that runs ahead writes the other one
        float s = 0.f;
        const int w0 = w / NW * NW;
#pragma unroll
        for (int i = 0; i < NW; ++i) s += red[parity * 16 + w0 + i];
        v = s;
    }
    return v;
}

template <typename T, int E, int LPR>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256)
    rms_forward_kernel(const T* __restrict__ X, int64_t ld_x, const T* __restrict__ RES, int64_t ld_res,
                       const float* __restrict__ Wt, T* __restrict__ Y, T* __restrict__ R, float* __restrict__ RSTD,
                       int8_t* __restrict__ Q, uint8_t* __restrict__ QE, int64_t rows, int C, float eps) {
    constexpr int V = Vec<T>::N, K = E / V;
    constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR;
    __shared__ float red[32];
    const int lane = threadIdx.x & (LPR - 1);
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    const bool live = row < rows;   // LPR > 64: RPB rows share the barriers, so no early return
    float v[K][V], w[K][V];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * LPR + lane) * V;
        const int n = live && c < C ? C - c : 0;
        load_n<T, V>(X + row * ld_x + c, n, v[k]);
        if (RES) {
            float t[V];
            load_n<T, V>(RES + row * ld_res + c, n, t);
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] += t[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) ss += v[k][i] * v[k][i];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * LPR + lane) * V;
        load_n<float, V>(Wt + c, c < C ? C - c : 0, w[k]);
    }
    ss = row_sum<LPR>(ss, red, 0);
    const float rstd = 1.f / sqrtf(ss / (float)C + eps);
    if (live && lane == 0 && RSTD) RSTD[row] = rstd;
    const int nb = (C + 127) / 128;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * LPR + lane) * V;
        const int n = live && c < C ? C - c : 0;
        if (R) store_n<T, V>(R + row * C + c, n, v[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] = v[k][i] * rstd * w[k][i];
        store_n<T, V>(Y + row * C + c, n, v[k]);
        if (Q) {   // 128 neighbours are 128 / V lanes of one wave (LPR >= 128 / V in every variant)
            float m = 0.f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                m = fmaxf(m, fabsf(v[k][i]));
                bad |= !(v[k][i] - v[k][i] == 0.f);
            }
#pragma unroll
            for (int off = 64 / V; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
            constexpr int GL = 128 / V;
            const uint64_t group = ((1ull << (GL - 1)) * 2 - 1) << ((threadIdx.x & 63) / GL * GL);
            const bool any_bad = (__ballot(bad) & group) != 0;
            const int eb = any_bad ? 255 : exponent_byte(m);
            const float inv = any_bad ? 0.f : exponent_inverse(eb);
            if (n > 0) {
                int8_t* o = Q + row * C + c;
                uint32_t word[V / 4];
#pragma unroll
                for (int j = 0; j < V / 4; ++j) word[j] = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int q = any_bad ? 0 : quantize8(v[k][i], inv, eb);
                    word[i / 4] |= (uint32_t)(uint8_t)q << (8 * (i % 4));
                }
                if (n >= V) {
                    typedef uint32_t u32b __attribute__((aligned(1)));
#pragma unroll
                    for (int j = 0; j < V / 4; ++j) *reinterpret_cast<u32b*>(o + 4 * j) = word[j];
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i < n) o[i] = (int8_t)(word[i / 4] >> (8 * (i % 4)));
                }
                if (lane % GL == 0) QE[row * nb + c / 128] = (uint8_t)eb;
            }
        }
    }
}

// One workgroup walks the rows of (group, split); its row slots keep their share of dw in registers and meet in LDS at the end.
// SUM: r is R + RES.  HAS_DR: DR is added to DX.  (Compiled in: a branch round a load is waited for before the next load.)
template <typename T, int E, int LPR, bool SUM, bool HAS_DR>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256, 4)
    rms_backward_kernel(const T* __restrict__ R, int64_t ld_r, const T* __restrict__ RES, int64_t ld_res,
                        const T* __restrict__ DY, int64_t ld_dy, const T* __restrict__ DR, int64_t ld_dr,
                        const float* __restrict__ Wt, const float* __restrict__ RSTD, T* __restrict__ DX, float* __restrict__ DW,
                        int64_t dw_stride, int64_t rows_per_group, int split, int C, float scale, int accumulate) {
    constexpr int V = Vec<T>::N, K = E / V;
    constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR;
    __shared__ float red[32];
    __shared__ float cols[RPB > 1 ? RPB * LPR * E : 1];
    const int lane = threadIdx.x & (LPR - 1), slot = threadIdx.x / LPR;
    const int64_t group = blockIdx.x / split, part = blockIdx.x % split;
    const int64_t lo = rows_per_group * part / split, hi = rows_per_group * (part + 1) / split;
    float w[K][V], dw[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * LPR + lane) * V;
        load_n<float, V>(Wt + c, c < C ? C - c : 0, w[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
    }
    const float inv_c = 1.f / (float)C;
    // two rows of a slot are under way where they fit the registers: 16 bytes a lane and row are too few to fill HBM's latency
    constexpr int NR = E <= 8 ? 2 : 1;
    for (int64_t r0 = lo; r0 < hi; r0 += RPB * NR) {
        float x[NR][K][V], s[NR][K][V], g[NR][K][V], d[NR][K][V], rstd[NR], dot[NR];
        bool live[NR];
        int64_t row[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            live[j] = r0 + j * RPB + slot < hi;
            row[j] = group * rows_per_group + (live[j] ? r0 + j * RPB + slot : lo);
            rstd[j] = RSTD[row[j]];
            dot[j] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * LPR + lane) * V;
                const int n = live[j] && c < C ? C - c : 0;
                load_n<T, V>(R + row[j] * ld_r + c, n, x[j][k]);
                if (SUM) load_n<T, V>(RES + row[j] * ld_res + c, n, s[j][k]);
                load_n<T, V>(DY + row[j] * ld_dy + c, n, g[j][k]);
                if (HAS_DR) load_n<T, V>(DR + row[j] * ld_dr + c, n, d[j][k]);
            }
        }
#pragma unroll
        for (int j = 0; j < NR; ++j) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (SUM) x[j][k][i] += s[j][k][i];
                    x[j][k][i] *= rstd[j];
                    dw[k][i] += g[j][k][i] * x[j][k][i];
                    g[j][k][i] *= w[k][i];
                    dot[j] += g[j][k][i] * x[j][k][i];
                }
            dot[j] = row_sum<LPR>(dot[j], red, NR == 2 ? j : (int)((r0 - lo) / RPB & 1)) * inv_c;
        }
        if (DX) {
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = (k * LPR + lane) * V;
                    const int n = live[j] && c < C ? C - c : 0;
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        o[i] = rstd[j] * (g[j][k][i] - x[j][k][i] * dot[j]);
                        if (HAS_DR) o[i] += d[j][k][i];
                    }
                    store_n<T, V>(DX + row[j] * C + c, n, o);
                }
        }
    }
    if (!DW) return;
    float* out = DW + (int64_t)blockIdx.x * dw_stride;
    if constexpr (RPB > 1) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) cols[slot * LPR * E + (k * LPR + lane) * V + i] = dw[k][i];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += NT) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < RPB; ++i) s += cols[i * LPR * E + c];
            out[c] = accumulate ? out[c] + scale * s : scale * s;
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * LPR + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < C) out[c + i] = accumulate ? out[c + i] + scale * dw[k][i] : scale * dw[k][i];
        }
    }
}

// Lanes per row and elements per lane: narrow rows take half a wave with one 16-byte access a lane (two rows a wave keep its lanes
// busy, and the 8-bit output's blocks of 128 stay whole), then a wave with up to 16 elements a lane, then 256 and 1024 lanes.
#define RMS_PICK(T, C, CALL)                                              \
    do {                                                                  \
        constexpr int V = Vec<T>::N;                                      \
        if (C <= 32 * V) { CALL(T, V, 32); }                              \
        else if (C <= 64 * V) { CALL(T, V, 64); }                         \
        else if (C <= 64 * 8) { CALL(T, 8, 64); }                         \
        else if (C <= 64 * 16) { CALL(T, 16, 64); }                       \
        else if (C <= 256 * 8) { CALL(T, 8, 256); }                       \
        else if (C <= 256 * 16) { CALL(T, 16, 256); }                     \
        else { CALL(T, 16, 1024); }                                       \
    } while (0)

}  // namespace

extern "C" int dpk_rms_norm_forward(const void* X, int64_t ld_x, const void* RES, int64_t ld_res, const float* W, void* Y, void* R,
                                    float* rstd, int8_t* Q, uint8_t* QE, int64_t rows, int C, float eps, int dtype, void* stream) {
    if (rows < 0 || C <= 0 || ld_x < 0 || ld_res < 0 || !(eps >= 0.f)) return DPK_EINVAL;
    if (rows == 0) return DPK_OK;
    if (!X || !W || !Y || (Q == nullptr) != (QE == nullptr)) return DPK_EINVAL;
    if (C > MAX_C || rows > 0x7fffffffLL) return DPK_ERANGE;
#define RMS_CALL(T, E, LPR)                                                                                                  \
    {                                                                                                                        \
        constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR;                                                            \
        if (!dpk_launchable((rows + RPB - 1) / RPB, NT)) return DPK_ERANGE;                                                  \
        hipLaunchKernelGGL((rms_forward_kernel<T, E, LPR>), dim3((unsigned)((rows + RPB - 1) / RPB)), dim3(NT), 0,           \
                           (hipStream_t)stream, (const T*)X, ld_x, (const T*)RES, ld_res, W, (T*)Y, (T*)R, rstd, Q, QE, rows, \
                           C, eps);                                                                                          \
    }
    DPK_DISPATCH_DTYPE(dtype, T, RMS_PICK(T, C, RMS_CALL);)
#undef RMS_CALL
    return dpk_launch_status();
}

// Workgroups a group's rows are spread over: enough for four a CU, with no fewer than 16 rows each (a part's row of dw costs as much
// as a row of the data); but while there are not two a CU, down to 2 rows each (184 rows of 3815 in 12 parts: 82 us a pass, in 92: 26).
extern "C" int dpk_rms_norm_split(int64_t groups, int64_t rows_per_group) {
    if (groups <= 0 || rows_per_group <= 0) return 1;
    int64_t s = (1024 + groups - 1) / groups;
    if (s > (rows_per_group + 15) / 16) s = (rows_per_group + 15) / 16;
    const int64_t few = (512 + groups - 1) / groups;
    if (s < few) s = few < (rows_per_group + 1) / 2 ? few : (rows_per_group + 1) / 2;
    return (int)(s < 1 ? 1 : s);
}

extern "C" int dpk_rms_norm_backward(const void* R, int64_t ld_r, const void* RES, int64_t ld_res, const void* DY,
                                     int64_t ld_dy, const void* DR, int64_t ld_dr, const float* W, const float* rstd, void* DX,
                                     float* DW, int64_t dw_stride, int64_t groups, int64_t rows_per_group, int split, int C,
                                     float scale, int accumulate, int dtype, void* stream) {
    if (groups < 0 || rows_per_group < 0 || split <= 0 || C <= 0 || ld_r < 0 || ld_res < 0 || ld_dy < 0 || ld_dr < 0)
        return DPK_EINVAL;
    if ((DW && dw_stride < C) || (RES && dtype == DPK_F32)) return DPK_EINVAL;
    if (groups == 0) return DPK_OK;
    if (!W || (rows_per_group > 0 && (!R || !DY || !rstd))) return DPK_EINVAL;
    if (C > MAX_C || groups > 0x7fffffffLL || !dpk_launchable(groups * split, C > 256 * 16 ? 1024 : 256)) return DPK_ERANGE;
#define RMS_GO(T, E, LPR, SUM, HAS_DR)                                                                                           \
    hipLaunchKernelGGL((rms_backward_kernel<T, E, LPR, SUM, HAS_DR>), dim3((unsigned)(groups * split)),                        \
                       dim3(LPR > 256 ? LPR : 256), 0, (hipStream_t)stream, (const T*)R, ld_r, (const T*)RES, ld_res,           \
                       (const T*)DY, ld_dy, (const T*)DR, ld_dr, W, rstd, (T*)DX, DW, dw_stride, rows_per_group, split, C, scale, \
                       accumulate)
#define RMS_CALL(T, E, LPR)                                    \
    if (RES && DX && DR)                                       \
        RMS_GO(T, E, LPR, (sizeof(T) == 2), true);             \
    else if (RES)                                              \
        RMS_GO(T, E, LPR, (sizeof(T) == 2), false);            \
    else if (DX && DR)                                         \
        RMS_GO(T, E, LPR, false, true);                        \
    else                                                       \
        RMS_GO(T, E, LPR, false, false)
    DPK_DISPATCH_DTYPE(dtype, T, RMS_PICK(T, C, RMS_CALL);)
#undef RMS_CALL
#undef RMS_GO
    return dpk_launch_status();
}
