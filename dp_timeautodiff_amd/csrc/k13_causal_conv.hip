// K13 — short causal depthwise convolution over time, its backward pass and its single-token form.
//
//   p_t = bias + sum_i w[i] * x_{t-W+1+i},  y = p or silu(p); x before the sequence comes from `state` (W-1 rows) or is 0.
//   backward: g = dy * act'(p); dx_t = sum_i w[i] * g_{t+W-1-i}; dw[i] = sum_t g_t * x_{t-W+1+i}; dbias = sum_t g_t
// Rows at and behind lengths[b] are not part of sequence b: y, dx there are 0 and they reach no gradient.  The state handed on is
// the last W-1 rows of the sequence itself.
//
// HBM-bound (one read and one write an element forward, two and one backward).  A lane owns 4 neighbouring channels and walks a
// stretch of time with the window in registers; a workgroup is CGL such lanes times 256 / CGL stretches, so the rows a
// neighbour's window needs again come out of the same CU's cache.  Parameter gradients are summed in registers along the stretch,
// then over the workgroup's stretches in a fixed order.
#include "ssm_common.h"

namespace {

constexpr int CV = 4;

struct ConvArgs {
    const void *x, *dy, *state, *dstate_out;
    const float *w, *bias;
    const int* lengths;
    void *y, *state_out, *dx, *dstate;
    float* dpar;   // rows of D * W weight gradients, then (if has_bias) at dbias_off the D bias gradients
    int64_t x_sb, x_st, dy_sb, dy_st, dpar_stride, dbias_off;
    int B, T, D, silu, seg, nseg, nct, accumulate;
    float scale;
};

__device__ __forceinline__ int seq_end(const ConvArgs& a, int b) {
    int n = a.lengths ? a.lengths[b] : a.T;
    return n < 0 ? 0 : n > a.T ? a.T : n;
}

// x row t (t may be negative: the state's rows); rows at or behind `end` are never asked for
template <typename T, int W>
__device__ __forceinline__ void load_x(const ConvArgs& a, int b, int t, int c, int n, float (&v)[CV]) {
    if (t >= 0) {
        load_n<T, CV>((const T*)a.x + (int64_t)b * a.x_sb + (int64_t)t * a.x_st + c, n, v);
    } else if (a.state) {
        load_n<T, CV>((const T*)a.state + ((int64_t)b * (W - 1) + (W - 1 + t)) * a.D + c, n, v);
    } else {
#pragma unroll
        for (int i = 0; i < CV; ++i) v[i] = 0.f;
    }
}

template <typename T, int W, int CGL>
__global__ void __launch_bounds__(256) conv_forward_kernel(ConvArgs a) {
    const int ct = blockIdx.x % a.nct, rest = blockIdx.x / a.nct;
    const int s = rest % a.nseg, b = rest / a.nseg;
    const int c = (ct * CGL + threadIdx.x % CGL) * CV;
    const int n = a.D - c;
    if (n <= 0) return;
    constexpr int NS = 256 / CGL;
    const int len = (a.seg + NS - 1) / NS;
    const int t0 = s * a.seg + (threadIdx.x / CGL) * len;
    int t1 = t0 + len;
    if (t1 > (s + 1) * a.seg) t1 = (s + 1) * a.seg;
    if (t1 > a.T) t1 = a.T;
    const int end = seq_end(a, b);
    float w[W][CV], bias[CV];
#pragma unroll
    for (int i = 0; i < CV; ++i) {
        const bool in = i < n;
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = in ? a.w[(int64_t)(c + i) * W + j] : 0.f;
        bias[i] = in && a.bias ? a.bias[c + i] : 0.f;
    }
    if (W > 1 && a.state_out && s == 0 && threadIdx.x < CGL) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            float v[CV];
            load_x<T, W>(a, b, end - (W - 1) + j, c, n, v);
            store_n<T, CV>((T*)a.state_out + ((int64_t)b * (W - 1) + j) * a.D + c, n, v);
        }
    }
    float win[W][CV];   // win[j] = x_{t-W+1+j}
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        if (t0 < end) {
            load_x<T, W>(a, b, t0 - (W - 1) + j, c, n, win[j + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < CV; ++i) win[j + 1][i] = 0.f;
        }
    }
    T* y = (T*)a.y + ((int64_t)b * a.T) * a.D + c;
    for (int t = t0; t < t1; ++t) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int i = 0; i < CV; ++i) win[j][i] = win[j + 1][i];
        float o[CV] = {0.f, 0.f, 0.f, 0.f};
        if (t < end) {
            load_x<T, W>(a, b, t, c, n, win[W - 1]);
#pragma unroll
            for (int i = 0; i < CV; ++i) {
                float p = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) p += w[j][i] * win[j][i];
                o[i] = a.silu ? p * sigmoid_f(p) : p;
            }
        }
        store_n<T, CV>(y + (int64_t)t * a.D, n, o);
    }
}

template <typename T, int W, int CGL>
__global__ void __launch_bounds__(256) conv_backward_kernel(ConvArgs a) {
    constexpr int NS = 256 / CGL;
    __shared__ float red[NS][CGL * CV * (W + 1)];
    const int ct = blockIdx.x % a.nct, rest = blockIdx.x / a.nct;
    const int s = rest % a.nseg, b = rest / a.nseg;
    const int cl = threadIdx.x % CGL, slot = threadIdx.x / CGL;
    const int c = (ct * CGL + cl) * CV;
    const int n = a.D - c > 0 ? a.D - c : 0;
    const int len = (a.seg + NS - 1) / NS;
    const int t0 = s * a.seg + slot * len;
    int t1 = t0 + len;
    if (t1 > (s + 1) * a.seg) t1 = (s + 1) * a.seg;
    if (t1 > a.T) t1 = a.T;
    const int end = seq_end(a, b);
    float dw[W][CV], db[CV];
#pragma unroll
    for (int i = 0; i < CV; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][i] = 0.f;
    }
    if (n > 0 && (t0 < t1 || (a.T == 0 && slot == 0))) {   // no rows at all: the state still passes its gradient on
        float w[W][CV], bias[CV];
#pragma unroll
        for (int i = 0; i < CV; ++i) {
            const bool in = i < n;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = in ? a.w[(int64_t)(c + i) * W + j] : 0.f;
            bias[i] = in && a.bias ? a.bias[c + i] : 0.f;
        }
        float win[W][CV], gw[W][CV];   // gw[j] = g_{t-W+1+j}
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < CV; ++i) {
                win[j][i] = 0.f;
                gw[j][i] = 0.f;
            }
        if (t0 < end) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) load_x<T, W>(a, b, t0 - (W - 1) + j, c, n, win[j + 1]);
        }
        // g runs W-1 rows past the stretch (those belong to the next one, which sums their parameter gradients); dx_{t-W+1} is
        // complete once g_t is known.  In the first stretch the rows before 0 are the state's.
        for (int t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int i = 0; i < CV; ++i) {
                    win[j][i] = win[j + 1][i];
                    gw[j][i] = gw[j + 1][i];
                }
#pragma unroll
            for (int i = 0; i < CV; ++i) gw[W - 1][i] = 0.f;
            if (t < end) {
                float dy[CV];
                load_x<T, W>(a, b, t, c, n, win[W - 1]);
                load_n<T, CV>((const T*)a.dy + (int64_t)b * a.dy_sb + (int64_t)t * a.dy_st + c, n, dy);
#pragma unroll
                for (int i = 0; i < CV; ++i) {
                    float p = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) p += w[j][i] * win[j][i];
                    const float sg = a.silu ? sigmoid_f(p) : 1.f;
                    const float g = a.silu ? dy[i] * sg * (1.f + p * (1.f - sg)) : dy[i];
                    gw[W - 1][i] = g;
                    if (t < t1) {
                        db[i] += g;
#pragma unroll
                        for (int j = 0; j < W; ++j) dw[j][i] += g * win[j][i];
                    }
                }
            }
            const int to = t - (W - 1);
            if (to >= (t0 == 0 ? -(W - 1) : t0) && to < t1) {
                float d[CV] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < CV; ++i)
#pragma unroll
                    for (int j = 0; j < W; ++j) d[i] += w[j][i] * gw[W - 1 - j][i];
                const int kept = to - (end - (W - 1));   // this row went out as row `kept` of the state
                if (a.dstate_out && kept >= 0 && kept < W - 1) {
                    float v[CV];
                    load_n<T, CV>((const T*)a.dstate_out + ((int64_t)b * (W - 1) + kept) * a.D + c, n, v);
#pragma unroll
                    for (int i = 0; i < CV; ++i) d[i] += v[i];
                }
                if (to >= 0)
                    store_n<T, CV>((T*)a.dx + ((int64_t)b * a.T + to) * a.D + c, n, d);
                else if (a.dstate)
                    store_n<T, CV>((T*)a.dstate + ((int64_t)b * (W - 1) + (W - 1 + to)) * a.D + c, n, d);
            }
        }
    }
    if (!a.dpar) return;
#pragma unroll
    for (int i = 0; i < CV; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) red[slot][(cl * CV + i) * W + j] = dw[j][i];
        red[slot][CGL * CV * W + cl * CV + i] = db[i];
    }
    __syncthreads();
    float* out = a.dpar + (int64_t)(b * a.nseg + s) * a.dpar_stride;
    for (int k = threadIdx.x; k < CGL * CV * (W + 1); k += 256) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) v += red[i][k];
        const bool is_w = k < CGL * CV * W;
        const int ch = ct * CGL * CV + (is_w ? k / W : k - CGL * CV * W);
        if (ch >= a.D || (!is_w && a.dbias_off < 0)) continue;
        float* o = is_w ? out + (int64_t)ct * CGL * CV * W + k : out + a.dbias_off + ch;
        *o = a.accumulate ? *o + a.scale * v : a.scale * v;
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(256) conv_step_kernel(const T* __restrict__ X, int64_t x_sb, T* __restrict__ S,
                                                        const float* __restrict__ Wt, const float* __restrict__ bias,
                                                        T* __restrict__ Y, int64_t total, int D, int silu) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t b = i / D;
    const int d = (int)(i - b * D);
    T* s = S + b * (W - 1) * D + d;
    T line[W];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) line[j] = s[(int64_t)j * D];
    line[W - 1] = X[b * x_sb + d];
    float p = bias ? bias[d] : 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) p += Wt[(int64_t)d * W + j] * to_f32(line[j]);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) s[(int64_t)j * D] = line[j + 1];
    Y[i] = (T)(silu ? p * sigmoid_f(p) : p);
}

constexpr int NARROW = 16, WIDE = 64;   // lanes across channels: 64 channels or 256

int check(int B, int T, int D, int W, int64_t sb, int64_t st) {
    if (B < 0 || T < 0 || D <= 0 || W <= 0 || sb < 0 || st < 0) return DPK_EINVAL;
    if (W > 4 || T > MAX_DIM || D > MAX_DIM) return DPK_ERANGE;
    return DPK_OK;
}

}  // namespace

#define CONV_W(W, CALL)           \
    switch (W) {                  \
        case 1: CALL(1) break;    \
        case 2: CALL(2) break;    \
        case 3: CALL(3) break;    \
        default: CALL(4) break;   \
    }

// Time segments per sequence: enough workgroups for four a CU, but no stretch shorter than 8 rows (a stretch reads W-1 rows
// of its neighbour as well).
extern "C" int dpk_causal_conv_segments(int B, int T, int D) {
    if (B <= 0 || T <= 0 || D <= 0) return 1;
    const int cgl = D <= NARROW * CV ? NARROW : WIDE;
    const int64_t have = (int64_t)B * ((D + cgl * CV - 1) / (cgl * CV));
    int64_t s = (1024 + have - 1) / have;
    const int64_t most = (T + 8 * (256 / cgl) - 1) / (8 * (256 / cgl));
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}

extern "C" int dpk_causal_conv_forward(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias,
                                       const void* state, const int* lengths, void* y, void* state_out, int B, int T, int D,
                                       int W, int silu, int dtype, void* stream) {
    const int rc = check(B, T, D, W, x_sb, x_st);
    if (rc) return rc;
    if (B == 0 || (T == 0 && (!state_out || W == 1))) return DPK_OK;
    if (!w || (T > 0 && (!x || !y))) return DPK_EINVAL;
    ConvArgs a = {};
    a.x = x; a.w = w; a.bias = bias; a.state = state; a.lengths = lengths; a.y = y; a.state_out = state_out;
    a.x_sb = x_sb; a.x_st = x_st; a.B = B; a.T = T; a.D = D; a.silu = silu;
    a.nseg = dpk_causal_conv_segments(B, T, D);
    a.seg = (T + a.nseg - 1) / a.nseg;
    const int cgl = D <= NARROW * CV ? NARROW : WIDE;
    a.nct = (D + cgl * CV - 1) / (cgl * CV);
    const int64_t grid = (int64_t)B * a.nseg * a.nct;
    if (!dpk_launchable(grid, 256)) return DPK_ERANGE;
#define CALL(WW)                                                                                                             \
    if (cgl == NARROW)                                                                                                       \
        hipLaunchKernelGGL((conv_forward_kernel<E, WW, NARROW>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a); \
    else                                                                                                                     \
        hipLaunchKernelGGL((conv_forward_kernel<E, WW, WIDE>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    DPK_DISPATCH_DTYPE(dtype, E, CONV_W(W, CALL))
#undef CALL
    return dpk_launch_status();
}

extern "C" int dpk_causal_conv_backward(const void* x, int64_t x_sb, int64_t x_st, const void* dy, int64_t dy_sb, int64_t dy_st,
                                        const float* w, const float* bias, const void* state, const void* dstate_out,
                                        const int* lengths, void* dx, void* dstate, float* dpar, int64_t dpar_stride,
                                        int64_t dbias_off, int segments, int B, int T, int D, int W, int silu, float scale,
                                        int accumulate, int dtype, void* stream) {
    const int rc = check(B, T, D, W, x_sb, x_st);
    if (rc) return rc;
    if (dy_sb < 0 || dy_st < 0 || segments <= 0 || (dpar && dpar_stride < (int64_t)D * W)) return DPK_EINVAL;
    if (B == 0) return DPK_OK;
    if (!w || (T > 0 && (!x || !dy || !dx))) return DPK_EINVAL;
    ConvArgs a = {};
    a.x = x; a.dy = dy; a.w = w; a.bias = bias; a.state = state; a.dstate_out = dstate_out; a.lengths = lengths;
    a.dx = dx; a.dstate = dstate; a.dpar = dpar; a.dpar_stride = dpar_stride; a.dbias_off = dbias_off;
    a.x_sb = x_sb; a.x_st = x_st; a.dy_sb = dy_sb; a.dy_st = dy_st;
    a.B = B; a.T = T; a.D = D; a.silu = silu; a.scale = scale; a.accumulate = accumulate;
    a.nseg = segments;
    a.seg = (T + segments - 1) / segments;
    const int cgl = D <= NARROW * CV ? NARROW : WIDE;
    a.nct = (D + cgl * CV - 1) / (cgl * CV);
    const int64_t grid = (int64_t)B * a.nseg * a.nct;
    if (!dpk_launchable(grid, 256)) return DPK_ERANGE;
#define CALL(WW)                                                                                                              \
    if (cgl == NARROW)                                                                                                        \
        hipLaunchKernelGGL((conv_backward_kernel<E, WW, NARROW>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a); \
    else                                                                                                                      \
        hipLaunchKernelGGL((conv_backward_kernel<E, WW, WIDE>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    DPK_DISPATCH_DTYPE(dtype, E, CONV_W(W, CALL))
#undef CALL
    return dpk_launch_status();
}

extern "C" int dpk_causal_conv_step(const void* x, int64_t x_sb, void* state, const float* w, const float* bias, void* y, int B,
                                    int D, int W, int silu, int dtype, void* stream) {
    const int rc = check(B, 1, D, W, x_sb, 0);
    if (rc) return rc;
    if (B == 0) return DPK_OK;
    if (!x || !w || !y || (W > 1 && !state)) return DPK_EINVAL;
    const int64_t total = (int64_t)B * D, grid = (total + 255) / 256;
    if (!dpk_launchable(grid, 256)) return DPK_ERANGE;
#define CALL(WW)                                                                                                               \
    hipLaunchKernelGGL((conv_step_kernel<E, WW>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const E*)x, x_sb, \
                       (E*)state, w, bias, (E*)y, total, D, silu);
    DPK_DISPATCH_DTYPE(dtype, E, CONV_W(W, CALL))
#undef CALL
    return dpk_launch_status();
}
