// K14 — selective state-space scan, its backward pass and its single-token form.
//
//   dt = softplus(delta + dt_bias) (or without the softplus), A = -exp(A_log), h_t = exp(dt A) h_{t-1} + dt B_t u_t,
//   y_t = C_t . h_t + D u_t, out = y silu(z); one state of N numbers per (sequence, channel)
//   backward, t descending: dy = dout silu(z), dz = dout y silu'(z), dh = C_t dy + (exp(dt A) dh) of t+1,
//   dC_t = sum_d dy h_t, dB_t = sum_d dh dt u, q = dh . B_t, du = q dt + D dy, e_n = dh_n exp(dt A_n) h_{t-1,n},
//   ddt = q u + sum_n e_n A_n, dA_log_n = A_n sum_t e_n dt, dD = sum dy u, ddelta = ddt sigmoid(delta + dt_bias)
// Rows at and behind lengths[b] have dt = 0: the state stays what it was, out and all gradients there are 0.
//
// A lane owns one channel and walks time with its N states in registers (rows of u, delta, z are contiguous over channels, so
// every access of a wave is one run of memory); B_t and C_t are the same for all channels and are staged in LDS for GROUP
// steps at a time.  Per state and step that is one v_exp_f32 (quarter rate) and four plain instructions forward, two and
// about thirteen backward: at N = 16 the vector ALU and HBM are about equally loaded forward, and the ALU bounds backward.
// The backward pass needs the states in reverse.  Undoing the recurrence would divide by decays near 0, so the forward pass
// keeps the state at the start of every group of 8 steps (8 bytes a channel and step at N = 16) and the backward pass
// recomputes a group into registers.
// Sequences x channels / 64 is the number of waves; few long sequences are cut into chunks of time: each chunk's effect is
// (decay, state from zero), which a short kernel joins in order, and the chunks then run side by side from their true states.
#include "ssm_common.h"

namespace {

constexpr int GROUP = 8;

struct ScanArgs {
    const void *u, *delta, *B, *C, *z, *dout;
    const float *A_log, *Dskip, *dt_bias, *h0, *dhT;
    const int* lengths;
    void *out, *du, *ddelta, *dB, *dC, *dz;
    float *hT, *dh0, *kept;     // kept: [b][group][n][d]
    float *edge, *span;         // chunk edges: [chunk][b][n][d] and sums of dt [chunk][b][d]
    float *dbc;                 // [d block][b][t][2N] partial sums of dB | dC, where a row of channels needs several workgroups
    float *dA, *dD, *dbias;     // parameter gradients, row (b * nchunk + chunk) of par_stride floats
    int64_t u_sb, u_st, delta_sb, delta_st, B_sb, B_st, C_sb, C_st, z_sb, z_st, dout_sb, dout_st, par_stride;
    int nb, T, D, N, softplus, nchunk, chunk, ndb, accumulate;
    float scale;
};

__device__ __forceinline__ int seq_end(const ScanArgs& a, int b) {
    const int n = a.lengths ? a.lengths[b] : a.T;
    return n < 0 ? 0 : n > a.T ? a.T : n;
}

// the block's place: blockIdx.x = (chunk * nb + b) * ndb + channel block
struct Place {
    int b, chunk, dblk, d, t0, t1;
    bool live;
    __device__ __forceinline__ Place(const ScanArgs& a) {
        dblk = blockIdx.x % a.ndb;
        const int rest = blockIdx.x / a.ndb;
        b = rest % a.nb;
        chunk = rest / a.nb;
        d = dblk * blockDim.x + threadIdx.x;
        live = d < a.D;
        t0 = chunk * a.chunk;
        t1 = t0 + a.chunk < a.T ? t0 + a.chunk : a.T;
    }
};

// rows [t0, t0 + GROUP) of B and C as fp32, zero behind the sequence and behind N: s[q][0..NT) = B, s[q][NT..2 NT) = C
template <typename T, int NT>
__device__ __forceinline__ void stage_bc(const ScanArgs& a, int b, int t0, int end, float (&s)[GROUP][2 * NT]) {
    for (int i = threadIdx.x; i < GROUP * 2 * NT; i += blockDim.x) {
        const int q = i / (2 * NT), r = i % (2 * NT), n = r % NT;
        float v = 0.f;
        if (t0 + q < end && n < a.N)
            v = r < NT ? to_f32(((const T*)a.B)[(int64_t)b * a.B_sb + (int64_t)(t0 + q) * a.B_st + n])
                       : to_f32(((const T*)a.C)[(int64_t)b * a.C_sb + (int64_t)(t0 + q) * a.C_st + n]);
        s[q][r] = v;
    }
}

template <typename T>
__device__ __forceinline__ float elem(const void* p, int64_t sb, int64_t st, int b, int t, int d) {
    return to_f32(((const T*)p)[(int64_t)b * sb + (int64_t)t * st + d]);
}

__device__ __forceinline__ float step_size(const ScanArgs& a, float pre) { return a.softplus ? softplus_f(pre) : pre; }

// EDGE: only the chunk's state from zero and its sum of dt, for the chunks' joining
template <typename T, int NT, bool EDGE>
__global__ void __launch_bounds__(256) scan_forward_kernel(ScanArgs a) {
    __shared__ float bc[2][GROUP][2 * NT];
    const Place p(a);
    const int end = seq_end(a, p.b);
    const int dd = p.live ? p.d : a.D - 1;   // lanes behind the last channel read it and store nothing
    float A2[NT], h[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        A2[n] = n < a.N ? -expf(a.A_log[(int64_t)dd * a.N + n]) * LOG2E : 0.f;
        h[n] = 0.f;
        if (!EDGE && n < a.N) {
            if (a.nchunk > 1)
                h[n] = a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + dd];
            else if (a.h0)
                h[n] = a.h0[((int64_t)p.b * a.D + dd) * a.N + n];
        }
    }
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f;
    const float skip = a.Dskip ? a.Dskip[dd] : 0.f;
    float span = 0.f;
    const int ngroup = (a.T + GROUP - 1) / GROUP;
    int ph = 0;
    for (int t0 = p.t0; t0 < p.t1; t0 += GROUP, ph ^= 1) {
        if (!EDGE && a.kept && p.live) {
            float* k = a.kept + (((int64_t)p.b * ngroup + t0 / GROUP) * a.N) * a.D + p.d;
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (n < a.N) k[(int64_t)n * a.D] = h[n];
        }
        if (t0 < end) {
            float u[GROUP], dt[GROUP], z[GROUP];
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const int t = t0 + q < end ? t0 + q : end - 1;
                u[q] = t0 + q < end ? elem<T>(a.u, a.u_sb, a.u_st, p.b, t, dd) : 0.f;
                dt[q] = elem<T>(a.delta, a.delta_sb, a.delta_st, p.b, t, dd);
                if (!EDGE && a.z) z[q] = elem<T>(a.z, a.z_sb, a.z_st, p.b, t, dd);
            }
            stage_bc<T, NT>(a, p.b, t0, end, bc[ph]);
            __syncthreads();
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                dt[q] = t0 + q < end ? step_size(a, dt[q] + bias) : 0.f;
                if (EDGE) span += dt[q];
            }
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const float x = dt[q] * u[q];
                float y = skip * u[q];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    h[n] = exp2_hw(dt[q] * A2[n]) * h[n] + x * bc[ph][q][n];
                    if (!EDGE) y += bc[ph][q][NT + n] * h[n];
                }
                if (!EDGE) {
                    if (a.z) y *= z[q] * sigmoid_f(z[q]);
                    if (p.live && t0 + q < p.t1)
                        ((T*)a.out)[((int64_t)p.b * a.T + t0 + q) * a.D + p.d] = (T)(t0 + q < end ? y : 0.f);
                }
            }
        } else if (!EDGE && p.live) {
#pragma unroll
            for (int q = 0; q < GROUP; ++q)
                if (t0 + q < p.t1) ((T*)a.out)[((int64_t)p.b * a.T + t0 + q) * a.D + p.d] = (T)0.f;
        }
    }
    if (!p.live) return;
    if (EDGE) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n < a.N) a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + p.d] = h[n];
        a.span[((int64_t)p.chunk * a.nb + p.b) * a.D + p.d] = span;
    } else if (a.hT && p.chunk == a.nchunk - 1) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n < a.N) a.hT[((int64_t)p.b * a.D + p.d) * a.N + n] = h[n];
    }
}

// Joins the chunks: edge[c] comes in as what chunk c makes of a zero start and goes out as its true start (forward) or the
// gradient that enters it from behind (reverse).
template <bool REVERSE>
__global__ void __launch_bounds__(256) scan_join_kernel(ScanArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t per = (int64_t)a.N * a.D;
    if (i >= a.nb * per) return;
    const int b = (int)(i / per);
    const int n = (int)(i % per / a.D), d = (int)(i % a.D);
    const float A2 = -expf(a.A_log[(int64_t)d * a.N + n]) * LOG2E;
    const float* first = REVERSE ? a.dhT : a.h0;
    float h = first ? first[((int64_t)b * a.D + d) * a.N + n] : 0.f;
    for (int k = 0; k < a.nchunk; ++k) {
        const int c = REVERSE ? a.nchunk - 1 - k : k;
        float* e = a.edge + (((int64_t)c * a.nb + b) * a.N + n) * a.D + d;
        const float own = *e;
        *e = h;
        h = own + exp2_hw(A2 * a.span[((int64_t)c * a.nb + b) * a.D + d]) * h;
    }
}

// what a chunk hands to the chunk before it if nothing enters it from behind
template <typename T, int NT>
__global__ void __launch_bounds__(256) scan_backward_edge_kernel(ScanArgs a) {
    __shared__ float bc[2][GROUP][2 * NT];
    const Place p(a);
    const int end = seq_end(a, p.b);
    const int dd = p.live ? p.d : a.D - 1;
    float A2[NT], dh[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        A2[n] = n < a.N ? -expf(a.A_log[(int64_t)dd * a.N + n]) * LOG2E : 0.f;
        dh[n] = 0.f;
    }
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f;
    float span = 0.f;
    int ph = 0;
    const int last = p.t0 + (p.t1 - p.t0 - 1) / GROUP * GROUP;
    for (int t0 = last; t0 >= p.t0; t0 -= GROUP, ph ^= 1) {
        if (t0 >= end) continue;
        float dy[GROUP], dt[GROUP];
#pragma unroll
        for (int q = 0; q < GROUP; ++q) {
            const int t = t0 + q < end ? t0 + q : end - 1;
            dt[q] = elem<T>(a.delta, a.delta_sb, a.delta_st, p.b, t, dd);
            dy[q] = elem<T>(a.dout, a.dout_sb, a.dout_st, p.b, t, dd);
            if (a.z) {
                const float z = elem<T>(a.z, a.z_sb, a.z_st, p.b, t, dd);
                dy[q] *= z * sigmoid_f(z);
            }
        }
        stage_bc<T, NT>(a, p.b, t0, end, bc[ph]);
        __syncthreads();
#pragma unroll
        for (int q = GROUP - 1; q >= 0; --q) {
            const float s = t0 + q < end ? step_size(a, dt[q] + bias) : 0.f;
            span += s;
#pragma unroll
            for (int n = 0; n < NT; ++n) dh[n] = exp2_hw(s * A2[n]) * (dh[n] + dy[q] * bc[ph][q][NT + n]);
        }
    }
    if (!p.live) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
        if (n < a.N) a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + p.d] = dh[n];
    a.span[((int64_t)p.chunk * a.nb + p.b) * a.D + p.d] = span;
}

// Sums each of V values over the 64 lanes of a wave; afterwards lane l holds the sum of value slot(l).  A step adds the halves
// of two values at once and leaves one register of the two, so V values take about 2 V instructions instead of 6 V.
template <int C>
__device__ __forceinline__ void fold32(float* v) {
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + C / 2]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}
template <int C>
__device__ __forceinline__ void fold16(float* v) {
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + C / 2]), false, false);
        v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}
// partner lane by the DPP control CTRL, which flips the lane bit BIT (and may flip lower ones)
template <int C, int CTRL, int BIT>
__device__ __forceinline__ void fold_dpp(float* v) {
    if constexpr (C == 1) {
        v[0] += dpp<CTRL>(v[0]);
    } else {
        const bool up = threadIdx.x & BIT;
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
            const float keep = up ? v[i + C / 2] : v[i], send = up ? v[i] : v[i + C / 2];
            v[i] = keep + dpp<CTRL>(send);
        }
    }
}
constexpr int half_of(int c) { return c > 1 ? c / 2 : 1; }
template <int V>   // V a power of two, 8..64
__device__ __forceinline__ void lane_sums(float* v) {
    constexpr int C3 = V / 4, C4 = half_of(C3), C5 = half_of(C4), C6 = half_of(C5);
    fold32<V>(v);
    fold16<V / 2>(v);
    fold_dpp<C3, 0x128, 8>(v);    // row_ror:8
    fold_dpp<C4, 0x141, 4>(v);    // row_half_mirror
    fold_dpp<C5, 0x4E, 2>(v);     // quad_perm 2,3,0,1
    fold_dpp<C6, 0xB1, 1>(v);     // quad_perm 1,0,3,2
}
template <int V>
__device__ __forceinline__ int lane_slot(int lane) {
    int s = 0, c = V;
#pragma unroll
    for (int bit = 32; bit >= 1; bit >>= 1) {
        c >>= 1;
        if (c >= 1 && (lane & bit)) s += c;
    }
    return s;
}
// one lane of each set that holds the same sum
template <int V>
__device__ __forceinline__ bool lane_writes(int lane) {
    return (lane & (64 / (V < 64 ? V : 64) - 1)) == 0;
}

template <typename T, int NT>
__global__ void __launch_bounds__(256) scan_backward_kernel(ScanArgs a) {
    __shared__ float bc[2][GROUP][2 * NT];
    __shared__ float part[2][4][GROUP][2 * NT];
    const Place p(a);
    const int end = seq_end(a, p.b);
    const int dd = p.live ? p.d : a.D - 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    float A2[NT], dh[NT], dA[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        A2[n] = n < a.N ? -expf(a.A_log[(int64_t)dd * a.N + n]) * LOG2E : 0.f;
        dA[n] = 0.f;
        dh[n] = 0.f;
        if (n < a.N) {
            if (a.nchunk > 1)
                dh[n] = a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + dd];
            else if (a.dhT)
                dh[n] = a.dhT[((int64_t)p.b * a.D + dd) * a.N + n];
        }
        if (!p.live) dh[n] = 0.f;   // nothing of these lanes may reach the sums over channels
    }
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f;
    const float skip = a.Dskip ? a.Dskip[dd] : 0.f;
    float dD = 0.f, dbias = 0.f;
    const int ngroup = (a.T + GROUP - 1) / GROUP;
    int ph = 0;
    const int last = p.t0 + (p.t1 - p.t0 - 1) / GROUP * GROUP;
    for (int t0 = last; t0 >= p.t0; t0 -= GROUP) {
        if (t0 >= end) {
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                if (t0 + q >= p.t1) break;
                if (p.live) {
                    const int64_t o = ((int64_t)p.b * a.T + t0 + q) * a.D + p.d;
                    ((T*)a.du)[o] = (T)0.f;
                    ((T*)a.ddelta)[o] = (T)0.f;
                    if (a.dz) ((T*)a.dz)[o] = (T)0.f;
                }
                for (int i = threadIdx.x; i < 2 * a.N; i += blockDim.x) {
                    const int64_t row = (int64_t)p.b * a.T + t0 + q;
                    if (a.ndb > 1)
                        a.dbc[((int64_t)p.dblk * a.nb * a.T + row) * 2 * a.N + i] = 0.f;
                    else if (i < a.N)
                        ((T*)a.dB)[row * a.N + i] = (T)0.f;
                    else
                        ((T*)a.dC)[row * a.N + i - a.N] = (T)0.f;
                }
            }
            continue;
        }
        float u[GROUP], pre[GROUP], dy[GROUP], z[GROUP], dt[GROUP], hist[GROUP][NT];
#pragma unroll
        for (int q = 0; q < GROUP; ++q) {
            // steps behind the sequence and lanes behind the last channel count as zeros, whatever lies there: neither may
            // bring an inf or NaN into the sums over channels
            const bool in = t0 + q < end && p.live;
            const int t = t0 + q < end ? t0 + q : end - 1;
            u[q] = in ? elem<T>(a.u, a.u_sb, a.u_st, p.b, t, dd) : 0.f;
            pre[q] = in ? elem<T>(a.delta, a.delta_sb, a.delta_st, p.b, t, dd) + bias : 0.f;
            dy[q] = in ? elem<T>(a.dout, a.dout_sb, a.dout_st, p.b, t, dd) : 0.f;
            z[q] = in && a.z ? elem<T>(a.z, a.z_sb, a.z_st, p.b, t, dd) : 0.f;
        }
        {
            const float* k = a.kept + (((int64_t)p.b * ngroup + t0 / GROUP) * a.N) * a.D + dd;
#pragma unroll
            for (int n = 0; n < NT; ++n) hist[0][n] = n < a.N && p.live ? k[(int64_t)n * a.D] : 0.f;
        }
        stage_bc<T, NT>(a, p.b, t0, end, bc[ph]);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < GROUP; ++q) dt[q] = t0 + q < end ? step_size(a, pre[q]) : 0.f;
#pragma unroll
        for (int q = 0; q + 1 < GROUP; ++q) {
            const float x = dt[q] * u[q];
#pragma unroll
            for (int n = 0; n < NT; ++n) hist[q + 1][n] = exp2_hw(dt[q] * A2[n]) * hist[q][n] + x * bc[ph][q][n];
        }
#pragma unroll
        for (int q = GROUP - 1; q >= 0; --q) {
            const float x = dt[q] * u[q];
            float g = dy[q], sg = 1.f;
            if (a.z) {
                sg = sigmoid_f(z[q]);
                g *= z[q] * sg;
            }
            float y = skip * u[q], into = 0.f, along = 0.f;
            float v[2 * NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float e = exp2_hw(dt[q] * A2[n]);
                const float eh = e * hist[q][n];
                const float h = eh + x * bc[ph][q][n];
                const float cn = bc[ph][q][NT + n];
                y += cn * h;
                dh[n] += g * cn;
                v[n] = dh[n] * x;
                v[NT + n] = g * h;
                into += dh[n] * bc[ph][q][n];
                const float t = dh[n] * eh;
                along += t * A2[n];
                dA[n] += t * dt[q];
                dh[n] *= e;
            }
            lane_sums<2 * NT>(v);
            if (lane_writes<2 * NT>(lane)) part[ph][wave][q][lane_slot<2 * NT>(lane)] = v[0];
            const bool in = t0 + q < end;
            const float ddt = into * u[q] + along * LN2;
            const float dpre = a.softplus ? ddt * sigmoid_f(pre[q]) : ddt;
            if (in) {
                dD += g * u[q];
                dbias += dpre;
            }
            if (p.live && t0 + q < p.t1) {
                const int64_t o = ((int64_t)p.b * a.T + t0 + q) * a.D + p.d;
                ((T*)a.du)[o] = (T)(in ? into * dt[q] + skip * g : 0.f);
                ((T*)a.ddelta)[o] = (T)(in ? dpre : 0.f);
                if (a.dz) ((T*)a.dz)[o] = (T)(in ? dy[q] * y * sg * (1.f + z[q] * (1.f - sg)) : 0.f);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < GROUP * 2 * NT; i += blockDim.x) {
            const int q = i / (2 * NT), r = i % (2 * NT), n = r % NT;
            if (n >= a.N || t0 + q >= p.t1) continue;
            float s = 0.f;
            if (t0 + q < end)
                for (int w = 0; w < nw; ++w) s += part[ph][w][q][r];
            const int64_t row = (int64_t)p.b * a.T + t0 + q;
            if (a.ndb > 1)
                a.dbc[((int64_t)p.dblk * a.nb * a.T + row) * 2 * a.N + (r < NT ? n : a.N + n)] = s;
            else if (r < NT)
                ((T*)a.dB)[row * a.N + n] = (T)s;
            else
                ((T*)a.dC)[row * a.N + n] = (T)s;
        }
        ph ^= 1;
    }
    if (!p.live) return;
    if (a.dh0 && p.chunk == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n < a.N) a.dh0[((int64_t)p.b * a.D + p.d) * a.N + n] = dh[n];
    }
    const int64_t row = ((int64_t)p.b * a.nchunk + p.chunk) * a.par_stride;
    if (a.dA) {
        float* o = a.dA + row + (int64_t)p.d * a.N;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n < a.N) o[n] = (a.accumulate ? o[n] : 0.f) + a.scale * (A2[n] * LN2) * dA[n];
    }
    if (a.dD) a.dD[row + p.d] = (a.accumulate ? a.dD[row + p.d] : 0.f) + a.scale * dD;
    if (a.dbias) a.dbias[row + p.d] = (a.accumulate ? a.dbias[row + p.d] : 0.f) + a.scale * dbias;
}

// dB and dC of all channel blocks, in their order
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_sum_kernel(const float* __restrict__ in, T* __restrict__ dB, T* __restrict__ dC,
                                                          int64_t rows, int N, int ndb) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t total = rows * 2 * N;
    if (i >= total) return;
    float s = 0.f;
    for (int k = 0; k < ndb; ++k) s += in[k * total + i];
    const int64_t row = i / (2 * N);
    const int r = (int)(i - row * 2 * N);
    if (r < N)
        dB[row * N + r] = (T)s;
    else
        dC[row * N + r - N] = (T)s;
}

// one token: L lanes a channel, 4 states a lane (a lane reads and writes 16 bytes of the state)
template <typename T, int L>
__global__ void __launch_bounds__(256) scan_step_kernel(ScanArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t ch = i / L;
    const bool live = ch < (int64_t)a.nb * a.D;
    const int64_t at = live ? ch : 0;
    const int b = (int)(at / a.D), d = (int)(at % a.D), n0 = (int)(i % L) * 4;
    const int n = live && n0 < a.N ? a.N - n0 : 0;
    const float u = elem<T>(a.u, a.u_sb, 0, b, 0, d);
    const float dt = step_size(a, elem<T>(a.delta, a.delta_sb, 0, b, 0, d) + (a.dt_bias ? a.dt_bias[d] : 0.f));
    float al[4], Bv[4], Cv[4], h[4];
    load_n<float, 4>(a.A_log + (int64_t)d * a.N + n0, n, al);
    load_n<T, 4>((const T*)a.B + (int64_t)b * a.B_sb + n0, n, Bv);
    load_n<T, 4>((const T*)a.C + (int64_t)b * a.C_sb + n0, n, Cv);
    float* hs = a.hT + at * a.N + n0;
    load_n<float, 4>(hs, n, h);
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        h[k] = exp2_hw(-expf(al[k]) * LOG2E * dt) * h[k] + dt * u * Bv[k];
        if (k < n) y += Cv[k] * h[k];
    }
    store_n<float, 4>(hs, n, h);
#pragma unroll
    for (int off = L / 2; off >= 1; off >>= 1) y += __shfl_xor(y, off, 64);
    if (live && n0 == 0) {
        if (a.Dskip) y += a.Dskip[d] * u;
        if (a.z) {
            const float z = elem<T>(a.z, a.z_sb, 0, b, 0, d);
            y *= z * sigmoid_f(z);
        }
        ((T*)a.out)[ch] = (T)y;
    }
}

int block_of(int D) { return D > 192 ? 256 : (D + 63) / 64 * 64; }

int check(const dpk_scan_desc* s) {
    if (!s || s->B < 0 || s->T < 0 || s->D <= 0 || s->N <= 0) return DPK_EINVAL;
    if (s->N > DPK_SCAN_MAX_STATE) return DPK_ERANGE;
    if (s->dtype != DPK_F32 && s->dtype != DPK_BF16 && s->dtype != DPK_F16) return DPK_EINVAL;
    if (s->nchunk <= 0 || s->chunk < 0 || s->chunk % GROUP || (int64_t)s->nchunk * s->chunk < s->T) return DPK_EINVAL;
    if (s->u_sb < 0 || s->u_st < 0 || s->delta_sb < 0 || s->delta_st < 0 || s->B_sb < 0 || s->B_st < 0 || s->C_sb < 0 ||
        s->C_st < 0 || s->z_sb < 0 || s->z_st < 0)
        return DPK_EINVAL;
    if (!s->A_log || (s->T > 0 && (!s->u || !s->delta || !s->Bm || !s->Cm))) return DPK_EINVAL;
    const int bl = block_of(s->D);
    if ((int64_t)s->B * s->nchunk * ((s->D + bl - 1) / bl) > 0x7fffffffLL) return DPK_ERANGE;
    if (((int64_t)s->B * s->N * s->D + 255) / 256 > 0x7fffffffLL) return DPK_ERANGE;
    return DPK_OK;
}

ScanArgs fill(const dpk_scan_desc* s) {
    ScanArgs a = {};
    a.u = s->u; a.delta = s->delta; a.B = s->Bm; a.C = s->Cm; a.z = s->z;
    a.A_log = s->A_log; a.Dskip = s->Dskip; a.dt_bias = s->dt_bias; a.h0 = s->h0; a.lengths = s->lengths;
    a.u_sb = s->u_sb; a.u_st = s->u_st; a.delta_sb = s->delta_sb; a.delta_st = s->delta_st;
    a.B_sb = s->B_sb; a.B_st = s->B_st; a.C_sb = s->C_sb; a.C_st = s->C_st; a.z_sb = s->z_sb; a.z_st = s->z_st;
    a.nb = s->B; a.T = s->T; a.D = s->D; a.N = s->N; a.softplus = s->softplus; a.nchunk = s->nchunk; a.chunk = s->chunk;
    const int bl = block_of(s->D);
    a.ndb = (s->D + bl - 1) / bl;
    a.kept = s->kept; a.edge = s->edge; a.span = s->span;
    return a;
}

}  // namespace

#define SCAN_N(N, CALL)           \
    if (N <= 4) { CALL(4) }       \
    else if (N <= 8) { CALL(8) }  \
    else if (N <= 16) { CALL(16) } \
    else { CALL(32) }

// Chunks of time a scan is cut into.  A whole pass costs a second reading of the inputs and most of its arithmetic again, so it
// has to win a factor of two in waves at least: only scans of fewer than 512 waves (half a wave a SIMD) are cut, into chunks of
// 64 steps or more.
extern "C" int dpk_selective_scan_chunks(int B, int T, int D, int* chunk) {
    if (B <= 0 || T <= 0 || D <= 0) {
        if (chunk) *chunk = (T > 0 ? (T + GROUP - 1) / GROUP * GROUP : 0);
        return 1;
    }
    const int64_t waves = (int64_t)B * ((D + 63) / 64);
    int64_t n = waves >= 512 ? 1 : 2048 / waves;
    const int64_t most = (T + 63) / 64;
    if (n > most) n = most;
    if (n < 3) n = 1;
    int64_t len = (T + n - 1) / n;
    len = (len + GROUP - 1) / GROUP * GROUP;
    n = (T + len - 1) / len;
    if (chunk) *chunk = (int)len;
    return (int)n;
}

extern "C" int dpk_selective_scan_group(void) { return GROUP; }
extern "C" int dpk_selective_scan_channel_blocks(int D) { return D <= 0 ? 0 : (D + block_of(D) - 1) / block_of(D); }

extern "C" int dpk_selective_scan_forward(const dpk_scan_desc* s, void* out, float* hT, void* stream) {
    const int rc = check(s);
    if (rc) return rc;
    if (s->B == 0) return DPK_OK;
    if (s->T > 0 && !out) return DPK_EINVAL;
    if (s->nchunk > 1 && (!s->edge || !s->span)) return DPK_EINVAL;
    ScanArgs a = fill(s);
    a.out = out; a.hT = hT;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(a.nb * a.nchunk * a.ndb)), block((unsigned)block_of(a.D));
    if (a.nchunk > 1) {
#define CALL(NT) hipLaunchKernelGGL((scan_forward_kernel<E, NT, true>), grid, block, 0, st, a);
        DPK_DISPATCH_DTYPE(s->dtype, E, SCAN_N(a.N, CALL))
#undef CALL
        hipLaunchKernelGGL(scan_join_kernel<false>, dim3((unsigned)(((int64_t)a.nb * a.N * a.D + 255) / 256)), dim3(256), 0, st, a);
    }
#define CALL(NT) hipLaunchKernelGGL((scan_forward_kernel<E, NT, false>), grid, block, 0, st, a);
    DPK_DISPATCH_DTYPE(s->dtype, E, SCAN_N(a.N, CALL))
#undef CALL
    return dpk_launch_status();
}

extern "C" int dpk_selective_scan_backward(const dpk_scan_desc* s, const dpk_scan_grads* g, void* stream) {
    const int rc = check(s);
    if (rc) return rc;
    if (!g || g->dout_sb < 0 || g->dout_st < 0) return DPK_EINVAL;
    if (s->B == 0) return DPK_OK;
    if (s->T > 0 && (!g->dout || !g->du || !g->ddelta || !g->dB || !g->dC || !s->kept || (s->z && !g->dz))) return DPK_EINVAL;
    if (s->nchunk > 1 && (!s->edge || !s->span)) return DPK_EINVAL;
    if ((g->dA || g->dD || g->dbias) && g->par_stride < s->D) return DPK_EINVAL;
    ScanArgs a = fill(s);
    if (a.ndb > 1 && s->T > 0 && !g->dbc) return DPK_EINVAL;
    a.dout = g->dout; a.dhT = g->dhT; a.du = g->du; a.ddelta = g->ddelta; a.dB = g->dB; a.dC = g->dC; a.dz = s->z ? g->dz : nullptr;
    a.dh0 = g->dh0; a.dbc = g->dbc; a.dA = g->dA; a.dD = g->dD; a.dbias = g->dbias; a.par_stride = g->par_stride;
    a.dout_sb = g->dout_sb; a.dout_st = g->dout_st; a.scale = g->scale; a.accumulate = g->accumulate;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(a.nb * a.nchunk * a.ndb)), block((unsigned)block_of(a.D));
    const int64_t sums = (int64_t)a.nb * a.T * 2 * a.N;
    if ((sums + 255) / 256 > 0x7fffffffLL) return DPK_ERANGE;
    if (a.nchunk > 1) {
#define CALL(NT) hipLaunchKernelGGL((scan_backward_edge_kernel<E, NT>), grid, block, 0, st, a);
        DPK_DISPATCH_DTYPE(s->dtype, E, SCAN_N(a.N, CALL))
#undef CALL
        hipLaunchKernelGGL(scan_join_kernel<true>, dim3((unsigned)(((int64_t)a.nb * a.N * a.D + 255) / 256)), dim3(256), 0, st, a);
    }
#define CALL(NT) hipLaunchKernelGGL((scan_backward_kernel<E, NT>), grid, block, 0, st, a);
    DPK_DISPATCH_DTYPE(s->dtype, E, SCAN_N(a.N, CALL))
#undef CALL
    if (a.ndb > 1 && sums > 0) {
        DPK_DISPATCH_DTYPE(s->dtype, E, hipLaunchKernelGGL(scan_bc_sum_kernel<E>, dim3((unsigned)((sums + 255) / 256)), dim3(256),
                                                           0, st, a.dbc, (E*)a.dB, (E*)a.dC, (int64_t)a.nb * a.T, a.N, a.ndb);)
    }
    return dpk_launch_status();
}

extern "C" int dpk_selective_scan_step(const dpk_scan_desc* s, float* state, void* out, void* stream) {
    const int rc = check(s);
    if (rc) return rc;
    if (s->T != 1) return DPK_EINVAL;
    if (s->B == 0) return DPK_OK;
    if (!state || !out) return DPK_EINVAL;
    ScanArgs a = fill(s);
    a.hT = state; a.out = out;
    const int lanes = s->N <= 4 ? 1 : s->N <= 8 ? 2 : s->N <= 16 ? 4 : 8;
    const int64_t grid = ((int64_t)a.nb * a.D * lanes + 255) / 256;
    if (grid > 0x7fffffffLL) return DPK_ERANGE;
#define CALL(L) hipLaunchKernelGGL((scan_step_kernel<E, L>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    DPK_DISPATCH_DTYPE(s->dtype, E, if (lanes == 1) { CALL(1) } else if (lanes == 2) { CALL(2) } else if (lanes == 4) { CALL(4) } else { CALL(8) })
#undef CALL
    return dpk_launch_status();
}
