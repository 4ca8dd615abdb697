// K14 — selective state-space scan, its backward pass and its single-token form.
//
//   dt = softplus(delta + dt_bias) (or without the softplus), A = -exp(A_log), h_t = exp(dt A) h_{t-1} + dt B_t u_t,
//   y_t = C_t . h_t + D u_t, out = y silu(z); one state of N numbers per (sequence, channel)
//   backward, t descending: dy = dout silu(z), dz = dout y silu'(z), dh = C_t dy + (exp(dt A) dh) of t+1,
//   dC_t = sum_d dy h_t, dB_t = sum_d dh dt u, q = dh . B_t, du = q dt + D dy, e_n = dh_n exp(dt A_n) h_{t-1,n},
//   ddt = q u + sum_n e_n A_n, dA_log_n = A_n sum_t e_n dt, dD = sum dy u, ddelta = ddt sigmoid(delta + dt_bias)
// Rows at and behind lengths[b] have dt = 0: the state stays what it was, out and all gradients there are 0.
//
// Forward, a lane owns one channel and walks time with its N states in registers (rows of u, delta, z are contiguous over
// channels, so every access of a wave is one run of memory); B_t and C_t are the same for all channels and are staged in LDS for
// GROUP steps at a time.
// The backward pass needs the states in reverse.  Undoing the recurrence would divide by decays near 0, so the forward pass
// keeps the state at the start of every group of 8 steps (8 bytes a channel and step at N = 16; not of the first group where it is
// 0), and the backward pass recomputes a group's states and decays into registers.  A channel's states lie on LS = N / 4 lanes there,
// so that three waves a SIMD fit (with all 16 on one lane, one wave a SIMD: 1887 us at 256 x 256 x 1024; with eight, the group spilled
// and waited for its spills: 3311); what a channel has once per step (softplus, gates, loads, stores) is dealt over those lanes by step, and passed round by
// lane swaps.
// Per state and step: forward one v_exp_f32 (quarter rate) and four plain instructions, backward one and twelve, and the sums
// over channels for dB and dC, a halving tree over the lanes (four more).  Measured at 256 x 256 x 1024, N = 16, fp32: forward
// 350 us = 4.5 TB/s with the kept states, backward 930 us, bound by the vector ALU (about 80 % busy), of which 2.4 GB of traffic are
// 500 us.
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
    float *hT, *dh0, *kept;     // kept: [b][group][n][d], from step kept_from on, n padded to 4, 8, 16 or 32
    float *edge, *span;         // chunk edges: [chunk][b][n][d] and sums of dt [chunk][b][d]
    float *dbc;                 // [d block][b][t][2N] partial sums of dB | dC, where a row of channels needs several workgroups
    float *dA, *dD, *dbias;     // parameter gradients, row (b * nchunk + chunk) of par_stride floats
    int64_t u_sb, u_st, delta_sb, delta_st, B_sb, B_st, C_sb, C_st, z_sb, z_st, dout_sb, dout_st, par_stride;
    int nb, T, D, N, softplus, gate, nchunk, chunk, ndb, accumulate;   // without a gate z is u: read, and not used
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

// The same in two halves, for workgroups of 256: fetched into registers, put into LDS once the group before is done with its half
// of the buffer.  (Smaller workgroups, of narrow layers, stage in one go.)
template <int NT>
struct Staged {
    static constexpr int K = GROUP * 2 * NT > 256 ? GROUP * 2 * NT / 256 : 1;
    float v[K];
};
// Operands are read and written relative to their group's first row: a 64-bit address that the wave shares and a 32-bit byte offset
// a lane.  GLOBAL: a store that the compiler takes for a flat one would be waited for with the next access to LDS.
#define GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ const char* group_row(const void* p, int64_t sb, int64_t st, int b, int t0) {
    return (const char*)p + (b * sb + t0 * st) * (int64_t)sizeof(T);
}
// rows of one sequence
template <typename T>
struct Rows {
    const char* first;
    uint32_t st;
    __device__ __forceinline__ Rows(const void* p, int64_t sb, int64_t st_, int b) : first((const char*)p + b * sb * (int64_t)sizeof(T)), st((uint32_t)st_) {
        asm("" : "+s"(first));
    }
    __device__ __forceinline__ const char* at(int t0) const { return first + (uint64_t)(uint32_t)t0 * st * sizeof(T); }
};
__device__ __forceinline__ char* out_row(void* p, int64_t at) {
    char* r = (char*)p + at;
    asm("" : "+s"(r));   // (else the lane's offset is added first and the row's becomes a 64-bit product per lane)
    return r;
}
template <typename T>
__device__ __forceinline__ float at(const char* row, uint32_t bytes) {
    return to_f32(*(GLOBAL const T*)(row + bytes));
}
template <typename T>
__device__ __forceinline__ void put(char* row, uint32_t bytes, float v) {
    *(GLOBAL T*)(row + bytes) = (T)v;
}

template <typename T, int NT>
__device__ __forceinline__ void fetch_bc(const ScanArgs& a, const Rows<T>& rb, const Rows<T>& rc, int t0, int end, Staged<NT>& r) {
    if (blockDim.x != 256) return;
    const char *gb = rb.at(t0), *gc = rc.at(t0);
#pragma unroll
    for (int k = 0; k < Staged<NT>::K; ++k) {
        const int i = threadIdx.x + k * 256;
        const int q = i / (2 * NT), c = i % (2 * NT), n = c % NT;
        const uint32_t row = i < GROUP * 2 * NT && t0 + q < end ? q : 0, col = n < a.N ? n : 0;   // others read and put 0
        r.v[k] = at<T>(c < NT ? gb : gc, (__umul24(row, c < NT ? rb.st : rc.st) + col) * (uint32_t)sizeof(T));
    }
}
template <typename T, int NT>
__device__ __forceinline__ void put_bc(const ScanArgs& a, int b, int t0, int end, const Staged<NT>& r, float (&s)[GROUP][2 * NT]) {
    if (blockDim.x != 256) {
        stage_bc<T, NT>(a, b, t0, end, s);
        return;
    }
#pragma unroll
    for (int k = 0; k < Staged<NT>::K; ++k) {
        const int i = threadIdx.x + k * 256;
        if (i < GROUP * 2 * NT) (&s[0][0])[i] = t0 + i / (2 * NT) < end && i % NT < a.N ? r.v[k] : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ float elem(const void* p, int64_t sb, int64_t st, int b, int t, int d) {
    return to_f32(((const T*)p)[(int64_t)b * sb + (int64_t)t * st + d]);
}

__device__ __forceinline__ float step_size(const ScanArgs& a, float pre) { return a.softplus ? softplus_f(pre).value : pre; }

// first step whose state the forward pass keeps: without h0 the first group's is 0
__device__ __forceinline__ int kept_from(const ScanArgs& a) { return a.h0 ? 0 : GROUP; }

// N numbers of a channel, which lie together: four at a time
template <int NT>
__device__ __forceinline__ void load_states(const float* __restrict__ p, int n, float (&v)[NT]) {
#pragma unroll
    for (int k = 0; k < NT; k += 4) {
        float t[4];
        load_n<float, 4>(p + k, n - k, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[k + i] = t[i];
    }
}
template <int NT>
__device__ __forceinline__ void store_states(float* __restrict__ p, int n, const float (&v)[NT]) {
#pragma unroll
    for (int k = 0; k < NT; k += 4) {
        const float t[4] = {v[k], v[k + 1], v[k + 2], v[k + 3]};
        store_n<float, 4>(p + k, n - k, t);
    }
}
// -exp(A_log) log2 e of states n0 ..., 0 behind N
template <int NT>
__device__ __forceinline__ void decay_rates(const ScanArgs& a, int d, int n0, float (&A2)[NT]) {
    load_states<NT>(a.A_log + (int64_t)d * a.N + n0, a.N - n0, A2);
#pragma unroll
    for (int n = 0; n < NT; ++n) A2[n] = n0 + n < a.N ? -expf(A2[n]) * LOG2E : 0.f;
}

// EDGE: only the chunk's state from zero and its sum of dt, for the chunks' joining
template <typename T, int NT, bool EDGE>
__global__ void __launch_bounds__(256, NT <= 16 ? 4 : 2) scan_forward_kernel(ScanArgs a) {
    __shared__ float bc[2][GROUP][2 * NT];
    const Place p(a);
    const int end = seq_end(a, p.b);
    const int dd = p.live ? p.d : a.D - 1;   // lanes behind the last channel read it and store nothing
    float A2[NT], h[NT];
    decay_rates<NT>(a, dd, 0, A2);
#pragma unroll
    for (int n = 0; n < NT; ++n) h[n] = 0.f;
    if (!EDGE && a.nchunk > 1) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n < a.N) h[n] = a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + dd];
    } else if (!EDGE && a.h0) {
        load_states<NT>(a.h0 + ((int64_t)p.b * a.D + dd) * a.N, a.N, h);
    }
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f;
    const float skip = a.Dskip ? a.Dskip[dd] : 0.f;
    float span = 0.f;
    const int k0 = kept_from(a), ngroup = (a.T - k0 + GROUP - 1) / GROUP;   // groups with a kept state
    const uint32_t lane_in = (uint32_t)dd * sizeof(T), lane_out = (uint32_t)p.d * sizeof(T);
    int ph = 0;
    for (int t0 = p.t0; t0 < p.t1; t0 += GROUP, ph ^= 1) {
        if (!EDGE && a.kept && p.live && t0 >= k0) {
            char* k = (char*)(a.kept + ((int64_t)p.b * ngroup + (t0 - k0) / GROUP) * NT * a.D);
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (n < a.N) put<float>(k + (int64_t)n * a.D * 4, (uint32_t)p.d * 4u, h[n]);
        }
        char* out = (char*)a.out + ((int64_t)p.b * a.T + t0) * a.D * (int64_t)sizeof(T);
        if (t0 < end) {
            float u[GROUP], dt[GROUP], z[GROUP];
            const char* gu = group_row<T>(a.u, a.u_sb, a.u_st, p.b, t0);
            const char* gd = group_row<T>(a.delta, a.delta_sb, a.delta_st, p.b, t0);
            const char* gz = group_row<T>(a.z, a.z_sb, a.z_st, p.b, t0);
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const uint32_t r = t0 + q < end ? q * (uint32_t)sizeof(T) : 0u;   // rows behind the sequence: the group's first
                u[q] = at<T>(gu, lane_in + r * (uint32_t)a.u_st);
                dt[q] = at<T>(gd, lane_in + r * (uint32_t)a.delta_st);
                if (!EDGE) z[q] = at<T>(gz, lane_in + r * (uint32_t)a.z_st);   // (with a gate or not: in a branch it is waited for)
            }
            stage_bc<T, NT>(a, p.b, t0, end, bc[ph]);
            __syncthreads();
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const bool in = t0 + q < end;
                u[q] = in ? u[q] : 0.f;
                dt[q] = in ? step_size(a, dt[q] + bias) : 0.f;
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
                    if (a.gate) y *= z[q] * sigmoid_f(z[q]);
                    if (p.live && t0 + q < p.t1) put<T>(out + (int64_t)q * a.D * (int64_t)sizeof(T), lane_out, t0 + q < end ? y : 0.f);
                }
            }
        } else if (!EDGE && p.live) {
#pragma unroll
            for (int q = 0; q < GROUP; ++q)
                if (t0 + q < p.t1) put<T>(out + (int64_t)q * a.D * (int64_t)sizeof(T), lane_out, 0.f);
        }
    }
    if (!p.live) return;
    if (EDGE) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if (n < a.N) a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + p.d] = h[n];
        a.span[((int64_t)p.chunk * a.nb + p.b) * a.D + p.d] = span;
    } else if (a.hT && p.chunk == a.nchunk - 1) {
        store_states<NT>(a.hT + ((int64_t)p.b * a.D + p.d) * a.N, a.N, h);
    }
}

constexpr int JOIN_RUN = 8;
// Joins the chunks: edge[c] comes in as what chunk c makes of a zero start and goes out as its true start (forward) or the
// gradient that enters it from behind (reverse).  LANES lanes share a state: each takes a run of eight chunks into registers, the
// runs' (decay, state from zero) are joined by lane shuffles, and each lane walks its run again from its true start.  As many lanes
// as there are runs, up to eight: the wave's other lanes are neighbouring states, so fewer runs make longer runs of memory (5 chunks
// of 50 x 16 x 1024 states: 79 us with eight lanes, 13 with one).
template <bool REVERSE, int LANES>
__global__ void __launch_bounds__(256) scan_join_kernel(ScanArgs a) {
    constexpr int RUN = JOIN_RUN, STATES = 64 / LANES;
    const int64_t per = (int64_t)a.N * a.D;
    const int run = (threadIdx.x & 63) / STATES, state = threadIdx.x % STATES;
    const int64_t i = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * STATES + state;
    const bool live = i < a.nb * per;
    const int64_t at = live ? i : 0;
    const int b = (int)(at / per);
    const int n = (int)(at % per / a.D), d = (int)(at % a.D);
    const float A2 = -expf(a.A_log[(int64_t)d * a.N + n]) * LOG2E;
    const float* first = REVERSE ? a.dhT : a.h0;
    float h = first ? first[((int64_t)b * a.D + d) * a.N + n] : 0.f;
    for (int k0 = 0; k0 < a.nchunk; k0 += RUN * LANES) {
        float own[RUN], decay[RUN];
        float f = 1.f, z = 0.f;   // the run as h -> f h + z
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            const int c = k0 + run * RUN + k;
            const bool in = c < a.nchunk;
            const int64_t cb = (int64_t)(REVERSE ? a.nchunk - 1 - (in ? c : 0) : (in ? c : 0)) * a.nb + b;
            const float o = a.edge[(cb * a.N + n) * a.D + d], s = a.span[cb * a.D + d];
            own[k] = in ? o : 0.f;
            decay[k] = in ? s : 0.f;
        }
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            decay[k] = exp2_hw(A2 * decay[k]);
            z = own[k] + decay[k] * z;
            f *= decay[k];
        }
#pragma unroll
        for (int off = 1; off < LANES; off <<= 1) {   // joined with all runs before it
            const float pf = __shfl_up(f, STATES * off, 64), pz = __shfl_up(z, STATES * off, 64);
            if (run >= off) {
                z = z + f * pz;
                f *= pf;
            }
        }
        float pf = 1.f, pz = 0.f;
        if constexpr (LANES > 1) {
            pf = __shfl_up(f, STATES, 64);
            pz = __shfl_up(z, STATES, 64);
        }
        float g = run ? pz + pf * h : h;
        const float lf = __shfl(f, 64 - STATES + state, 64), lz = __shfl(z, 64 - STATES + state, 64);
        h = lz + lf * h;
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
            const int c = k0 + run * RUN + k;
            if (c < a.nchunk && live) {
                const int64_t cb = (int64_t)(REVERSE ? a.nchunk - 1 - c : c) * a.nb + b;
                a.edge[(cb * a.N + n) * a.D + d] = g;
            }
            g = own[k] + decay[k] * g;
        }
    }
}

// what a chunk hands to the chunk before it if nothing enters it from behind
template <typename T, int NT>
__global__ void __launch_bounds__(256, 2) scan_backward_edge_kernel(ScanArgs a) {
    __shared__ float bc[2][GROUP][2 * NT];
    const Place p(a);
    const int end = seq_end(a, p.b);
    const int dd = p.live ? p.d : a.D - 1;
    float A2[NT], dh[NT];
    decay_rates<NT>(a, dd, 0, A2);
#pragma unroll
    for (int n = 0; n < NT; ++n) dh[n] = 0.f;
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f;
    const uint32_t lane_in = (uint32_t)dd * sizeof(T);
    float span = 0.f;
    auto fetch = [&](int t0, float (&dt)[GROUP], float (&dy)[GROUP], float (&z)[GROUP]) {
        const char* gd = group_row<T>(a.delta, a.delta_sb, a.delta_st, p.b, t0);
        const char* go = group_row<T>(a.dout, a.dout_sb, a.dout_st, p.b, t0);
        const char* gz = group_row<T>(a.z, a.z_sb, a.z_st, p.b, t0);
#pragma unroll
        for (int q = 0; q < GROUP; ++q) {
            const uint32_t r = t0 + q < end ? q * (uint32_t)sizeof(T) : 0u;
            dt[q] = at<T>(gd, lane_in + r * (uint32_t)a.delta_st);
            dy[q] = at<T>(go, lane_in + r * (uint32_t)a.dout_st);
            z[q] = at<T>(gz, lane_in + r * (uint32_t)a.z_st);
        }
    };
    const Rows<T> rb(a.B, a.B_sb, a.B_st, p.b), rc(a.C, a.C_sb, a.C_st, p.b);
    float ndt[GROUP], ndy[GROUP], nz[GROUP];
    Staged<NT> nbc;
    int ph = 0, t0 = p.t0 + (p.t1 - p.t0 - 1) / GROUP * GROUP;
    while (t0 >= p.t0 && t0 >= end) t0 -= GROUP;
    if (t0 >= p.t0) {
        fetch(t0, ndt, ndy, nz);
        fetch_bc<T, NT>(a, rb, rc, t0, end, nbc);
    }
    for (; t0 >= p.t0; t0 -= GROUP) {
        float dy[GROUP], dt[GROUP], z[GROUP];
#pragma unroll
        for (int q = 0; q < GROUP; ++q) {
            dt[q] = ndt[q];
            dy[q] = ndy[q];
            z[q] = nz[q];
        }
        put_bc<T, NT>(a, p.b, t0, end, nbc, bc[ph]);
        const int next = t0 - GROUP >= p.t0 ? t0 - GROUP : t0;   // (the first group is fetched twice)
        fetch(next, ndt, ndy, nz);
        fetch_bc<T, NT>(a, rb, rc, next, end, nbc);
        __syncthreads();
#pragma unroll
        for (int q = GROUP - 1; q >= 0; --q) {
            __builtin_amdgcn_sched_barrier(0);
            const bool in = t0 + q < end;
            const float s = in ? step_size(a, dt[q] + bias) : 0.f;
            const float g = in ? (a.dz ? dy[q] * (z[q] * sigmoid_f(z[q])) : dy[q]) : 0.f;
            span += s;
#pragma unroll
            for (int n = 0; n < NT; ++n) dh[n] = exp2_hw(s * A2[n]) * (dh[n] + g * bc[ph][q][NT + n]);
        }
        ph ^= 1;
    }
    if (!p.live) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
        if (n < a.N) a.edge[(((int64_t)p.chunk * a.nb + p.b) * a.N + n) * a.D + p.d] = dh[n];
    a.span[((int64_t)p.chunk * a.nb + p.b) * a.D + p.d] = span;
}

// Sums each of V values over lanes; afterwards lane l holds the sum of value lane_slot(l).  A step adds the halves of two values
// at once and leaves one register of the two, so V values take about 2 V instructions instead of one per value and lane bit.
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
// Four values each of two steps over the 64 / LS low lanes.  At N = 16 (LS = 4) the halving is by DPP adds that write only the banks
// (four lanes) a value stays on, which the compiler does not form from a choice and an add.  A DPP operand may be read two wait
// states after its write: the other step's adds and the s_nops keep that.
template <int LS>
__device__ __forceinline__ float lane_sums(float (&v)[4]) {
    constexpr int C1 = LS == 1 ? 2 : 4, C2 = LS <= 2 ? half_of(C1) : 4, C3 = LS <= 4 ? half_of(C2) : 4;
    constexpr int C4 = half_of(C3), C5 = half_of(C4);
    if constexpr (LS == 1) fold32<4>(v);
    if constexpr (LS <= 2) fold16<C1>(v);
    if constexpr (LS <= 4) fold_dpp<C2, 0x128, 8>(v);   // row_ror:8
    fold_dpp<C3, 0x141, 4>(v);                          // row_half_mirror
    fold_dpp<C4, 0x4E, 2>(v);                           // quad_perm 2,3,0,1
    fold_dpp<C5, 0xB1, 1>(v);                           // quad_perm 1,0,3,2
    return v[0];
}
template <int LS>
__device__ __forceinline__ void lane_sums(float (&v)[2][4], float& s0, float& s1) {
    if constexpr (LS == 4) {
        float a, b, c, d, r, s;
        asm("s_nop 1\n\t"
            "v_add_f32_dpp %0, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %1, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %2, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %3, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %0, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
            "v_add_f32_dpp %1, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
            "v_add_f32_dpp %2, %12, %12 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
            "v_add_f32_dpp %3, %13, %13 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
            "v_add_f32_dpp %4, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %4, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
            "v_add_f32_dpp %5, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %5, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
            "s_nop 0\n\t"
            "v_add_f32_dpp %0, %4, %4 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %2, %5, %5 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
            "s_nop 0\n\t"
            "v_add_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
            "v_add_f32_dpp %2, %2, %2 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf"
            : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(r), "=&v"(s)
            : "v"(v[0][0]), "v"(v[0][1]), "v"(v[0][2]), "v"(v[0][3]), "v"(v[1][0]), "v"(v[1][1]), "v"(v[1][2]), "v"(v[1][3]));
        s0 = a;
        s1 = c;
    } else {
        s0 = lane_sums<LS>(v[0]);
        s1 = lane_sums<LS>(v[1]);
    }
}
template <int LS>
__device__ __forceinline__ int lane_slot(int lane) {   // which of the four values the lane ends up with
    int s = 0, c = 4;
#pragma unroll
    for (int bit = 32 / LS; bit >= 1; bit >>= 1) {
        c >>= 1;
        if (c >= 1 && (lane & bit)) s += c;
    }
    return s;
}

// Lane part s = lane / (64 / LS) of a channel owns the steps s * GROUP / LS ...; all[q] becomes every lane's copy of step q.
template <int LS>
__device__ __forceinline__ void spread(const float (&own)[GROUP / LS], float (&all)[GROUP]) {
    constexpr int OWN = GROUP / LS;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        float v8[LS == 8 ? 2 : 1];
        if constexpr (LS == 8) {
            const float other = dpp<0x128>(own[i]);
            const bool up = threadIdx.x & 8;
            v8[0] = up ? other : own[i];
            v8[1] = up ? own[i] : other;
        } else {
            v8[0] = own[i];
        }
        constexpr int N8 = LS == 8 ? 2 : 1, N16 = LS >= 4 ? 2 : 1, N32 = LS >= 2 ? 2 : 1;
#pragma unroll
        for (int k8 = 0; k8 < N8; ++k8) {
            float v16[2] = {v8[k8], 0.f};
            if constexpr (LS >= 4) {
                const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v8[k8]), __float_as_uint(v8[k8]), false, false);
                v16[0] = __uint_as_float(r[0]);
                v16[1] = __uint_as_float(r[1]);
            }
#pragma unroll
            for (int k16 = 0; k16 < N16; ++k16) {
                float v32[2] = {v16[k16], 0.f};
                if constexpr (LS >= 2) {
                    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v16[k16]), __float_as_uint(v16[k16]), false, false);
                    v32[0] = __uint_as_float(r[0]);
                    v32[1] = __uint_as_float(r[1]);
                }
#pragma unroll
                for (int k32 = 0; k32 < N32; ++k32) all[((k32 * N16 + k16) * N8 + k8) * OWN + i] = v32[k32];
            }
        }
    }
}
// The sums over a channel's lanes, each step's at its owner; leaves them in all[0 .. GROUP / LS).  The first halving pairs steps q
// and q + GROUP / 2 (pair), as soon as both are there.
template <int LS>
__device__ __forceinline__ void pair(float (&all)[GROUP], int q) {
    if constexpr (LS >= 2) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(all[q]), __float_as_uint(all[q + GROUP / 2]), false, false);
        all[q] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}
template <int LS>
__device__ __forceinline__ void collect(float (&all)[GROUP]) {
    if constexpr (LS >= 4) fold16<GROUP / 2>(all);
    if constexpr (LS >= 8) fold_dpp<GROUP / 4, 0x128, 8>(all);
}

template <typename T, int LS>
__global__ void __launch_bounds__(256, LS >= 4 ? 3 : 2) scan_backward_kernel(ScanArgs a) {
    constexpr int S = 4, NT = S * LS, CPW = 64 / LS, OWN = GROUP / LS;
    __shared__ float bc[2][GROUP][2 * NT];
    __shared__ float part[2][4][GROUP][2 * NT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int sb = lane / CPW, n0 = sb * S, q0 = sb * OWN;
    const int part_slot = lane_slot<LS>(lane) + n0;
    const int dblk = blockIdx.x % a.ndb, rest = blockIdx.x / a.ndb;
    const int b = rest % a.nb, chunk = rest / a.nb;
    const int d = (dblk * nw + wave) * CPW + lane % CPW;
    const bool live = d < a.D;
    const int dd = live ? d : a.D - 1;
    const int lo = chunk * a.chunk, hi = lo + a.chunk < a.T ? lo + a.chunk : a.T;
    float A2[S], dh[S], dA[S];
    decay_rates<S>(a, dd, n0, A2);
#pragma unroll
    for (int j = 0; j < S; ++j) dA[j] = 0.f;
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f;
    const float skip = a.Dskip ? a.Dskip[dd] : 0.f;
    float dD = 0.f, dbias = 0.f;
    const int k0 = kept_from(a), ngroup = (a.T - k0 + GROUP - 1) / GROUP;   // groups with a kept state
    int ph = 0;
    const int end = seq_end(a, b);
#pragma unroll
    for (int j = 0; j < S; ++j) dh[j] = 0.f;
    if (live) {   // lanes behind the last channel stay 0: nothing of them may reach the sums over channels
        if (a.nchunk > 1) {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (n0 + j < a.N) dh[j] = a.edge[(((int64_t)chunk * a.nb + b) * a.N + n0 + j) * a.D + dd];
        } else if (a.dhT) {
            load_states<S>(a.dhT + ((int64_t)b * a.D + dd) * a.N + n0, a.N - n0, dh);
        }
    }
    // The group being fetched, as it lies in memory.  Steps behind the sequence read the group's first row instead and count as
    // zeros where the group is taken up, as do lanes behind the last channel.  (Not here: a choice right behind a load becomes a
    // branch round it and a wait for it, in the middle of the arithmetic that is to hide it.)
    float nu[OWN], npre[OWN], ndy[OWN], nz[OWN], nh[S];
    Staged<NT> nbc;
    const uint32_t lane_out = ((uint32_t)q0 * a.D + d) * sizeof(T);
    const uint32_t out_step = (uint32_t)a.D * sizeof(T);
    char *du_b = out_row(a.du, (int64_t)b * a.T * out_step), *dd_b = out_row(a.ddelta, (int64_t)b * a.T * out_step);
    // sums over this workgroup's channels: dB and dC themselves, or one row of both for every channel block
    const bool blocks = a.ndb > 1;
    const uint32_t sum_step = blocks ? 8u * a.N : (uint32_t)a.N * sizeof(T);
    char* sums_b = blocks ? out_row(a.dbc, ((int64_t)dblk * a.nb + b) * a.T * sum_step) : out_row(a.dB, (int64_t)b * a.T * sum_step);
    char* dc_b = out_row(a.dC, (int64_t)b * a.T * sum_step);   // (not used with channel blocks)
    char* dz_b = out_row(a.dz, (int64_t)b * a.T * out_step);
    const uint32_t lane_kept = ((uint32_t)n0 * a.D + dd) * 4u;
    const Rows<T> ru(a.u, a.u_sb, a.u_st, b), rd(a.delta, a.delta_sb, a.delta_st, b), ro(a.dout, a.dout_sb, a.dout_st, b);
    const bool gate = a.dz != nullptr;
    const Rows<T> rz(a.z, a.z_sb, a.z_st, b), rb(a.B, a.B_sb, a.B_st, b), rc(a.C, a.C_sb, a.C_st, b);
    const float* kept_b = a.kept + (int64_t)b * ngroup * NT * a.D;
    auto fetch = [&](int t0) {
        const char *gu = ru.at(t0), *gd = rd.at(t0), *go = ro.at(t0), *gz = rz.at(t0);
        uint32_t q = q0, kept = lane_kept;
        asm volatile("" : "+v"(q), "+v"(kept));   // offsets are made here: held over the group they would be spilled, and waited for
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const uint32_t r = (int)(t0 + q + i) < end ? q + i : 0u;
            nu[i] = at<T>(gu, (__umul24(r, ru.st) + dd) * (uint32_t)sizeof(T));
            npre[i] = at<T>(gd, (__umul24(r, rd.st) + dd) * (uint32_t)sizeof(T));
            ndy[i] = at<T>(go, (__umul24(r, ro.st) + dd) * (uint32_t)sizeof(T));
            nz[i] = at<T>(gz, (__umul24(r, rz.st) + dd) * (uint32_t)sizeof(T));
        }
        const char* k = (const char*)(kept_b + (int64_t)(t0 > k0 ? (t0 - k0) / GROUP : 0) * (NT * a.D));
#pragma unroll
        for (int j = 0; j < S; ++j) nh[j] = at<float>(k, kept + (uint32_t)j * (uint32_t)a.D * 4u);
    };
    int t0 = lo + (hi - lo - 1) / GROUP * GROUP;
    for (; t0 >= lo && t0 >= end; t0 -= GROUP) {   // groups behind the sequence
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            if (live && t0 + q0 + i < hi) {
                const int64_t o = ((int64_t)b * a.T + t0 + i) * a.D * (int64_t)sizeof(T);
                put<T>((char*)a.du + o, lane_out, 0.f);
                put<T>((char*)a.ddelta + o, lane_out, 0.f);
                if (a.dz) put<T>((char*)a.dz + o, lane_out, 0.f);
            }
        }
        for (int i = threadIdx.x; i < GROUP * 2 * a.N; i += blockDim.x) {
            const int q = i / (2 * a.N), r = i % (2 * a.N);
            if (t0 + q >= hi) continue;
            const int64_t bt = (int64_t)b * a.T + t0 + q;
            if (a.ndb > 1)
                a.dbc[((int64_t)dblk * a.nb * a.T + bt) * 2 * a.N + r] = 0.f;
            else if (r < a.N)
                ((T*)a.dB)[bt * a.N + r] = (T)0.f;
            else
                ((T*)a.dC)[bt * a.N + r - a.N] = (T)0.f;
        }
    }
    if (t0 >= lo) {
        fetch(t0);
        fetch_bc<T, NT>(a, rb, rc, t0, end, nbc);
        put_bc<T, NT>(a, b, t0, end, nbc, bc[ph]);
        __syncthreads();
    }
    for (; t0 >= lo; t0 -= GROUP) {
        float u[OWN], slope[OWN], gs[OWN], dts[OWN], zf[OWN];
        float dt[GROUP], x[GROUP], g[GROUP], into[GROUP], along[GROUP], y[GROUP];
        float e[GROUP][S], eh[GROUP][S];   // decay, and what it leaves of the state before the step
        const int next = t0 - GROUP >= lo ? t0 - GROUP : t0;   // (the first group is fetched twice)
        uint32_t to = lane_out;
        asm volatile("" : "+v"(to));
        const int64_t out_at = (int64_t)t0 * a.D * (int64_t)sizeof(T);
        fetch_bc<T, NT>(a, rb, rc, next, end, nbc);
        {
            float xs[OWN];
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const bool in = t0 + q0 + i < end && live;
                const float z = in ? nz[i] : 0.f, dy = in ? ndy[i] : 0.f, sg = sigmoid_f(z);
                const float pre = npre[i] + bias;
                const Softplus s = softplus_f(in ? pre : 0.f);
                u[i] = in ? nu[i] : 0.f;
                dts[i] = in ? (a.softplus ? s.value : pre) : 0.f;
                slope[i] = a.softplus ? s.slope : 1.f;
                gs[i] = gate ? dy * z * sg : dy;
                zf[i] = dy * sg * (1.f + z * (1.f - sg));
                xs[i] = dts[i] * u[i];
                dD += gs[i] * u[i];
            }
            spread<LS>(dts, dt);
            spread<LS>(xs, x);
            spread<LS>(gs, g);
        }
        // Steps are kept apart for the scheduler, which would otherwise fetch all of a group's B and C at once.
        {
            float h[S], v[2][S];
            int first_state = live ? n0 : a.N;
            asm volatile("" : "+v"(first_state));   // compared here: masks held over the loop are scalar registers spilled
#pragma unroll
            for (int j = 0; j < S; ++j) h[j] = first_state + j < a.N && t0 >= k0 ? nh[j] : 0.f;
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                __builtin_amdgcn_sched_barrier(0);
                y[q] = 0.f;
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    e[q][j] = exp2_hw(dt[q] * A2[j]);
                    eh[q][j] = e[q][j] * h[j];
                    h[j] = eh[q][j] + x[q] * bc[ph][q][n0 + j];
                    y[q] += bc[ph][q][NT + n0 + j] * h[j];
                    v[q & 1][j] = g[q] * h[j];
                }
                if (q & 1) lane_sums<LS>(v, part[ph][wave][q - 1][NT + part_slot], part[ph][wave][q][NT + part_slot]);
                if (q >= GROUP / 2) pair<LS>(y, q - GROUP / 2);   // lanes that hold the same sum write it to the same place
            }
        }
        collect<LS>(y);
        if (gate) {
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const int t = t0 + q0 + i;
                if (live && t < hi) put<T>(out_row(dz_b, out_at), to + i * out_step, t < end ? zf[i] * (y[i] + skip * u[i]) : 0.f);
            }
        }
        float v[2][S];
        asm volatile("" ::: "memory");   // B and C are read from LDS again rather than held for all steps
#pragma unroll
        for (int q = GROUP - 1; q >= 0; --q) {
            __builtin_amdgcn_sched_barrier(0);
            // half of the group's registers are free again: the next group's operands come in behind the other half
            if (q == GROUP / 2 - 1) fetch(next);
            into[q] = along[q] = 0.f;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                dh[j] += g[q] * bc[ph][q][NT + n0 + j];
                v[q & 1][j] = dh[j] * x[q];
                into[q] += dh[j] * bc[ph][q][n0 + j];
                const float t = dh[j] * eh[q][j];
                along[q] += t * A2[j];
                dA[j] += t * dt[q];
                dh[j] *= e[q][j];
                asm volatile("" : "+v"(dA[j]));   // summed here, not behind the group with eight steps' t held until then
            }
            if (!(q & 1)) lane_sums<LS>(v, part[ph][wave][q][part_slot], part[ph][wave][q + 1][part_slot]);
            if (q < GROUP / 2) {
                pair<LS>(into, q);
                pair<LS>(along, q);
            }
        }
        // Wait for the next group's operands here, before this group's stores: a wait behind them would be one for them as well.
#pragma unroll
        for (int i = 0; i < OWN; ++i) asm volatile("" : "+v"(nu[i]), "+v"(npre[i]), "+v"(ndy[i]), "+v"(nz[i]));
#pragma unroll
        for (int j = 0; j < S; ++j) asm volatile("" : "+v"(nh[j]));
        put_bc<T, NT>(a, b, next, end, nbc, bc[ph ^ 1]);
        collect<LS>(into);
        collect<LS>(along);
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const int t = t0 + q0 + i;
            const bool in = t < end;
            const float dpre = (into[i] * u[i] + along[i] * LN2) * slope[i];
            if (in) dbias += dpre;
            if (live && t < hi) {
                put<T>(out_row(du_b, out_at), to + i * out_step, in ? into[i] * dts[i] + skip * gs[i] : 0.f);
                put<T>(out_row(dd_b, out_at), to + i * out_step, in ? dpre : 0.f);
            }
        }
        __syncthreads();   // the group's sums are written, the next group's B and C staged
        char* sums = out_row(sums_b, (int64_t)t0 * sum_step);
        char* sums_c = blocks ? sums : out_row(dc_b, (int64_t)t0 * sum_step);
        for (int i = threadIdx.x; i < GROUP * 2 * NT; i += blockDim.x) {
            const int q = i / (2 * NT), r = i % (2 * NT), n = r % NT;
            if (n >= a.N || t0 + q >= hi) continue;
            float s = 0.f;
            if (t0 + q < end)
                for (int w = 0; w < nw; ++w) s += part[ph][w][q][r];
            const uint32_t row = __umul24(q, sum_step);
            if (blocks)
                put<float>(sums, row + (r < NT ? n : a.N + n) * 4u, s);
            else
                put<T>(r < NT ? sums : sums_c, row + n * (uint32_t)sizeof(T), s);
        }
        ph ^= 1;
    }
    if (a.dh0 && chunk == 0 && live) store_states<S>(a.dh0 + ((int64_t)b * a.D + d) * a.N + n0, a.N - n0, dh);
    // dD and dbias are spread over the channel's lanes by step
#pragma unroll
    for (int off = CPW; off < 64; off <<= 1) {
        dD += __shfl_xor(dD, off, 64);
        dbias += __shfl_xor(dbias, off, 64);
    }
    if (!live) return;
    const int64_t at = ((int64_t)b * a.nchunk + chunk) * a.par_stride;
    if (a.dA && n0 < a.N) {
        float* o = a.dA + at + (int64_t)d * a.N + n0;
        float old[S];
#pragma unroll
        for (int j = 0; j < S; ++j) old[j] = 0.f;
        if (a.accumulate) load_states<S>(o, a.N - n0, old);
#pragma unroll
        for (int j = 0; j < S; ++j) dA[j] = old[j] + a.scale * (A2[j] * LN2) * dA[j];
        store_states<S>(o, a.N - n0, dA);
    }
    if (sb > 0) return;
    if (a.dD) a.dD[at + d] = (a.accumulate ? a.dD[at + d] : 0.f) + a.scale * dD;
    if (a.dbias) a.dbias[at + d] = (a.accumulate ? a.dbias[at + d] : 0.f) + a.scale * dbias;
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
        if (a.gate) {
            const float z = elem<T>(a.z, a.z_sb, 0, b, 0, d);
            y *= z * sigmoid_f(z);
        }
        ((T*)a.out)[ch] = (T)y;
    }
}

int block_of(int D) { return D > 192 ? 256 : (D + 63) / 64 * 64; }
// backward: lanes a channel's states lie on, threads of a workgroup, workgroups a row of channels needs
int lanes_of(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8; }
int back_block_of(int D, int N) { return block_of(D > 1024 ? 1024 : D * lanes_of(N)); }
// lanes that share a state where chunks are joined
int join_lanes(int nchunk) { return nchunk <= JOIN_RUN ? 1 : nchunk <= 2 * JOIN_RUN ? 2 : nchunk <= 4 * JOIN_RUN ? 4 : 8; }
int back_blocks_of(int D, int N) {
    const int per = back_block_of(D, N) / lanes_of(N);
    return (D + per - 1) / per;
}

int check(const dpk_scan_desc* s) {
    if (!s || s->B < 0 || s->T < 0 || s->D <= 0 || s->N <= 0) return DPK_EINVAL;
    if (s->N > DPK_SCAN_MAX_STATE || s->T > MAX_DIM) return DPK_ERANGE;
    if (s->dtype != DPK_F32 && s->dtype != DPK_BF16 && s->dtype != DPK_F16) return DPK_EINVAL;
    if (s->nchunk <= 0 || s->chunk < 0 || s->chunk % GROUP || (int64_t)s->nchunk * s->chunk < s->T) return DPK_EINVAL;
    if (s->u_sb < 0 || s->u_st < 0 || s->delta_sb < 0 || s->delta_st < 0 || s->B_sb < 0 || s->B_st < 0 || s->C_sb < 0 ||
        s->C_st < 0 || s->z_sb < 0 || s->z_st < 0)
        return DPK_EINVAL;
    // a lane's byte offset within a group of rows is 32 bits, a product with a row's distance takes 24 of it (at the full rate)
    const int64_t row_limit = (int64_t)1 << 24;
    if (s->D >= row_limit || (int64_t)s->D * s->N >= (int64_t)1 << 29 || s->u_st >= row_limit || s->delta_st >= row_limit ||
        s->z_st >= row_limit || s->B_st >= row_limit || s->C_st >= row_limit)
        return DPK_ERANGE;
    if (!s->A_log || (s->T > 0 && (!s->u || !s->delta || !s->Bm || !s->Cm))) return DPK_EINVAL;
    return DPK_OK;
}

// whether every launch of a direction can be made (looked at before the first one)
bool launches(const dpk_scan_desc* s, bool backward) {
    const int64_t runs = (int64_t)s->B * s->nchunk;
    const int bl = block_of(s->D), back = back_block_of(s->D, s->N), per = 256 / join_lanes(s->nchunk);
    const int64_t states = (int64_t)s->B * s->N * s->D;
    if (runs > 0x7fffffffLL) return false;
    if ((!backward || s->nchunk > 1) && !dpk_launchable(runs * ((s->D + bl - 1) / bl), bl)) return false;
    if (s->nchunk > 1 && !dpk_launchable((states + per - 1) / per, 256)) return false;
    if (!backward) return true;
    const int blocks = back_blocks_of(s->D, s->N);
    return dpk_launchable(runs * blocks, back) && (blocks == 1 || dpk_launchable(((int64_t)s->B * s->T * 2 * s->N + 255) / 256, 256));
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
    a.gate = s->z != nullptr;
    if (!a.gate) { a.z = a.u; a.z_sb = a.u_sb; a.z_st = a.u_st; }
    a.kept = s->kept; a.edge = s->edge; a.span = s->span;
    return a;
}

template <bool REVERSE>
void join(const ScanArgs& a, hipStream_t st) {
    const int64_t states = (int64_t)a.nb * a.N * a.D;
#define CALL(LANES)                                                                                                             \
    hipLaunchKernelGGL((scan_join_kernel<REVERSE, LANES>), dim3((unsigned)((states + 256 / LANES - 1) / (256 / LANES))), dim3(256), \
                       0, st, a)
    switch (join_lanes(a.nchunk)) {
        case 1: CALL(1); break;
        case 2: CALL(2); break;
        case 4: CALL(4); break;
        default: CALL(8); break;
    }
#undef CALL
}

}  // namespace

#define SCAN_N(N, CALL)           \
    if (N <= 4) { CALL(4) }       \
    else if (N <= 8) { CALL(8) }  \
    else if (N <= 16) { CALL(16) } \
    else { CALL(32) }

// Chunks of time a scan is cut into.  Cutting costs a second reading of the inputs and most of the arithmetic again, so it has to
// win a factor of two or three in waves.  Times of whole calls at N = 16, bf16 where no type is named.  Forward into up to 4096 waves
// (four a SIMD; 1 x 8192 x 1024: 87 us, 86 with 2048, 3520 in one piece) of chunks as short as 32 steps (2 x 4096 x 500: 53 us, 65
// with 64), from fewer than 800 (10 x 2000 x 4096, 640 waves: 606 us, 919 in one piece; 16 x 1000 x 4096, 1024 waves: 467 in one
// piece, 457 in four), of short sequences fewer than 512 (50 x 256 x 1024 fp32, 800 waves: 120 in one piece, 127 in five).
// Backward into up to 2048 of at least 64 steps (1 x 8192 x 1024: 203 us, 213 with 32; 2 x 4096 x 500: 131, 120 with 32) from
// fewer than 512 (8 x 1000 x 4096: 783 us in one piece, 756 in four).  The backward numbers are those of N from 9 to 16, whose waves
// hold 16 channels; the rule does not go by N, and is off where they hold 64 (N = 4, 8 x 2000 x 4096: 1556 us in one piece, as it says,
// 657 in four) or 8 (N = 32, 4 x 2000 x 4096: 1994 us in eight, as it says, 1299 in one).
extern "C" int dpk_selective_scan_chunks(int B, int T, int D, int backward, int* chunk) {
    if (B <= 0 || T <= 0 || D <= 0) {
        if (chunk) *chunk = (T > 0 ? (T + GROUP - 1) / GROUP * GROUP : 0);
        return 1;
    }
    const int64_t waves = (int64_t)B * ((D + 63) / 64);
    int64_t n = waves >= (backward || T < 512 ? 512 : 800) ? 1 : (backward ? 2048 : 4096) / waves;
    const int shortest = backward ? 64 : 32;
    const int64_t most = (T + shortest - 1) / shortest;
    if (n > most) n = most;
    if (n < 3) n = 1;
    int64_t len = (T + n - 1) / n;
    len = (len + GROUP - 1) / GROUP * GROUP;
    n = (T + len - 1) / len;
    if (chunk) *chunk = (int)len;
    return (int)n;
}

extern "C" int dpk_selective_scan_group(void) { return GROUP; }
extern "C" int dpk_selective_scan_state_rows(int N) { return N <= 0 || N > DPK_SCAN_MAX_STATE ? 0 : 4 * lanes_of(N); }
extern "C" int dpk_selective_scan_channel_blocks(int D, int N) {
    return D <= 0 || N <= 0 || N > DPK_SCAN_MAX_STATE ? 0 : back_blocks_of(D, N);
}

extern "C" int dpk_selective_scan_forward(const dpk_scan_desc* s, void* out, float* hT, void* stream) {
    const int rc = check(s);
    if (rc) return rc;
    if (s->B == 0) return DPK_OK;
    if (s->T > 0 && !out) return DPK_EINVAL;
    if (s->nchunk > 1 && (!s->edge || !s->span)) return DPK_EINVAL;
    if (!launches(s, false)) return DPK_ERANGE;
    ScanArgs a = fill(s);
    a.out = out; a.hT = hT;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(a.nb * a.nchunk * a.ndb)), block((unsigned)block_of(a.D));
    if (a.nchunk > 1) {
#define CALL(NT) hipLaunchKernelGGL((scan_forward_kernel<E, NT, true>), grid, block, 0, st, a);
        DPK_DISPATCH_DTYPE(s->dtype, E, SCAN_N(a.N, CALL))
#undef CALL
        join<false>(a, st);
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
    if (g->dout_st >= (int64_t)1 << 24) return DPK_ERANGE;
    if (s->B == 0) return DPK_OK;
    if (s->T > 0 && (!g->dout || !g->du || !g->ddelta || !g->dB || !g->dC || !s->kept || (s->z && !g->dz))) return DPK_EINVAL;
    if (s->nchunk > 1 && (!s->edge || !s->span)) return DPK_EINVAL;
    if ((g->dA || g->dD || g->dbias) && g->par_stride < s->D) return DPK_EINVAL;
    if (!launches(s, true)) return DPK_ERANGE;
    ScanArgs a = fill(s);
    const int blocks = back_blocks_of(s->D, s->N);
    if (blocks > 1 && s->T > 0 && !g->dbc) return DPK_EINVAL;
    a.dout = g->dout; a.dhT = g->dhT; a.du = g->du; a.ddelta = g->ddelta; a.dB = g->dB; a.dC = g->dC; a.dz = s->z ? g->dz : nullptr;
    a.dh0 = g->dh0; a.dbc = g->dbc; a.dA = g->dA; a.dD = g->dD; a.dbias = g->dbias; a.par_stride = g->par_stride;
    a.dout_sb = g->dout_sb; a.dout_st = g->dout_st; a.scale = g->scale; a.accumulate = g->accumulate;
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(a.nb * a.nchunk * a.ndb)), block((unsigned)block_of(a.D));
    const int64_t sums = (int64_t)a.nb * a.T * 2 * a.N;
    if (a.nchunk > 1) {
#define CALL(NT) hipLaunchKernelGGL((scan_backward_edge_kernel<E, NT>), grid, block, 0, st, a);
        DPK_DISPATCH_DTYPE(s->dtype, E, SCAN_N(a.N, CALL))
#undef CALL
        join<true>(a, st);
    }
    a.ndb = blocks;
    const dim3 bgrid((unsigned)(a.nb * a.nchunk * a.ndb)), bblock((unsigned)back_block_of(a.D, a.N));
#define CALL(NT) hipLaunchKernelGGL((scan_backward_kernel<E, NT / 4>), bgrid, bblock, 0, st, a);
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
    if (!dpk_launchable(grid, 256)) return DPK_ERANGE;
#define CALL(L) hipLaunchKernelGGL((scan_step_kernel<E, L>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    DPK_DISPATCH_DTYPE(s->dtype, E, if (lanes == 1) { CALL(1) } else if (lanes == 2) { CALL(2) } else if (lanes == 4) { CALL(4) } else { CALL(8) })
#undef CALL
    return dpk_launch_status();
}
