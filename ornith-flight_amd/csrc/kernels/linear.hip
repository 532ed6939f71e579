// SPDX-License-Identifier: MIT
//
// Linear attention with a decay for each head (ornith_hip.h).
#include "common.h"
#include "launch.h"

namespace {

__device__ __forceinline__ void report(const ornk_linear_args &a, int what, int b)
{
    *(volatile int *)(a.err + what) = 1 + b;
}

// Sequence b: its first token, their number (-1: left out), and where its state
// comes from and goes to (-1: zeros, nowhere).
struct Seq {
    int t0, n, in, out;
};

__device__ __forceinline__ Seq seq_of(const ornk_linear_args &a, int b)
{
    Seq s = {b, 1, -1, -1};
    if (a.starts) {
        s.t0 = a.starts[b];
        const int t1 = a.starts[b + 1];
        s.n = t1 - s.t0;
        if (s.t0 < 0 || t1 < s.t0 || t1 > a.n_tokens || s.n > a.max_len) {
            report(a, ORNK_KV_ERR_START, b);
            s.n = -1;
        }
    }
    if (a.in) s.in = a.in[b];
    if (a.out_slots) s.out = a.out_slots[b];
    if (s.in < -1 || s.in >= a.n_slots || s.out < -1 || s.out >= a.n_slots) {
        report(a, ORNK_KV_ERR_STATE, b);
        s.n = -1;
    }
    return s;
}

// Token by token: a group of 4 waves holds 64 columns of a head's state, a wave a
// quarter of its rows.
__global__ void __launch_bounds__(256) k_linear_steps(ornk_linear_args a)
{
    __shared__ float q[256], k[256], part[4][64];
    const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int w = tid >> 6, col = blockIdx.z * 64 + (tid & 63);
    const Seq seq = seq_of(a, b);
    if (seq.n < 0) return;
    const bool on = col < a.dv;
    const int hq = h / (a.heads / a.qh), hk = h / (a.heads / a.kh), hv = h / (a.heads / a.vh);
    const size_t size = (size_t)a.dk * a.dv;
    float s[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const int r = 4 * i + w;
        s[i] = on && r < a.dk && seq.in >= 0
                   ? a.S[((size_t)seq.in * a.heads + h) * size + (size_t)r * a.dv + col]
                   : 0.0f;
    }
    for (int j = 0; j < seq.n; ++j) {
        const size_t t = (size_t)seq.t0 + j;
        __syncthreads();
        if (tid < a.dk) {
            q[tid] = a.q[(t * a.qh + hq) * a.dk + tid] * a.scale;
            k[tid] = a.k[(t * a.kh + hk) * a.dk + tid];
        }
        __syncthreads();
        const float g = a.decay[a.per_token ? t * a.heads + h : h];
        const float f = expf(g);
        float v = on ? a.v[(t * a.vh + hv) * a.dv + col] : 0.0f, o = 0.0f;
        if (a.complement) v *= -expm1f(g);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
            const int r = 4 * i + w;
            if (r < a.dk) {
                s[i] = fmaf(k[r], v, f * s[i]);
                o = fmaf(q[r], s[i], o);
            }
        }
        part[w][tid & 63] = o;
        __syncthreads();
        if (w == 0 && on)
            a.out[(t * a.heads + h) * a.dv + col] = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    }
    if (seq.out < 0 || !on) return;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const int r = 4 * i + w;
        if (r < a.dk) a.S[((size_t)seq.out * a.heads + h) * size + (size_t)r * a.dv + col] = s[i];
    }
}

}  // namespace

extern "C" size_t ornk_linear_ws(const ornk_linear_args *a) { return 0; }

extern "C" int ornk_linear(const ornk_linear_args *a, hipStream_t s)
{
    hipLaunchKernelGGL(k_linear_steps, dim3(a->n_seqs, a->heads, (a->dv + 63) / 64), dim3(256), 0, s, *a);
    return hipGetLastError();
}
