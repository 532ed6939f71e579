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

// ---- chunks ------------------------------------------------------------------
// C tokens at a time, on the fp32 matrix cores.  With G_i the sum of a chunk's decays
// up to token i (base 2, in 64 bits), S the state before it and P_ij = q_i k_j:
//   o_i = scale (2^G_i q_i S + sum_(j <= i) 2^(G_i - G_j) b_j P_ij v_j)
//   S  <- 2^G_C S + sum_j 2^(G_C - G_j) b_j k_j v_j^T
// Exponents are differences of tokens in order, so no factor overflows before the
// formula does.  A group of 4 waves takes a head's 64 CB columns of V, a wave 16 CB of
// them, in its lanes' order: lane 16 g + c holds column CB c + j of its wave in
// register j, and the accumulators' rows 4 g + r.  So S's accumulators are the second
// operand of q S as they are, P's (formed as K Q^T) the first of P V, and V never
// leaves its registers.  K and Q are in LDS; each wave forms P over its share of the
// key's dimensions, and the shares meet in LDS.
constexpr int C = 32;

struct Decays {
    double G[C];
    float q[C];  // 2^G_i scale
    float k[C];  // 2^(G_C - G_j) b_j
    float b[C];  // b_j scale
    float all;   // 2^G_C
};

// 2^x for x <= 0 (or the formula's overflow), relative error 2^-23: the part of x that
// fp32 leaves out counts, too
__device__ __forceinline__ float exp2_of(double x)
{
    const float hi = (float)x, lo = (float)(x - (double)hi);
    const float e = __builtin_amdgcn_exp2f(hi);
    return hi == lo ? e : fmaf(e, lo * 0.693147181f, e);
}

// Token i's decay of a chunk in base 2: 0 behind its n tokens.  Where 2^x is 0 a
// smaller x changes nothing but the sums' digits.
__device__ __forceinline__ double decay2(const ornk_linear_args &a, size_t t, int h, bool on)
{
    if (!on) return 0.0;
    const double x = (double)a.decay[a.per_token ? t * a.heads + h : h] * 1.4426950408889634;
    return x < -16384.0 ? -16384.0 : x;
}

// One wave, lanes i and i + 32 alike: the chunk's sums and factors.
__device__ __forceinline__ double fill_decays(const ornk_linear_args &a, Decays &d, double x, bool on)
{
    const int i = threadIdx.x & (C - 1);
    double G = x;
#pragma unroll
    for (int o = 1; o < C; o <<= 1) {
        const double y = __shfl_up(G, o, C);
        if (i >= o) G += y;
    }
    const double end = __shfl(G, C - 1, C);
    const float b = !on ? 0.0f : a.complement ? -expm1f((float)(x * 0.6931471805599453)) : 1.0f;
    d.G[i] = G;
    d.q[i] = exp2_of(G) * a.scale;
    d.k[i] = exp2_of(end - G) * b;
    d.b[i] = b * a.scale;
    if (!i) d.all = exp2_of(end);
    return end;
}

#define MFMA4(A, B, C) __builtin_amdgcn_mfma_f32_16x16x4f32(A, B, C, 0, 0, 0)

struct Cut {
    int segs, len;     // parts of a sequence that are done side by side, and their tokens
    float *states;     // [n_seqs][heads][segs][dk][dv]: what a part adds, then what it begins with
    float *decays;     // [n_seqs][heads][segs]: what a part leaves of a state
};

// SUMS: only what a part adds to a state that begins with zeros.
template <int KB, int CB, bool VEC, bool SUMS>
__global__ void __launch_bounds__(256, 2) k_linear_chunks(ornk_linear_args a, Cut cut)
{
    constexpr int LD = 16 * KB + 4;          // floats of a row in LDS
    constexpr int NL = C * 4 * KB / 256 > 0 ? C * 4 * KB / 256 : 1;  // float4s of a chunk per thread
    __shared__ __align__(16) float Ks[C][LD];
    __shared__ __align__(16) float Qs[SUMS ? 1 : C][LD];
    __shared__ __align__(16) v4f part[SUMS ? 1 : 4][3][64];
    __shared__ Decays dec[2];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const int b = blockIdx.x, h = blockIdx.y;
    const int blocks = (a.dv + 64 * CB - 1) / (64 * CB);
    const int sg = blockIdx.z / blocks, col0 = (blockIdx.z - sg * blocks) * 64 * CB + w * 16 * CB + c * CB;
    const Seq seq = seq_of(a, b);
    const int first = sg * cut.len;
    if (seq.n < 0 || (sg && first >= seq.n)) return;
    if (SUMS && first + cut.len >= seq.n) return;  // nothing begins behind it
    const int last = min(seq.n, first + cut.len);
    const int hq = h / (a.heads / a.qh), hk = h / (a.heads / a.kh), hv = h / (a.heads / a.vh);
    const bool busy = col0 - c * CB < a.dv;  // the wave has columns
    const size_t size = (size_t)a.dk * a.dv;
    float *const mine = cut.segs > 1 ? cut.states + (((size_t)b * a.heads + h) * cut.segs + sg) * size : nullptr;

    v4f S[KB][CB];
    {
        const float *from = SUMS ? nullptr : cut.segs > 1 ? mine
                            : seq.in >= 0 ? a.S + ((size_t)seq.in * a.heads + h) * size : nullptr;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * kb + 4 * g + r;
#pragma unroll
                for (int j = 0; j < CB; ++j)
                    S[kb][j][r] = from && row < a.dk && col0 + j < a.dv ? from[(size_t)row * a.dv + col0 + j] : 0.0f;
            }
    }

    v4f kn[NL], qn[SUMS ? 1 : NL];  // the next chunk's rows of K and Q on their way
    float vn[2][4][CB];
    double xn = 0.0;
    bool on_n = false;
    auto fetch = [&](int t) {  // the chunk from token t of the sequence on
        const size_t row0 = (size_t)seq.t0 + t;
        const int n = last - t;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int at = tid + 256 * i, row = at / (4 * KB), col = 4 * (at - row * 4 * KB);
            v4f x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            if (row < C && row < n) {
                const float *kp = a.k + ((row0 + row) * a.kh + hk) * a.dk + col;
                const float *qp = a.q + ((row0 + row) * a.qh + hq) * a.dk + col;
                if (VEC) {
                    if (col < a.dk) {
                        x = *reinterpret_cast<const v4f *>(kp);
                        if (!SUMS) y = *reinterpret_cast<const v4f *>(qp);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < a.dk) {
                            x[e] = kp[e];
                            if (!SUMS) y[e] = qp[e];
                        }
                }
            }
            kn[i] = x;
            if (!SUMS) qn[i] = y;
        }
        if (busy) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * tb + 4 * g + r;
                    const float *vp = a.v + ((row0 + row) * a.vh + hv) * a.dv + col0;
#pragma unroll
                    for (int j = 0; j < CB; ++j) vn[tb][r][j] = row < n && col0 + j < a.dv ? vp[j] : 0.0f;
                }
        }
        if (w == 3) {
            const int i = lane & (C - 1);
            on_n = i < n;
            xn = decay2(a, row0 + i, h, on_n);
        }
    };
    double left = 0.0;  // wave 3: the part's decays
    auto stage = [&](int p) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int at = tid + 256 * i, row = at / (4 * KB), col = 4 * (at - row * 4 * KB);
            if (row < C) {
                *reinterpret_cast<v4f *>(&Ks[row][col]) = kn[i];
                if (!SUMS) *reinterpret_cast<v4f *>(&Qs[row][col]) = qn[i];
            }
        }
    };

    int p = 0;
    if (first < last) {
        fetch(first);
        if (w == 3) left += fill_decays(a, dec[0], xn, on_n);
        stage(0);
    }
    for (int t = first; t < last; t += C, p ^= 1) {
        __syncthreads();
        float v[2][4][CB];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < CB; ++j) v[tb][r][j] = vn[tb][r][j];
        if (t + C < last) fetch(t + C);
        const Decays &d = dec[p];
        if (!SUMS) {
            // P over this wave's dimensions: keys jb x queries ib
            v4f P[3] = {};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                if ((kb & 3) != w) continue;
                const int at = 16 * kb + 4 * g;
                const v4f k0 = *reinterpret_cast<const v4f *>(&Ks[c][at]);
                const v4f k1 = *reinterpret_cast<const v4f *>(&Ks[16 + c][at]);
                const v4f q0 = *reinterpret_cast<const v4f *>(&Qs[c][at]);
                const v4f q1 = *reinterpret_cast<const v4f *>(&Qs[16 + c][at]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    P[0] = MFMA4(k0[r], q0[r], P[0]);
                    P[1] = MFMA4(k0[r], q1[r], P[1]);
                    P[2] = MFMA4(k1[r], q1[r], P[2]);
                }
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) part[w][i][lane] = P[i];
            // q S
            v4f O[2][CB] = {};
            if (busy) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const int at = 16 * kb + 4 * g;
                    const v4f q0 = *reinterpret_cast<const v4f *>(&Qs[c][at]);
                    const v4f q1 = *reinterpret_cast<const v4f *>(&Qs[16 + c][at]);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < CB; ++j) {
                            O[0][j] = MFMA4(q0[r], S[kb][j][r], O[0][j]);
                            O[1][j] = MFMA4(q1[r], S[kb][j][r], O[1][j]);
                        }
                }
#pragma unroll
                for (int ib = 0; ib < 2; ++ib) {
                    const v4f f = *reinterpret_cast<const v4f *>(&d.q[16 * ib + 4 * g]);
#pragma unroll
                    for (int j = 0; j < CB; ++j) O[ib][j] *= f;
                }
            }
            __syncthreads();
            if (busy) {
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    const int ib = i > 0, jb = i > 1;
                    P[i] = (part[0][i][lane] + part[1][i][lane]) + (part[2][i][lane] + part[3][i][lane]);
                    const double Gi = d.G[16 * ib + c];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = 4 * g + r;
                        const float f = exp2_of(Gi - d.G[16 * jb + j]) * d.b[16 * jb + j];
                        P[i][r] = ib != jb || c >= j ? P[i][r] * f : 0.0f;
                    }
                }
                // A value that is not finite would reach tokens before it, as 0 times itself:
                // those of a diagonal block are added one by one.
                float z = 0.0f;
#pragma unroll
                for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < CB; ++j) z = fmaf(v[tb][r][j], 0.0f, z);
                if (!__any(z != z)) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < CB; ++j) {
                            O[0][j] = MFMA4(P[0][r], v[0][r][j], O[0][j]);
                            O[1][j] = MFMA4(P[1][r], v[0][r][j], O[1][j]);
                            O[1][j] = MFMA4(P[2][r], v[1][r][j], O[1][j]);
                        }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < CB; ++j) O[1][j] = MFMA4(P[1][r], v[0][r][j], O[1][j]);
                    for (int key = 0; key < 16; ++key) {
                        const int at = 16 * (key >> 2), kr = key & 3;
#pragma unroll
                        for (int ib = 0; ib < 2; ++ib) {
                            const v4f pk = P[2 * ib];
                            const float ps = kr == 0 ? pk[0] : kr == 1 ? pk[1] : kr == 2 ? pk[2] : pk[3];
                            float vs[CB];
#pragma unroll
                            for (int j = 0; j < CB; ++j) {
                                const float x = kr == 0 ? v[ib][0][j] : kr == 1 ? v[ib][1][j]
                                                : kr == 2 ? v[ib][2][j] : v[ib][3][j];
                                vs[j] = __shfl(x, at + c, 64);
                            }
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float pr = __shfl(ps, at + 4 * g + r, 64);
#pragma unroll
                                for (int j = 0; j < CB; ++j)
                                    if (4 * g + r >= key) O[ib][j][r] = fmaf(pr, vs[j], O[ib][j][r]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int ib = 0; ib < 2; ++ib)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = 16 * ib + 4 * g + r;
                        if (t + row >= last) continue;
                        float *op = a.out + (((size_t)seq.t0 + t + row) * a.heads + h) * a.dv + col0;
#pragma unroll
                        for (int j = 0; j < CB; ++j)
                            if (col0 + j < a.dv) op[j] = O[ib][j][r];
                    }
            }
        }
        if (busy) {
            const float all = d.all;
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                const v4f f = *reinterpret_cast<const v4f *>(&d.k[16 * tb + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < CB; ++j) v[tb][r][j] *= f[r];
            }
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                for (int j = 0; j < CB; ++j) S[kb][j] *= all;
#pragma unroll
                for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float k = Ks[16 * tb + 4 * g + r][16 * kb + c];
#pragma unroll
                        for (int j = 0; j < CB; ++j) S[kb][j] = MFMA4(k, v[tb][r][j], S[kb][j]);
                    }
            }
        }
        if (t + C < last) {
            if (w == 3) left += fill_decays(a, dec[p ^ 1], xn, on_n);
            __syncthreads();
            stage(p ^ 1);
        }
    }

    float *to = nullptr;
    if (SUMS) {
        to = mine;
        if (tid == 192 && blockIdx.z == sg * blocks)
            cut.decays[((size_t)b * a.heads + h) * cut.segs + sg] = exp2_of(left);
    } else if (last == seq.n && seq.out >= 0) {
        to = a.S + ((size_t)seq.out * a.heads + h) * size;
    }
    if (!to || !busy) return;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * kb + 4 * g + r;
#pragma unroll
            for (int j = 0; j < CB; ++j)
                if (row < a.dk && col0 + j < a.dv) to[(size_t)row * a.dv + col0 + j] = S[kb][j][r];
        }
}

// From what each part adds to what each part begins with, an element per thread.
__global__ void __launch_bounds__(256) k_linear_join(ornk_linear_args a, Cut cut)
{
    const int b = blockIdx.x, h = blockIdx.y, e = blockIdx.z * 256 + threadIdx.x;
    const Seq seq = seq_of(a, b);
    const int size = a.dk * a.dv;
    if (seq.n < 0 || e >= size) return;
    const size_t at = ((size_t)b * a.heads + h) * cut.segs;
    float s = seq.in >= 0 ? a.S[((size_t)seq.in * a.heads + h) * size + e] : 0.0f;
    for (int i = 0; i == 0 || i * cut.len < seq.n; ++i) {
        float *p = cut.states + (at + i) * size + e;
        const bool more = (i + 1) * cut.len < seq.n;
        const float add = more ? *p : 0.0f, keep = more ? cut.decays[at + i] : 0.0f;
        *p = s;
        s = fmaf(keep, s, add);
    }
}

// Sequences are cut where their heads and columns leave CUs idle: into parts of at
// least 256 tokens, until there are two groups for each CU.
Cut cut_of(const ornk_linear_args &a, int cb)
{
    const long long groups = (long long)a.n_seqs * a.heads * ((a.dv + 64 * cb - 1) / (64 * cb));
    long long segs = 512 / groups;
    if (segs > a.max_len / 256) segs = a.max_len / 256;
    Cut c = {1, a.max_len, nullptr, nullptr};
    if (segs < 2) return c;
    c.len = (int)(((a.max_len + segs - 1) / segs + C - 1) / C * C);
    c.segs = (a.max_len - 1) / c.len + 1;
    return c;
}

int columns(const ornk_linear_args &a) { return a.dv > 64 && a.dk <= 128 ? 2 : 1; }

template <int KB, int CB, bool VEC>
void launch(const ornk_linear_args &a, const Cut &cut, hipStream_t s)
{
    const int blocks = (a.dv + 64 * CB - 1) / (64 * CB);
    const dim3 grid(a.n_seqs, a.heads, cut.segs * blocks);
    if (cut.segs > 1) {
        hipLaunchKernelGGL((k_linear_chunks<KB, CB, VEC, true>), grid, dim3(256), 0, s, a, cut);
        hipLaunchKernelGGL(k_linear_join, dim3(a.n_seqs, a.heads, (a.dk * a.dv + 255) / 256), dim3(256), 0, s,
                           a, cut);
    }
    hipLaunchKernelGGL((k_linear_chunks<KB, CB, VEC, false>), grid, dim3(256), 0, s, a, cut);
}

template <int KB, int CB>
void launch(const ornk_linear_args &a, const Cut &cut, hipStream_t s)
{
    if (a.dk % 4) launch<KB, CB, false>(a, cut, s);
    else launch<KB, CB, true>(a, cut, s);
}

}  // namespace

extern "C" size_t ornk_linear_ws(const ornk_linear_args *a)
{
    const Cut c = cut_of(*a, columns(*a));
    return c.segs < 2 ? 0 : sizeof(float) * a->n_seqs * a->heads * c.segs * ((size_t)a->dk * a->dv + 1);
}

extern "C" int ornk_linear(const ornk_linear_args *a, hipStream_t s)
{
    if (a->max_len <= 1) {
        hipLaunchKernelGGL(k_linear_steps, dim3(a->n_seqs, a->heads, (a->dv + 63) / 64), dim3(256), 0, s, *a);
        return hipGetLastError();
    }
    const int cb = columns(*a);
    Cut c = cut_of(*a, cb);
    c.states = static_cast<float *>(a->ws);
    if (c.segs > 1) c.decays = c.states + (size_t)a->n_seqs * a->heads * c.segs * a->dk * a->dv;
    if (a->dk > 128) launch<16, 1>(*a, c, s);
    else if (cb == 2) a->dk > 64 ? launch<8, 2>(*a, c, s) : launch<4, 2>(*a, c, s);
    else a->dk > 64 ? launch<8, 1>(*a, c, s) : launch<4, 1>(*a, c, s);
    return hipGetLastError();
}
