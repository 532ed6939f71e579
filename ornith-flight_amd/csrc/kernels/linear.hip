// SPDX-License-Identifier: MIT
//
// Linear attention with a decay for each head (ornith_hip.h).
#include <type_traits>

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

// 2^x for x <= 0 (or the formula's overflow): the part of x that fp32 leaves out counts, too.
// Relative error 2^-23 from 2^-126 on; below it is 0.
__device__ __forceinline__ float exp2_of(double x)
{
    const float hi = (float)x, lo = (float)(x - (double)hi);
    const float e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e, lo * 0.693147181f, e);
}

// 2^x as m 2^e, for what is large enough to leave something below that: e is 0 but for x
// from -1024 to -126.
struct Factor {
    float m;
    int e;
};

__device__ __forceinline__ int exponent_of(double x) { return x < -126.0 && x > -1024.0 ? (int)ceil(x) : 0; }

__device__ __forceinline__ Factor factor_of(double x)
{
    const int e = exponent_of(x);
    return {exp2_of(x - e), e};
}

// Token i's decay of a chunk in base 2: 0 behind its n tokens.  Where 2^x is 0 a
// smaller x changes nothing but the sums' digits.
__device__ __forceinline__ double decay2(float decay, bool on)
{
    const double x = (double)decay * 1.4426950408889634;
    return !on ? 0.0 : x < -16384.0 ? -16384.0 : x;
}

// One token of each sequence (or none): V columns per lane, L lanes to a row of the
// state, 256 / L rows at a time and up to 16 of them in flight per thread.  q and k come
// through LDS, and the row groups' shares of q S meet there.  Bound by memory, the state in
// and out: 64 sequences of 32 heads of 128 x 128 move 272 MB in 59 us (4.6 TB/s; a copy 5.1),
// one 6.7 us.
template <int V, int L>
__global__ void __launch_bounds__(256) k_linear_step(ornk_linear_args a)
{
    typedef float vec __attribute__((ext_vector_type(V)));
    constexpr int G = 256 / L, R = 16;
    __shared__ float q[256], k[256];
    __shared__ vec part[G][L];
    const int blocks = (a.dv + V * L - 1) / (V * L), tid = threadIdx.x, g = tid / L;
    const int b = blockIdx.y, h = blockIdx.x / blocks;
    const int col = V * ((blockIdx.x - h * blocks) * L + tid - g * L);
    const Seq seq = seq_of(a, b);
    if (seq.n < 0) return;
    const size_t t = seq.t0, size = (size_t)a.dk * a.dv;
    const float *from = seq.in >= 0 ? a.S + ((size_t)seq.in * a.heads + h) * size + col : nullptr;
    float *to = seq.out >= 0 ? a.S + ((size_t)seq.out * a.heads + h) * size + col : nullptr;
    const bool on = col < a.dv;
    float f = 1.0f;
    int exponent = 0;
    vec v = 0.0f, o = 0.0f;
    if (!seq.n && tid < a.dk) q[tid] = k[tid] = 0.0f;
    if (seq.n) {
        if (tid < a.dk) {
            q[tid] = a.q[(t * a.qh + h / (a.heads / a.qh)) * a.dk + tid] * a.scale;
            k[tid] = a.k[(t * a.kh + h / (a.heads / a.kh)) * a.dk + tid];
        }
        if (on) v = *reinterpret_cast<const vec *>(a.v + (t * a.vh + h / (a.heads / a.vh)) * a.dv + col);
        const float decay = a.decay[a.per_token ? t * a.heads + h : h];
        const double x = decay2(decay, true);
        exponent = __builtin_amdgcn_readfirstlane(exponent_of(x));
        f = exponent ? exp2_of(x - exponent) : expf(decay);
        if (a.complement) v *= -expm1f(decay);
    }
    vec s[R];
    auto load = [&](int r0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = r0 + G * i;
            s[i] = 0.0f;
            if (from && on && r < a.dk) s[i] = *reinterpret_cast<const vec *>(from + (size_t)r * a.dv);
        }
    };
    load(g);
    __syncthreads();
    for (int r0 = 0;; load(r0 + g)) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = r0 + g + G * i;
            if (r < a.dk) {
                const float kr = k[r], qr = q[r];
                if (exponent)
#pragma unroll
                    for (int e = 0; e < V; ++e) s[i][e] = ldexpf(f * s[i][e], exponent);
                else
                    s[i] *= f;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    s[i][e] = fmaf(kr, v[e], s[i][e]);
                    o[e] = fmaf(qr, s[i][e], o[e]);
                }
                if (to && on) *reinterpret_cast<vec *>(to + (size_t)r * a.dv) = s[i];
            }
        }
        r0 += G * R;
        if (r0 >= a.dk) break;
    }
    if (!seq.n) return;
    part[g][tid - g * L] = o;
    __syncthreads();
    if (tid < L && on) {
        vec sum = part[0][tid];
        for (int i = 1; i < G; ++i) sum += part[i][tid];
        *reinterpret_cast<vec *>(a.out + (t * a.heads + h) * a.dv + col) = sum;
    }
}

// Groups of 128 columns where that gives every CU two of them, else of 32 (one sequence of
// 32 heads of 128: 11.0 us in groups of 64 columns, 6.7).
template <int V, int L>
void launch_step(const ornk_linear_args &a, hipStream_t s)
{
    const int blocks = (a.dv + V * L - 1) / (V * L);
    hipLaunchKernelGGL((k_linear_step<V, L>), dim3((unsigned)a.heads * blocks, a.n_seqs), dim3(256), 0, s, a);
}

// ---- chunks ------------------------------------------------------------------
// C tokens at a time, on the matrix cores.  With G_i the sum of a chunk's decays
// up to token i (base 2, in 64 bits), S the state before it and P_ij = q_i k_j:
//   o_i = scale (2^G_i q_i S + sum_(j <= i) 2^(G_i - G_j) b_j P_ij v_j)
//   S  <- 2^G_C S + sum_j 2^(G_C - G_j) b_j k_j v_j^T
// Exponents are differences of tokens in order, so no factor overflows before the
// formula's own factors together do.  A group of 4 waves takes 64 CB columns of a head's
// V, a wave 16 CB of them: lane 16 g + c has columns CB c + j, and rows 4 g + r of a block
// of 16 in its registers [r][j].  So S's accumulators are the second operand of q S as they are, P's
// (formed as K Q^T) the first of P V, and V never leaves its registers.  K and Q are in
// LDS.  P has three blocks of 16 x 16 (keys and queries of the first half, first and
// second, of the second), one for each of three waves; the fourth sums the next chunk's
// decays meanwhile.
//
// With fp32 operands it was bound by the matrix cores, which take 15 ns for a 16x16x4
// product of a SIMD (140 TFLOP/s): 24 x up to 1501 tokens, 32 heads of 128 (18,210 tokens in
// all) 431 us.  With three bf16 parts (8 ns for 16x16x32, six products) it takes 346 to 360, by
// the run: 1.28 GB are moved at 3.7 TB/s, and each wave's 232 matrix instructions and 1170 others
// of a chunk wait for three barriers, with one other group on the CU.  C = 32 costs 19 % more
// than the recurrence (P, P V).  Later loads of V, addresses of whole chunks kept apart, K and Q
// staged before S's products, and heads that share K and Q on one XCD made no difference.
constexpr int C = 32;

// A chunk is far where its decays together are below 2^FAR: factors times small numbers lose
// digits there, and below 2^-126 they are 0, which shows in what large numbers leave.  So where
// one of its numbers passes 2^16 (if none does, what is lost is below 2^-94 of each token), its
// part is done again in chunks that end before they are far: within those no factor is small
// but the first token's, which the state alone takes, as a mantissa and an exponent.  Looking
// for large numbers takes 1 to 5 % (8191 tokens, 16 heads of 128 142 -> 143 us, 4 x 2000, 8 of
// 256 x 256 288 -> 301), chunks cut so from the start nearly twice as long where decays are
// strong (548).
constexpr double FAR = -64.0;
constexpr float LARGE = 65536.0f;

struct alignas(16) Decays {
    double G[C]; // behind the chunk's last token as there
    float q[C];  // 2^G_i scale (in chunks that are cut the mantissa)
    float k[C];  // 2^(G_C - G_j) b_j
    float b[C];  // b_j scale
    float all;   // 2^G_C (or its mantissa)
    int far;
    int n;       // tokens
};

// x of the lane that a DPP step names, 0 where there is none or its row takes none
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double x)
{
    const uint64_t u = __double_as_longlong(x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((uint64_t)hi << 32 | lo);
}

// The sum of x up to each lane's, lanes i and i + 32 alike.
__device__ __forceinline__ double sums(double x)
{
    x += dpp<0x111, 0xf>(x);  // row_shr:1
    x += dpp<0x112, 0xf>(x);
    x += dpp<0x114, 0xf>(x);
    x += dpp<0x118, 0xf>(x);
    x += dpp<0x142, 0xa>(x);  // row_bcast:15, the second row of each half
    return x;
}

__device__ __forceinline__ double lane_of(double x, int lane)
{
    const uint64_t u = __double_as_longlong(x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __longlong_as_double((uint64_t)hi << 32 | lo);
}

// One wave, lanes i and i + 32 alike: the sums and factors of a chunk of up to n tokens; with
// CUT only as many of them as are not far.  The chunk's sum.
template <bool CUT>
__device__ __forceinline__ double fill_decays(const ornk_linear_args &a, Decays &d, double x, int &n)
{
    const int i = threadIdx.x & (C - 1);
    double G = sums(x), span = G;  // span: without growth, and without what clears any state
    double end = lane_of(G, C - 1);
    const bool plain = x <= 0.0 && x > -300.0;
    bool far = end < FAR;
    if (__any(!plain)) {
        span = sums(plain ? x : 0.0);
        far = lane_of(span, C - 1) < FAR;
    }
    if (CUT && far) {
        const uint32_t near = (uint32_t)__ballot(i == 0 || span - lane_of(span, 0) >= FAR);
        n = min(n, __builtin_ctzll(~(uint64_t)near));
        end = lane_of(G, n - 1);
        if (i >= n) G = end;
    }
    const float b = i >= n ? 0.0f : a.complement ? -expm1f((float)(x * 0.6931471805599453)) : 1.0f;
    d.G[i] = G;
    d.q[i] = (CUT && far ? factor_of(G).m : exp2_of(G)) * a.scale;
    d.k[i] = exp2_of(end - G) * b;
    d.b[i] = b * a.scale;
    if (!i) {
        d.all = CUT && far ? factor_of(end).m : exp2_of(end);
        d.far = far;
        d.n = n;
    }
    return end;
}

#define MFMA4(A, B, C) __builtin_amdgcn_mfma_f32_16x16x4f32(A, B, C, 0, 0, 0)

struct Cut {
    int segs, len;     // parts of a sequence that are done side by side, and their tokens
    bool joined;       // by a launch of its own; else each part joins those before it
    float *states;     // [n_seqs][heads][segs][dk][dv]: what a part adds, then (joined) what it
                       // begins with; of the last part what the sequence begins with
    Factor *decays;    // [n_seqs][heads][segs]: what a part leaves of a state
};

// N floats at p; without VEC only those before `left`, and 0 for the others.
template <int N, bool VEC>
__device__ __forceinline__ void load(float (&x)[N], const float *p, int left = N)
{
    typedef float vec __attribute__((ext_vector_type(N)));
    if (VEC) {
        const vec y = *reinterpret_cast<const vec *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = ((const float *)&y)[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? p[i] : 0.0f;
    }
}

template <int N, bool VEC>
__device__ __forceinline__ void store(float *p, const float (&x)[N], int left)
{
    typedef float vec __attribute__((ext_vector_type(N)));
    if (VEC) {
        vec y;
#pragma unroll
        for (int i = 0; i < N; ++i) ((float *)&y)[i] = x[i];
        *reinterpret_cast<vec *>(p) = y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = x[i];
    }
}

// O += P V within a block of 16 tokens, one key after the other: for values that are
// not finite, which the matrix cores would carry to tokens before them as 0 times
// themselves.
template <int CB>
__device__ __forceinline__ void add_in_order(v4f (&O)[CB], v4f P, const float (&v)[4][CB])
{
    const int g = (threadIdx.x & 63) >> 4, c = threadIdx.x & 15;
#pragma unroll 1
    for (int key = 0; key < 16; ++key) {
        const int kr = key & 3, at = 16 * (key >> 2);
        const float ps = kr == 0 ? P[0] : kr == 1 ? P[1] : kr == 2 ? P[2] : P[3];
        float vs[CB];
#pragma unroll
        for (int j = 0; j < CB; ++j)
            vs[j] = __shfl(kr == 0 ? v[0][j] : kr == 1 ? v[1][j] : kr == 2 ? v[2][j] : v[3][j], at + c, 64);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float pr = __shfl(ps, at + 4 * g + r, 64);
#pragma unroll
            for (int j = 0; j < CB; ++j)
                if (4 * g + r >= key) O[j][r] = fmaf(pr, vs[j], O[j][r]);
        }
    }
}

// The sequence of rank `rank` by length, the longest first: groups that start late are
// then short ones (24 x up to 1501 tokens 557 -> 449 us).  Up to 256 sequences; of more the
// order makes little difference.
__device__ __forceinline__ int by_length(const ornk_linear_args &a, int rank, int *lens)
{
    if (!a.starts || a.n_seqs > 256) return rank;
    const int i = threadIdx.x;
    if (i < a.n_seqs) lens[i] = a.starts[i + 1] - a.starts[i];
    __syncthreads();
    int before = 0;
    if (i < a.n_seqs) {
        const int n = lens[i];
        for (int j = 0; j < a.n_seqs; ++j) before += lens[j] > n || (lens[j] == n && j < i);
    }
    __syncthreads();
    if (i < a.n_seqs && before == rank) lens[0] = i;
    __syncthreads();
    const int b = lens[0];
    __syncthreads();
    return b;
}

// What a group has: a part of a sequence, and 64 CB columns of a head.
struct Part {
    Seq seq;
    int h, sg, block, first, last;  // tokens first to last - 1 of the sequence
    size_t at;                      // of the head's parts in the work buffers, the first
};

template <int CB>
__device__ __forceinline__ Part part_of(const ornk_linear_args &a, const Cut &cut, int *lens)
{
    Part p;
    const int blocks = (a.dv + 64 * CB - 1) / (64 * CB), rest = blockIdx.x / a.heads;
    p.h = blockIdx.x - rest * a.heads;
    p.sg = rest / blocks;
    p.block = rest - p.sg * blocks;
    const int b = cut.segs > 1 ? blockIdx.y : by_length(a, blockIdx.y, lens);
    p.seq = seq_of(a, b);
    p.first = p.sg * cut.len;
    p.last = min(p.seq.n, p.first + cut.len);
    p.at = ((size_t)b * a.heads + p.h) * cut.segs;
    return p;
}

// The state that a part begins with; whether it is known to be 0.
template <int KB, int CB, bool VEC, bool SUMS>
__device__ __forceinline__ bool begin_state(const ornk_linear_args &a, const Cut &cut, const Part &p, int col0,
                                            v4f (&S)[KB][CB])
{
    const int g = (threadIdx.x & 63) >> 4, cols = a.dv - col0;
    const size_t size = (size_t)a.dk * a.dv;
    const float *from = p.seq.in >= 0 ? a.S + ((size_t)p.seq.in * a.heads + p.h) * size : nullptr;
    if (SUMS) from = nullptr;
    else if (cut.segs > 1 && cut.joined) from = cut.states + (p.at + p.sg) * size;
    else if (cut.segs > 1 && from) from = cut.states + (p.at + (p.seq.n ? (p.seq.n - 1) / cut.len : 0)) * size;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < CB; ++j) S[kb][j] = v4f{0, 0, 0, 0};
    auto add = [&](const float *y, Factor keep) {  // all loads on their way at once
        float x[KB][4][CB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                load<CB, VEC>(x[kb][r], y + (size_t)min(16 * kb + 4 * g + r, a.dk - 1) * a.dv + col0, cols);
        if (__builtin_amdgcn_readfirstlane(keep.e))
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int j = 0; j < CB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[kb][j][r] = ldexpf(S[kb][j][r], keep.e);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < CB; ++j) S[kb][j][r] = fmaf(keep.m, S[kb][j][r], x[kb][r][j]);
    };
    if (from && cols > 0) add(from, {0.0f, 0});
    const bool joins = !SUMS && cut.segs > 1 && !cut.joined;
    if (joins) {
#pragma unroll 1
        for (int i = 0; i < p.sg; ++i)
            if (cols > 0) add(cut.states + (p.at + i) * size, cut.decays[p.at + i]);
    }
    if (a.dk < 16 * KB) {  // rows behind the key's dimensions stay 0
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < CB; ++j)
                    if (16 * kb + 4 * g + r >= a.dk) S[kb][j][r] = 0.0f;
    }
    return !from && !(joins && p.sg);
}

template <int KB, int CB, bool VEC>
__device__ __forceinline__ void end_state(const ornk_linear_args &a, float *to, int col0, const v4f (&S)[KB][CB])
{
    const int g = (threadIdx.x & 63) >> 4, cols = a.dv - col0;
    if (cols <= 0) return;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * kb + 4 * g + r;
            float x[CB];
#pragma unroll
            for (int j = 0; j < CB; ++j) x[j] = S[kb][j][r];
            if (row < a.dk) store<CB, VEC>(to + (size_t)row * a.dv + col0, x, cols);
        }
}

template <bool SUMS>
__device__ __forceinline__ float *state_of(const ornk_linear_args &a, const Cut &cut, const Part &p)
{
    const size_t size = (size_t)a.dk * a.dv;
    return SUMS ? cut.states + (p.at + p.sg) * size : a.S + ((size_t)p.seq.out * a.heads + p.h) * size;
}

template <int KB, bool SUMS>
struct Exact {
    static constexpr int LD = 16 * KB + 4;    // floats of a row in LDS
    static constexpr int NK = KB > 8 ? 1 : 2; // K of the next chunk beside this one's where two groups still fit a CU
    __align__(16) float Ks[NK][C][LD];
    __align__(16) float Qs[SUMS ? 1 : C][LD];
    __align__(16) v4f Ps[SUMS ? 1 : 3][64];
    __align__(16) Decays dec[2];
};

__device__ __forceinline__ float larger(float most, float x) { return fmaxf(most, fabsf(x)); }

template <int KB, int CB>
__device__ __forceinline__ float largest(float most, const float (&v)[2][4][CB], const v4f (&S)[KB][CB])
{
#pragma unroll
    for (int i = 0; i < 8 * CB; ++i) most = larger(most, (&v[0][0][0])[i]);
#pragma unroll
    for (int i = 0; i < 4 * KB * CB; ++i) most = larger(most, S[i / (4 * CB)][i / 4 % CB][i & 3]);
    return most;
}

// With fp32 operands: what 32-bit arithmetic gives, infinities and NaN included.  CUT: chunks
// end before they are far.  false: they have to, and nothing of the state is stored.
template <int KB, int CB, bool VEC, bool SUMS, bool CUT>
__device__ __forceinline__ bool exact_chunks(const ornk_linear_args &a, const Cut &cut, const Part &part, Exact<KB, SUMS> &lds)
{
    constexpr int LD = Exact<KB, SUMS>::LD, NK = Exact<KB, SUMS>::NK;
    constexpr int RS = 64 / KB;        // rows that the threads load at a time, a float4 each
    constexpr int NL = C / RS;
    auto &Ks = lds.Ks;
    auto &Qs = lds.Qs;
    auto &Ps = lds.Ps;
    auto &dec = lds.dec;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const Seq &seq = part.seq;
    const int h = part.h, first = part.first, last = part.last, block = part.block;
    const int col0 = block * 64 * CB + w * 16 * CB + c * CB, cols = a.dv - col0;
    const int hq = h / (a.heads / a.qh), hk = h / (a.heads / a.kh), hv = h / (a.heads / a.vh);
    const bool busy = block * 64 * CB + w * 16 * CB < a.dv;  // the wave has columns
    const bool stored = SUMS || (last == seq.n && seq.out >= 0);  // the state is, in the end
    v4f S[KB][CB];
    bool zero = begin_state<KB, CB, VEC, SUMS>(a, cut, part, col0, S);  // the state is, still

    // Rows of a chunk: uniform addresses, and each lane's place in them.  Where every load
    // is whole (VEC), lanes without columns load others' and rows behind the end the last
    // one, and what they get is dropped.
    const size_t ks = (size_t)a.kh * a.dk, qs = (size_t)a.qh * a.dk, vs = (size_t)a.vh * a.dv,
                 os = (size_t)a.heads * a.dv;
    const int lr = tid / (4 * KB), lc = 4 * (tid - lr * 4 * KB), left_k = a.dk - lc;
    const float *kp = a.k + ((size_t)seq.t0 + first) * ks + hk * a.dk, *qp = a.q + ((size_t)seq.t0 + first) * qs + hq * a.dk,
                *vp = a.v + ((size_t)seq.t0 + first) * vs + hv * a.dv;
    float *op = a.out + ((size_t)seq.t0 + first) * os + h * a.dv;
    const uint32_t lcv = VEC && left_k <= 0 ? 0 : lc, colv = VEC && cols <= 0 ? 0 : col0;
    float kn[NL][4], qn[SUMS ? 1 : NL][4], v[2][4][CB], vn[2][4][CB];
    // K and Q of the next chunk, `skip` tokens behind this one's first; n are left from there on
    auto fetch = [&](int n, int skip) {
        kp += skip * ks;
        qp += skip * qs;
        const uint32_t ko = lr * (uint32_t)ks + lcv, qo = lr * (uint32_t)qs + lcv;
        if (VEC && n >= C) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                load<4, true>(kn[i], kp + i * RS * ks + ko);
                if (!SUMS) load<4, true>(qn[i], qp + i * RS * qs + qo);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int row = min(lr + i * RS, n - 1);
                load<4, VEC>(kn[i], kp + row * ks + lcv, left_k);
                if (!SUMS) load<4, VEC>(qn[i], qp + row * qs + lcv, left_k);
                if (lr + i * RS >= n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) kn[i][e] = 0.0f;
            }
        }
    };
    auto fetch_v = [&](int n, int skip) {
        vp += skip * vs;
        const uint32_t vo = 4 * g * (uint32_t)vs + colv;
        if (VEC && n >= C) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int r = 0; r < 4; ++r) load<CB, true>(vn[tb][r], vp + (16 * tb + r) * vs + vo);
        } else {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * tb + 4 * g + r;
                    load<CB, VEC>(vn[tb][r], vp + min(row, n - 1) * vs + colv, cols);
                    if (row >= n)
#pragma unroll
                        for (int j = 0; j < CB; ++j) vn[tb][r][j] = 0.0f;
                }
        }
    };
    float xn = 0.0f;     // wave 3: a decay of the chunk that it sums next
    double left = 0.0;   // and the part's sum
    auto fetch_decays = [&](int t) {
        const int i = lane & (C - 1);
        const size_t tok = (size_t)seq.t0 + t + (i < last - t ? i : 0);
        xn = a.decay[a.per_token ? tok * a.heads + h : h];
    };
    auto fill = [&](int p, int t) {
        int n = min(C, last - t);
        const double x = decay2(xn, (lane & (C - 1)) < n);
        left += fill_decays<CUT>(a, dec[p], x, n);
        if (t + n < last) fetch_decays(t + n);
    };
    float own_k = 0.0f;  // the largest of the K staged
    auto stage_k = [&](int p) {
        own_k = 0.0f;
        if (left_k <= 0) return;
        if (!CUT)
#pragma unroll
            for (int i = 0; i < 4 * NL; ++i) own_k = larger(own_k, kn[i >> 2][i & 3]);
#pragma unroll
        for (int i = 0; i < NL; ++i)
            *reinterpret_cast<v4f *>(&Ks[p & (NK - 1)][lr + i * RS][lc]) = v4f{kn[i][0], kn[i][1], kn[i][2], kn[i][3]};
    };
    auto stage_q = [&] {
        if (SUMS || left_k <= 0) return;
#pragma unroll
        for (int i = 0; i < (SUMS ? 0 : NL); ++i)
            *reinterpret_cast<v4f *>(&Qs[lr + i * RS][lc]) = v4f{qn[i][0], qn[i][1], qn[i][2], qn[i][3]};
    };

    float most = 0.0f;  // the largest of far chunks' numbers
    int p = 0, n = C;
    if (first < last) {
        fetch(last - first, 0);
        if (w == 3) fetch_decays(first);
        fetch_v(last - first, 0);
        if (w == 3) fill(0, first);
        if (left_k <= 0) {  // columns behind the key's dimensions stay 0
            const v4f z = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                for (int k = 0; k < NK; ++k) *reinterpret_cast<v4f *>(&Ks[k][lr + i * RS][lc]) = z;
                if (!SUMS) *reinterpret_cast<v4f *>(&Qs[lr + i * RS][lc]) = z;
            }
        }
        stage_k(0);
        stage_q();
    }
    for (int t = first; t < last; t += n, p ^= 1) {
        float(*const K)[LD] = Ks[p & (NK - 1)];
        __syncthreads();
        const Decays &d = dec[p];
        if (CUT) n = __builtin_amdgcn_readfirstlane(d.n);
        const bool more = t + n < last, far = CUT && __builtin_amdgcn_readfirstlane(d.far);
        float own = own_k;  // the largest of this chunk's
#pragma unroll
        for (int i = 0; i < 8 * CB; ++i) (&v[0][0][0])[i] = (&vn[0][0][0])[i];
        if (CUT && n < C && more) {  // cut: the tokens behind are the next chunk's
            if (left_k > 0)
#pragma unroll
                for (int i = 0; i < NL; ++i)
                    if (lr + i * RS >= n) *reinterpret_cast<v4f *>(&K[lr + i * RS][lc]) = v4f{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (16 * (i >> 2) + 4 * g + (i & 3) >= n)
#pragma unroll
                    for (int j = 0; j < CB; ++j) v[i >> 2][i & 3][j] = 0.0f;
            __syncthreads();
        }
        if (more) {
            fetch(last - t - n, n);
            fetch_v(last - t - n, n);
        }
        v4f O[2][CB];
        if (w == 3) {
            if (more) fill(p ^ 1, t + n);
        } else if (!SUMS) {
            const int i = w, query = 16 * (i > 0) + c, key = 16 * (i > 1) + 4 * g;
            const float *kr = K[16 * (i > 1) + c], *qr = Qs[16 * (i > 0) + c];
            v4f P0 = {0, 0, 0, 0}, P1 = {0, 0, 0, 0}, f;
            const double G = d.G[query];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                f[r] = query >= key + r ? exp2_of(G - d.G[key + r]) * d.b[key + r] : 0.0f;
            v4f kq[2][4];
            auto read = [&](v4f (&y)[4], int x) {
                y[0] = *reinterpret_cast<const v4f *>(kr + 16 * x + 4 * g);
                y[1] = *reinterpret_cast<const v4f *>(qr + 16 * x + 4 * g);
                y[2] = *reinterpret_cast<const v4f *>(kr + 16 * x + 4 * g + 16);
                y[3] = *reinterpret_cast<const v4f *>(qr + 16 * x + 4 * g + 16);
            };
            read(kq[0], 0);
#pragma unroll
            for (int x = 0; x < KB; x += 2) {
                if (x + 2 < KB) read(kq[x / 2 + 1 & 1], x + 2);
                __builtin_amdgcn_sched_barrier(0);
                const v4f(&y)[4] = kq[x / 2 & 1];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    P0 = MFMA4(y[0][r], y[1][r], P0);
                    P1 = MFMA4(y[2][r], y[3][r], P1);
                }
            }
            P0 += P1;
            if (!CUT)
#pragma unroll
                for (int r = 0; r < 4; ++r) own = larger(own, P0[r]);
#pragma unroll
            for (int r = 0; r < 4; ++r) P0[r] = query >= key + r ? P0[r] * f[r] : 0.0f;
            Ps[i][lane] = P0;
        }
        if (!SUMS && busy) {  // q S
#pragma unroll
            for (int ib = 0; ib < 2; ++ib)
#pragma unroll
                for (int j = 0; j < CB; ++j) O[ib][j] = v4f{0, 0, 0, 0};
        }
        if (!SUMS && busy && !zero) {
            v4f q[2][2];
            auto read = [&](v4f (&y)[2], int kb) {
                y[0] = *reinterpret_cast<const v4f *>(&Qs[c][16 * kb + 4 * g]);
                y[1] = *reinterpret_cast<const v4f *>(&Qs[16 + c][16 * kb + 4 * g]);
            };
            read(q[0], 0);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                if (kb + 1 < KB) read(q[kb + 1 & 1], kb + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < CB; ++j) {
                        O[0][j] = MFMA4(q[kb & 1][0][r], S[kb][j][r], O[0][j]);
                        O[1][j] = MFMA4(q[kb & 1][1][r], S[kb][j][r], O[1][j]);
                    }
            }
#pragma unroll
            for (int ib = 0; ib < 2; ++ib) {
                const v4f f = *reinterpret_cast<const v4f *>(&d.q[16 * ib + 4 * g]);
                if (!CUT)
#pragma unroll
                    for (int i = 0; i < 4 * CB; ++i) own = larger(own, O[ib][i >> 2][i & 3]);
#pragma unroll
                for (int j = 0; j < CB; ++j) O[ib][j] *= f;
                if (CUT && far)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int exponent = exponent_of(d.G[16 * ib + 4 * g + r]);
#pragma unroll
                        for (int j = 0; j < CB; ++j) O[ib][j][r] = ldexpf(O[ib][j][r], exponent);
                    }
            }
        }
        __syncthreads();
        stage_q();
        if (NK > 1) stage_k(p ^ 1);
        if (busy) {
            if (!SUMS) {
                const v4f P0 = Ps[0][lane], P1 = Ps[1][lane], P2 = Ps[2][lane];
                float z = 0.0f;
#pragma unroll
                for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < CB; ++j) z = fmaf(v[tb][r][j], 0.0f, z);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < CB; ++j) O[1][j] = MFMA4(P1[r], v[0][r][j], O[1][j]);
                if (!__any(z != z)) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int j = 0; j < CB; ++j) {
                            O[0][j] = MFMA4(P0[r], v[0][r][j], O[0][j]);
                            O[1][j] = MFMA4(P2[r], v[1][r][j], O[1][j]);
                        }
                } else {
                    add_in_order(O[0], P0, v[0]);
                    add_in_order(O[1], P2, v[1]);
                }
                const int rows = CUT ? n : last - t;
                const uint32_t oo = 4 * g * (uint32_t)os + col0;
                auto put = [&](int ib, int r) {
                    float x[CB];
#pragma unroll
                    for (int j = 0; j < CB; ++j) x[j] = O[ib][j][r];
                    store<CB, VEC>(op + (16 * ib + r) * os + oo, x, cols);
                };
                if (cols > 0) {
                    if (rows >= C) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) put(i >> 2, i & 3);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (16 * (i >> 2) + 4 * g + (i & 3) < rows) put(i >> 2, i & 3);
                    }
                }
                op += n * os;
            }
        }
        if (!CUT && __builtin_amdgcn_readfirstlane(d.far)) {
            if (busy) own = largest(own, v, S);
            most = fmaxf(most, own);
        }
        if (busy && (more || stored)) {
            const float all = d.all;
            if (CUT && far) {
                const int exponent = exponent_of(d.G[C - 1]);
#pragma unroll
                for (int i = 0; i < 4 * KB * CB; ++i) {
                    float y = S[i / (4 * CB)][i / 4 % CB][i & 3];
                    S[i / (4 * CB)][i / 4 % CB][i & 3] = ldexpf(y, exponent);
                }
            }
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
                        const float k = K[16 * tb + 4 * g + r][16 * kb + c];
#pragma unroll
                        for (int j = 0; j < CB; ++j) S[kb][j] = MFMA4(k, v[tb][r][j], S[kb][j]);
                    }
            }
        }
        zero = false;
        if (NK == 1) {
            __syncthreads();
            stage_k(0);
        }
    }

    if (!CUT && __syncthreads_or(most > LARGE)) return false;
    if (SUMS && tid == 192 && !block) cut.decays[part.at + part.sg] = factor_of(left);
    if (stored) end_state<KB, CB, VEC>(a, state_of<SUMS>(a, cut, part), col0, S);
    return true;
}

// With operands of three bf16 parts, which hold the 24 bits of an fp32 number (of those
// below 2^-110 fewer), and the six products of parts that reach its last bit: what is left
// out is at most 2^-22 of a product.  16 x the rate, so 2.7 x the speed.  Parts of an
// infinity are no numbers, so whatever is not finite shows in the results, and the part is
// done again with fp32 operands, as where a far chunk's numbers are large.
template <int KB, bool SUMS>
struct Split {
    // [part][row][pair of dimensions]: of 32 dimensions those that a lane group of the
    // state's rows has, 4 g + r and 16 + 4 g + r, side by side; a row's 16 bytes turned by its number
    __align__(16) uint32_t K[SUMS ? 1 : 3][C][8 * KB];
    __align__(16) uint32_t Q[SUMS ? 1 : 3][C][8 * KB];
    // [part][four dimensions][a dimension's pairs of tokens], tokens in the same order
    __align__(16) uint32_t T[SUMS ? 2 : 1][3][4 * KB][64 + 4];
    __align__(16) uint2 P[SUMS ? 1 : 3][3][64];
    __align__(16) Decays dec[2];
};

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

// Part Z of two numbers, of which the parts before it are taken off, and what it leaves,
// exactly.  The second is rounded to nearest, so that what the products leave out has either
// sign; the others are the leading 8 bits (an instruction that issues in half the time: all
// three rounded take 3 % longer).
template <int Z>
__device__ __forceinline__ uint32_t take(float &x, float &y)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const uint32_t p = Z == 1 ? __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), b2))
                              : __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    x -= __uint_as_float(Z == 1 ? p << 16 : __float_as_uint(x) & 0xffff0000u);
    y -= __uint_as_float(Z == 1 ? p & 0xffff0000u : __float_as_uint(y) & 0xffff0000u);
    return p;
}

// F(Z) for each of the parts.
template <class F>
__device__ __forceinline__ void each_part(F f)
{
    f(std::integral_constant<int, 0>());
    f(std::integral_constant<int, 1>());
    f(std::integral_constant<int, 2>());
}

// Eight numbers as three operands of the matrix cores.
__device__ __forceinline__ void split8(u4 (&o)[3], float (&x)[8])
{
    each_part([&](auto z) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[z][i] = take<z>(x[2 * i], x[2 * i + 1]);
    });
}

__device__ __forceinline__ v4f mfma(u4 a, u4 b, v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// The parts of a product, the small ones first.
#define PRODUCTS(F) F(0, 2) F(2, 0) F(1, 1) F(0, 1) F(1, 0) F(0, 0)

// false: something was not finite, or large in a far chunk, and nothing of the state is stored.
template <int KB, int CB, bool SUMS>
__device__ __forceinline__ bool split_chunks(const ornk_linear_args &a, const Cut &cut, const Part &part, Split<KB, SUMS> &lds)
{
    constexpr int M = 2 * KB - 1;  // 16-byte words of a row, less one
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
    const Seq &seq = part.seq;
    const int h = part.h, first = part.first, last = part.last, block = part.block;
    const int col0 = block * 64 * CB + w * 16 * CB + c * CB, cols = a.dv - col0;
    const int hq = h / (a.heads / a.qh), hk = h / (a.heads / a.kh), hv = h / (a.heads / a.vh);
    const bool busy = block * 64 * CB + w * 16 * CB < a.dv;
    const bool stored = SUMS || (last == seq.n && seq.out >= 0);
    v4f S[KB][CB];
    bool zero = begin_state<KB, CB, true, SUMS>(a, cut, part, col0, S);

    // a thread has four dimensions of four tokens of K and Q
    const int lr = tid / (4 * KB), ld = tid - lr * 4 * KB;
    const bool loads = lr < C / 4;
    const bool filled = 4 * ld < a.dk;
    const size_t ks = (size_t)a.kh * a.dk, qs = (size_t)a.qh * a.dk, vs = (size_t)a.vh * a.dv,
                 os = (size_t)a.heads * a.dv;
    const float *kp = a.k + ((size_t)seq.t0 + first) * ks + hk * a.dk, *qp = a.q + ((size_t)seq.t0 + first) * qs + hq * a.dk,
                *vp = a.v + ((size_t)seq.t0 + first) * vs + hv * a.dv;
    float *op = a.out + ((size_t)seq.t0 + first) * os + h * a.dv;
    const uint32_t lcv = filled ? 4 * ld : 0, colv = cols <= 0 ? 0 : col0;
    float kn[4][4], qn[SUMS ? 1 : 4][4], v[2][4][CB], vn[2][4][CB];
    auto fetch = [&](int n) {
        if (loads) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t row = min(4 * lr + e, n - 1);
                load<4, true>(kn[e], kp + (row * (uint32_t)ks + lcv));
                if (!SUMS) load<4, true>(qn[e], qp + (row * (uint32_t)qs + lcv));
            }
            if (n < C || !filled) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (4 * lr + e >= n || !filled) kn[e][i] = 0.0f;
                        if (!SUMS && !filled) qn[e][i] = 0.0f;
                    }
            }
        }
        kp += C * ks;
        qp += C * qs;
    };
    auto fetch_v = [&](int n) {
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row = min(16 * tb + 4 * g + r, n - 1);
                load<CB, true>(vn[tb][r], vp + (row * (uint32_t)vs + colv));
            }
        if (n < C) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < CB; ++j)
                        if (16 * tb + 4 * g + r >= n) vn[tb][r][j] = 0.0f;
        }
        vp += C * vs;
    };
    float xn = 0.0f;
    double left = 0.0;
    auto fetch_decays = [&](int t) {
        const int i = lane & (C - 1);
        const size_t tok = (size_t)seq.t0 + t + (i < last - t ? i : 0);
        xn = a.decay[a.per_token ? tok * a.heads + h : h];
    };
    auto fill = [&](int p, int t) {
        int n = min(C, last - t);
        left += fill_decays<false>(a, lds.dec[p], decay2(xn, (lane & (C - 1)) < n), n);
        if (t + C < last) fetch_decays(t + C);
    };
    float own = 0.0f;  // the largest of this chunk's
    auto stage = [&](int p) {
        own = 0.0f;
        if (!loads) return;
#pragma unroll
        for (int i = 0; i < 16; ++i) own = larger(own, kn[i >> 2][i & 3]);
        const int word = (4 * (ld >> 3) + (ld & 3)), half = ld >> 2 & 1;
        auto rows = [&](auto z, uint32_t (&to)[SUMS ? 1 : 3][C][8 * KB], float (&x)[4][4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 4 * lr + e;
                const uint32_t y0 = take<z>(x[e][0], x[e][1]), y1 = take<z>(x[e][2], x[e][3]);
                *reinterpret_cast<uint2 *>(&to[z][row][4 * (word ^ (row & M)) + 2 * half]) = uint2{y0, y1};
            }
        };
        each_part([&](auto z) {
            if constexpr (!SUMS) {
                float x[4][4];
#pragma unroll
                for (int i = 0; i < 16; ++i) (&x[0][0])[i] = (&kn[0][0])[i];
                rows(z, lds.K, x);
                rows(z, lds.Q, qn);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t y0 = take<z>(kn[0][i], kn[1][i]), y1 = take<z>(kn[2][i], kn[3][i]);
                *reinterpret_cast<uint2 *>(&lds.T[SUMS ? p : 0][z][ld][16 * i + 4 * (lr & 3) + 2 * (lr >> 2)]) =
                    uint2{y0, y1};
            }
        });
    };
    auto row_of = [&](const uint32_t (&from)[SUMS ? 1 : 3][C][8 * KB], int part, int row, int x) {
        return *reinterpret_cast<const u4 *>(&from[part][row][4 * ((4 * x + g) ^ (row & M))]);
    };

    float bad = 0.0f;   // 0, or a NaN
    float most = 0.0f;  // the largest of far chunks' numbers
    int p = 0;
    if (first < last) {
        fetch(last - first);
        if (w == 3) fetch_decays(first);
        fetch_v(last - first);
        if (w == 3) fill(0, first);
    }
    for (int t = first; t < last; t += C, p ^= 1) {
        const bool more = t + C < last;
        stage(p);
#pragma unroll
        for (int i = 0; i < 8 * CB; ++i) (&v[0][0][0])[i] = (&vn[0][0][0])[i];
        __syncthreads();
        if (more) {
            fetch(last - t - C);
            fetch_v(last - t - C);
        }
        const Decays &d = lds.dec[p];
        v4f O[2][CB];
        if (w == 3) {
            if (more) fill(p ^ 1, t + C);
        } else if constexpr (!SUMS) {
            const int i = w, query = 16 * (i > 0) + c, key = 16 * (i > 1) + 4 * g, kr = 16 * (i > 1) + c;
            v4f P0 = {0, 0, 0, 0}, P1 = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < KB / 2; ++x) {
                u4 k[3], q[3];
#pragma unroll
                for (int y = 0; y < 3; ++y) {
                    k[y] = row_of(lds.K, y, kr, x);
                    q[y] = row_of(lds.Q, y, query, x);
                }
                v4f &P = x & 1 ? P1 : P0;
#define F(A, B) P = mfma(k[A], q[B], P);
                PRODUCTS(F)
#undef F
            }
            P0 += P1;
#pragma unroll
            for (int r = 0; r < 4; ++r) own = larger(own, P0[r]);
            const double G = d.G[query];
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                y[r] = query >= key + r ? P0[r] * (exp2_of(G - d.G[key + r]) * d.b[key + r]) : 0.0f;
            each_part([&](auto z) {
                const uint32_t y0 = take<z>(y[0], y[1]), y1 = take<z>(y[2], y[3]);
                lds.P[i][z][lane] = uint2{y0, y1};
            });
        }
        if constexpr (!SUMS) {
#pragma unroll
            for (int ib = 0; ib < 2; ++ib)
#pragma unroll
                for (int j = 0; j < CB; ++j) O[ib][j] = v4f{0, 0, 0, 0};
            if (busy && !zero) {  // q S
#pragma unroll
                for (int x = 0; x < KB / 2; ++x) {
                    u4 q[2][3], s[CB][3];
#pragma unroll
                    for (int y = 0; y < 3; ++y) {
                        q[0][y] = row_of(lds.Q, y, c, x);
                        q[1][y] = row_of(lds.Q, y, 16 + c, x);
                    }
#pragma unroll
                    for (int j = 0; j < CB; ++j) {
                        float y[8];
#pragma unroll
                        for (int r = 0; r < 8; ++r) y[r] = S[2 * x + (r >> 2)][j][r & 3];
                        split8(s[j], y);
                    }
#define F(A, B)                                                                     \
    _Pragma("unroll") for (int j = 0; j < CB; ++j)                                  \
    {                                                                               \
        O[0][j] = mfma(q[0][A], s[j][B], O[0][j]);                                  \
        O[1][j] = mfma(q[1][A], s[j][B], O[1][j]);                                  \
    }
                    PRODUCTS(F)
#undef F
                }
#pragma unroll
                for (int ib = 0; ib < 2; ++ib) {
                    const v4f f = *reinterpret_cast<const v4f *>(&d.q[16 * ib + 4 * g]);
#pragma unroll
                    for (int i = 0; i < 4 * CB; ++i) own = larger(own, O[ib][i >> 2][i & 3]);
#pragma unroll
                    for (int j = 0; j < CB; ++j) O[ib][j] *= f;
                }
            }
            __syncthreads();
            if (busy) {
                u4 m[2][3];
#pragma unroll
                for (int z = 0; z < 3; ++z) {
                    const uint2 x0 = lds.P[0][z][lane], x1 = lds.P[1][z][lane], x2 = lds.P[2][z][lane];
                    m[0][z] = u4{x0.x, x0.y, 0, 0};
                    m[1][z] = u4{x1.x, x1.y, x2.x, x2.y};
                }
                u4 s[CB][3];
#pragma unroll
                for (int j = 0; j < CB; ++j) {
                    float y[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) y[r] = v[r >> 2][r & 3][j];
                    split8(s[j], y);
                }
#define F(A, B)                                                                     \
    _Pragma("unroll") for (int j = 0; j < CB; ++j)                                  \
    {                                                                               \
        O[0][j] = mfma(m[0][A], s[j][B], O[0][j]);                                  \
        O[1][j] = mfma(m[1][A], s[j][B], O[1][j]);                                  \
    }
                PRODUCTS(F)
#undef F
                const int n = last - t;
                const uint32_t oo = 4 * g * (uint32_t)os + col0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ib = i >> 2, r = i & 3;
                    float x[CB];
#pragma unroll
                    for (int j = 0; j < CB; ++j) {
                        x[j] = O[ib][j][r];
                        bad = fmaf(x[j], 0.0f, bad);
                    }
                    if (cols > 0 && 16 * ib + 4 * g + r < n) store<CB, true>(op + (16 * ib + r) * os + oo, x, cols);
                }
                op += C * os;
            }
        }
        if (__builtin_amdgcn_readfirstlane(d.far)) {
            if (busy) own = largest(own, v, S);
            most = fmaxf(most, own);
        }
        if (busy && (more || stored)) {
            const float all = d.all;
            u4 s[CB][3];
#pragma unroll
            for (int j = 0; j < CB; ++j) {
                float y[8];
#pragma unroll
                for (int tb = 0; tb < 2; ++tb) {
                    const v4f f = *reinterpret_cast<const v4f *>(&d.k[16 * tb + 4 * g]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[4 * tb + r] = v[tb][r][j] * f[r];
                }
                split8(s[j], y);
            }
#pragma unroll
            for (int kb = 0; kb < KB; kb += 2) {
                u4 k[2][3];
#pragma unroll
                for (int z = 0; z < 3; ++z)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        k[i][z] = *reinterpret_cast<const u4 *>(
                            &lds.T[SUMS ? p : 0][z][4 * (kb + i) + (c >> 2)][16 * (c & 3) + 4 * g]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < CB; ++j) S[kb + i][j] *= all;
#define F(A, B)                                                                     \
    _Pragma("unroll") for (int i = 0; i < 2; ++i)                                   \
        _Pragma("unroll") for (int j = 0; j < CB; ++j)                              \
            S[kb + i][j] = mfma(k[i][A], s[j][B], S[kb + i][j]);
                PRODUCTS(F)
#undef F
            }
        }
        zero = false;
        if (!SUMS) __syncthreads();
    }
    if (stored && busy) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int j = 0; j < CB; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) bad = fmaf(S[kb][j][r], 0.0f, bad);
    }
    if (__syncthreads_or(bad != bad || most > LARGE)) return false;
    if (SUMS && tid == 192 && !block) cut.decays[part.at + part.sg] = factor_of(left);
    if (stored) end_state<KB, CB, true>(a, state_of<SUMS>(a, cut, part), col0, S);
    return true;
}
#undef PRODUCTS

// SUMS: only what a part adds to a state that begins with zeros.  VEC: rows of K and Q
// are whole float4s, those of V whole vectors of CB.
template <int KB, int CB, bool VEC, bool SUMS>
__global__ void __launch_bounds__(256, 2) k_linear_chunks(ornk_linear_args a, Cut cut)
{
    constexpr bool FAST = VEC && KB <= 8;
    __shared__ union Lds {
        int lens[256];
        Exact<KB, SUMS> exact;
        Split<FAST ? KB : 1, SUMS> split;
        __device__ Lds() {}
    } lds;
    const Part part = part_of<CB>(a, cut, lds.lens);
    if (part.seq.n < 0 || (part.sg && part.first >= part.seq.n)) return;
    if (SUMS && part.first + cut.len >= part.seq.n) {
        // Nothing begins behind it; but where each part joins those before it, its place
        // holds what the sequence begins with, whose slot may be written before all have begun.
        if (cut.joined || part.seq.in < 0) return;
        const size_t size = (size_t)a.dk * a.dv;
        const float *from = a.S + ((size_t)part.seq.in * a.heads + part.h) * size;
        float *to = cut.states + (part.at + part.sg) * size;
        const int col = part.block * 64 * CB + (threadIdx.x & 63), n = min(a.dv, (part.block + 1) * 64 * CB);
        for (int row = threadIdx.x >> 6; row < a.dk; row += 4)
            for (int i = col; i < n; i += 64) to[(size_t)row * a.dv + i] = from[(size_t)row * a.dv + i];
        return;
    }
    if constexpr (FAST)
        if (split_chunks<KB, CB, SUMS>(a, cut, part, lds.split)) return;
    if constexpr (!FAST)
        if (exact_chunks<KB, CB, VEC, SUMS, false>(a, cut, part, lds.exact)) return;
    exact_chunks<KB, CB, VEC, SUMS, true>(a, cut, part, lds.exact);
}

// From what each part adds to what each part begins with, an element per thread (16 heads
// of 128 x 128 in 32 parts 16 us, 67 MB).
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
        const float add = more ? *p : 0.0f;
        const Factor keep = more ? cut.decays[at + i] : Factor{0.0f, 0};
        *p = s;
        s = keep.e ? ldexpf(keep.m * s, keep.e) + add : fmaf(keep.m, s, add);
    }
}

// Parts of a sequence that join those before them by themselves, which saves a launch (5 x
// 333, 12 heads of 96 x 80: 42 -> 39 us); with 8 of them it takes longer (1 x 512, 32 heads of
// 128: 51 us, by a launch 42).
constexpr int JOIN = 4;

// Sequences are cut where their heads and columns leave CUs idle: into parts of at
// least 64 tokens, until there are two groups for each CU.  What the parts add to a state
// is formed first, and their tokens after that from what they begin with, which takes 1.4
// times the products.  One prompt of 8191 tokens, 16 heads of 128: 143 us (alone, under a
// profiler, sums 41, joining 16, tokens 93); with one group for each CU 159.  5 x 333, 12
// heads of 96 x 80: 39; with parts of 128 tokens 50.
Cut cut_of(const ornk_linear_args &a, int cb)
{
    const long long groups = (long long)a.n_seqs * a.heads * ((a.dv + 64 * cb - 1) / (64 * cb));
    long long segs = 512 / groups;
    if (segs > a.max_len / 64) segs = a.max_len / 64;
    Cut c = {1, a.max_len, false, nullptr, nullptr};
    if (segs < 2) return c;
    c.len = (int)(((a.max_len + segs - 1) / segs + C - 1) / C * C);
    c.segs = (a.max_len - 1) / c.len + 1;
    c.joined = c.segs > JOIN;
    return c;
}

// Blocks of 16 columns of a wave: two, where there is then a group for each CU, and the
// state's registers leave room for another group.  Two share a group's P and its waits (one
// prompt of 8191 tokens, 16 heads of 128: 143 us, with one block 158); one gives twice the
// groups (1 x 512, 16 heads of 128: 29, with two 33).
int blocks_of(const ornk_linear_args &a)
{
    if (a.dv <= 64 || a.dk > 128) return 1;
    return (long long)a.n_seqs * a.heads * ((a.dv + 127) / 128) * cut_of(a, 2).segs >= 256 ? 2 : 1;
}

template <int KB, int CB, bool VEC>
void launch(const ornk_linear_args &a, const Cut &cut, hipStream_t s)
{
    const int blocks = (a.dv + 64 * CB - 1) / (64 * CB);
    const dim3 grid((unsigned)a.heads * cut.segs * blocks, a.n_seqs);
    if (cut.segs > 1) {
        hipLaunchKernelGGL((k_linear_chunks<KB, CB, VEC, true>), grid, dim3(256), 0, s, a, cut);
        if (cut.joined)
            hipLaunchKernelGGL(k_linear_join, dim3(a.n_seqs, a.heads, (a.dk * a.dv + 255) / 256), dim3(256), 0,
                               s, a, cut);
    }
    hipLaunchKernelGGL((k_linear_chunks<KB, CB, VEC, false>), grid, dim3(256), 0, s, a, cut);
}

template <int KB, int CB>
void launch(const ornk_linear_args &a, const Cut &cut, hipStream_t s)
{
    if (a.dk % 4 || a.dv % CB) launch<KB, CB, false>(a, cut, s);
    else launch<KB, CB, true>(a, cut, s);
}

}  // namespace

extern "C" size_t ornk_linear_ws(const ornk_linear_args *a)
{
    const Cut c = cut_of(*a, blocks_of(*a));
    if (c.segs < 2) return 0;
    return (size_t)a->n_seqs * a->heads * c.segs * (sizeof(float) * a->dk * a->dv + sizeof(Factor));
}

extern "C" int ornk_linear(const ornk_linear_args *a, hipStream_t s)
{
    if (a->max_len <= 1) {
        if (a->dv % 4) launch_step<1, 32>(*a, s);
        else if ((long long)a->n_seqs * a->heads >= 512 && a->dv > 32) launch_step<4, 32>(*a, s);
        else launch_step<4, 8>(*a, s);
        return hipGetLastError();
    }
    const int cb = blocks_of(*a);
    Cut c = cut_of(*a, cb);
    c.states = static_cast<float *>(a->ws);
    if (c.segs > 1)
        c.decays = reinterpret_cast<Factor *>(c.states + (size_t)a->n_seqs * a->heads * c.segs * a->dk * a->dv);
    if (a->dk > 128) launch<16, 1>(*a, c, s);
    else if (cb == 2) a->dk > 64 ? launch<8, 2>(*a, c, s) : launch<4, 2>(*a, c, s);
    else a->dk > 64 ? launch<8, 1>(*a, c, s) : launch<4, 1>(*a, c, s);
    return hipGetLastError();
}
