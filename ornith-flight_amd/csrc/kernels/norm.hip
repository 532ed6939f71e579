// SPDX-License-Identifier: MIT
//
// Norms of the query and key heads with the rotation, and the append to the paged
// key-value cache, in one pass (ornith_hip.h).
#include "kv.h"

namespace {

constexpr int NT = 256;

// A token's row: query heads, then key heads, then value heads.
struct Row {
    const float *x, *w;  // w: weights, NULL: ones
    float *out;          // NULL: only the cache
    void *cache;         // the row's place there, NULL: not stored
    float scale;
    bool norm;
};

template <int TYPE>
__device__ __forceinline__ Row row_of(const ornk_kv_pages &p, const ornk_rope_args &a, int t, int slot,
                                      int i)
{
    typedef typename KvElem<TYPE>::T T;
    const int hd = a.hd;
    Row r;
    r.cache = nullptr;
    r.scale = 1.0f;
    if (i < a.heads) {
        const size_t at = ((size_t)t * a.heads + i) * hd;
        r.x = a.q + at;
        r.out = a.q_out + at;
        r.w = a.qw ? a.qw + (a.per_head ? (size_t)i * hd : 0) : nullptr;
        r.norm = true;
        return r;
    }
    i -= a.heads;
    r.norm = i < a.kv;
    const int h = r.norm ? i : i - a.kv;
    const size_t at = ((size_t)t * a.kv + h) * hd;
    r.x = (r.norm ? a.k : a.v) + at;
    r.out = r.norm && a.k_out ? a.k_out + at : nullptr;
    r.w = r.norm && a.kw ? a.kw + (a.per_head ? (size_t)h * hd : 0) : nullptr;
    if (slot >= 0) {
        r.cache = static_cast<T *>(r.norm ? p.k : p.v) +
                  kv_at(p, slot >> p.page_log2, h, slot & (p.page - 1));
        r.scale = r.norm ? p.k_scale : p.v_scale;
    }
    return r;
}

// What a row is divided by: sqrt(sum or mean of squares + eps).  Where that square is not a
// 32-bit number, or so small that squares lost digits, it is formed of the row times c,
// 2^-70 or 2^100: scaled(c) is the sum of the squares of that.
struct Norm {
    float s, per, c;  // per = 1 / s
    template <class F>
    __device__ __forceinline__ Norm(const ornk_rope_args &a, float ss, bool norm, F scaled)
    {
        const float n = a.norm == 1 ? (float)a.hd : 1.0f;
        float m = ss / n + a.eps;
        c = 1.0f;
        if (norm && !(m >= 0x1p-100f && m < INFINITY)) {
            c = m < 1.0f ? 0x1p100f : 0x1p-70f;
            m = scaled(c) / n + a.eps * c * c;
        }
        s = sqrtf(m);
        per = 1.0f / s;
    }
    // x / s; the product with 1 / s alone rounds once more (of 4099 tokens' heads of 128
    // 4.9e-8 of the whole instead of 4.2e-8)
    template <int N, class T>
    __device__ __forceinline__ void divide(T &x) const
    {
        if (c == 1.0f) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float q = x[e] * per;
                x[e] = fmaf(fmaf(-q, s, x[e]), per, q);
            }
            return;
        }
        const bool exact = s < INFINITY && per < INFINITY;  // the quotient's remainder is a number
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float y = c > 1.0f ? x[e] * c : x[e];
            float q = y * per;
            if (exact) q = fmaf(fmaf(-q, s, y), per, q);
            x[e] = c < 1.0f ? q * c : q;
        }
    }
};

// Rows that are no whole float4s (or halves of pairs that are not four): a wave per
// row, an element or a pair per lane, which reads the row a second time after its sum.  The
// token's angles are formed once, in LDS.  Bound by its loads of one element per lane, twice:
// 4099 tokens of 32 + 8 heads of 66 65 us (87 MB, 17 at the copy's rate).
template <int TYPE>
__global__ void __launch_bounds__(NT) k_norm_append_any(ornk_kv_pages p, ornk_rope_args a, int rows)
{
    typedef KvElem<TYPE> E;
    __shared__ float2 cs[ORN_ROPE_MAX_PAIRS];
    const int lane = threadIdx.x & 63, hd = a.hd, R = a.R;
    const int r0 = (int)((long long)rows * blockIdx.y / gridDim.y);
    const int r1 = (int)((long long)rows * (blockIdx.y + 1) / gridDim.y);
    for (long long at = blockIdx.x; at < a.T; at += gridDim.x) {
        const int t = (int)at;
        for (int i = threadIdx.x; i < R; i += NT) cs[i] = rope_cs(a, t, i);
        const int slot = a.slots ? kv_slot(p, a.slots, t) : -1;
        __syncthreads();
        for (int i = r0 + (threadIdx.x >> 6); i < r1; i += NT / 64) {
            const Row r = row_of<TYPE>(p, a, t, slot, i);
            float ss = 0.0f;
            if (r.norm)
                for (int d = lane; d < hd; d += 64) ss = fmaf(r.x[d], r.x[d], ss);
            const Norm norm(a, orn_wave_sum(ss), r.norm, [&](float c) {
                float sum = 0.0f;
                for (int d = lane; d < hd; d += 64) sum = fmaf(r.x[d] * c, r.x[d] * c, sum);
                return orn_wave_sum(sum);
            });
            auto get = [&](int d) {
                float x[1] = {r.x[d]};
                if (!r.norm) return x[0];
                norm.template divide<1>(x);
                return r.w ? x[0] * r.w[d] : x[0];
            };
            auto put = [&](int d, float x) {
                if (r.out) r.out[d] = x;
                if (r.cache) static_cast<typename E::T *>(r.cache)[d] = E::put(x, r.scale);
            };
            const int n_rot = r.norm ? R : 0;
            for (int d = lane; d < hd - n_rot; d += 64) {
                if (d >= n_rot) {
                    put(d + n_rot, get(d + n_rot));
                    continue;
                }
                const int i0 = a.halves ? d : 2 * d, i1 = a.halves ? d + R : 2 * d + 1;
                const float u = get(i0), v = get(i1);
                put(i0, u * cs[d].x - v * cs[d].y);
                put(i1, u * cs[d].y + v * cs[d].x);
            }
        }
        __syncthreads();  // the token's angles are consumed
    }
}

// A row by 2^g lanes, an item of it per lane: a float4, with HALVES two of one pair's
// four (R apart).  A row of more than 64 items is read a second time after its sum.
// Bound by memory: 8190 tokens of 32 + 8 heads of 128 with the append to f16 move 369 MB in
// 75 us (4.9 TB/s; a copy 5.1), 4099 of 16 + 16 heads without rotation 134 MB in 32 us.  One
// token of 16 + 2 heads takes 7.0 us, the launch and the caller's side (kernel 4.9).
template <int TYPE, bool HALVES>
__global__ void __launch_bounds__(NT, 8) k_norm_append(ornk_kv_pages p, ornk_rope_args a, int rows, int g)
{
    typedef typename KvElem<TYPE>::T T;
    __shared__ __align__(16) float2 cs[ORN_ROPE_MAX_PAIRS];
    const int hd = a.hd, R = a.R, G = 1 << g;
    const int n_norm = (HALVES ? hd - R : hd) / 4, n_val = hd / 4;
    const int li = threadIdx.x & (G - 1);
    const int r0 = (int)((long long)rows * blockIdx.y / gridDim.y);
    const int r1 = (int)((long long)rows * (blockIdx.y + 1) / gridDim.y);

    for (long long at = blockIdx.x; at < a.T; at += gridDim.x) {
        const int t = (int)at;
        const int slot = a.slots ? kv_slot(p, a.slots, t) : -1;
        for (int i = threadIdx.x; i < R; i += NT) cs[i] = rope_cs(a, t, i);
        __syncthreads();
        // every lane of a row's group goes through the loop alike; groups past r1 idle
        for (int base = r0; base < r1; base += NT >> g) {
            const int i = base + (threadIdx.x >> g);
            const bool on = i < r1;
            const Row r = row_of<TYPE>(p, a, t, slot, on ? i : r0);
            const int items = !on ? 0 : r.norm ? n_norm : n_val;
            auto column = [&](int it, bool &two) {
                two = HALVES && r.norm && 4 * it < R;
                return 4 * it + (HALVES && r.norm && !two ? R : 0);
            };
            v4f x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            float ss = 0.0f;
            auto load = [&](int it) {
                bool two;
                const int c = column(it, two);
                x = *reinterpret_cast<const v4f *>(r.x + c);
                if (two) y = *reinterpret_cast<const v4f *>(r.x + c + R);
                else y = v4f{0, 0, 0, 0};
            };
            for (int it = li; it < items; it += G) {
                load(it);
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fmaf(y[e], y[e], fmaf(x[e], x[e], ss));
            }
            for (int o = G >> 1; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const Norm norm(a, ss, on && r.norm, [&](float c) {
                float sum = 0.0f;
                for (int it = li; it < items; it += G) {
                    if (items > G) load(it);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum = fmaf(y[e] * c, y[e] * c, fmaf(x[e] * c, x[e] * c, sum));
                }
                for (int o = G >> 1; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
                return sum;
            });
            for (int it = li; it < items; it += G) {
                if (items > G) load(it);
                bool two;
                const int c = column(it, two);
                if (r.norm) {
                    norm.template divide<4>(x);
                    if (HALVES) norm.template divide<4>(y);
                    if (r.w) {
                        x *= *reinterpret_cast<const v4f *>(r.w + c);
                        if (two) y *= *reinterpret_cast<const v4f *>(r.w + c + R);
                    }
                    if (HALVES) {
                        if (two) {
                            const v4f u = x, v = y;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 q = cs[c + e];
                                x[e] = u[e] * q.x - v[e] * q.y;
                                y[e] = u[e] * q.y + v[e] * q.x;
                            }
                        }
                    } else {
                        const v4f u = x;
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            if (c + e >= 2 * R) continue;  // past the last pair
                            const float2 q = cs[(c + e) / 2];
                            x[e] = u[e] * q.x - u[e + 1] * q.y;
                            x[e + 1] = u[e] * q.y + u[e + 1] * q.x;
                        }
                    }
                }
                if (r.out) {
                    *reinterpret_cast<v4f *>(r.out + c) = x;
                    if (two) *reinterpret_cast<v4f *>(r.out + c + R) = y;
                }
                if (r.cache) {
                    T *o = static_cast<T *>(r.cache) + c;
                    put4<TYPE>(o, x, r.scale);
                    if (two) put4<TYPE>(o + R, y, r.scale);
                }
            }
        }
        __syncthreads();  // the token's angles are consumed
    }
}

constexpr int MAX_GROUPS = 1 << 20;  // of a launch; more tokens take turns

template <int TYPE>
int launch(const ornk_kv_pages &p, const ornk_rope_args &a, hipStream_t s)
{
    const int rows = a.heads + a.kv * (a.slots ? 2 : 1);
    const bool any = a.hd % 4 || (a.halves && a.R % 4);
    int g = any ? 6 : 0;
    while (g < 6 && 4 << g < (a.halves ? a.hd - a.R : a.hd)) ++g;
    // A token's rows in one group, so that its angles are formed once, unless the
    // tokens leave CUs without one.
    const long long per = NT >> g;
    long long y = (rows + per - 1) / per;
    if (y * a.T > 512) y = a.T < 512 ? 512 / a.T : 1;
    const dim3 grid(a.T < MAX_GROUPS ? a.T : MAX_GROUPS, (unsigned)(y < 1 ? 1 : y));
    if (any)
        hipLaunchKernelGGL(k_norm_append_any<TYPE>, grid, dim3(NT), 0, s, p, a, rows);
    else if (a.halves)
        hipLaunchKernelGGL((k_norm_append<TYPE, true>), grid, dim3(NT), 0, s, p, a, rows, g);
    else
        hipLaunchKernelGGL((k_norm_append<TYPE, false>), grid, dim3(NT), 0, s, p, a, rows, g);
    return hipGetLastError();
}

}  // namespace

extern "C" int ornk_norm_append(const ornk_kv_pages *pp, const ornk_rope_args *a, hipStream_t s)
{
    ornk_kv_pages p = {};
    if (pp) p = *pp;
    switch (p.type) {
    case ORN_KV_F32: return launch<ORN_KV_F32>(p, *a, s);
    case ORN_KV_F16: return launch<ORN_KV_F16>(p, *a, s);
    case ORN_KV_BF16: return launch<ORN_KV_BF16>(p, *a, s);
    default: return launch<ORN_KV_E4M3>(p, *a, s);
    }
}
