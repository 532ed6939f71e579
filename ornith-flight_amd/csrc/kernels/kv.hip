// SPDX-License-Identifier: MIT
//
// Rotary positions of several axes, and the append to the paged key-value
// cache (ornith_hip.h).
#include "kv.h"

namespace {

// cos and sin of pair i's angle at token t.  The turn is formed in 64 bits and
// reduced before it is rounded, so far positions keep their digits.  The reduced turn,
// its cosine and its sine are fp32: an output is off by 1.3 times what it is with
// these in 64 bits, too (of 4099 tokens 5.4e-8 of the whole instead of 4.2e-8), which
// took 7 % longer there (28.4 us) and 5 % with 8190 tokens' append (71.0 us).
__device__ __forceinline__ float2 rope_cs(const ornk_rope_args &a, int t, int i)
{
    const double turn = (double)a.pos[(size_t)a.axis[i] * a.T + t] * a.turns[i];
    float2 r;
    sincospif(2.0f * (float)(turn - rint(turn)), &r.y, &r.x);
    return r;
}

// Heads whose pairs are not whole float4s: one work group per token and row
// (query heads, key heads, value heads), an element or a pair per thread.  Bound by the
// angles, formed again for every head: 4099 tokens of 32 + 8 heads of 66 in halves 68 us,
// with the append to f16 91 (of 64, by k_rope_append, 17); of 16 tokens 7.4, as any.
template <int TYPE>
__global__ void __launch_bounds__(128) k_rope_append_any(ornk_kv_pages p, ornk_rope_args a, int rows)
{
    typedef KvElem<TYPE> E;
    const int tid = threadIdx.x, hd = a.hd, R = a.R;
    for (long long at = blockIdx.x; at < (long long)a.T * rows; at += gridDim.x) {
        const int t = (int)(at / rows);
        int head = (int)(at - (long long)t * rows), part = 0;  // 0 query, 1 key, 2 value
        if (head >= a.heads) {
            head -= a.heads;
            part = 1;
            if (head >= a.kv) {
                head -= a.kv;
                part = 2;
            }
        }
        const int heads = part ? a.kv : a.heads;
        const float *x = (part == 0 ? a.q : part == 1 ? a.k : a.v) + ((size_t)t * heads + head) * hd;
        float *y = part == 0 ? a.q_out : part == 1 ? a.k_out : nullptr;
        if (y) y += ((size_t)t * heads + head) * hd;
        typename E::T *c = nullptr;
        float scale = 1.0f;
        if (part && a.slots) {
            const int slot = kv_slot(p, a.slots, t);
            if (slot >= 0) {
                c = static_cast<typename E::T *>(part == 1 ? p.k : p.v) +
                    kv_at(p, slot >> p.page_log2, head, slot & (p.page - 1));
                scale = part == 1 ? p.k_scale : p.v_scale;
            }
        }
        auto put = [&](int i, float v) {
            if (y) y[i] = v;
            if (c) c[i] = E::put(v, scale);
        };
        const int n_rot = part == 2 ? 0 : R;
        for (int i = tid; i < hd - n_rot; i += 128) {
            if (i >= n_rot) {
                const int d = i + n_rot;
                put(d, x[d]);
                continue;
            }
            const float2 cs = rope_cs(a, t, i);
            const int i0 = a.halves ? i : 2 * i, i1 = a.halves ? i + R : 2 * i + 1;
            const float u = x[i0], v = x[i1];
            put(i0, u * cs.x - v * cs.y);
            put(i1, u * cs.y + v * cs.x);
        }
    }
}

// Four elements rounded to the cache's type, in one store.
template <int TYPE>
__device__ __forceinline__ void put4(typename KvElem<TYPE>::T *c, v4f x, float scale)
{
    typedef typename KvElem<TYPE>::T T;
    typedef T vec __attribute__((ext_vector_type(4)));
    vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = KvElem<TYPE>::put(x[i], scale);
    *reinterpret_cast<vec *>(c) = v;
}

// Work groups (token, share of its items): an item is a float4 of a row, with
// HALVES two float4s of one (pairs p..p+3 lie R apart).  The first items are on
// their way while the group forms the token's cosines and sines in LDS, once
// for all its heads.
//
// Bound by memory: 4099 tokens of 32 + 8 heads of 128 move 168 MB in 33 us (5.0
// TB/s), 8190 with the append to e4m3 352 MB in 68 us (5.2 TB/s; a copy 4.7); the
// division by the scale there takes 0.7 us more than a product, of 512 tokens 0.3.
// One item per thread at a time and eight groups per CU: with two items (and
// 64 registers) 39 and 83 us, with four and five groups 46 and 103 us.
constexpr int RT = 256;
constexpr int MAX_GROUPS = 1 << 20;  // of a launch; more tokens take turns

template <int TYPE, bool HALVES>
__global__ void __launch_bounds__(RT, 8) k_rope_append(ornk_kv_pages p, ornk_rope_args a)
{
    __shared__ __align__(16) float2 cs[ORN_ROPE_MAX_PAIRS];
    const int tid = threadIdx.x, hd = a.hd, R = a.R;
    const int nr = (HALVES ? hd - R : hd) / 4, nv = hd / 4;  // items of a rotated row, of a value row
    const int rot = (a.heads + a.kv) * nr, items = rot + (a.slots ? a.kv * nv : 0);
    const int i0 = (int)((long long)items * blockIdx.y / gridDim.y);
    const int i1 = (int)((long long)items * (blockIdx.y + 1) / gridDim.y);

    struct Item {
        v4f x, y;    // y: the other half
        int row, c;  // row: query heads, key heads, value heads; first element
        bool two;
    };
    auto load = [&](Item &it, int t, int i) {
        if (i < rot) {
            it.row = i / nr;
            it.c = 4 * (i - it.row * nr);
            it.two = HALVES && it.c < R;
            if (HALVES && !it.two) it.c += R;
        } else {
            i -= rot;
            it.row = i / nv;
            it.c = 4 * (i - it.row * nv);
            it.row += a.heads + a.kv;
            it.two = false;
        }
        const float *x;
        if (it.row < a.heads) x = a.q + ((size_t)t * a.heads + it.row) * hd;
        else if (it.row < a.heads + a.kv) x = a.k + ((size_t)t * a.kv + it.row - a.heads) * hd;
        else x = a.v + ((size_t)t * a.kv + it.row - a.heads - a.kv) * hd;
        it.x = *reinterpret_cast<const v4f *>(x + it.c);
        if (it.two) it.y = *reinterpret_cast<const v4f *>(x + it.c + R);
    };
    for (long long at = blockIdx.x; at < a.T; at += gridDim.x) {
        const int t = (int)at;
        Item it;
        if (i0 + tid < i1) load(it, t, i0 + tid);
        for (int i = tid; i < R; i += RT) cs[i] = rope_cs(a, t, i);
        const int slot = a.slots ? kv_slot(p, a.slots, t) : -1;
        __syncthreads();
        for (int i = i0 + tid; i < i1; i += RT) {
            if (i != i0 + tid) load(it, t, i);
            const int kvh = it.row - a.heads;  // key heads, then value heads
            v4f x = it.x, y = it.y;
            if (kvh < a.kv) {
                if (HALVES) {
                    if (it.two) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 r = cs[it.c + e];
                            x[e] = it.x[e] * r.x - it.y[e] * r.y;
                            y[e] = it.x[e] * r.y + it.y[e] * r.x;
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        if (it.c + e >= 2 * R) continue;  // past the last pair
                        const float2 r = cs[(it.c + e) / 2];
                        x[e] = it.x[e] * r.x - it.x[e + 1] * r.y;
                        x[e + 1] = it.x[e] * r.y + it.x[e + 1] * r.x;
                    }
                }
            }
            float *out = kvh < 0 ? a.q_out + ((size_t)t * a.heads + it.row) * hd
                         : kvh < a.kv && a.k_out ? a.k_out + ((size_t)t * a.kv + kvh) * hd : nullptr;
            if (out) {
                *reinterpret_cast<v4f *>(out + it.c) = x;
                if (it.two) *reinterpret_cast<v4f *>(out + it.c + R) = y;
            }
            if (kvh >= 0 && slot >= 0) {
                typedef typename KvElem<TYPE>::T T;
                const bool key = kvh < a.kv;
                T *c = static_cast<T *>(key ? p.k : p.v) +
                       kv_at(p, slot >> p.page_log2, key ? kvh : kvh - a.kv, slot & (p.page - 1)) + it.c;
                put4<TYPE>(c, x, key ? p.k_scale : p.v_scale);
                if (it.two) put4<TYPE>(c + R, y, p.k_scale);
            }
        }
        __syncthreads();  // the token's angles are consumed
    }
}

template <int TYPE>
int launch(const ornk_kv_pages &p, const ornk_rope_args &a, hipStream_t s)
{
    const int rows = a.heads + a.kv * (a.slots ? 2 : 1);
    if (a.hd % 4 || (a.halves && a.R % 4)) {
        const long long n = (long long)a.T * rows;
        hipLaunchKernelGGL(k_rope_append_any<TYPE>, dim3((unsigned)(n < MAX_GROUPS ? n : MAX_GROUPS)),
                           dim3(128), 0, s, p, a, rows);
        return hipGetLastError();
    }
    // A token's items in one group, so that its angles are formed once, unless
    // the tokens leave CUs without one; then in as many as have RT items each.
    const long long items = (long long)rows * (a.hd / 4);
    long long y = (items + RT - 1) / RT;
    if (y * a.T > 512) y = a.T < 512 ? 512 / a.T : 1;
    const dim3 grid(a.T < MAX_GROUPS ? a.T : MAX_GROUPS, (unsigned)(y < 1 ? 1 : y));
    if (a.halves)
        hipLaunchKernelGGL((k_rope_append<TYPE, true>), grid, dim3(RT), 0, s, p, a);
    else
        hipLaunchKernelGGL((k_rope_append<TYPE, false>), grid, dim3(RT), 0, s, p, a);
    return hipGetLastError();
}

}  // namespace

extern "C" int ornk_rope_append(const ornk_kv_pages *pp, const ornk_rope_args *a, hipStream_t s)
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
