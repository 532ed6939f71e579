// SPDX-License-Identifier: MIT
//
// Device-side view of the paged key-value cache: element types, checked page
// numbers and rotary angles.  Only included from .hip translation units.
#pragma once

#include "../../../include/ornith/ornith_hip.h"
#include "common.h"
#include "launch.h"

template <int TYPE>
struct KvElem;
template <>
struct KvElem<ORN_KV_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(T x) { return x; }
    static __device__ __forceinline__ T put(float x, float) { return x; }
};
template <>
struct KvElem<ORN_KV_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float get(T x) { return (float)x; }
    static __device__ __forceinline__ T put(float x, float) { return (T)x; }
};
template <>
struct KvElem<ORN_KV_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float get(T x) { return (float)x; }
    static __device__ __forceinline__ T put(float x, float) { return (T)x; }
};
template <>
struct KvElem<ORN_KV_E4M3> {
    typedef uint8_t T;
    static __device__ __forceinline__ float get(T x)
    {
        return __builtin_amdgcn_cvt_f32_fp8((int)x, 0);
    }
    // the quotient in fp32 (a rounded 1 / scale would round twice, and move values
    // next to a middle of two); clamped by comparisons, which leave a NaN one
    static __device__ __forceinline__ T put(float x, float scale)
    {
        x /= scale;
        x = x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x;
        return (T)(__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xff);
    }
};

// Records the first argument out of range that a thread meets (any one of
// several threads'; host memory, read after the stream has ended).
__device__ __forceinline__ void kv_error(const ornk_kv_pages &p, int what, int at)
{
    *(volatile int *)(p.err + what) = 1 + at;
}

// Sequence b's length within [0, max_len].
__device__ __forceinline__ int kv_len(const ornk_kv_pages &p, int n, int b, int max_len)
{
    if (n >= 0 && n <= max_len) return n;
    kv_error(p, ORNK_KV_ERR_LEN, b);
    return n < 0 ? 0 : max_len;
}

// A table entry: the page, or -1 where it is none.
__device__ __forceinline__ int kv_page(const ornk_kv_pages &p, int id, int b)
{
    if ((unsigned)id < (unsigned)p.n_pages) return id;
    kv_error(p, ORNK_KV_ERR_PAGE, b);
    return -1;
}

// First element of slot i of a page, for one kv head.
__device__ __forceinline__ size_t kv_at(const ornk_kv_pages &p, int page, int h, int i)
{
    return ((((size_t)page * p.kv + h) << p.page_log2) + i) * p.hd;
}

// Token t's slot, -1 where it is not stored.
__device__ __forceinline__ int kv_slot(const ornk_kv_pages &p, const int *slots, int t)
{
    const int slot = slots[t];
    if (slot >= 0 && slot < p.n_pages * p.page) return slot;
    if (slot != -1) kv_error(p, ORNK_KV_ERR_SLOT, t);
    return -1;
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

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x)
{
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return x;
}
