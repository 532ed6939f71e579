// SPDX-License-Identifier: MIT
//
// Rotary positions of several axes, and the append to the paged key-value
// cache (ornith_hip.h).
#include "kv.h"

namespace {

// One work group per token and head: query heads, key heads, value heads.
template <int TYPE>
__global__ void __launch_bounds__(128) k_kv_append(ornk_kv_pages p, ornk_rope_args a)
{
    typedef KvElem<TYPE> E;
    const int t = blockIdx.x, tid = threadIdx.x, hd = a.hd, R = a.R;
    int head = blockIdx.y, part = 0;  // 0 query, 1 key, 2 value
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
    float inv = 1.0f;
    if (part && a.slots) {
        const int slot = a.slots[t];
        if (slot >= 0 && slot < p.n_pages * p.page) {
            c = static_cast<typename E::T *>(part == 1 ? p.k : p.v) +
                kv_at(p, slot >> p.page_log2, head, slot & (p.page - 1));
            inv = 1.0f / (part == 1 ? p.k_scale : p.v_scale);
        } else if (slot != -1) {
            kv_error(p, ORNK_KV_ERR_SLOT, t);
        }
    }
    auto put = [&](int i, float v) {
        if (y) y[i] = v;
        if (c) c[i] = E::put(v, inv);
    };
    const int n_rot = part == 2 ? 0 : R;
    for (int i = tid; i < hd - n_rot; i += 128) {
        if (i >= n_rot) {
            const int d = i + n_rot;
            put(d, x[d]);
            continue;
        }
        const double turn = (double)a.pos[(size_t)a.axis[i] * a.T + t] * a.turns[i];
        float s, co;
        sincospif(2.0f * (float)(turn - rint(turn)), &s, &co);
        const int i0 = a.halves ? i : 2 * i, i1 = a.halves ? i + R : 2 * i + 1;
        const float u = x[i0], v = x[i1];
        put(i0, u * co - v * s);
        put(i1, u * s + v * co);
    }
}

}  // namespace

extern "C" int ornk_rope_append(const ornk_kv_pages *pp, const ornk_rope_args *a, hipStream_t s)
{
    ornk_kv_pages p = {};
    if (pp) p = *pp;
    const int rows = a->heads + a->kv * (a->slots ? 2 : 1);
    // a grid's y ends at 65535
    if (rows > 65535) return hipErrorInvalidValue;
    const dim3 grid(a->T, rows), block(128);
    switch (p.type) {
    case ORN_KV_F32: hipLaunchKernelGGL(k_kv_append<ORN_KV_F32>, grid, block, 0, s, p, *a); break;
    case ORN_KV_F16: hipLaunchKernelGGL(k_kv_append<ORN_KV_F16>, grid, block, 0, s, p, *a); break;
    case ORN_KV_BF16: hipLaunchKernelGGL(k_kv_append<ORN_KV_BF16>, grid, block, 0, s, p, *a); break;
    default: hipLaunchKernelGGL(k_kv_append<ORN_KV_E4M3>, grid, block, 0, s, p, *a); break;
    }
    return hipGetLastError();
}
