// SPDX-License-Identifier: MIT
//
// Attention of one new token per sequence over the paged key-value cache
// (ornith_hip.h): out = sum_t w_t V[t], w = softmax(scale * q . K[t]), the sums
// over the sequence's tokens, query heads sharing kv heads.
#include "kv.h"

namespace {

constexpr int WAVES = 4;

struct AttendWs {
    float *s;   // [n_seqs][heads][max_len] scores (only where the weights are asked for)
    float2 *ml; // [n_seqs][heads] maximum and sum
};

// One work group per sequence and query head.
template <int TYPE>
__global__ void __launch_bounds__(64 * WAVES) k_kv_attend(ornk_kv_pages p, ornk_attend_args a,
                                                          AttendWs w)
{
    typedef KvElem<TYPE> E;
    __shared__ float so[WAVES][256], sm[WAVES], sl[WAVES];
    const int b = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = head / (a.heads / p.kv), hd = p.hd;
    const int len = kv_len(p, a.lens, b, a.max_len);
    const float *q = a.q + ((size_t)b * a.heads + head) * hd;
    float qr[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        qr[j] = lane + 64 * j < hd ? q[lane + 64 * j] * a.scale * p.k_scale : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int t = wave; t < len; t += WAVES) {
        const int page = kv_page(p, a.table[(size_t)b * a.max_pages + (t >> p.page_log2)], b);
        float sc = -INFINITY;
        const size_t at = page < 0 ? 0 : kv_at(p, page, h, t & (p.page - 1));
        if (page >= 0) {
            const typename E::T *k = static_cast<const typename E::T *>(p.k) + at;
            sc = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (lane + 64 * j < hd) sc = fmaf(qr[j], E::get(k[lane + 64 * j]), sc);
            sc = orn_wave_sum(sc);
        }
        if (w.s && lane == 0) w.s[((size_t)b * a.heads + head) * a.max_len + t] = sc;
        if (page < 0) continue;
        const float mn = fmaxf(m, sc);
        const bool none = mn == -INFINITY;
        const float corr = none ? 1.0f : expf(m - mn), pr = none ? 0.0f : expf(sc - mn);
        l = l * corr + pr;
        m = mn;
        const typename E::T *v = static_cast<const typename E::T *>(p.v) + at;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < hd) o[j] = fmaf(pr, E::get(v[lane + 64 * j]), o[j] * corr);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) so[wave][lane + 64 * j] = o[j];
    if (lane == 0) {
        sm[wave] = m;
        sl[wave] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int i = 0; i < WAVES; ++i) M = fmaxf(M, sm[i]);
    float acc = 0.0f;
    for (int i = 0; i < WAVES; ++i) {
        const float f = sm[i] == -INFINITY ? 0.0f : expf(sm[i] - M);
        L += sl[i] * f;
        acc += so[i][tid] * f;
    }
    if (tid < hd)
        a.out[((size_t)b * a.heads + head) * hd + tid] = L != 0.0f ? acc / L * p.v_scale : 0.0f;
    if (w.s && tid == 0) w.ml[(size_t)b * a.heads + head] = make_float2(M, L);
}

// The weights each token got, summed over a kv head's query heads.
__global__ void k_kv_score(ornk_kv_pages p, ornk_attend_args a, AttendWs w)
{
    const int t = blockIdx.x * blockDim.x + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    if (t >= kv_len(p, a.lens, b, a.max_len)) return;
    const int G = a.heads / p.kv;
    float sum = 0.0f;
    for (int g = 0; g < G; ++g) {
        const size_t row = (size_t)b * a.heads + h * G + g;
        const float2 ml = w.ml[row];
        const float s = w.s[row * a.max_len + t];
        sum += s == -INFINITY ? 0.0f : expf(s - ml.x) / ml.y;
    }
    const size_t i = ((size_t)b * p.kv + h) * a.score_stride + t;
    a.score_out[i] = a.score_in ? fmaf(a.decay, a.score_in[i], sum) : sum;
}

}  // namespace

extern "C" size_t ornk_kv_attend_ws(const ornk_kv_pages *p, const ornk_attend_args *a)
{
    if (!a->score_out) return 0;
    const size_t rows = (size_t)a->n_seqs * a->heads;
    return rows * 8 + rows * a->max_len * 4;
}

extern "C" int ornk_kv_attend(const ornk_kv_pages *p, const ornk_attend_args *a, hipStream_t s)
{
    AttendWs w = {};
    if (a->score_out) {
        w.ml = static_cast<float2 *>(a->ws);
        w.s = reinterpret_cast<float *>(w.ml + (size_t)a->n_seqs * a->heads);
    }
    const dim3 grid(a->n_seqs, a->heads), block(64 * WAVES);
    switch (p->type) {
    case ORN_KV_F32: hipLaunchKernelGGL(k_kv_attend<ORN_KV_F32>, grid, block, 0, s, *p, *a, w); break;
    case ORN_KV_F16: hipLaunchKernelGGL(k_kv_attend<ORN_KV_F16>, grid, block, 0, s, *p, *a, w); break;
    case ORN_KV_BF16: hipLaunchKernelGGL(k_kv_attend<ORN_KV_BF16>, grid, block, 0, s, *p, *a, w); break;
    default: hipLaunchKernelGGL(k_kv_attend<ORN_KV_E4M3>, grid, block, 0, s, *p, *a, w); break;
    }
    if (a->score_out && a->max_len)
        hipLaunchKernelGGL(k_kv_score, dim3((a->max_len + 255) / 256, p->kv, a->n_seqs), dim3(256),
                           0, s, *p, *a, w);
    return hipGetLastError();
}
