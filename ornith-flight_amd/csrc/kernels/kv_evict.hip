// SPDX-License-Identifier: MIT
//
// Eviction from the paged key-value cache by accumulated attention weight
// (ornith_hip.h): per sequence and kv head the tokens that stay are chosen
// (k_evict_choose) and moved to the front of the destination pages
// (k_evict_move).
#include "kv.h"

namespace {

constexpr int CT = 1024;  // threads of the choosing work group

// Order of the scores as unsigned integers: a NaN is 0, -0 counts as +0.
__device__ __forceinline__ uint32_t order_key(float f)
{
    if (f != f) return 0u;
    const uint32_t u = __float_as_uint(f + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One work group per kv head and sequence.  Where the tokens are more than
// `keep`, four rounds of eight bits find the key of the lowest score that
// stays and how many of its equals do; a last pass numbers the kept tokens in
// order.
__global__ void __launch_bounds__(CT) k_evict_choose(ornk_kv_pages p, ornk_evict_args a)
{
    __shared__ int hist[256], wsum[CT / 64], sh[2];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = kv_len(p, a.lens, b, a.max_len), n = min(len, a.keep);
    const float *score = a.score + ((size_t)b * p.kv + h) * a.score_stride;
    float *ds = a.dst_score ? a.dst_score + ((size_t)b * p.kv + h) * a.dst_stride : nullptr;
    int *kept = a.kept + ((size_t)b * p.kv + h) * a.keep;
    if (h == 0 && tid == 0) a.counts[b] = n;
    const int lo = a.sink, hi = len - a.recent;  // the tokens that the scores decide on
    uint32_t key = 0;                            // the lowest key that stays
    int ties = 0;                                // and how many tokens of that key
    if (len > a.keep) {
        int left = a.keep - a.sink - a.recent;
        if (left == 0) {
            key = 0xffffffffu;  // above every key
        } else {
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = tid; i < 256; i += CT) hist[i] = 0;
                __syncthreads();
                for (int i = lo + tid; i < hi; i += CT) {
                    const uint32_t k = order_key(score[i]);
                    if (shift == 24 || k >> (shift + 8) == key >> (shift + 8))
                        atomicAdd(&hist[(k >> shift) & 255], 1);
                }
                __syncthreads();
                if (tid == 0) {
                    int d = 255, above = 0;
                    while (d > 0 && above + hist[d] < left) above += hist[d--];
                    sh[0] = d;
                    sh[1] = above;
                }
                __syncthreads();
                key |= (uint32_t)sh[0] << shift;
                left -= sh[1];
                __syncthreads();
            }
            ties = left;
        }
    }
    int base = 0, eq_base = 0;  // kept for certain, and ties, before this stretch
    for (int i0 = 0; i0 < len; i0 += CT) {
        const int i = i0 + tid;
        const float f = i < len ? score[i] : 0.0f;
        bool sure = false, tie = false;
        if (i < len) {
            const uint32_t k = order_key(f);
            sure = len <= a.keep || i < lo || i >= hi || k > key;
            tie = !sure && ties && k == key;
        }
        const uint64_t bs = __ballot(sure), bt = __ballot(tie);
        if (lane == 0) wsum[wave] = __popcll(bs) | __popcll(bt) << 16;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < CT / 64; ++w) {
            if (w < wave) before += wsum[w];
            all += wsum[w];
        }
        const uint64_t mask = ((uint64_t)1 << lane) - 1;
        const int eq = eq_base + (before >> 16) + __popcll(bt & mask);
        const int at = base + (before & 0xffff) + __popcll(bs & mask) + min(eq, ties);
        // every score of this stretch has been read: an earlier place may be written
        if (sure || (tie && eq < ties)) {
            kept[at] = i;
            if (ds) ds[at] = f;
        }
        base += all & 0xffff;
        eq_base += all >> 16;
        __syncthreads();
    }
    for (int i = n + tid; i < a.keep; i += CT) kept[i] = -1;
}

// One work group per kv head, sequence and K or V.  Within a sequence's own
// pages a row moves towards the front or stays, so a stretch of rows is read
// before any of it is written and nothing that a later stretch reads is.
__global__ void __launch_bounds__(256) k_evict_move(ornk_kv_pages p, ornk_evict_args a, int row_bytes)
{
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int n = a.counts[b];
    const int *kept = a.kept + ((size_t)b * p.kv + h) * a.keep;
    uint8_t *pool = static_cast<uint8_t *>(blockIdx.z ? p.v : p.k);
    if (h == 0 && blockIdx.z == 0 && tid == 0) a.dst_lens[b] = n;
    const size_t es = row_bytes / p.hd;
    auto row = [&](const int *table, int pages, int i) {
        const int page = kv_page(p, table[(size_t)b * pages + (i >> p.page_log2)], b);
        return page < 0 ? nullptr : pool + kv_at(p, page, h, i & (p.page - 1)) * es;
    };
    for (int j = 0; j < n; ++j) {
        const uint8_t *from = row(a.table, a.max_pages, kept[j]);
        uint8_t *to = row(a.dst_table, a.dst_pages, j);
        uint8_t v[4];
        if (from && to)
            for (int i = tid, k = 0; i < row_bytes; i += 256, ++k) v[k] = from[i];
        __syncthreads();
        if (from && to)
            for (int i = tid, k = 0; i < row_bytes; i += 256, ++k) to[i] = v[k];
        __syncthreads();
    }
}

}  // namespace

extern "C" int ornk_kv_evict(const ornk_kv_pages *p, const ornk_evict_args *a, hipStream_t s)
{
    if (a->n_seqs > 65535) return hipErrorInvalidValue;
    const int es = p->type == ORN_KV_F32 ? 4 : p->type == ORN_KV_E4M3 ? 1 : 2;
    hipLaunchKernelGGL(k_evict_choose, dim3(p->kv, a->n_seqs), dim3(CT), 0, s, *p, *a);
    hipLaunchKernelGGL(k_evict_move, dim3(p->kv, a->n_seqs, 2), dim3(256), 0, s, *p, *a, es * p->hd);
    return hipGetLastError();
}
