// SPDX-License-Identifier: MIT
//
// Eviction from the paged key-value cache by accumulated attention weight
// (ornith_hip.h): per sequence and kv head the tokens that stay are chosen
// (k_evict_choose) and moved to the front of the destination pages
// (k_evict_move).
#include "kv.h"

namespace {

constexpr int CT = 1024;  // threads of the choosing work group
constexpr int BINS = 2048;

// Order of the scores as unsigned integers: a NaN is 0, -0 counts as +0.
__device__ __forceinline__ uint32_t order_key(float f)
{
    const uint32_t u = __float_as_uint(f + 0.0f);
    return f != f ? 0u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
// One work group per kv head and sequence; a thread holds PER scores of a
// stretch of CT * PER, every CT-th one.  Where the tokens are more than `keep`,
// up to three rounds of counting (11, 11 and 10 bits of the keys, from the top)
// find the lowest key that stays and how many of its equals do; then one scan over
// the waves' counts numbers the kept tokens in order.  Sequences longer than a
// stretch read their scores (from L2) again in every round.
//
// Up to 4096 tokens bound by latency: lengths, scores, then a dozen barriers, 7 us
// for one sequence or 64; beyond by the instructions of one CU, about 30 per score
// and round (one sequence, with the move of few tokens into other pages: 4096 11 us, 8192 14, 16,384
// 20, 32,768 33, 131,072 97).  PER 4 up to 4096 tokens (8: 12 us) and 8 beyond (4:
// 8192 15 us; 16 and 32 hold longer sequences, for 19.5 and 31.5 us at 16,384 and
// 32,768, but take 16 and 21 us at 8192, as what is unrolled is run).
template <int PER>
__global__ void __launch_bounds__(CT) k_evict_choose(ornk_kv_pages p, ornk_evict_args a)
{
    constexpr int NW = CT / 64, NC = PER * NW;  // waves; counts of a stretch
    __shared__ uint32_t hist[3][BINS], wsum[2][NW], sh[3];
    __shared__ uint2 count[NC];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int len = kv_len(p, a.lens[b], b, a.max_len), n = min(len, a.keep);
    const float *score = a.score + ((size_t)b * p.kv + h) * a.score_stride;
    float *ds = a.dst_score ? a.dst_score + ((size_t)b * p.kv + h) * a.dst_stride : nullptr;
    int *kept = a.kept + ((size_t)b * p.kv + h) * a.keep;
    if (h == 0 && tid == 0) a.counts[b] = n;
    // the tokens that the scores decide on: `some` from `lo` on
    const int lo = a.sink;
    const uint32_t some = len > a.keep ? len - a.recent - lo : 0;
    const bool one = len <= CT * PER;
    float f[PER];
    auto load = [&](int i0) {  // (lengths leave room for a stretch below 2^31)
#pragma unroll
        for (int e = 0; e < PER; ++e) f[e] = score[min(i0 + e * CT + tid, len - 1)];
    };
    // the sums of x and y over the work group's threads before this one
    auto before = [&](uint32_t &x, uint32_t &y) {
        const uint32_t sx = wave_scan(x), sy = wave_scan(y);
        if (lane == 63) wsum[0][wave] = sx, wsum[1][wave] = sy;
        __syncthreads();
        x = sx - x;
        y = sy - y;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            x += w < wave ? wsum[0][w] : 0;
            y += w < wave ? wsum[1][w] : 0;
        }
    };

    uint32_t key = 0;  // the lowest key that stays
    int ties = 0;      // and how many tokens of that key
    if (one && len) load(0);
    if (some) {
        for (int i = tid; i < 3 * BINS; i += CT) hist[i / BINS][i % BINS] = 0;
        __syncthreads();
        int left = a.keep - a.sink - a.recent;
        if (left == 0) key = 0xffffffffu;  // above every key
#pragma unroll 1
        for (int round = 0; round < 3 && left; ++round) {
            const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
            const uint32_t mask = round == 2 ? 1023u : 2047u;
            const uint32_t width = round == 0 ? ~0u : round == 1 ? (1u << 21) - 1 : 1023u;
            uint32_t *bins = hist[round];
            for (int i0 = 0; i0 < len; i0 += CT * PER) {
                if (!one) load(i0);
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    if (i0 + e * CT >= len) break;
                    const uint32_t k = order_key(f[e]);
                    if ((uint32_t)(i0 + e * CT + tid - lo) < some && k - key <= width)
                        atomicAdd(&bins[(k >> shift) & mask], 1u);
                }
            }
            __syncthreads();
            // two bins a thread, from the highest down: one holds the key that is `left` from the top
            const int d = BINS - 2 - 2 * tid;
            const int c0 = bins[d], c1 = bins[d + 1];
            uint32_t sum = c0 + c1, none = 0;
            before(sum, none);
            const int above = sum;
            if (above < left && left <= above + c1) sh[0] = d + 1, sh[1] = above, sh[2] = c1;
            else if (above + c1 < left && left <= above + c1 + c0) sh[0] = d, sh[1] = above + c1, sh[2] = c0;
            __syncthreads();
            key |= sh[0] << shift;
            left -= sh[1];
            if ((int)sh[2] == left) {  // every one of this bin stays: those above the key before it
                key -= 1;
                left = 0;
            }
        }
        ties = left;
    }
    int base = 0, eq_base = 0;  // kept for certain, and ties, before this stretch
    for (int i0 = 0; i0 < len; i0 += CT * PER) {
        if (!one) load(i0);
        uint64_t sure = 0, tie = 0;  // bit e
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int i = i0 + e * CT + tid;
            const uint32_t k = order_key(f[e]);
            const bool open = (uint32_t)(i - lo) < some;
            const bool s = i < len && (!open || k > key);
            const bool t = open && k == key;
            const uint64_t bs = __ballot(s), bt = __ballot(t);
            if (lane == 0) count[e * NW + wave] = make_uint2(__popcll(bs), __popcll(bt));
            sure |= (uint64_t)s << e;
            tie |= (uint64_t)t << e;
        }
        __syncthreads();  // also: every score of this stretch has been read
        const uint2 c = tid < NC ? count[tid] : make_uint2(0, 0);
        uint32_t cs = c.x, ct = c.y;
        before(cs, ct);
        if (tid < NC) count[tid] = make_uint2(cs, ct);
        if (tid == CT - 1) sh[0] = cs + c.x, sh[1] = ct + c.y;
        __syncthreads();
        const uint64_t mine = ((uint64_t)1 << lane) - 1;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const bool s = sure >> e & 1, t = tie >> e & 1;
            const uint64_t bs = __ballot(s), bt = __ballot(t);
            if (!(bs | bt)) continue;
            const uint2 c = count[e * NW + wave];
            const int eq = eq_base + (int)c.y + __popcll(bt & mine);
            if (s || (t && eq < ties)) {
                const int j = base + (int)c.x + __popcll(bs & mine) + min(eq, ties);
                kept[j] = i0 + e * CT + tid;
                if (ds) ds[j] = f[e];
            }
        }
        base += sh[0];
        eq_base += sh[1];
        __syncthreads();
    }
    for (long long i = n + tid; i < a.keep; i += CT) kept[i] = -1;
}

// The kept rows to their new places, in words of WORD.  A work group takes rows
// of one kv head, sequence and K or V, a stretch at a time: the rows' places go
// through LDS, then every thread has up to MB words in flight.
//
// Into other pages, each group takes one stretch of whole rows, up to MAX_GROUPS of
// them a launch (rows of 129 words and more have stretches of 4).  Within a
// sequence's own pages (IN_PLACE) a row moves towards the front or stays: a
// group takes every row, one stretch after the other, of SLICE bytes of the
// columns; a stretch is read whole before any of it is written, and no later
// stretch reads what it writes.
//
// Bound by memory: 32 sequences' up to 4096 rows of 8 kv heads of 128 in f16, 0.94
// GB read and written, take 198 us (4.75 TB/s; a copy 4.72); 2048 rows of 2 heads
// of 256 in bf16, 8.4 MB, 4.4 us, most of them the start and the chain of kept,
// table and row.  IN_PLACE it is bound by that chain, one stretch after the other in
// few groups: with the choice, the 32 sequences take 275 us (into other pages 218),
// 2048 rows of 2 heads of 256 24 (12), 16,384 rows 168 (43), 65,536 rows 640 (159).
// The words are a vector type of the compiler: a struct of four was put into LDS with
// a wait after each load (17 us).
constexpr int MT = 256, MB = 4, SLICE = 64;
constexpr int MAX_GROUPS = 1 << 20;  // of a launch's x: 2^28 threads

// Rows of a stretch, of `words` words each (at most MT): MB for every thread.
__host__ __device__ inline int stretch_rows(int words)
{
    const int n = MB * (MT / words);
    return n < MT ? n : MT;
}

template <class WORD, bool IN_PLACE>
__global__ void __launch_bounds__(MT) k_evict_move(ornk_kv_pages p, ornk_evict_args a, int row_bytes,
                                                    int group0)
{
    constexpr int WB = sizeof(WORD);
    __shared__ size_t from[MT], to[MT];  // bytes into the pages; NONE: the row stays where it is
    constexpr size_t NONE = ~(size_t)0;
    const int h = blockIdx.y % p.kv, b = blockIdx.z, tid = threadIdx.x;
    const int *kept = a.kept + ((size_t)b * p.kv + h) * a.keep;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) a.dst_lens[b] = a.counts[b];
    const int es = row_bytes / p.hd, most = min(a.keep, a.max_len);
    const int c0 = IN_PLACE ? blockIdx.x * SLICE : 0;
    const int words = (IN_PLACE ? min(SLICE, row_bytes - c0) : row_bytes) / WB;
    const int pass = MT / words, mr = stretch_rows(words);
    const int r0 = tid / words < pass ? tid / words : MT, col = tid % words * WB;
    uint8_t *pool = static_cast<uint8_t *>(blockIdx.y >= p.kv ? p.v : p.k) + c0;
    for (int j0 = IN_PLACE ? 0 : (group0 + blockIdx.x) * mr; j0 < most; j0 += mr) {
        const int rows = min(mr, most - j0);
        int some = 0;  // (kept is -1 past the sequence's last)
        if (tid < rows) {
            const int j = j0 + tid, i = kept[j];
            some = i >= 0;
            size_t f = NONE, t = NONE;
            if (some && !(IN_PLACE && i == j)) {
                const int pf = kv_page(p, a.table[(size_t)b * a.max_pages + (i >> p.page_log2)], b);
                const int pt = kv_page(p, a.dst_table[(size_t)b * a.dst_pages + (j >> p.page_log2)], b);
                if (pf >= 0 && pt >= 0) {
                    f = kv_at(p, pf, h, i & (p.page - 1)) * es;
                    t = kv_at(p, pt, h, j & (p.page - 1)) * es;
                }
            }
            from[tid] = f;
            to[tid] = t;
        }
        if (!__syncthreads_or(some)) break;
        WORD v[MB];
        size_t f[MB];
#pragma unroll
        for (int k = 0; k < MB; ++k) {
            const int r = r0 + k * pass;
            f[k] = r < rows ? from[r] : NONE;
        }
#pragma unroll
        for (int k = 0; k < MB; ++k)
            if (f[k] != NONE) v[k] = *reinterpret_cast<const WORD *>(pool + f[k] + col);
        if (IN_PLACE) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < MB; ++k)
            if (f[k] != NONE) *reinterpret_cast<WORD *>(pool + to[r0 + k * pass] + col) = v[k];
        if (!IN_PLACE) break;
        __syncthreads();
    }
}

template <class WORD>
void move(const ornk_kv_pages &p, const ornk_evict_args &a, int row_bytes, hipStream_t s)
{
    const int most = a.keep < a.max_len ? a.keep : a.max_len;
    const unsigned y = 2 * p.kv, z = a.n_seqs;
    if (a.in_place) {
        hipLaunchKernelGGL((k_evict_move<WORD, true>), dim3((row_bytes + SLICE - 1) / SLICE, y, z),
                           dim3(MT), 0, s, p, a, row_bytes, 0);
        return;
    }
    const int mr = stretch_rows(row_bytes / (int)sizeof(WORD));
    const int x = most ? (most + mr - 1) / mr : 1;
    for (int x0 = 0; x0 < x; x0 += MAX_GROUPS)
        hipLaunchKernelGGL((k_evict_move<WORD, false>), dim3(x - x0 < MAX_GROUPS ? x - x0 : MAX_GROUPS, y, z),
                           dim3(MT), 0, s, p, a, row_bytes, x0);
}

}  // namespace

extern "C" int ornk_kv_evict(const ornk_kv_pages *p, const ornk_evict_args *a, hipStream_t s)
{
    const int rb = p->hd * (p->type == ORN_KV_F32 ? 4 : p->type == ORN_KV_E4M3 ? 1 : 2);
    if (a->max_len <= 4 * CT)
        hipLaunchKernelGGL(k_evict_choose<4>, dim3(p->kv, a->n_seqs), dim3(CT), 0, s, *p, *a);
    else
        hipLaunchKernelGGL(k_evict_choose<8>, dim3(p->kv, a->n_seqs), dim3(CT), 0, s, *p, *a);
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    if (rb % 16 == 0) move<u4>(*p, *a, rb, s);
    else if (rb % 4 == 0) move<uint32_t>(*p, *a, rb, s);
    else if (rb % 2 == 0) move<uint16_t>(*p, *a, rb, s);
    else move<uint8_t>(*p, *a, rb, s);
    return hipGetLastError();
}
