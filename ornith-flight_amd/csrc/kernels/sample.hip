// SPDX-License-Identifier: MIT
//
// A token for each row of logits by temperature, top-k, top-p and min-p (ornith_hip.h).
#include "../../../include/ornith/ornith_hip.h"
#include "common.h"
#include "launch.h"

namespace {

// A logit as a whole number of the same order; equal logits (-0 and 0) are equal, a
// NaN is the lowest with -infinity.
__device__ __forceinline__ uint32_t key_of(float x)
{
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 + 0 = 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^x for x <= 0 in 64 bits: the series of 2^f on [-1/2, 1/2], whose first term left
// out is below 2^-52.
__device__ __forceinline__ double exp2_of(double x)
{
    const double n = rint(x), f = x - n;
    double p = 2.5678435993488206e-11;  // ln(2)^12 / 12!
    p = fma(p, f, 4.4455382718708112e-10);
    p = fma(p, f, 7.0549116208011234e-09);
    p = fma(p, f, 1.0178086009239699e-07);
    p = fma(p, f, 1.3215486790144309e-06);
    p = fma(p, f, 1.5252733804059841e-05);
    p = fma(p, f, 1.5403530393381608e-04);
    p = fma(p, f, 1.3333558146428443e-03);
    p = fma(p, f, 9.6181291076284772e-03);
    p = fma(p, f, 5.5504108664821580e-02);
    p = fma(p, f, 2.4022650695910071e-01);
    p = fma(p, f, 6.9314718055994531e-01);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}

constexpr int NB = 1024;   // bins of a row's logits
constexpr int CAP = 8192;  // tokens that are put in order

// A row, its request and its largest logit.
struct Row {
    const float *x;
    int n;
    ornith_sample_request q;
    float u;
    float top;         // the largest logit
    uint32_t top_key;
    double per;        // log2(e) / temperature
    double unit;       // weights are whole multiples of 1 / unit; n of them fit 62 bits
    float scale;       // bins per logit
    float reach;       // tokens farther below the largest take no part in the order
    bool by_rank;      // the top_k are few: all of them are put in order, and bins only count
    uint32_t cut, ties;  // by passes: kept are keys above `cut`, and the first `ties` of it
};

// 2^((x - largest) log2(e) / temperature)
__device__ __forceinline__ double weight(const Row &r, float x)
{
    if (x == r.top) return 1.0;
    const double y = ((double)x - (double)r.top) * r.per;
    return y > -60.0 ? exp2_of(y) : 0.0;  // also where x is a NaN
}

__device__ __forceinline__ uint64_t fixed(const Row &r, double w) { return (uint64_t)(w * r.unit + 0.5); }

// Bins are equal stretches of the logits, the largest in bin 0.
__device__ __forceinline__ int bin_at(const Row &r, float below)
{
    const float b = below * r.scale;
    return b < (float)(NB - 1) ? (int)b : NB - 1;
}

__device__ __forceinline__ int bin_of(const Row &r, float x) { return x == r.top ? 0 : bin_at(r, r.top - x); }

__device__ __forceinline__ bool valid(const ornith_sample_request &q, float u)
{
    return q.temperature >= 0.0f && q.temperature < INFINITY && q.top_p >= 0.0f && q.top_p <= 1.0f &&
           q.min_p >= 0.0f && q.min_p <= 1.0f && u >= 0.0f && u < 1.0f;
}

__device__ __forceinline__ Row row_of(const ornk_sample_args &a, int row)
{
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.n = a.n;
    r.q = static_cast<const ornith_sample_request *>(a.requests)[row];
    r.u = a.u[row];
    r.unit = a.unit;
    r.cut = r.ties = 0;
    return r;
}

// The row's largest and least logits known: what the weights and bins need, and how far
// below the largest a border of the choice may lie, which is where the bins end:
// - a weight below 2^-53 of the largest is 0;
// - the tokens below (1 - top_p) / 2 n are less than half of what top_p leaves out;
// - min_p leaves out what is below it.
// Where the top_k are few the first alone holds; where they are many, too, since their
// own border may lie anywhere.
__device__ __forceinline__ void scale_row(Row &r, uint32_t top, uint32_t low)
{
    r.top_key = top;
    r.top = logit_of(top);
    const double T = r.q.temperature;
    r.per = 1.4426950408889634 / T;
    r.by_rank = r.q.top_k > 0 && r.q.top_k <= CAP / 2;
    r.reach = 37.0f * r.q.temperature;
    if (r.q.top_k <= 0 || r.q.top_k >= r.n) {
        r.by_rank = false;
        if (r.q.top_p < 1.0f)
            r.reach = fminf(r.reach, (float)(-log((1.0 - (double)r.q.top_p) / (2.0 * r.n)) * T));
        if (r.q.min_p > 0.0f) r.reach = fminf(r.reach, (float)(-log((double)r.q.min_p) * T * 1.0001));
    }
    const float all = r.top - logit_of(low);
    const float range = all < r.reach ? all : r.reach;
    const float s = (float)NB / range;
    r.scale = range > 0.0f ? s < 1e30f ? s : 1e30f : 0.0f;
}

// A logit's distance below the largest; a NaN counts as far.
__device__ __forceinline__ float below(const Row &r, float x) { return x == r.top ? 0.0f : r.top - x; }
__device__ __forceinline__ bool within(const Row &r, float x)
{
    return below(r, x) <= r.reach && x > -INFINITY;
}

__device__ __forceinline__ void put_result(const ornk_sample_args &a, int row, int token, float prob)
{
    a.tokens[row] = token;
    if (a.prob) a.prob[row] = prob;
}

__device__ __forceinline__ float share(const Row &r, double w, uint64_t all)
{
    return (float)(w * r.unit / (double)all);
}

// The largest (key, then the least index) and the least key of a row.
struct Ends {
    uint64_t top;  // key << 32 | ~index; 0: every logit is -infinity
    uint32_t low;
};

__device__ __forceinline__ void extend(Ends &e, float x, int i)
{
    const uint32_t key = key_of(x);
    if (!key) return;
    const uint64_t t = (uint64_t)key << 32 | (uint32_t)~i;
    e.top = t > e.top ? t : e.top;
    e.low = key < e.low ? key : e.low;
}

__device__ __forceinline__ Ends join(Ends a, Ends b)
{
    return {a.top > b.top ? a.top : b.top, a.low < b.low ? a.low : b.low};
}

template <int NT>
__device__ __forceinline__ Ends block_ends(Ends e, Ends *tmp)
{
    for (int o = 32; o; o >>= 1) e = join(e, {__shfl_xor(e.top, o, 64), __shfl_xor(e.low, o, 64)});
    __syncthreads();
    if (!(threadIdx.x & 63)) tmp[threadIdx.x >> 6] = e;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) e = join(e, tmp[i]);
    return e;
}

// ---- what bins decide ----------------------------------------------------------
// Sums of weights and numbers of tokens before each bin, and the bins whose tokens have
// to be put in order: those where a border of the choice may lie.
struct Bins {
    uint64_t w[NB + 1];
    uint32_t c[NB + 1];
    uint32_t marked[NB / 32];
    uint64_t tmp[16];
    uint32_t tmp32[16];
    int found;
    int min_lo, min_hi;  // min_p's border is in these
    bool by_k;           // top_k leaves some out
};

// w and c from each bin's own to what is before it.
template <int NT>
__device__ __forceinline__ void sums_before(Bins &s)
{
    constexpr int PER = NB / NT > 0 ? NB / NT : 1;
    const int tid = threadIdx.x, lane = tid & 63;
    const bool on = tid * PER < NB;
    uint64_t w = 0;
    uint32_t c = 0;
    uint64_t ws[PER];
    uint32_t cs[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        ws[i] = on ? s.w[tid * PER + i] : 0;
        cs[i] = on ? s.c[tid * PER + i] : 0;
        w += ws[i];
        c += cs[i];
    }
    uint64_t wi = w;
    uint32_t ci = c;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up(wi, o, 64);
        const uint32_t z = __shfl_up(ci, o, 64);
        if (lane >= o) wi += y, ci += z;
    }
    if (lane == 63) s.tmp[tid >> 6] = wi, s.tmp32[tid >> 6] = ci;
    __syncthreads();
    wi -= w, ci -= c;
    for (int i = 0; i < tid >> 6; ++i) wi += s.tmp[i], ci += s.tmp32[i];
    if (on) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s.w[tid * PER + i] = wi;
            s.c[tid * PER + i] = ci;
            wi += ws[i];
            ci += cs[i];
        }
        if (tid * PER + PER == NB) s.w[NB] = wi, s.c[NB] = ci;
    }
    __syncthreads();
}

// The bin in which the sum passes `limit`.  All threads; limit is below the whole.
template <int NT, class T>
__device__ __forceinline__ int find(Bins &s, const T *sum, T limit)
{
    for (int i = threadIdx.x; i < NB; i += NT)
        if (sum[i] <= limit && limit < sum[i + 1]) s.found = i;
    __syncthreads();
    const int f = s.found;
    __syncthreads();
    return f;
}

__device__ __forceinline__ void mark(Bins &s, int lo, int hi)
{
    for (int i = lo + (int)threadIdx.x; i <= hi; i += blockDim.x) atomicOr(&s.marked[i >> 5], 1u << (i & 31));
}

// top_p's share of a sum, as a number of units that the kept tokens reach
__device__ __forceinline__ uint64_t least_of(const Row &r, uint64_t all)
{
    const uint64_t p = (uint64_t)ceil((double)r.q.top_p * (double)all);
    return p < 1 ? 1 : p > all ? all : p;
}

__device__ __forceinline__ uint64_t target_of(const Row &r, uint64_t all)
{
    const uint64_t t = (uint64_t)((double)r.u * (double)all);
    return t < all ? t : all - 1;
}

// Intervals follow from bins alone: every sum below is known up to the bins marked.
template <int NT>
__device__ __forceinline__ void mark_bins(const Row &r, Bins &s)
{
    for (int i = threadIdx.x; i < NB / 32; i += NT) s.marked[i] = 0;
    const uint64_t all = s.w[NB];
    uint64_t lo = all, hi = all;
    s.by_k = r.q.top_k > 0 && (uint32_t)r.q.top_k < s.c[NB];
    __syncthreads();
    if (r.by_rank) {
        mark(s, 0, s.by_k ? find<NT, uint32_t>(s, s.c, (uint32_t)r.q.top_k - 1) : NB - 1);
        __syncthreads();
        return;
    }
    if (s.by_k) {
        const int b = find<NT, uint32_t>(s, s.c, (uint32_t)r.q.top_k - 1);
        mark(s, b, b);
        lo = s.w[b];
        hi = s.w[b + 1];
    }
    if (r.q.top_p < 1.0f) {
        const int b0 = find<NT, uint64_t>(s, s.w, (lo ? least_of(r, lo) : 1) - 1);
        const int b1 = find<NT, uint64_t>(s, s.w, least_of(r, hi) - 1);
        mark(s, b0, b1);
        lo = s.w[b0];
        hi = s.w[b1 + 1] < hi ? s.w[b1 + 1] : hi;
    }
    if (r.q.min_p > 0.0f) {
        const int b = bin_at(r, (float)(-log((double)r.q.min_p) * (double)r.q.temperature));
        s.min_lo = b > 0 ? b - 1 : 0;  // the logarithm's rounding may move the border to the next bin
        s.min_hi = b < NB - 1 ? b + 1 : b;
        mark(s, s.min_lo, s.min_hi);
        lo = s.w[s.min_lo] < lo ? s.w[s.min_lo] : lo;
        hi = s.w[s.min_hi + 1] < hi ? s.w[s.min_hi + 1] : hi;
    }
    const int b0 = find<NT, uint64_t>(s, s.w, lo ? target_of(r, lo) : 0);
    const int b1 = find<NT, uint64_t>(s, s.w, target_of(r, hi));
    mark(s, b0, b1);
    __syncthreads();
}

__device__ __forceinline__ bool is_marked(const Bins &s, int bin) { return s.marked[bin >> 5] >> (bin & 31) & 1; }

// ---- a row by its marked tokens ------------------------------------------------
constexpr int RT = 1024;  // threads of a group that has a row

struct Choice {
    uint64_t list[CAP];      // ~key << 32 | index: ascending is the order of the choice
    uint64_t first_w[NB];    // the list's sum before a bin's first token
    uint32_t first[NB];      // and its place
    uint64_t tmp[RT / 64];
    uint64_t whole, end, by_min;
    uint32_t count;
};

// The list of m tokens, m <= CAP, in order.
__device__ __forceinline__ void sort(Choice &s, int m)
{
    int size = 2;
    while (size < m) size <<= 1;
    for (int i = m + (int)threadIdx.x; i < size; i += RT) s.list[i] = ~0ull;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int e = threadIdx.x; e < size / 2; e += RT) {
                const int i = 2 * e - (e & (j - 1)), o = i + j;
                const uint64_t x = s.list[i], y = s.list[o];
                if ((x > y) == !(i & k)) s.list[i] = y, s.list[o] = x;
            }
        }
    __syncthreads();
}

// The token from the list of all tokens in marked bins.
__device__ __forceinline__ void choose(const ornk_sample_args &a, int row, const Row &r, Bins &b, Choice &s, int m)
{
    constexpr int PER = CAP / RT;
    const int tid = threadIdx.x, lane = tid & 63;
    sort(s, m);
    const int per = (m + RT - 1) / RT;  // of a thread, in a row
    double e[PER];
    uint64_t w[PER], sum = 0;
    int bin[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = tid * per + i;
        w[i] = 0;
        if (i >= per || at >= m) continue;
        const float x = logit_of(~(uint32_t)(s.list[at] >> 32));
        e[i] = weight(r, x);
        w[i] = fixed(r, e[i]);
        bin[i] = bin_of(r, x);
        sum += w[i];
    }
    uint64_t before = sum;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up(before, o, 64);
        if (lane >= o) before += y;
    }
    if (lane == 63) s.tmp[tid >> 6] = before;
    __syncthreads();
    before -= sum;
    for (int i = 0; i < tid >> 6; ++i) before += s.tmp[i];
    if (tid == RT - 1) {
        s.whole = r.by_rank ? before + sum : b.w[NB];
        s.by_min = r.q.min_p == 0.0f ? ~0ull : r.by_rank ? 0 : b.w[b.min_lo];
    }
    uint64_t run = before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = tid * per + i;
        if (i >= per || at >= m) continue;
        const int left = i ? bin[i - 1] : at ? bin_of(r, logit_of(~(uint32_t)(s.list[at - 1] >> 32))) : -1;
        if (left != bin[i]) s.first_w[bin[i]] = run, s.first[bin[i]] = at;
        run += w[i];
    }
    __syncthreads();
    // each of the thread's tokens: f(its place in w[], the sum before it, its rank)
    auto each = [&](auto f) {
        uint64_t run = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = tid * per + i;
            if (i >= per || at >= m) continue;
            if (r.by_rank) f(i, run, (uint32_t)at);
            else f(i, b.w[bin[i]] + (run - s.first_w[bin[i]]), b.c[bin[i]] + (at - s.first[bin[i]]));
            run += w[i];
        }
    };
    if (b.by_k) {
        each([&](int i, uint64_t at, uint32_t rank) {
            if (rank == (uint32_t)r.q.top_k - 1) s.whole = at + w[i];
        });
        __syncthreads();
    }
    if (!tid) s.end = s.whole;  // also where top_p's border lies behind min_p's
    __syncthreads();
    if (r.q.top_p < 1.0f) {
        const uint64_t least = least_of(r, s.whole);
        each([&](int i, uint64_t at, uint32_t) {
            if (at < least && least <= at + w[i]) s.end = at + w[i];
        });
    }
    if (r.q.min_p > 0.0f)
        each([&](int i, uint64_t at, uint32_t) {
            if ((r.by_rank || (bin[i] >= b.min_lo && bin[i] <= b.min_hi)) && e[i] >= (double)r.q.min_p)
                atomicMax((unsigned long long *)&s.by_min, (unsigned long long)(at + w[i]));
        });
    __syncthreads();
    const uint64_t all = s.end < s.by_min ? s.end : s.by_min, target = target_of(r, all);
    each([&](int i, uint64_t at, uint32_t) {
        if (at <= target && target < at + w[i])
            put_result(a, row, (int)(uint32_t)s.list[tid * per + i], share(r, e[i], all));
    });
}

// ---- a row by passes -------------------------------------------------------------
// Where the marked tokens are too many to put in order (a great many logits alike):
// every border is found by three passes over the row, a digit of the keys each.
__device__ __forceinline__ uint64_t kept_weight(const Row &r, uint32_t key)
{
    const double w = weight(r, logit_of(key));
    return w >= (double)r.q.min_p ? fixed(r, w) : 0;
}

__device__ uint64_t block_sum(uint64_t v, uint64_t *tmp)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if (!(threadIdx.x & 63)) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < RT / 64; ++i) v += tmp[i];
    return v;
}

// The first key, from the largest down, up to which f's sum is more than `limit`; *above:
// the sum of the keys above it.  The whole sum is more than `limit`.
template <class F>
__device__ uint32_t descend(const Row &r, uint64_t limit, uint64_t *above, uint64_t *hist, uint64_t *tmp,
                            F f)
{
    uint32_t found = 0;
    uint64_t sum = 0;
    for (int shift = 21; ; shift = shift == 21 ? 10 : 0) {
        const int bits = shift ? 11 : 10;
        __syncthreads();
        for (int i = threadIdx.x; i < 2048; i += RT) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < r.n; i += RT) {
            const uint32_t key = key_of(r.x[i]);
            if (!key || (shift < 21 && (key ^ found) >> (shift + bits))) continue;
            const uint64_t v = f(key);
            if (v) atomicAdd((unsigned long long *)&hist[key >> shift & ((1u << bits) - 1)], v);
        }
        __syncthreads();
        // thread i: bins 2i and 2i + 1 from the top
        const int top = (1 << bits) - 1, b0 = top - 2 * threadIdx.x;
        const uint64_t h0 = b0 >= 0 ? hist[b0] : 0, h1 = b0 > 0 ? hist[b0 - 1] : 0;
        uint64_t incl = h0 + h1;
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t u = __shfl_up(incl, o, 64);
            if ((threadIdx.x & 63) >= o) incl += u;
        }
        if ((threadIdx.x & 63) == 63) tmp[threadIdx.x >> 6] = incl;
        __syncthreads();
        for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) incl += tmp[i];
        const uint64_t excl = sum + incl - h0 - h1;
        if (excl <= limit && excl + h0 + h1 > limit) {
            const bool first = excl + h0 > limit;
            tmp[RT / 64] = first ? b0 : b0 - 1;
            tmp[RT / 64 + 1] = first ? excl : excl + h0;
        }
        __syncthreads();
        found |= (uint32_t)tmp[RT / 64] << shift;
        sum = tmp[RT / 64 + 1];
        if (!shift) break;
    }
    *above = sum;
    return found;
}

template <class F>
__device__ uint64_t total(const Row &r, uint64_t *tmp, F f)
{
    uint64_t v = 0;
    for (int i = threadIdx.x; i < r.n; i += RT) {
        const uint32_t key = key_of(r.x[i]);
        if (key > r.cut) v += f(key);
    }
    return block_sum(v, tmp) + (r.cut ? r.ties * f(r.cut) : 0);
}

__device__ void choose_by_passes(const ornk_sample_args &a, int row, Row &r, uint64_t *hist, uint64_t *tmp)
{
    const int tid = threadIdx.x;
    auto plain = [&](uint32_t key) { return fixed(r, weight(r, logit_of(key))); };
    auto kept = [&](uint32_t key) { return kept_weight(r, key); };
    uint64_t above;
    uint64_t alive = 0;
    for (int i = tid; i < r.n; i += RT) {
        const uint32_t key = key_of(r.x[i]);
        alive += key && plain(key);
    }
    if (r.q.top_k > 0 && (uint64_t)r.q.top_k < block_sum(alive, tmp)) {
        r.cut = descend(r, r.q.top_k - 1, &above, hist, tmp, [&](uint32_t key) { return (uint64_t)(plain(key) != 0); });
        r.ties = r.q.top_k - (uint32_t)above;
    }
    if (r.q.top_p < 1.0f) {
        const uint64_t least = least_of(r, total(r, tmp, plain));
        const uint32_t cut = descend(r, least - 1, &above, hist, tmp, plain);
        const uint64_t w = plain(cut), n = (least - above + w - 1) / w;
        r.ties = (uint32_t)n;
        r.cut = cut;
    }
    const uint64_t all = total(r, tmp, kept), target = target_of(r, all);
    const uint32_t key = descend(r, target, &above, hist, tmp, kept);
    const uint32_t rank = (uint32_t)((target - above) / kept(key));
    // the token: the rank-th of this key
    uint32_t before = 0;
    for (int base = 0; base < r.n; base += RT) {
        const int i = base + tid;
        const bool is = i < r.n && key_of(r.x[i]) == key;
        const uint64_t m = __ballot(is);
        __syncthreads();
        if (!(tid & 63)) tmp[tid >> 6] = __popcll(m);
        __syncthreads();
        uint32_t at = before + __popcll(m & ((1ull << (tid & 63)) - 1));
        for (int w = 0; w < RT / 64; ++w) {
            if (w < tid >> 6) at += (uint32_t)tmp[w];
            before += (uint32_t)tmp[w];
        }
        if (is && at == rank) put_result(a, row, i, share(r, weight(r, logit_of(key)), all));
        if (before > rank) break;
    }
}

// A row's end: what is known of it after its bins are filled and its list is made.
struct Work {
    union {
        Choice c;
        struct {
            uint64_t hist[2048], tmp[RT / 64 + 2];
        } p;
    };
};

typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));

// A float4 of the row from token i on; -infinity behind its end.
__device__ __forceinline__ v4f load4(const float *x, int n, int i)
{
    if (i + 4 <= n) return *reinterpret_cast<const v4u *>(x + i);
    v4f y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = i + e < n ? x[i + e] : -INFINITY;
    return y;
}

// Tokens i0 to end - 1 of a row, by a group of NT threads.
template <int NT>
__device__ __forceinline__ Ends ends_of(const float *x, int i0, int end)
{
    Ends e = {0, ~0u};
#pragma unroll 4
    for (int i = i0 + 4 * (int)threadIdx.x; i < end; i += 4 * NT) {
        const v4f y = load4(x, end, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) extend(e, y[j], i + j);
    }
    return e;
}

// Into the bins of w and c, which are in LDS.  What is out of reach belongs to the sum
// that top_p is a share of, behind all bins' tokens.
template <int NT>
__device__ __forceinline__ void fill_bins(const Row &r, int i0, int end, uint64_t *w, uint32_t *c)
{
    uint64_t rest = 0;
#pragma unroll 2
    for (int i = i0 + 4 * (int)threadIdx.x; i < end; i += 4 * NT) {
        const v4f y = load4(r.x, end, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = within(r, y[j]);
            if (r.by_rank) {
                if (in) atomicAdd(&c[bin_of(r, y[j])], 1u);
                continue;
            }
            if (!in && r.q.top_p == 1.0f) continue;
            const uint64_t v = fixed(r, weight(r, y[j]));
            if (in) {
                const int bin = bin_of(r, y[j]);
                atomicAdd((unsigned long long *)&w[bin], (unsigned long long)v);
                if (r.q.top_k > 0) atomicAdd(&c[bin], 1u);
            } else {
                rest += v;
            }
        }
    }
    if (r.by_rank || r.q.top_p == 1.0f) return;
    for (int o = 32; o; o >>= 1) rest += __shfl_xor(rest, o, 64);
    if (!(threadIdx.x & 63) && rest) atomicAdd((unsigned long long *)&w[NB - 1], (unsigned long long)rest);
}

// Those in marked bins: f(token's place in the order).
template <int NT, class F>
__device__ __forceinline__ void gather(const Row &r, const Bins &b, int i0, int end, F f)
{
#pragma unroll 2
    for (int i = i0 + 4 * (int)threadIdx.x; i < end; i += 4 * NT) {
        const v4f y = load4(r.x, end, i);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (within(r, y[j]) && is_marked(b, bin_of(r, y[j]))) f((uint64_t)~key_of(y[j]) << 32 | (uint32_t)(i + j));
    }
}

// Shorter rows: a group each, in one launch.
__global__ void __launch_bounds__(RT) k_sample_row(ornk_sample_args a)
{
    __shared__ Bins b;
    __shared__ Work s;
    __shared__ Ends ends[RT / 64];
    const int row = blockIdx.x, tid = threadIdx.x;
    Row r = row_of(a, row);
    if (!valid(r.q, r.u)) {
        if (!tid) *(volatile int *)(a.err + ORNK_KV_ERR_SAMPLE) = 1 + row, put_result(a, row, -1, 0.0f);
        return;
    }
    const Ends e = block_ends<RT>(ends_of<RT>(r.x, 0, r.n), ends);
    if (!e.top || r.q.temperature == 0.0f) {
        if (!tid) put_result(a, row, e.top ? (int)~(uint32_t)e.top : -1, e.top ? 1.0f : 0.0f);
        return;
    }
    scale_row(r, (uint32_t)(e.top >> 32), e.low);
    for (int i = tid; i < NB; i += RT) b.w[i] = 0, b.c[i] = 0;
    if (!tid) s.c.count = 0;
    __syncthreads();
    fill_bins<RT>(r, 0, r.n, b.w, b.c);
    __syncthreads();
    sums_before<RT>(b);
    mark_bins<RT>(r, b);
    gather<RT>(r, b, 0, r.n, [&](uint64_t t) {
        const uint32_t at = atomicAdd(&s.c.count, 1u);
        if (at < CAP) s.c.list[at] = t;
    });
    __syncthreads();
    const uint32_t m = s.c.count;
    __syncthreads();
    if (m <= CAP) choose(a, row, r, b, s.c, m);
    else choose_by_passes(a, row, r, s.p.hist, s.p.tmp);
}

// ---- longer rows: in slices ------------------------------------------------------
constexpr int SL = 256;       // threads of a slice's group
constexpr int MAX_SLICES = 256;

// Work buffers of a row.
struct Slices {
    int n, len;              // number of a row's slices, their tokens (a multiple of 4 * SL)
    Ends *ends;              // [rows][n]
    uint64_t *w;             // [rows][NB]
    uint32_t *c;             // [rows][NB]
    uint64_t *list;          // [rows][CAP]
    uint32_t *count;         // [rows]
};

__device__ __forceinline__ Ends row_ends(const Slices &s, int row, Ends *tmp)
{
    Ends e = {0, ~0u};
    if ((int)threadIdx.x < s.n) e = s.ends[(size_t)row * s.n + threadIdx.x];
    for (int o = 32; o; o >>= 1) e = join(e, {__shfl_xor(e.top, o, 64), __shfl_xor(e.low, o, 64)});
    if (threadIdx.x < MAX_SLICES && !(threadIdx.x & 63)) tmp[threadIdx.x >> 6] = e;
    __syncthreads();
    e = tmp[0];
    for (int i = 1; i < MAX_SLICES / 64; ++i) e = join(e, tmp[i]);
    return e;
}

// The slices' ends; the row's bins and list emptied.
__global__ void __launch_bounds__(SL) k_sample_ends(ornk_sample_args a, Slices s)
{
    __shared__ Ends tmp[SL / 64];
    const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * s.len;
    for (int i = blockIdx.x * SL + tid; i < NB; i += s.n * SL) {
        s.w[(size_t)row * NB + i] = 0;
        s.c[(size_t)row * NB + i] = 0;
    }
    if (!blockIdx.x && !tid) s.count[row] = 0;
    const Ends e = block_ends<SL>(ends_of<SL>(a.logits + (size_t)row * a.stride, i0, min(i0 + s.len, a.n)), tmp);
    if (!tid) s.ends[(size_t)row * s.n + blockIdx.x] = e;
}

// The row as the later launches take it; false: it needs no bins.
__device__ __forceinline__ bool row_ready(const ornk_sample_args &a, const Slices &s, int row, Row &r, Ends &e, Ends *tmp)
{
    r = row_of(a, row);
    if (!valid(r.q, r.u)) return e.top = 0, false;
    e = row_ends(s, row, tmp);
    if (!e.top || r.q.temperature == 0.0f) return false;
    scale_row(r, (uint32_t)(e.top >> 32), e.low);
    return true;
}

__global__ void __launch_bounds__(SL) k_sample_bins(ornk_sample_args a, Slices s)
{
    __shared__ uint64_t w[NB];
    __shared__ uint32_t c[NB];
    __shared__ Ends tmp[MAX_SLICES / 64];
    const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * s.len;
    Row r;
    Ends e;
    if (!row_ready(a, s, row, r, e, tmp)) return;
    for (int i = tid; i < NB; i += SL) w[i] = 0, c[i] = 0;
    __syncthreads();
    fill_bins<SL>(r, i0, min(i0 + s.len, a.n), w, c);
    __syncthreads();
    for (int i = tid; i < NB; i += SL) {
        if (w[i]) atomicAdd((unsigned long long *)&s.w[(size_t)row * NB + i], (unsigned long long)w[i]);
        if (c[i]) atomicAdd(&s.c[(size_t)row * NB + i], c[i]);
    }
}

template <int NT>
__device__ __forceinline__ void load_bins(const Slices &s, int row, const Row &r, Bins &b)
{
    for (int i = threadIdx.x; i < NB; i += NT) {
        b.w[i] = s.w[(size_t)row * NB + i];
        b.c[i] = s.c[(size_t)row * NB + i];
    }
    __syncthreads();
    sums_before<NT>(b);
    mark_bins<NT>(r, b);
}

// The marked tokens to the row's list: those of a group together, as long as LDS holds
// them (an atomic of its own for each token took 110 us for 16 rows of 2000).
__global__ void __launch_bounds__(SL) k_sample_gather(ornk_sample_args a, Slices s)
{
    constexpr int MINE = 1024;
    __shared__ Bins b;
    __shared__ Ends tmp[MAX_SLICES / 64];
    __shared__ uint64_t mine[MINE];
    __shared__ uint32_t count, base;
    const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * s.len;
    Row r;
    Ends e;
    if (!row_ready(a, s, row, r, e, tmp)) return;
    if (!tid) count = 0;
    load_bins<SL>(s, row, r, b);
    uint64_t *list = s.list + (size_t)row * CAP;
    gather<SL>(r, b, i0, min(i0 + s.len, a.n), [&](uint64_t t) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < MINE) {
            mine[at] = t;
        } else {
            const uint32_t to = atomicAdd(&s.count[row], 1u);
            if (to < CAP) list[to] = t;
        }
    });
    __syncthreads();
    const uint32_t m = count < MINE ? count : MINE;
    if (!tid && m) base = atomicAdd(&s.count[row], m);
    __syncthreads();
    for (uint32_t i = tid; i < m; i += SL)
        if (base + i < CAP) list[base + i] = mine[i];
}

__global__ void __launch_bounds__(RT) k_sample_choose(ornk_sample_args a, Slices s)
{
    __shared__ Bins b;
    __shared__ Work k;
    __shared__ Ends tmp[MAX_SLICES / 64];
    const int row = blockIdx.x, tid = threadIdx.x;
    Row r;
    Ends e;
    if (!row_ready(a, s, row, r, e, tmp)) {
        if (tid) return;
        if (!valid(r.q, r.u)) *(volatile int *)(a.err + ORNK_KV_ERR_SAMPLE) = 1 + row;
        put_result(a, row, e.top ? (int)~(uint32_t)e.top : -1, e.top ? 1.0f : 0.0f);
        return;
    }
    const uint32_t m = s.count[row];
    if (m > CAP) return choose_by_passes(a, row, r, k.p.hist, k.p.tmp);
    load_bins<RT>(s, row, r, b);
    for (int i = tid; i < (int)m; i += RT) k.c.list[i] = s.list[(size_t)row * CAP + i];
    choose(a, row, r, b, k.c, m);
}

constexpr int ROW_MAX = 32768;  // tokens of a row that one group takes

Slices slices_of(const ornk_sample_args &a)
{
    const long long want = ((long long)a.rows * a.n / 1024 + 4 * SL - 1) / (4 * SL);  // for 1024 groups
    const long long least = ((long long)a.n + 4 * SL * MAX_SLICES - 1) / (4 * SL * MAX_SLICES);
    long long k = want < 1 ? 1 : want > 16 ? 16 : want;
    if (k < least) k = least;
    Slices s = {};
    s.len = (int)k * 4 * SL;
    s.n = (a.n + s.len - 1) / s.len;
    return s;
}

}  // namespace

extern "C" size_t ornk_sample_ws(const ornk_sample_args *a)
{
    if (a->n <= ROW_MAX) return 0;
    const size_t per = NB * 12 + CAP * 8 + sizeof(Ends) * slices_of(*a).n + 8;
    return a->rows * per;
}

extern "C" int ornk_sample(const ornk_sample_args *a, hipStream_t st)
{
    if (a->n <= ROW_MAX) {
        hipLaunchKernelGGL(k_sample_row, dim3(a->rows), dim3(RT), 0, st, *a);
        return hipGetLastError();
    }
    Slices s = slices_of(*a);
    const size_t R = a->rows;
    s.list = static_cast<uint64_t *>(a->ws);
    s.w = s.list + R * CAP;
    s.ends = reinterpret_cast<Ends *>(s.w + R * NB);
    s.c = reinterpret_cast<uint32_t *>(s.ends + R * s.n);
    s.count = s.c + R * NB;
    const dim3 grid(s.n, a->rows);
    hipLaunchKernelGGL(k_sample_ends, grid, dim3(SL), 0, st, *a, s);
    hipLaunchKernelGGL(k_sample_bins, grid, dim3(SL), 0, st, *a, s);
    hipLaunchKernelGGL(k_sample_gather, grid, dim3(SL), 0, st, *a, s);
    hipLaunchKernelGGL(k_sample_choose, dim3(a->rows), dim3(RT), 0, st, *a, s);
    return hipGetLastError();
}
