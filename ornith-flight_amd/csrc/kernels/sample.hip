// SPDX-License-Identifier: MIT
//
// A token for each row of logits by temperature, top-k, top-p and min-p (ornith_hip.h).
//
// The order of the choice is that of the logits, so a row is never sorted.  Its logits
// fall into bins of equal stretches; a bin's weights are summed as whole numbers, in which
// the order of the additions does not show.  The bins tell each border of the choice
// (top_k, top_p, min_p, the random number's) up to one or a few of them; only the tokens
// there are listed, and the borders found among them.  Rows of which a small top_k is
// asked need no bins: the k-th largest of the largest logits of many parts of a row is a bound
// that k tokens reach and few more.
#include "../../../include/ornith/ornith_hip.h"
#include "common.h"
#include "launch.h"

namespace {

constexpr int NB = 1024;   // bins of a row's logits
constexpr int CAP = 4096;  // tokens of a row that are listed
constexpr int ST = 1024;   // threads of a group that has a row
constexpr int CT = 256;    // those of them that work on bins and on a list: with more waves
                           // the same steps wait for each other's instructions

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

// 2^x for x <= 0 in 64 bits: the series of 2^f on [-1/2, 1/2], whose first term left
// out is below 2^-52.
__device__ __forceinline__ double exp2_of(double x)
{
    const double n = rint(x), f = x - n;
    const double f2 = f * f, f4 = f2 * f2, f8 = f4 * f4;  // c_k = ln(2)^k / k!
    const double a0 = fma(6.9314718055994531e-01, f, 1.0), a1 = fma(5.5504108664821580e-02, f, 2.4022650695910071e-01);
    const double a2 = fma(1.3333558146428443e-03, f, 9.6181291076284772e-03);
    const double a3 = fma(1.5252733804059841e-05, f, 1.5403530393381608e-04);
    const double a4 = fma(1.0178086009239699e-07, f, 1.3215486790144309e-06);
    const double a5 = fma(4.4455382718708112e-10, f, 7.0549116208011234e-09);
    const double b0 = fma(a1, f2, a0), b1 = fma(a3, f2, a2), b2 = fma(a5, f2, a4);
    return ldexp(fma(fma(2.5678435993488206e-11, f4, b2), f8, fma(b1, f4, b0)), (int)n);
}

// A row, its request and its largest logit.
struct Row {
    const float *x;
    int n;
    ornith_sample_request q;
    float u;
    bool valid;
    float top;     // the largest logit
    double per;    // log2(e) / temperature
    double unit;   // weights are whole multiples of 1 / unit; n of them fit 62 bits
    float scale;   // bins to `below`
    float reach;   // tokens farther below are behind every border
    bool by_rank;  // the top_k are few: all of them are listed
};

__device__ __forceinline__ Row row_of(const ornk_sample_args &a, int row)
{
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.n = a.n;
    r.q = static_cast<const ornith_sample_request *>(a.requests)[row];
    r.u = a.u[row];
    r.unit = a.unit;
    r.valid = r.q.temperature >= 0.0f && r.q.temperature < INFINITY && r.q.top_p >= 0.0f && r.q.top_p <= 1.0f &&
              r.q.min_p >= 0.0f && r.q.min_p <= 1.0f && r.u >= 0.0f && r.u < 1.0f;
    r.by_rank = r.q.top_k > 0 && r.q.top_k < r.n && r.q.top_k <= CAP / 2;
    return r;
}

// Half of how far below a row's largest logit another lies (the whole may pass the largest
// number); for a NaN a NaN.
__device__ __forceinline__ float below(const Row &r, float x)
{
    if (r.top == INFINITY) return x == INFINITY ? 0.0f : INFINITY;
    return fmaf(-0.5f, x, 0.5f * r.top);
}

__device__ __forceinline__ int bin_at(const Row &r, float below)
{
    const float b = below * r.scale;
    return b < (float)(NB - 1) ? (int)b : NB - 1;
}

__device__ __forceinline__ int bin_of(const Row &r, float x) { return bin_at(r, below(r, x)); }

// A token's weight, exp((x - largest) / temperature), as a whole number of units.
__device__ __forceinline__ double weight(const Row &r, float x)
{
    if (r.top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    const double y = ((double)x - (double)r.top) * r.per;
    return y > -60.0 ? exp2_of(y) : 0.0;  // also where x is a NaN
}

// To the nearest whole number, which is at most 2^51: the low bits of its sum with 2^52.
__device__ __forceinline__ uint64_t fixed(const Row &r, double w)
{
    return __double_as_longlong(fma(w, r.unit, 0x1p52)) & 0xfffffffffffffull;
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

__device__ __forceinline__ void put_result(const ornk_sample_args &a, int row, int token, float prob)
{
    a.tokens[row] = token;
    if (a.prob) a.prob[row] = prob;
}

// The largest and least logit of some tokens that are above -infinity.
struct Ends {
    float top, low;  // -infinity and infinity where there is none
};

__device__ __forceinline__ Ends join(Ends a, Ends b) { return {fmaxf(a.top, b.top), fminf(a.low, b.low)}; }

__device__ __forceinline__ Ends wave_ends(Ends e)
{
    for (int o = 32; o; o >>= 1) e = join(e, {__shfl_xor(e.top, o, 64), __shfl_xor(e.low, o, 64)});
    return e;
}

// What the weights and bins need, and how far below the largest a border of the choice
// may lie, which is where the bins end:
// - a weight below 2^-53 of the largest (37 temperatures) is 0;
// - the tokens below (1 - top_p) / 2 n are less than half of what top_p leaves out;
// - min_p leaves out what is below it.
// Where the top_k are few, `bound` is a key that as many tokens have or pass (0: none is
// known); where they are many, their own border may lie anywhere.
__device__ __forceinline__ void scale_row(Row &r, Ends e, uint32_t bound)
{
    const float T = r.q.temperature;
    r.top = e.top;
    r.per = 1.4426950408889634 / (double)T;
    r.reach = fminf(18.5f * T, 3.4028234e38f);
    if (r.by_rank) {
        if (bound) r.reach = fminf(r.reach, below(r, logit_of(bound)));
    } else if (r.q.top_k <= 0 || r.q.top_k >= r.n) {
        if (r.q.top_p < 1.0f) r.reach = fminf(r.reach, -logf((1.0f - r.q.top_p) / (2.0f * r.n)) * T * 0.50005f);
        if (r.q.min_p > 0.0f) r.reach = fminf(r.reach, -logf(r.q.min_p) * T * 0.50005f);
    }
    const float range = fminf(below(r, e.low), r.reach), s = (float)NB / range;
    r.scale = range > 0.0f ? fminf(s, 1e30f) : 0.0f;
}

// ---- what bins decide ----------------------------------------------------------
// Sums of weights and numbers of tokens before each bin, and the bins whose tokens are
// listed: those where a border of the choice may lie.
struct Bins {
    uint64_t w[NB + 1];
    uint32_t c[NB + 1];
    uint32_t marked[NB / 32];
    uint64_t tmp[CT / 64];
    uint32_t tmp32[CT / 64];
    int found;
    int last;            // the last bin marked
    int min_lo, min_hi;  // min_p's border is in these
};

// w and c from each bin's own to what is before it.
__device__ __forceinline__ void sums_before(Bins &s)
{
    constexpr int PER = NB / CT;
    const int tid = threadIdx.x, lane = tid & 63;
    uint64_t w = 0, ws[PER];
    uint32_t c = 0, cs[PER];
    if (tid < CT) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            w += ws[i] = s.w[tid * PER + i];
            c += cs[i] = s.c[tid * PER + i];
        }
        uint64_t wi = w;
        uint32_t ci = c;
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t y = __shfl_up(wi, o, 64);
            const uint32_t z = __shfl_up(ci, o, 64);
            if (lane >= o) wi += y, ci += z;
        }
        if (lane == 63) s.tmp[tid >> 6] = wi, s.tmp32[tid >> 6] = ci;
        w = wi - w;
        c = ci - c;
    }
    __syncthreads();
    if (tid < CT) {
        for (int i = 0; i < tid >> 6; ++i) w += s.tmp[i], c += s.tmp32[i];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s.w[tid * PER + i] = w;
            s.c[tid * PER + i] = c;
            w += ws[i];
            c += cs[i];
        }
        if (tid == CT - 1) s.w[NB] = w, s.c[NB] = c;
    }
    __syncthreads();
}

// Whether the k-th of the parts' largest logits is a bound of the top_k: of tokens in any
// order about parts * ln(parts / (parts - k)) pass it, which have to fit the list.
__device__ __forceinline__ bool is_bound(const Row &r, int parts)
{
    return r.by_rank && r.q.top_k < parts && -logf(1.0f - (float)r.q.top_k / (float)parts) * (float)parts < 0.75f * CAP;
}

// The bin in which a sum passes `limit`, which is below the whole.  All threads.
template <class T>
__device__ __forceinline__ int find(Bins &s, const T *sum, T limit)
{
    if (threadIdx.x < CT)
        for (int i = threadIdx.x; i < NB; i += CT)
            if (sum[i] <= limit && limit < sum[i + 1]) s.found = i;
    __syncthreads();
    const int f = s.found;
    __syncthreads();
    return f;
}

__device__ __forceinline__ void mark(Bins &s, int lo, int hi)
{
    if (threadIdx.x >= CT) return;
    for (int i = lo + (int)threadIdx.x; i <= hi; i += CT) atomicOr(&s.marked[i >> 5], 1u << (i & 31));
    if (!threadIdx.x) s.last = s.last > hi ? s.last : hi;
}

// Every sum below is known up to the bins marked, so those of the next border are.
// counted: only that the bins hold the top_k is known.  min_bin: min_p's.
__device__ __forceinline__ void mark_bins(const Row &r, Bins &s, bool counted, int min_bin)
{
    if (threadIdx.x < NB / 32) s.marked[threadIdx.x] = 0;
    if (!threadIdx.x) s.last = 0;
    __syncthreads();
    const bool by_k = r.q.top_k > 0 && (uint32_t)r.q.top_k < s.c[NB];
    if (counted) {
        mark(s, 0, by_k ? find<uint32_t>(s, s.c, (uint32_t)r.q.top_k - 1) : NB - 1);
        __syncthreads();
        return;
    }
    uint64_t lo = s.w[NB], hi = lo;
    if (by_k) {
        const int b = find<uint32_t>(s, s.c, (uint32_t)r.q.top_k - 1);
        mark(s, b, b);
        lo = s.w[b];
        hi = s.w[b + 1];
    }
    if (r.q.min_p > 0.0f) {
        s.min_lo = min_bin > 0 ? min_bin - 1 : 0;  // the logarithm's rounding may move it to the next bin
        s.min_hi = min_bin < NB - 1 ? min_bin + 1 : min_bin;
        mark(s, s.min_lo, s.min_hi);
    }
#pragma unroll 1
    for (int target = r.q.top_p == 1.0f; target < 2; ++target) {
        if (target && r.q.min_p > 0.0f) {
            lo = s.w[s.min_lo] < lo ? s.w[s.min_lo] : lo;
            hi = s.w[s.min_hi + 1] < hi ? s.w[s.min_hi + 1] : hi;
        }
        const int b0 = find<uint64_t>(s, s.w, !lo ? 0 : target ? target_of(r, lo) : least_of(r, lo) - 1);
        const int b1 = find<uint64_t>(s, s.w, target ? target_of(r, hi) : least_of(r, hi) - 1);
        mark(s, b0, b1);
        lo = s.w[b0];
        hi = s.w[b1 + 1] < hi ? s.w[b1 + 1] : hi;
    }
    __syncthreads();
}

__device__ __forceinline__ float min_below(const Row &r) { return -logf(r.q.min_p) * r.q.temperature * 0.5f; }

__device__ __forceinline__ bool is_marked(const Bins &s, int bin) { return s.marked[bin >> 5] >> (bin & 31) & 1; }

__device__ __forceinline__ uint64_t wave_sum(uint64_t v)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// ---- passes over logits, tokens i0 to end - 1 of a row by a group ------------------
template <int NT>
__device__ __forceinline__ Ends ends_of(const float *x, int i0, int end)
{
    Ends e = {-INFINITY, INFINITY};
#pragma unroll 4
    for (int i = i0 + 4 * (int)threadIdx.x; i < end; i += 4 * NT) {
        const v4f y = load4(x, end, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            e.top = fmaxf(e.top, y[j]);  // which a NaN leaves as it is
            e.low = y[j] > -INFINITY ? fminf(e.low, y[j]) : e.low;
        }
    }
    return e;
}

// f(logit, token) of those within reach, g(logit) of the others; one copy of each in a
// loop, the next float4 on its way.
template <int NT, class F, class G>
__device__ __forceinline__ void each_token(const Row &r, int i0, int end, F f, G g)
{
    int i = i0 + 4 * (int)threadIdx.x;
    if (i >= end) return;
    v4f next = load4(r.x, end, i);
#pragma unroll 1
    for (; i < end; i += 4 * NT) {
        v4f y = next;
        if (i + 4 * NT < end) next = load4(r.x, end, i + 4 * NT);
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
            if (below(r, y[0]) <= r.reach) f(y[0], i + j);
            else g(y[0]);
            y = v4f{y[1], y[2], y[3], y[0]};
        }
    }
}

// Into the bins of w and c, which are in LDS.  What is out of reach belongs to the sum
// that top_p is a share of, behind all bins' tokens.
template <int NT>
__device__ __forceinline__ void fill_bins(const Row &r, int i0, int end, uint64_t *w, uint32_t *c)
{
    uint64_t rest = 0;
    const bool sums = !r.by_rank && r.q.top_p < 1.0f;
    each_token<NT>(
        r, i0, end,
        [&](float x, int) {
            const int bin = bin_of(r, x);
            if (!r.by_rank) {
                const uint64_t v = fixed(r, weight(r, x));
                if (!v) return;
                atomicAdd((unsigned long long *)&w[bin], (unsigned long long)v);
            }
            if (r.q.top_k > 0) atomicAdd(&c[bin], 1u);
        },
        [&](float x) {
            if (sums) rest += fixed(r, weight(r, x));
        });
    if (!sums) return;
    rest = wave_sum(rest);
    if (!(threadIdx.x & 63) && rest) atomicAdd((unsigned long long *)&w[NB - 1], (unsigned long long)rest);
}

// ---- the choice ------------------------------------------------------------------
// By CT threads, of a list in LDS, or (where more than CAP tokens lie next to a border: a
// great many logits alike) of the whole row.  Loops stay loops: a group runs this once,
// and code that is not yet in the instruction cache takes longer than its work.
struct Choice {
    uint64_t list[CAP];  // key << 32 | index
    uint64_t w[CAP];     // their weights
    uint64_t hist[256], tmp[3][CT / 64], found[2];
    uint32_t keys[2][CT / 64];
    uint32_t count;
};

__device__ __forceinline__ uint64_t wave_scan(uint64_t v)
{
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up(v, o, 64);
        if ((threadIdx.x & 63) >= o) v += y;
    }
    return v;
}

__device__ __forceinline__ float share(const Row &r, uint32_t key, uint64_t all)
{
    return (float)(weight(r, logit_of(key)) * r.unit / (double)all);
}

// At most CT tokens: each finds its place by counting those before it.
template <class F>
__device__ __forceinline__ void choose_few(const ornk_sample_args &a, int row, const Row &r, const Bins &b, Choice &s, int m,
                                           bool binned, F place_of)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const bool on = tid < m;
    auto order = [&](int i) { return s.list[i] ^ 0xffffffffu; };  // the key, then the least index
    int place = 0;
    if (on) {
        const uint64_t mine = order(tid);
#pragma unroll 4
        for (int i = 0; i < m; ++i) place += order(i) > mine;
        s.w[place] = s.list[tid];  // m <= CT: apart from the sums below
    }
    __syncthreads();
    // thread i: the i-th token
    const uint64_t token = on ? s.w[tid] : 0;
    const uint32_t key = (uint32_t)(token >> 32);
    const double e = on ? weight(r, logit_of(key)) : 0.0;
    const uint64_t w = on ? fixed(r, e) : 0, run = wave_scan(w);
    const int bin = binned && on ? place_of(logit_of(key)) : -1;
    if (lane == 63) s.tmp[0][tid >> 6] = run;
    __syncthreads();
    uint64_t lo = run - w, all = 0;  // the sum before it
    for (int i = 0; i < CT / 64; ++i) {
        if (i < tid >> 6) lo += s.tmp[0][i];
        all += s.tmp[0][i];
    }
    uint32_t rank = tid;
    if (binned) {
        uint64_t *first_w = s.w + CT;                                       // of a bin's tokens in the list
        uint32_t *first = reinterpret_cast<uint32_t *>(s.w + CT + NB);
        if (on && (!tid || place_of(logit_of((uint32_t)(s.w[tid - 1] >> 32))) != bin)) first_w[bin] = lo, first[bin] = tid;
        __syncthreads();
        if (on) {
            lo = b.w[bin] + lo - first_w[bin];
            rank = b.c[bin] + tid - first[bin];
        }
    }
    const uint64_t hi = lo + w;
    uint64_t whole = binned ? b.w[NB] : all, by_min = ~0ull;
    if (r.q.top_k > 0 && (binned ? (uint32_t)r.q.top_k < b.c[NB] : r.q.top_k < m)) {
        if (on && rank == (uint32_t)r.q.top_k - 1) s.found[0] = hi;
        __syncthreads();
        whole = s.found[0];
    }
    if (r.q.min_p > 0.0f) {
        const bool kept = on && e >= (double)r.q.min_p && (!binned || (bin >= b.min_lo && bin <= b.min_hi));
        uint64_t last = kept ? hi : binned ? b.w[b.min_lo] : 0;
        for (int o = 32; o; o >>= 1) {
            const uint64_t y = __shfl_xor(last, o, 64);
            last = y > last ? y : last;
        }
        if (!lane) s.tmp[1][tid >> 6] = last;
        __syncthreads();
        by_min = 0;
        for (int i = 0; i < CT / 64; ++i) by_min = s.tmp[1][i] > by_min ? s.tmp[1][i] : by_min;
    }
    uint64_t end = whole;
    if (r.q.top_p < 1.0f) {
        const uint64_t least = least_of(r, whole);
        if (!tid) s.found[1] = whole;  // where min_p's border comes first
        __syncthreads();
        if (on && lo < least && least <= hi) s.found[1] = hi;
        __syncthreads();
        end = s.found[1];
    }
    const uint64_t kept = end < by_min ? end : by_min, target = target_of(r, kept);
    if (on && lo <= target && target < hi) put_result(a, row, (int)(uint32_t)token, share(r, key, kept));
}

// More: every border is the first key, from the largest down, up to which a sum (of
// tokens, or of their weights) passes a limit.  Its bin is known; the key is found by passes
// over the bin's tokens, 8 bits of the keys' distance from the least each.  Of the whole row
// (m > CAP) a bin's tokens are listed first, if they are few; the many of one that does not
// fit are mostly alike, and need one pass for a border and one for the index.  64 rows of
// 248,320 logits and a top_p: 373 us where all are equal, 461 where they are multiples of 1/4.
template <class F>
__device__ __forceinline__ void choose_many(const ornk_sample_args &a, int row, const Row &r, Bins &b, Choice &s, uint32_t m,
                                            F place_of)
{
    const int tid = threadIdx.x, lane = tid & 63;
    bool listed = m <= CAP;
    int n = listed ? (int)m : r.n;
    // f(key, index, place in the list) of the list's tokens, or of the row's within reach
    auto each = [&](auto f) {
        const int step = listed ? 1 : 4;
        v4f x, next;
        if (!listed) next = load4(r.x, n, 4 * tid);
#pragma unroll 1
        for (int i = step * tid; i < n; i += step * CT) {
            if (!listed) x = next, next = load4(r.x, n, i + 4 * CT);
#pragma unroll 1
            for (int j = 0; j < step; ++j) {
                const uint64_t t = listed ? s.list[i] : (uint64_t)key_of(x[0]) << 32 | (i + j);
                if (listed || below(r, x[0]) <= r.reach) f((uint32_t)(t >> 32), (uint32_t)t, i);
                if (!listed) x = __builtin_shufflevector(x, x, 1, 2, 3, 0);
            }
        }
    };
    uint32_t seen = 0;  // of a row's tokens the last key, which many may share, and its weight
    uint64_t seen_units = 0;
    auto units = [&](uint32_t key, int at) {
        if (listed) return s.w[at];
        if (key != seen) seen = key, seen_units = fixed(r, weight(r, logit_of(key)));
        return seen_units;
    };
    auto weigh = [&] {  // the list
#pragma unroll 1
        for (int i = tid; i < n; i += CT) s.w[i] = fixed(r, weight(r, logit_of((uint32_t)(s.list[i] >> 32))));
    };
    if (listed) weigh();
    auto group_sum = [&](uint64_t v) {
        v = wave_sum(v);
        if (!lane) s.tmp[1][tid >> 6] = v;
        __syncthreads();
        v = 0;
        for (int i = 0; i < CT / 64; ++i) v += s.tmp[1][i];
        __syncthreads();
        return v;
    };
    uint64_t by_min = ~0ull;
    if (r.q.min_p > 0.0f) {
        uint64_t sum = 0;
        each([&](uint32_t key, uint32_t, int at) {
            const int bin = place_of(logit_of(key));
            if (bin >= b.min_lo && bin <= b.min_hi && weight(r, logit_of(key)) >= (double)r.q.min_p) sum += units(key, at);
        });
        by_min = b.w[b.min_lo] + group_sum(sum);
    }
    uint64_t whole = b.w[NB], end = whole;

    enum { TOP_K, TOP_P, TARGET, INDEX };
    uint64_t all = 0;   // of the kept
    uint32_t key = 0;   // the token's
    uint64_t rank = 0;  // and its place among those of the same key
    int bin = 0;
#pragma unroll 1
    for (int stage = TOP_K; stage <= INDEX; ++stage) {
        uint64_t limit, base = 0;
        if (stage == TOP_K) {
            if (r.q.top_k <= 0 || (uint32_t)r.q.top_k >= b.c[NB]) continue;
            bin = find<uint32_t>(b, b.c, (uint32_t)r.q.top_k - 1);
            limit = r.q.top_k - 1 - b.c[bin];
        } else if (stage == INDEX) {
            limit = rank;
            if (!listed) break;
        } else {
            if (stage == TOP_P) {
                end = whole;
                if (r.q.top_p == 1.0f) continue;
                limit = least_of(r, whole) - 1;
                if (by_min <= limit) continue;  // min_p's border comes first
            } else {
                all = end < by_min ? end : by_min;
                limit = target_of(r, all);
            }
            bin = find<uint64_t>(b, b.w, limit);
            base = b.w[bin];
            limit -= base;
        }
        // f(key, weight) of this stage's tokens; of INDEX the keys are the largest index
        // there may be, less theirs
        auto those = [&](auto f) {
            each([&](uint32_t k, uint32_t index, int at) {
                if (stage == INDEX ? k != key : place_of(logit_of(k)) != bin) return;
                const uint64_t v = units(k, at);
                if (v) f(stage == INDEX ? ORN_SAMPLE_MAX_VOCAB - 1 - index : k, v);
            });
        };
        uint32_t low = ~0u, high = 0;
        const bool fill = m > CAP && stage != INDEX;
        if (fill) {
            listed = false;
            n = r.n;
            if (!tid) s.count = 0;
            __syncthreads();
            v4f next = load4(r.x, n, 4 * tid);
#pragma unroll 1
            for (int i = 4 * tid; i < n; i += 4 * CT) {
                const v4f x = next;
                next = load4(r.x, n, i + 4 * CT);
                int in = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t k = key_of(x[j]);
                    const bool on = below(r, x[j]) <= r.reach && bin_of(r, x[j]) == bin;
                    in |= on << j;
                    low = on && k < low ? k : low;
                    high = on && k > high ? k : high;
                }
                if (!in || *(volatile uint32_t *)&s.count > CAP) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!(in >> j & 1)) continue;
                    const uint32_t at = atomicAdd(&s.count, 1u);
                    if (at < CAP) s.list[at] = (uint64_t)key_of(x[j]) << 32 | (i + j);
                }
            }
        } else {
            those([&](uint32_t k, uint64_t) {
                low = k < low ? k : low;
                high = k > high ? k : high;
            });
        }
        for (int o = 32; o; o >>= 1) {
            const uint32_t x = __shfl_xor(low, o, 64), y = __shfl_xor(high, o, 64);
            low = x < low ? x : low;
            high = y > high ? y : high;
        }
        if (!lane) s.keys[0][tid >> 6] = low, s.keys[1][tid >> 6] = high;
        __syncthreads();
        for (int i = 0; i < CT / 64; ++i) {
            low = s.keys[0][i] < low ? s.keys[0][i] : low;
            high = s.keys[1][i] > high ? s.keys[1][i] : high;
        }
        if (fill && s.count <= CAP) {
            listed = true;
            n = (int)s.count;
            weigh();
            __syncthreads();
        }
        // the border: a key's distance from the least, and the sum above it
        uint32_t found = 0;
        uint64_t above = 0;
        int known = low == high ? 0 : 32 - __clz((int)(high - low));  // bits from this one on are known
#pragma unroll 1
        while (known > 0) {
            const int shift = known > 8 ? known - 8 : 0;
            s.hist[tid] = 0;
            __syncthreads();
            those([&](uint32_t k, uint64_t v) {
                k -= low;
                if ((uint64_t)(k ^ found) >> known) return;
                atomicAdd((unsigned long long *)&s.hist[k >> shift & 255],
                          stage == TOP_K || stage == INDEX ? 1ull : (unsigned long long)v);
            });
            __syncthreads();
            // thread i: digit i from the top (with less than 8 bits to go, those known
            // are the same for all)
            const uint64_t h = s.hist[255 - tid], in = wave_scan(h);
            if (lane == 63) s.tmp[0][tid >> 6] = in;
            __syncthreads();
            uint64_t run = in + above - h;
            for (int i = 0; i < tid >> 6; ++i) run += s.tmp[0][i];
            if (run <= limit && limit < run + h) s.found[0] = 255 - tid, s.found[1] = run;
            __syncthreads();
            found |= (uint32_t)s.found[0] << shift;
            above = s.found[1];
            known = shift;
        }
        found += low;
        if (stage == INDEX) {
            if (!tid) put_result(a, row, ORN_SAMPLE_MAX_VOCAB - 1 - found, share(r, key, all));
            return;
        }
        const uint64_t w = fixed(r, weight(r, logit_of(found)));
        if (stage == TOP_K) {
            uint64_t more = 0;
            if (low != high)
                those([&](uint32_t k, uint64_t v) {
                    if (k > found) more += v;
                });
            whole = end = b.w[bin] + group_sum(more) + (limit + 1 - above) * w;
        } else if (stage == TOP_P) {
            end = base + above + ((limit - above) / w + 1) * w;
        } else {
            key = found;
            rank = (limit - above) / w;
        }
        __syncthreads();
    }

    // The index in a row: each wave counts the key's tokens in stretches of 256, one of which
    // has the rank.
    uint32_t *counts = reinterpret_cast<uint32_t *>(s.w);
    constexpr int PER = ORN_SAMPLE_MAX_VOCAB / 256 / CT;
    for (int i = 0; i < PER; ++i) counts[CT * i + tid] = 0;
    __syncthreads();
    v4f next = load4(r.x, r.n, 4 * tid), after = load4(r.x, r.n, 4 * tid + 4 * CT);
#pragma unroll 1
    for (int i0 = 0; i0 < r.n; i0 += 4 * CT) {
        const v4f x = next;
        next = after;
        after = load4(r.x, r.n, i0 + 4 * tid + 8 * CT);
        int c = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) c += __popcll(__ballot(key_of(x[j]) == key));
        if (!lane) counts[(i0 >> 8) + (tid >> 6)] = c;
    }
    __syncthreads();
    uint32_t mine = 0;
    for (int i = 0; i < PER; ++i) mine += counts[PER * tid + i];
    uint64_t run = wave_scan(mine);
    if (lane == 63) s.tmp[0][tid >> 6] = run;
    __syncthreads();
    run -= mine;
    for (int i = 0; i < tid >> 6; ++i) run += s.tmp[0][i];
    if (run <= rank && rank < run + mine) {
        int i = PER * tid;
        for (; rank >= run + counts[i]; ++i) run += counts[i];
        s.found[0] = i;
        s.found[1] = run;
    }
    __syncthreads();
    if (tid >= 64) return;
    const int i = 256 * (int)s.found[0] + 4 * lane;
    const v4f x = load4(r.x, r.n, i);
    int in = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) in += key_of(x[j]) == key;
    run = s.found[1] + wave_scan(in) - in;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (key_of(x[j]) == key && run++ == rank) put_result(a, row, i + j, share(r, key, all));
}

// Which part of a bin: the marked bins (without bins: all of the reach) in as many equal
// stretches as NB allows.
struct Fine {
    int parts;       // of a bin; 1: the bins are as they were
    uint32_t before[NB / 32];
};

__device__ __forceinline__ int fine_at(const Row &r, const Bins &b, const Fine &f, float below)
{
    const int bin = bin_at(r, below), in = (int)((below * r.scale - (float)bin) * (float)f.parts);
    const uint32_t word = b.marked[bin >> 5];
    return (int)(f.before[bin >> 5] + __popc(word & ((1u << (bin & 31)) - 1))) * f.parts + (in < f.parts ? in : f.parts - 1);
}

// The choice from a list.  A longer one is divided once more, by finer bins.  Where too many
// tokens pass the bound of the top_k, the bins are filled after all.
__device__ __forceinline__ void choose(const ornk_sample_args &a, int row, Row &r, const Ends &e, Bins &b, Bins &c,
                                       Fine &f, Choice &s, uint32_t m)
{
    const int tid = threadIdx.x, lane = tid & 63;
    bool binned = !r.by_rank;
    const bool fine = m > CT && m <= CAP;
    if (fine) {
        if (r.by_rank) {  // the list's own bins
            if (tid < NB / 32) b.marked[tid] = ~0u;
            for (int i = tid; i <= NB; i += CT) b.w[i] = b.c[i] = 0;
        }
        for (int i = tid; i < NB; i += CT) c.w[i] = c.c[i] = 0;
        if (!tid) s.count = 0;
        __syncthreads();
        if (tid < 64) {
            const uint32_t n = lane < NB / 32 ? __popc(b.marked[lane]) : 0;
            const uint32_t to = (uint32_t)wave_scan(n);
            if (lane < NB / 32) f.before[lane] = to - n;
            if (lane == NB / 32 - 1) f.parts = NB / (int)to;
        }
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < (int)m; i += CT) {
            const float x = logit_of((uint32_t)(s.list[i] >> 32));
            const int bin = fine_at(r, b, f, below(r, x));
            const uint64_t v = fixed(r, weight(r, x));
            if (!v) continue;
            atomicAdd((unsigned long long *)&c.w[bin], (unsigned long long)v);
            atomicAdd(&c.c[bin], 1u);
        }
        __syncthreads();
        sums_before(c);
        if (binned) {
            // from the list's sums to the row's: what lies between marked bins
            uint64_t *dw = s.w;
            uint32_t *dc = reinterpret_cast<uint32_t *>(s.w + NB);
            for (int bin = tid; bin < NB; bin += CT) {
                if (!is_marked(b, bin)) continue;
                const int o = (int)(f.before[bin >> 5] + __popc(b.marked[bin >> 5] & ((1u << (bin & 31)) - 1)));
                dw[o] = b.w[bin] - c.w[o * f.parts];
                dc[o] = b.c[bin] - c.c[o * f.parts];
            }
            __syncthreads();
            const int used = (int)(f.before[NB / 32 - 1] + __popc(b.marked[NB / 32 - 1])) * f.parts;
            for (int i = tid; i <= NB; i += CT) {
                c.w[i] = i < used ? c.w[i] + dw[i / f.parts] : b.w[NB];
                c.c[i] = i < used ? c.c[i] + dc[i / f.parts] : b.c[NB];
            }
            __syncthreads();
        }
        binned = true;
        mark_bins(r, c, false, r.q.min_p > 0.0f ? fine_at(r, b, f, min_below(r)) : 0);
#pragma unroll 1
        for (int i = tid; i < (int)m; i += CT) {
            const uint64_t t = s.list[i];
            if (!is_marked(c, fine_at(r, b, f, below(r, logit_of((uint32_t)(t >> 32)))))) continue;
            const uint32_t at = atomicAdd(&s.count, 1u);
            s.w[at] = t;
        }
        __syncthreads();
        m = s.count;
        for (int i = tid; i < (int)m; i += CT) s.list[i] = s.w[i];
        __syncthreads();
    }
    if (m > CAP && r.by_rank) {
        r.by_rank = false;
        scale_row(r, e, 0);
        for (int i = tid; i < NB; i += CT) b.w[i] = b.c[i] = 0;
        __syncthreads();
        fill_bins<CT>(r, 0, r.n, b.w, b.c);
        __syncthreads();
        sums_before(b);
        mark_bins(r, b, false, bin_at(r, min_below(r)));
    }
    auto place_of = [&](float x) { return fine ? fine_at(r, b, f, below(r, x)) : bin_of(r, x); };
    if (m <= CT) choose_few(a, row, r, fine ? c : b, s, (int)m, binned, place_of);
    else choose_many(a, row, r, fine ? c : b, s, m, place_of);
}

// ---- lists ----------------------------------------------------------------------
// Those in marked bins, or (b is NULL) all within reach: f(key << 32 | token).
template <int NT, class F>
__device__ __forceinline__ void gather(const Row &r, const Bins *b, int i0, int end, F f)
{
    const float last = b && b->last < NB - 1 ? (float)(b->last + 1) : INFINITY;
    each_token<NT>(
        r, i0, end,
        [&](float x, int i) {
            if (!b || (below(r, x) * r.scale < last && is_marked(*b, bin_of(r, x))))
                f((uint64_t)key_of(x) << 32 | (uint32_t)i);
        },
        [](float) {});
}

// A lower bound of the k-th largest of the group's keys, P of a thread: its upper 16
// bits.  0 where there are less.
template <int P>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[P], uint32_t k, uint32_t *hist)
{
    const int tid = threadIdx.x;
    uint32_t found = 0, left = k;
#pragma unroll 1
    for (int shift = 24; shift >= 16; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (key[i] && (shift == 24 || key[i] >> 24 == found >> 24)) atomicAdd(&hist[key[i] >> shift & 255], 1u);
        __syncthreads();
        uint32_t c = 0, before = 0;
        if (tid < 256) {
            c = hist[255 - tid];
            before = c;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(before, o, 64);
                if ((tid & 63) >= o) before += y;
            }
            if ((tid & 63) == 63) hist[256 + (tid >> 6)] = before;
        }
        if (tid == 0) hist[260] = 256;
        __syncthreads();
        if (tid < 256) {
            before -= c;
            for (int i = 0; i < tid >> 6; ++i) before += hist[256 + i];
            if (before < left && left <= before + c) hist[260] = 255 - tid, hist[261] = before;
        }
        __syncthreads();
        if (hist[260] == 256) return 0;
        found |= hist[260] << shift;
        left -= hist[261];
        __syncthreads();
    }
    return found;
}

// The first token that has the largest logit.
template <int NT>
__device__ __forceinline__ void first_of(const Row &r, float top, int i0, int end, uint32_t *first)
{
#pragma unroll 1
    for (int i = i0 + (int)threadIdx.x; i < end; i += NT)
        if (r.x[i] == top) {
            atomicMin(first, (uint32_t)i);
            return;
        }
}

// ---- shorter rows: a group each, in one launch -------------------------------------
__global__ void __launch_bounds__(ST) k_sample_row(ornk_sample_args a)
{
    __shared__ Bins b, fine;
    __shared__ Fine parts;
    __shared__ Choice s;
    __shared__ Ends ends[ST / 64];
    const int row = blockIdx.x, tid = threadIdx.x;
    Row r = row_of(a, row);
    if (!r.valid) {
        if (!tid) *(volatile int *)(a.err + ORNK_KV_ERR_SAMPLE) = 1 + row, put_result(a, row, -1, 0.0f);
        return;
    }
    const Ends own = ends_of<ST>(r.x, 0, r.n);
    Ends e = wave_ends(own);
    if (!(tid & 63)) ends[tid >> 6] = e;
    if (!tid) s.count = r.q.temperature == 0.0f ? ~0u : 0;
    __syncthreads();
    for (int i = 0; i < ST / 64; ++i) e = join(e, ends[i]);
    if (!(e.top > -INFINITY)) {
        if (!tid) put_result(a, row, -1, 0.0f);
        return;
    }
    if (r.q.temperature == 0.0f) {
        first_of<ST>(r, e.top, 0, r.n, &s.count);
        __syncthreads();
        if (!tid) put_result(a, row, (int)s.count, 1.0f);
        return;
    }
    uint32_t bound = 0;
    if (is_bound(r, min(ST, r.n / 4))) {
        const uint32_t key[1] = {key_of(own.top)};
        bound = kth_largest(key, r.q.top_k, b.c);
    }
    scale_row(r, e, bound);
    if (!bound) {
        for (int i = tid; i < NB; i += ST) b.w[i] = 0, b.c[i] = 0;
        __syncthreads();
        fill_bins<ST>(r, 0, r.n, b.w, b.c);
        __syncthreads();
        sums_before(b);
        mark_bins(r, b, r.by_rank, bin_at(r, min_below(r)));
    }
    gather<ST>(r, bound ? nullptr : &b, 0, r.n, [&](uint64_t t) {
        const uint32_t at = atomicAdd(&s.count, 1u);
        if (at < CAP) s.list[at] = t;
    });
    __syncthreads();
    const uint32_t m = s.count;
    __syncthreads();
    if (tid < CT) choose(a, row, r, e, b, fine, parts, s, m);
}

// ---- longer rows: in slices ------------------------------------------------------
constexpr int SL = 512;  // threads of a slice's group: 64 rows of 248,320 take 68 us, with 1024 or 256 73
constexpr int MAX_SLICES = 256;
constexpr int MAX_TOPS = 4096;

// Work buffers of a row.
struct Slices {
    int n, len;       // number of a row's slices, their tokens (a multiple of 4 * SL)
    int per;          // parts of a slice whose largest keys are kept: 1 << per threads have one
    Ends *ends;       // [rows][n]
    uint64_t *w;      // [rows][NB]
    uint32_t *c;      // [rows][NB]
    uint64_t *list;   // [rows][CAP]
    uint32_t *count;  // [rows]: of the list
    uint32_t *first;  // [rows]: the first token that has the largest logit
    uint32_t *tops;   // [rows][MAX_TOPS]: the parts' largest keys
    uint32_t *bound;  // [rows]
};

// The slices' ends and largest keys; the row's bins and list emptied.
__global__ void __launch_bounds__(SL) k_sample_ends(ornk_sample_args a, Slices s)
{
    __shared__ Ends tmp[SL / 64];
    const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * s.len;
    for (int i = blockIdx.x * SL + tid; i < NB; i += s.n * SL) {
        s.w[(size_t)row * NB + i] = 0;
        s.c[(size_t)row * NB + i] = 0;
    }
    if (!blockIdx.x && !tid) s.count[row] = 0, s.first[row] = ~0u;
    const Ends own = ends_of<SL>(a.logits + (size_t)row * a.stride, i0, min(i0 + s.len, a.n));
    float top = own.top;
    for (int o = 1; o < 1 << s.per; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (!(tid & ((1 << s.per) - 1)))
        s.tops[(size_t)row * MAX_TOPS + blockIdx.x * (SL >> s.per) + (tid >> s.per)] = key_of(top);
    Ends e = wave_ends(own);
    if (!(tid & 63)) tmp[tid >> 6] = e;
    __syncthreads();
    for (int i = 0; i < SL / 64; ++i) e = join(e, tmp[i]);
    if (!tid) s.ends[(size_t)row * s.n + blockIdx.x] = e;
}

__device__ __forceinline__ Ends own_ends(const Slices &s, int row)
{
    const Ends none = {-INFINITY, INFINITY};
    return (int)threadIdx.x < s.n ? s.ends[(size_t)row * s.n + threadIdx.x] : none;
}

__device__ __forceinline__ Ends row_ends(Ends e, Ends *tmp)
{
    if (threadIdx.x < MAX_SLICES) {
        e = wave_ends(e);
        if (!(threadIdx.x & 63)) tmp[threadIdx.x >> 6] = e;
    }
    __syncthreads();
    e = tmp[0];
    for (int i = 1; i < MAX_SLICES / 64; ++i) e = join(e, tmp[i]);
    return e;
}

__global__ void __launch_bounds__(SL) k_sample_bins(ornk_sample_args a, Slices s)
{
    __shared__ uint64_t w[NB];
    __shared__ uint32_t c[NB];
    __shared__ Ends tmp[MAX_SLICES / 64];
    const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * s.len;
    Row r = row_of(a, row);
    const Ends own = own_ends(s, row);
    if (!r.valid || r.q.temperature == 0.0f) return;
    const int tops = s.n * (SL >> s.per);
    uint32_t bound = 0;
    if (is_bound(r, tops)) {
        uint32_t key[MAX_TOPS / SL];
#pragma unroll
        for (int i = 0; i < MAX_TOPS / SL; ++i)
            key[i] = tid + SL * i < tops ? s.tops[(size_t)row * MAX_TOPS + tid + SL * i] : 0;
        bound = kth_largest(key, r.q.top_k, c);
    }
    if (!blockIdx.x && !tid) s.bound[row] = bound;
    if (bound) return;  // the top_k are found by it
    const Ends e = row_ends(own, tmp);
    if (!(e.top > -INFINITY)) return;
    scale_row(r, e, 0);
    for (int i = tid; i < NB; i += SL) w[i] = 0, c[i] = 0;
    __syncthreads();
    fill_bins<SL>(r, i0, min(i0 + s.len, a.n), w, c);
    __syncthreads();
    for (int i = tid; i < NB; i += SL) {
        if (w[i]) atomicAdd((unsigned long long *)&s.w[(size_t)row * NB + i], (unsigned long long)w[i]);
        if (c[i]) atomicAdd(&s.c[(size_t)row * NB + i], c[i]);
    }
}

// A thread's bins of the row, on their way.
template <int NT>
struct OwnBins {
    uint64_t w[NB / NT];
    uint32_t c[NB / NT];
    __device__ __forceinline__ OwnBins(const Slices &s, int row)
    {
#pragma unroll
        for (int i = 0; i < NB / NT; ++i) {
            w[i] = s.w[(size_t)row * NB + threadIdx.x + NT * i];
            c[i] = s.c[(size_t)row * NB + threadIdx.x + NT * i];
        }
    }
    __device__ __forceinline__ void put(const Row &r, Bins &b) const
    {
#pragma unroll
        for (int i = 0; i < NB / NT; ++i) {
            b.w[threadIdx.x + NT * i] = w[i];
            b.c[threadIdx.x + NT * i] = c[i];
        }
        __syncthreads();
        sums_before(b);
        mark_bins(r, b, r.by_rank, bin_at(r, min_below(r)));
    }
};

// The tokens in marked bins, or those that pass the bound, to the row's list: those of a
// group together (an atomic of its own for each token took 110 us for 16 rows of 2000).
__global__ void __launch_bounds__(SL) k_sample_gather(ornk_sample_args a, Slices s)
{
    __shared__ Bins b;
    __shared__ Ends tmp[MAX_SLICES / 64];
    __shared__ uint32_t mine[CAP];
    __shared__ uint32_t count, base;
    const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * s.len, end = min(i0 + s.len, a.n);
    Row r = row_of(a, row);
    const Ends own = own_ends(s, row);
    const OwnBins<SL> bins(s, row);
    const uint32_t bound = s.bound[row];
    if (!r.valid) return;
    const Ends e = row_ends(own, tmp);
    if (!(e.top > -INFINITY)) return;
    if (r.q.temperature == 0.0f) {
        if (s.ends[(size_t)row * s.n + blockIdx.x].top == e.top) first_of<SL>(r, e.top, i0, end, &s.first[row]);
        return;
    }
    scale_row(r, e, r.by_rank ? bound : 0);
    if (!tid) count = 0;
    const bool binned = !(r.by_rank && bound);
    if (binned) bins.put(r, b);
    __syncthreads();
    gather<SL>(r, binned ? &b : nullptr, i0, end, [&](uint64_t t) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < CAP) mine[at] = (uint32_t)t;
    });
    __syncthreads();
    const uint32_t m = count;
    if (!tid && m) base = atomicAdd(&s.count[row], m);
    __syncthreads();
    if (m > CAP || base >= CAP) return;
    uint64_t *list = s.list + (size_t)row * CAP + base;
    for (uint32_t i = tid; i < min(m, CAP - base); i += SL) list[i] = (uint64_t)key_of(r.x[mine[i]]) << 32 | mine[i];
}

// All that the choice needs is loaded at once: each wait for memory is longer than most
// of its steps.
__global__ void __launch_bounds__(CT) k_sample_choose(ornk_sample_args a, Slices s)
{
    __shared__ Bins b, fine;
    __shared__ Fine parts;
    __shared__ Choice k;
    __shared__ Ends tmp[MAX_SLICES / 64];
    const int row = blockIdx.x, tid = threadIdx.x;
    Row r = row_of(a, row);
    const Ends own = own_ends(s, row);
    const OwnBins<CT> bins(s, row);
    const uint32_t m = s.count[row], first = s.first[row], bound = s.bound[row];
    const uint64_t *list = s.list + (size_t)row * CAP;
    const uint64_t mine = list[tid];
    const Ends e = row_ends(own, tmp);
    if (!r.valid || !(e.top > -INFINITY) || r.q.temperature == 0.0f) {
        if (tid) return;
        const bool none = !r.valid || !(e.top > -INFINITY);
        if (!r.valid) *(volatile int *)(a.err + ORNK_KV_ERR_SAMPLE) = 1 + row;
        put_result(a, row, none ? -1 : (int)first, none ? 0.0f : 1.0f);
        return;
    }
    scale_row(r, e, r.by_rank ? bound : 0);
    k.list[tid] = mine;
#pragma unroll 1
    for (int i = tid + CT; i < min((int)m, CAP); i += 8 * CT) {
        uint64_t t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = list[min(i + CT * j, CAP - 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + CT * j < CAP) k.list[i + CT * j] = t[j];
    }
    if (!r.by_rank) bins.put(r, b);
    __syncthreads();
    choose(a, row, r, e, b, fine, parts, k, m);
}

constexpr int ROW_MAX = 32768;  // tokens of a row that one group takes

Slices slices_of(const ornk_sample_args &a)
{
    // 4096 to 32768 tokens each, for 1536 groups: shorter slices add more bins than they
    // count (16 rows of 100,000 in slices of 2048 take 61 us, of 4096 53).
    constexpr int UNIT = 4 * SL;
    const long long want = ((long long)a.rows * a.n / 1536 + UNIT - 1) / UNIT;
    const long long least = ((long long)a.n + UNIT * MAX_SLICES - 1) / (UNIT * MAX_SLICES);
    long long k = want < 4096 / UNIT ? 4096 / UNIT : want > 32768 / UNIT ? 32768 / UNIT : want;
    if (k > a.n / (8 * UNIT)) k = a.n / (8 * UNIT);  // 8 slices at least: parts whose bound a top_k of 1600 has
    if (k < least) k = least;
    Slices s = {};
    s.len = (int)k * UNIT;
    s.n = (a.n + s.len - 1) / s.len;
    while (s.n * (SL >> s.per) > MAX_TOPS) ++s.per;
    return s;
}

}  // namespace

extern "C" size_t ornk_sample_ws(const ornk_sample_args *a)
{
    if (a->n <= ROW_MAX) return 0;
    const size_t per = CAP * 8 + NB * 12 + sizeof(Ends) * slices_of(*a).n + MAX_TOPS * 4 + 12;
    return a->rows * per;
}

extern "C" int ornk_sample(const ornk_sample_args *a, hipStream_t st)
{
    if (a->n <= ROW_MAX) {
        hipLaunchKernelGGL(k_sample_row, dim3(a->rows), dim3(ST), 0, st, *a);
        return hipGetLastError();
    }
    Slices s = slices_of(*a);
    const size_t R = a->rows;
    s.list = static_cast<uint64_t *>(a->ws);
    s.w = s.list + R * CAP;
    s.ends = reinterpret_cast<Ends *>(s.w + R * NB);
    s.c = reinterpret_cast<uint32_t *>(s.ends + R * s.n);
    s.tops = s.c + R * NB;
    s.count = s.tops + R * MAX_TOPS;
    s.first = s.count + R;
    s.bound = s.first + R;
    const dim3 grid(s.n, a->rows);
    hipLaunchKernelGGL(k_sample_ends, grid, dim3(SL), 0, st, *a, s);
    hipLaunchKernelGGL(k_sample_bins, grid, dim3(SL), 0, st, *a, s);
    hipLaunchKernelGGL(k_sample_gather, grid, dim3(SL), 0, st, *a, s);
    hipLaunchKernelGGL(k_sample_choose, dim3(a->rows), dim3(CT), 0, st, *a, s);
    return hipGetLastError();
}
