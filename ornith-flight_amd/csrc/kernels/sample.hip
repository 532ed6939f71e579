// SPDX-License-Identifier: MIT
//
// A token for each row of logits by temperature, top-k, top-p and min-p (ornith_hip.h).
#include "../../../include/ornith/ornith_hip.h"
#include "common.h"
#include "launch.h"

namespace {

constexpr int ST = 1024;

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

// A row's request and what the passes over it have found.
struct Row {
    const float *x;
    int n;
    uint32_t top;      // largest key
    double per_temp;   // 1 / temperature
    double unit;       // weights are whole multiples of 1 / unit; n of them fit 62 bits
    uint32_t cut;      // kept: keys above it, and the first `ties` of its own
    uint32_t ties;
    double min_p;
};

// exp((x - largest) / temperature)
__device__ __forceinline__ double weight(const Row &r, uint32_t key)
{
    if (key == r.top) return 1.0;
    if (!key) return 0.0;
    return exp(((double)logit_of(key) - (double)logit_of(r.top)) * r.per_temp);
}

__device__ __forceinline__ uint64_t fixed(const Row &r, double w) { return (uint64_t)(w * r.unit + 0.5); }

__device__ __forceinline__ uint64_t kept_weight(const Row &r, uint32_t key)
{
    const double w = weight(r, key);
    return w >= r.min_p ? fixed(r, w) : 0;
}

__device__ uint64_t block_sum(uint64_t v, uint64_t *tmp)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if (!(threadIdx.x & 63)) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < ST / 64; ++i) v += tmp[i];
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
        for (int i = threadIdx.x; i < 2048; i += ST) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < r.n; i += ST) {
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
            tmp[ST / 64] = first ? b0 : b0 - 1;
            tmp[ST / 64 + 1] = first ? excl : excl + h0;
        }
        __syncthreads();
        found |= (uint32_t)tmp[ST / 64] << shift;
        sum = tmp[ST / 64 + 1];
        if (!shift) break;
    }
    *above = sum;
    return found;
}

template <class F>
__device__ uint64_t total(const Row &r, uint64_t *tmp, F f)
{
    uint64_t v = 0;
    for (int i = threadIdx.x; i < r.n; i += ST) {
        const uint32_t key = key_of(r.x[i]);
        if (key > r.cut) v += f(key);
    }
    return block_sum(v, tmp) + (r.cut ? r.ties * f(r.cut) : 0);
}

// A row per work group, every step a pass over it.
__global__ void __launch_bounds__(ST) k_sample_passes(ornk_sample_args a)
{
    __shared__ uint64_t hist[2048], tmp[ST / 64 + 2];
    const int row = blockIdx.x, tid = threadIdx.x;
    const ornith_sample_request q = static_cast<const ornith_sample_request *>(a.requests)[row];
    const float u = a.u[row];
    Row r = {a.logits + (size_t)row * a.stride, a.n, 0, 0.0, a.unit, 0, 0, q.min_p};
    int token = -1;
    float prob = 0.0f;
    auto done = [&] {
        if (tid) return;
        a.tokens[row] = token;
        if (a.prob) a.prob[row] = prob;
    };
    if (!(q.temperature >= 0.0f && q.temperature < INFINITY && q.top_p >= 0.0f && q.top_p <= 1.0f &&
          q.min_p >= 0.0f && q.min_p <= 1.0f && u >= 0.0f && u < 1.0f)) {
        if (!tid) *(volatile int *)(a.err + ORNK_KV_ERR_SAMPLE) = 1 + row;
        return done();
    }
    uint32_t top = 0, count = 0;
    for (int i = tid; i < r.n; i += ST) {
        const uint32_t key = key_of(r.x[i]);
        top = key > top ? key : top;
        count += key != 0;
    }
    for (int o = 32; o; o >>= 1) {
        const uint32_t v = __shfl_xor(top, o, 64);
        top = v > top ? v : top;
    }
    if (!(tid & 63)) hist[tid >> 6] = top;
    __syncthreads();
    for (int i = 0; i < ST / 64; ++i) top = hist[i] > top ? (uint32_t)hist[i] : top;
    r.top = top;
    count = (uint32_t)block_sum(count, tmp);
    if (!top) return done();
    const bool greedy = q.temperature == 0.0f;
    r.per_temp = greedy ? 0.0 : 1.0 / (double)q.temperature;
    auto plain = [&](uint32_t key) { return fixed(r, weight(r, key)); };
    auto kept = [&](uint32_t key) { return kept_weight(r, key); };
    uint64_t above;
    if (greedy) {
        r.cut = top;
        r.ties = 1;
    } else if (q.top_k > 0 && (uint32_t)q.top_k < count) {
        r.cut = descend(r, q.top_k - 1, &above, hist, tmp, [](uint32_t) { return (uint64_t)1; });
        r.ties = q.top_k - (uint32_t)above;
    }
    if (!greedy && q.top_p < 1.0f) {
        const uint64_t all = total(r, tmp, plain);
        uint64_t least = (uint64_t)ceil((double)q.top_p * (double)all);
        least = least < 1 ? 1 : least > all ? all : least;
        const uint32_t cut = descend(r, least - 1, &above, hist, tmp, plain);
        const uint64_t w = plain(cut), n = (least - above + w - 1) / w;
        if (cut != r.cut || n < r.ties) r.ties = (uint32_t)n;
        r.cut = cut;
    }
    const uint64_t all = total(r, tmp, kept);
    uint64_t target = (uint64_t)((double)u * (double)all);
    target = target < all ? target : all - 1;
    const uint32_t key = descend(r, target, &above, hist, tmp, kept);
    const uint32_t rank = (uint32_t)((target - above) / kept(key));
    // the token: the rank-th of this key
    uint32_t before = 0;
    for (int base = 0; base < r.n; base += ST) {
        const int i = base + tid;
        const bool is = i < r.n && key_of(r.x[i]) == key;
        const uint64_t m = __ballot(is);
        __syncthreads();
        if (!(tid & 63)) tmp[tid >> 6] = __popcll(m);
        __syncthreads();
        uint32_t at = before + __popcll(m & ((1ull << (tid & 63)) - 1));
        for (int w = 0; w < ST / 64; ++w) {
            if (w < tid >> 6) at += (uint32_t)tmp[w];
            before += (uint32_t)tmp[w];
        }
        if (is && at == rank) {
            a.tokens[row] = i;
            if (a.prob) a.prob[row] = (float)(weight(r, key) * r.unit / (double)all);
        }
        if (before > rank) break;
    }
}

}  // namespace

extern "C" size_t ornk_sample_ws(const ornk_sample_args *a) { return 0; }

extern "C" int ornk_sample(const ornk_sample_args *a, hipStream_t s)
{
    hipLaunchKernelGGL(k_sample_passes, dim3(a->rows), dim3(ST), 0, s, *a);
    return hipGetLastError();
}
