// SPDX-License-Identifier: MIT
//
// Attention of one new token per sequence over the paged key-value cache
// (ornith_hip.h): out = sum_t w_t V[t], w = softmax(scale * q . K[t]), the sums
// over the sequence's tokens, query heads sharing kv heads.
//
// Work: the tokens of every sequence, kv head and tile of 16 of its query heads
// ("pair") in units of 64 to 256, one after the other on a line.  W work groups
// take equal stretches of the line, whatever the lengths are; a pair that one
// group covers is finished there, of the others the groups leave O, m and l of
// their part, which k_kv_finish puts together:
//   M = max m_i, L = sum l_i 2^(m_i - M), out = sum O_i 2^(m_i - M) / L.
// (Exponents are base 2: log2 e is in the query's scale.)  The parts' places and
// the order of their sums depend on the lengths alone: equal calls give equal bits.
// Stretches whose sums are not finite are done once more (Shares).
//
// Bound by the reading of K and V where the cache is large: 64 sequences of up to
// 8192 tokens, 32 heads over 8 of 128, 1.04 GB of bf16 in 192 us (5.4 TB/s; a
// streaming read 6.3, a copy 4.7), of f16 in 205; one of 131,071, 16 heads over 2 of
// 256 in bf16, 268 MB in 52 us and 6 more for the joining; 32 of up to 16,384, 64
// heads over 4 of 128 in e4m3, 280 MB in 61 + 6 us (of a CU's cycles vector
// instructions take half there, mostly unpacking, and MFMA a fifth; in f16 44% and
// 17%).  Short calls are bound by latency: lengths, table, K and V, the waves'
// joining, 8 us for 37 tokens.
#include "kv.h"

namespace {

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
// A unit has more tokens than below where that keeps the line below 2^22 units
// (32-bit products with a group's number).
constexpr int LINE_LOG2 = 22;
constexpr int MAX_SEGMENTS = (1 << (LINE_LOG2 - 8)) + 32;  // of one of 2^8 groups or more
// Work groups per CU, as log2: one's start and end under another's stream.  What
// registers allow: K, V and O of a tile and their addresses take all of one
// wave's per SIMD at 256 columns (two groups with tiles of 16 keys: 131,071
// tokens of bf16 64 us instead of 52), and two waves' at 128 (four spill: 209 ->
// 393 us); the fp32 path of 64 columns leaves room for four (5 x 2047 tokens of
// 12 kv heads 20.0 -> 18.2 us), the others of 64 do not (126 -> 144 us).  What spills
// is fp32 of fewer than 64 columns, 6 registers of the 128, and 56 where its rows are
// not whole 16-byte words.
constexpr int groups_log2(int type, int HD)
{
    return HD == 256 ? 0 : HD == 64 && type == ORN_KV_F32 ? 2 : 1;
}
constexpr int CUS_LOG2 = 8;
// Tokens of a unit, as log2: a tile for each wave; of the fp32 cache, whose tiles
// are 16 keys, two at 64 columns (four: 32 sequences of up to 8000 tokens, 4 heads,
// 66.3 instead of 60.9 us; 5 of 2047, 12 heads, 17.0 and 17.9) and one beyond (two:
// 100 of up to 600, 2 heads of 128, 27.7 instead of 22.7 us; 5 of 2047, 4 heads of
// 256, 31.9 and 27.6; one of 4000, 8 heads of 128, 14.1 and 16.5: more parts).
constexpr int unit_log2(int type, int HD)
{
    return type == ORN_KV_F32 ? HD == 64 ? 7 : 6 : HD == 64 ? 8 : 7;
}

struct AttendWs {
    uint32_t *cum;   // [n_seqs + 1] units before each sequence, per pair of it
    float2 *part_ml; // [2 W][16] of the parts: of the pair a group goes on with, of the one it begins
    float *part_o;   // [2 W][16][row]
    int w_log2, row, unit_log2;  // W; floats of a row of part_o; a unit
    uint32_t whole;  // units of a pair that is not cut, at least
    float2 *ml;      // [n_seqs][heads] and scores [n_seqs][heads][s_len], for the weights
    float *s;
    size_t s_len;
};

// The line of T units: the first of group w's stretch, and the group of unit u.
// A line shorter than the groups gives one unit to each of the first T.
__device__ __forceinline__ uint32_t line_at(uint32_t T, int w_log2, uint32_t w)
{
    return T >> w_log2 ? T * w >> w_log2 : min(w, T);
}
__device__ __forceinline__ uint32_t line_group(uint32_t T, int w_log2, uint32_t u)
{
    return T >> w_log2 ? (((u + 1) << w_log2) - 1) / T : u;
}

// Pairs of up to so many units are not cut: a bound of a group's stretch that
// falls into one moves to its nearer end.  Up to a group's share of the line, as
// parts of two pairs take a group about twice as long as a whole one (256 rows of
// up to 300 tokens, 8 kv heads of 128 in bf16: 59.3 -> 55.9 us; 100 of up to 600,
// 2 heads: 20.1 -> 21.0); at most 4, since a group waits for the longest (8: the
// same times).  `least`: all of them, where max_len alone says that they are
// short; then there is nothing to join either.  Pairs of 2 units always (one row
// of 250 tokens, 8 heads of 128: 10.8 -> 8.9 us), pairs of 8 where there are half
// as many as groups (200 rows of up to 1000: 103 -> 91; 8 rows: 13.2 -> 18.3).
__device__ __forceinline__ uint32_t line_whole(uint32_t T, int w_log2, uint32_t least)
{
    const uint32_t share = T >> w_log2;
    return max(least, share ? min(share + 1, 4u) : 1);
}

struct Seg {  // part of one pair
    int b, h, j0, rows;  // sequence, kv head, first query head, query heads
    int len, k0, k1;     // the sequence's tokens; this part's
    size_t score;        // first score of query head j0
};

// 2^x (results below 2^-126: zero)
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// The factor of sums relative to m in sums relative to M >= m: 1 also where
// both are -inf (no weight yet; but a NaN's sum is one).
__device__ __forceinline__ float weight_from(float m, float M) { return m == M ? 1.0f : exp2_(m - M); }

__device__ __forceinline__ uint32_t top16(float hi, float lo)
{
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float rest16(float x)
{
    return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}
__device__ __forceinline__ v8b as_v8b(u4 x) { return __builtin_bit_cast(v8b, x); }

// N bytes (4, 8, 16) into words.
template <int N>
__device__ __forceinline__ void load_words(uint32_t *w, const uint8_t *p)
{
    typedef uint32_t vec __attribute__((ext_vector_type(N / 4)));
    const vec v = *reinterpret_cast<const vec *>(p);
    if constexpr (N == 4) w[0] = v[0];
    else
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = v[i];
}

template <int TYPE>
constexpr int elem_size = (int)sizeof(typename KvElem<TYPE>::T);

// Four consecutive elements in words -> fp32.
template <int TYPE>
__device__ __forceinline__ void unpack4(float *f, const uint32_t *w)
{
    if constexpr (TYPE == ORN_KV_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else if constexpr (TYPE == ORN_KV_BF16) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else if constexpr (TYPE == ORN_KV_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const h2 h = __builtin_bit_cast(h2, w[i]);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    } else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[0], false);
        const f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[0], true);
        f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1];
    }
}

// ---------------------------------------------------------------------------
// A wave's tile: KT keys by the 16 query heads of the pair.  Scores are formed
// transposed, S^T = K Q^T, so that lane (g = lane / 16, n = lane % 16) holds the
// scores of query head n for keys 16 i + 4 g + r: the row maximum and sum are
// two exchanges away, and the weights are the A operand of O = P V as they
// are.  Both paths read K and V from memory straight into operand registers.
// ---------------------------------------------------------------------------

// fp32 operands (v_mfma_f32_16x16x4_f32): what 32-bit arithmetic gives, with
// infinities and NaN where it has them.  The path of the fp32 cache; of heads
// whose rows are not whole 16-byte words (VEC = false); and, as Shares, of what
// neither path gives.  16 keys per tile.
template <int TYPE, int HD, bool VEC, bool FULL>
struct Exact {
    static constexpr int KT = 16, NJ = HD / 16, NV = HD / 64, NO = HD / 16;
    static constexpr int ES = elem_size<TYPE>;
    static constexpr size_t Q_BYTES = 16 * HD * 4;
    static constexpr bool full = FULL, vec = VEC, shares = false, ahead = TYPE == ORN_KV_F32 && VEC;
    float k[NJ][4], v[4][NV][4];

    // Past the row: any of its elements.  Of V they are columns that are not
    // stored; of K zeros take their places in scores, as here each load would be
    // waited for before the next (122 rows of up to 358 tokens, 8 kv heads of 192
    // in fp32: 174 us, and 99 so).
    static __device__ __forceinline__ void load4(float *f, const uint8_t *p, int c, int hd)
    {
        if constexpr (VEC) {
            uint32_t w[ES];
            load_words<4 * ES>(w, p + (FULL || c < hd ? c : 0) * ES);
            unpack4<TYPE>(f, w);
        } else {
            const typename KvElem<TYPE>::T *e = reinterpret_cast<const typename KvElem<TYPE>::T *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = KvElem<TYPE>::get(e[min(c + i, hd - 1)]);
        }
    }
    // row: this lane's key of each 16
    __device__ __forceinline__ void load_k(const uint8_t *const *row, int g, int hd)
    {
#pragma unroll
        for (int j = 0; j < NJ; ++j) load4(k[j], row[0], 16 * j + 4 * g, hd);
    }
    // row: this lane's four keys of each 16
    __device__ __forceinline__ void load_v(const uint8_t *const *row, int n, int hd)
    {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NV; ++j) load4(v[r][j], row[r], 64 * j + 4 * n, hd);
    }
    // dimensions d .. d + 3 of query n: [16 j][n][4 g + i], so that a lane's four
    // steps are one word
    static __device__ __forceinline__ void put_q(void *lds, int n, int d, v4f q)
    {
        *reinterpret_cast<v4f *>(static_cast<float *>(lds) + (d / 16) * 256 + n * 16 + d % 16) = q;
    }
    __device__ __forceinline__ void scores(float *s, const void *lds, int lane, int hd) const
    {
        const int g = lane >> 4, n = lane & 15;
        const v4f *q = reinterpret_cast<const v4f *>(static_cast<const float *>(lds) + n * 16 + 4 * g);
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const v4f b = q[64 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = FULL || 16 * j + 4 * g + i < hd ? k[j][i] : 0.0f;
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x, b[i], acc, 0, 0, 0);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = acc[r];
    }
    // A key that is left out has the weight 0, and 0 times an infinity is none:
    // its values count as zeros.  (Parts: such a segment comes to Shares.)
    __device__ __forceinline__ void leave_out(int r)
    {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][j][i] = 0.0f;
    }
    __device__ __forceinline__ void pv(v4f *o, const float *p) const
    {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[4 * j + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[r], v[r][j][i], o[4 * j + i],
                                                                        0, 0, 0);
    }
    // column of o[c] in lane n; four at a time are consecutive
    static __device__ __forceinline__ int col(int c, int n) { return 64 * (c / 4) + 4 * n + c % 4; }
};

// A segment whose sums were not finite, once more.  There are two reasons: an
// infinity or a NaN, which Parts' operands cannot be; and weights relative to a
// maximum that still grows, up to 2^6 each, whose sums with values near the largest
// number pass it though the mean does not.  So the maximum and the sum are found
// first (the scores are formed twice), and O is the sum of shares of it.  An infinite
// value takes the call of 131,071 tokens from 51 to 237 us, and in every sequence the
// batch of 64 from 244 to 800.
template <int TYPE, int HD, bool VEC, bool FULL>
struct Shares : Exact<TYPE, HD, VEC, FULL> {
    static constexpr bool shares = true, ahead = false;
};

// bf16 operands (v_mfma_f32_16x16x32_bf16) for the caches of 16 and 8 bits.  A
// cached value is one bf16 part (bf16, e4m3) or two (f16: 8 and 3 bits), a query
// or a weight three: the top 8 bits, of the rest the top 8, and the rest.  Each
// part has fp32's exponents, so 24 bits stay at every size, and the sums are
// fp32.  Of the f16 products the smallest, second part by third, is left out
// (2^-24 of the whole).  Parts of an infinity are no numbers: a segment whose
// sums are not finite is left to Shares.  32 or 64 keys per tile.
//
// Reduction indexes are permuted alike in both operands: a lane's 16 bytes of a
// K row are its dimensions of one step (of two, for e4m3), and key 16 i + 4 g + r
// is place 8 g + 4 i + r of the reduction over keys, so that the weights stay
// where they are.  V's 8 rows by CW columns in a lane's registers are turned
// into CW operands of 8 keys there (v_perm_b32).
// Keys of a tile: more bytes on their way for every wave where short rows leave
// registers for them (98 sequences of 10,699, e4m3, 64 columns: 126 us with 32
// keys, 117 with 64; 128 columns of e4m3 70 and 74 us).
constexpr int parts_keys(int HD) { return HD == 64 ? 64 : 32; }

template <int TYPE, int HD, bool FULL>
struct Parts {
    static constexpr int ES = elem_size<TYPE>, KT = parts_keys(HD), NI = KT / 16, NG = KT / 32;
    static constexpr int NS = HD / 32, NO = HD / 16;
    static constexpr int DL = 16 / ES, NL = HD / (4 * DL);             // K: dimensions of a load, loads
    static constexpr int CW = HD / 16 < DL ? HD / 16 : DL, NH = HD / (16 * CW);  // V: columns, loads of a row
    static constexpr int VW = CW * ES / 4;
    static constexpr int NP = TYPE == ORN_KV_F16 ? 2 : 1;
    static constexpr size_t Q_BYTES = 3 * 16 * HD * 2;
    static constexpr bool full = FULL, vec = true, shares = false, ahead = true;
    uint32_t k[NI][NL][4], v[4 * NI][NH][VW];

    __device__ __forceinline__ void load_k(const uint8_t *const *row, int g, int hd)
    {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                // past the row: its start, which meets zeros of the query
                const int c = (4 * j + g) * DL;
                load_words<16>(k[i][j], row[i] + (FULL || c < hd ? c : 0) * ES);
            }
    }
    __device__ __forceinline__ void load_v(const uint8_t *const *row, int n, int hd)
    {
#pragma unroll
        for (int r = 0; r < 4 * NI; ++r)
#pragma unroll
            for (int j = 0; j < NH; ++j) {
                const int c = CW * (16 * j + n);  // past the row: a column that is not stored
                load_words<4 * VW>(v[r][j], row[r] + (FULL || c < hd ? c : 0) * ES);
            }
    }
    // dimensions d .. d + 3 of query n: [part][step][lane][8]
    static __device__ __forceinline__ void put_q(void *lds, int n, int d, v4f q)
    {
        const int j = d / (4 * DL), g = d / DL % 4, e = d % DL;
        const int step = j * (DL / 8) + e / 8;
        uint8_t *at = static_cast<uint8_t *>(lds) + (step * 64 + 16 * g + n) * 16 + e % 8 * 2;
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            *reinterpret_cast<uint2 *>(at + part * NS * 1024) = make_uint2(top16(q[1], q[0]), top16(q[3], q[2]));
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = rest16(q[i]);
        }
    }
    // operand of step `st`, keys of half i
    __device__ __forceinline__ void k_parts(v8b *out, int i, int st) const
    {
        if constexpr (TYPE == ORN_KV_BF16) {
            out[0] = as_v8b((u4){k[i][st][0], k[i][st][1], k[i][st][2], k[i][st][3]});
        } else if constexpr (TYPE == ORN_KV_F16) {
            u4 hi, lo;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float f[4];
                unpack4<TYPE>(f, &k[i][st][2 * w]);
                hi[2 * w] = top16(f[1], f[0]), hi[2 * w + 1] = top16(f[3], f[2]);
                lo[2 * w] = top16(rest16(f[1]), rest16(f[0]));
                lo[2 * w + 1] = top16(rest16(f[3]), rest16(f[2]));
            }
            out[0] = as_v8b(hi), out[1] = as_v8b(lo);
        } else {
            u4 hi;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float f[4];
                unpack4<TYPE>(f, &k[i][st / 2][2 * (st % 2) + w]);
                hi[2 * w] = top16(f[1], f[0]), hi[2 * w + 1] = top16(f[3], f[2]);
            }
            out[0] = as_v8b(hi);
        }
    }
    static __device__ __forceinline__ v4f mma(v8b a, v8b b, v4f c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ void scores(float *s, const void *lds, int lane, int) const
    {
        const v8b *q = static_cast<const v8b *>(lds) + lane;
        v4f x[NI], y[NI];  // the products of the first parts; the others
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i] = y[i] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            v8b kk[NI][NP], qq[3];
#pragma unroll
            for (int i = 0; i < NI; ++i) k_parts(kk[i], i, st);
#pragma unroll
            for (int part = 0; part < 3; ++part) qq[part] = q[64 * (part * NS + st)];
            auto add = [&](v4f *z, int kp, int qp) {
#pragma unroll
                for (int i = 0; i < NI; ++i) z[i] = mma(kk[i][kp], qq[qp], z[i]);
            };
            add(x, 0, 0);
            add(y, 0, 2);
            add(y, 0, 1);
            if constexpr (NP == 2) {
                add(y, 1, 1);
                add(y, 1, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * i + r] = x[i][r] + y[i][r];
    }
    __device__ __forceinline__ void leave_out(int) {}
    __device__ __forceinline__ void pv(v4f *o, const float *p) const
    {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
            v8b pp[3];
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[8 * gr + e];
#pragma unroll
            for (int part = 0; part < 3; ++part) {
                u4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = top16(x[2 * e + 1], x[2 * e]);
                pp[part] = as_v8b(w);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = rest16(x[e]);
            }
#pragma unroll
            for (int j = 0; j < NH; ++j)
#pragma unroll
                for (int c = 0; c < CW; c += 4) pv4(o + j * CW + c, pp, v + 8 * gr, j, c);
        }
    }
    // Four columns of O: their operands are V's rows turned.
    static __device__ __forceinline__ void pv4(v4f *o, const v8b *pp, const uint32_t (*v)[NH][VW], int j,
                                               int c)
    {
        u4 hi[4], lo[4];
        if constexpr (TYPE == ORN_KV_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    hi[i][e] = __builtin_amdgcn_perm(v[2 * e + 1][j][(c + i) / 2], v[2 * e][j][(c + i) / 2],
                                                     i % 2 ? 0x07060302u : 0x05040100u);
        } else {
            float f[8][4];
#pragma unroll
            for (int e = 0; e < 8; ++e) unpack4<TYPE>(f[e], &v[e][j][c * ES / 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[i][e] = top16(f[2 * e + 1][i], f[2 * e][i]);
                    if constexpr (NP == 2) lo[i][e] = top16(rest16(f[2 * e + 1][i]), rest16(f[2 * e][i]));
                }
        }
        auto add = [&](int part, const u4 *b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = mma(pp[part], as_v8b(b[i]), o[i]);
        };
        add(2, hi);
        if constexpr (NP == 2) add(1, lo);
        add(1, hi);
        if constexpr (NP == 2) add(0, lo);
        add(0, hi);
    }
    static __device__ __forceinline__ int col(int c, int n) { return CW * (16 * (c / CW) + n) + c % CW; }
};

// ---------------------------------------------------------------------------
// Returns whether one of this thread's sums is not finite.
template <int TYPE, int HD, class Path>
__device__ bool attend_segment(const ornk_kv_pages &p, const ornk_attend_args &a, const AttendWs &w,
                               const Seg &sg, uint8_t *lds, int slot, int tid)
{
    constexpr int KT = Path::KT, NI = KT / 16, NO = Path::NO, ES = elem_size<TYPE>;
    __shared__ float sm[WAVES][16], sl[WAVES][16];
    const int lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hd = p.hd, len = sg.len;

    // Pages: lane i holds the page of place page0 + i of the table.  A tile's
    // tokens are in places of one such 64 (their first is a multiple of KT).
    const int *table = a.table + (size_t)sg.b * a.max_pages;
    const uint32_t row_bytes = hd * ES, page_bytes = (row_bytes << p.page_log2) * p.kv;
    const size_t head = (size_t)(row_bytes << p.page_log2) * sg.h;
    const uint8_t *kp = static_cast<const uint8_t *>(p.k) + head;
    const uint8_t *vp = static_cast<const uint8_t *>(p.v) + head;
    int page0 = -1, ids = 0;
    auto pages_for = [&](int t) {
        const int want = (t >> p.page_log2) & ~63;
        if (want == page0) return;
        page0 = want;
        const int i = want + lane;
        ids = i <= (len - 1) >> p.page_log2 ? kv_page(p, table[i], sg.b) : -1;
    };
    // the row of token t, through its page (page 0 for one that is none)
    auto place = [&](const uint8_t *base, int t, bool &ok) {
        const int id = __builtin_amdgcn_ds_bpermute(4 * ((t >> p.page_log2) & 63), ids);
        ok = id >= 0;
        return base + (size_t)(uint32_t)max(id, 0) * page_bytes + (uint32_t)(t & (p.page - 1)) * row_bytes;
    };

    Path x;
    bool ok[NI];  // whether this lane's four tokens of each 16 have a page
    auto load_k = [&](int t) {  // past the sequence's last token: that one again
        const uint8_t *row[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            bool any;
            row[i] = place(kp, min(t + 16 * i + n, len - 1), any);
        }
        x.load_k(row, g, hd);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load_v = [&](int t) {
        const uint8_t *row[4 * NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int at = min(t + 16 * i + 4 * g, (len - 1) & ~3);  // four of one page
            const uint8_t *first = place(vp, at, ok[i]);
#pragma unroll
            for (int r = 0; r < 4; ++r) row[4 * i + r] = first + (uint32_t)min(r, len - 1 - at) * row_bytes;
        }
        x.load_v(row, n, hd);
        __builtin_amdgcn_sched_barrier(0);
    };

    // On their way together: the table, the queries, then the first K and V.
    int t = sg.k0 + KT * wave;
    if (t < sg.k1) pages_for(t);
    v4f q[HD / 64];
    {
        const float *src = a.q + ((size_t)sg.b * a.heads + sg.j0) * hd;
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
            const int at = tid + 64 * WAVES * i, row = at / (HD / 4), d = at % (HD / 4) * 4;
            q[i] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};  // of heads past the last too
            if (row >= sg.rows) continue;
            if (hd % 4 == 0) {
                if (d < hd) q[i] = *reinterpret_cast<const v4f *>(src + (size_t)row * hd + d);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < hd) q[i][e] = src[(size_t)row * hd + d + e];
            }
        }
    }
    if (Path::ahead && t < sg.k1) {
        load_k(t);
        load_v(t);
    }
    __syncthreads();  // what the last segment left in LDS is consumed
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        const int at = tid + 64 * WAVES * i;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[i][e] = q[i][e] * (a.scale * 1.44269504088896341f) * p.k_scale;
        Path::put_q(lds, at / (HD / 4), at % (HD / 4) * 4, q[i]);
    }
    __syncthreads();

    v4f o[NO];
#pragma unroll
    for (int c = 0; c < NO; ++c) o[c] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    float s[4 * NI];
    v4f raw[NI];
    // A tile's scores kept for the weights: after the next tile's loads, which
    // would wait for a store before them (they are counted in order).
    auto keep = [&](int t) {
        if (w.s && n < sg.rows) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
                *reinterpret_cast<v4f *>(w.s + sg.score + n * w.s_len + t + 16 * i + 4 * g) = raw[i];
        }
    };
    // a tile's scores without the keys that are left out
    auto mask = [&](int t) {
        bool all = t + KT <= len;
#pragma unroll
        for (int i = 0; i < NI; ++i) all = all && ok[i];
        if (__any(!all)) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!ok[i] || t + 16 * i + 4 * g + r >= len) {
                        s[4 * i + r] = -INFINITY;
                        x.leave_out(4 * i + r);
                    }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) raw[i] = (v4f){s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
    };
    auto tile_max = [&]() {
        float tm = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * NI; ++i) tm = fmaxf(tm, s[i]);
        tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
        tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
        return tm;
    };
    // the softmax of a tile's scores, and its O
    auto rest = [&](int t) {
        mask(t);
        const float tm = tile_max();
        // the reference moves only when the maximum has passed it by a factor
        // of 2^6 (weights up to that stay): O is left alone in most tiles
        const float mn = tm > m + 6.0f ? tm : m;
        if (__any(mn != m)) {
            const float corr = weight_from(m, mn);
            l *= corr;
            float cr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) cr[r] = __shfl(corr, 4 * g + r, 64);
#pragma unroll
            for (int c = 0; c < NO; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[c][r] *= cr[r];
            m = mn;
        }
#pragma unroll
        for (int i = 0; i < 4 * NI; ++i) {
            s[i] = s[i] == -INFINITY ? 0.0f : exp2_(s[i] - mn);
            l += s[i];
        }
        x.pv(o, s);
    };
    if constexpr (Path::shares) {
        auto tile = [&](int t) {
            asm volatile("" ::: "memory");
            pages_for(t);
            load_k(t);
            load_v(t);
            x.scores(s, lds, lane, hd);
            mask(t);
        };
        auto weight = [&](float v) { return v == -INFINITY ? 0.0f : exp2_(v - m); };
        for (int u = t; u < sg.k1; u += KT * WAVES) {
            tile(u);
            const float mn = fmaxf(m, tile_max());
            l *= weight_from(m, mn);
            m = mn;
#pragma unroll
            for (int i = 0; i < 4 * NI; ++i) l += weight(s[i]);
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) {
            sm[wave][n] = m;
            sl[wave][n] = l;
        }
        __syncthreads();
        const float M = fmaxf(fmaxf(sm[0][n], sm[1][n]), fmaxf(sm[2][n], sm[3][n]));
        float L = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) L += sl[v][n] * weight_from(sm[v][n], M);
        l *= weight_from(m, M);
        m = M;
        const float share = L != 0.0f ? 1.0f / L : 0.0f;
        for (; t < sg.k1; t += KT * WAVES) {
            tile(t);
#pragma unroll
            for (int i = 0; i < 4 * NI; ++i) s[i] = weight(s[i]) * share;
            x.pv(o, s);
            keep(t);
        }
    } else if constexpr (Path::ahead) {
        // the next tile's K is on its way from the scores on, its V from O on
        if (t < sg.k1) {
            for (; t + KT * WAVES < sg.k1; t += KT * WAVES) {
                asm volatile("" ::: "memory");  // the queries are read from LDS in every tile
                x.scores(s, lds, lane, hd);
                pages_for(t + KT * WAVES);
                load_k(t + KT * WAVES);
                rest(t);
                load_v(t + KT * WAVES);
                keep(t);
            }
            x.scores(s, lds, lane, hd);
            rest(t);
            keep(t);
        }
    } else {
        for (; t < sg.k1; t += KT * WAVES) {
            asm volatile("" ::: "memory");
            pages_for(t);
            load_k(t);
            load_v(t);
            x.scores(s, lds, lane, hd);
            rest(t);
            keep(t);
        }
    }
    if constexpr (!Path::shares) {
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
    }

    __syncthreads();  // the queries are consumed
    if (g == 0) {
        sm[wave][n] = m;
        sl[wave][n] = l;
    }
    float *ob = reinterpret_cast<float *>(lds);  // [wave][rows][HD]
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = 4 * g + r;
        if (row >= sg.rows) continue;
#pragma unroll
        for (int c = 0; c < NO; c += 4) {
            const v4f v = {o[c][r], o[c + 1][r], o[c + 2][r], o[c + 3][r]};
            *reinterpret_cast<v4f *>(ob + ((size_t)wave * sg.rows + row) * HD + Path::col(c, n)) = v;
        }
    }
    __syncthreads();
    const int c = 4 * (tid % (HD / 4));
    float z = 0.0f;
#pragma unroll
    for (int row = tid / (HD / 4); row < 16; row += 64 * WAVES / (HD / 4)) {
        if (row >= sg.rows) break;
        v4f part[WAVES];
        float pm[WAVES], pl[WAVES];
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            part[v] = *reinterpret_cast<const v4f *>(ob + (v * sg.rows + row) * HD + c);
            pm[v] = sm[v][row];
            pl[v] = sl[v][row];
        }
        const float M = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
        float L = 0.0f;
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            const float f = weight_from(pm[v], M);  // (a wave without tokens holds zeros)
            L += pl[v] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(part[v][e], f, acc[e]);
        }
        z += L * 0.0f + (acc[0] * 0.0f + acc[1] * 0.0f) + (acc[2] * 0.0f + acc[3] * 0.0f);
        float2 *ml;
        if (slot < 0) {  // the whole pair
            const size_t at = (size_t)sg.b * a.heads + sg.j0 + row;
            float *out = a.out + at * hd + c;
            const float f = Path::shares ? 1.0f : 1.0f / L;
#pragma unroll
            for (int e = 0; e < 4; ++e)  // (no weight: zeros, also of an infinity)
                acc[e] = L != 0.0f ? acc[e] * f * p.v_scale : 0.0f;
            if (hd % 4 == 0) {
                if (c < hd) *reinterpret_cast<v4f *>(out) = acc;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < hd) out[e] = acc[e];
            }
            ml = w.ml ? w.ml + at : nullptr;
        } else {
            const size_t at = (size_t)slot * 16 + row;
            if (c < w.row) *reinterpret_cast<v4f *>(w.part_o + at * w.row + c) = acc;
            ml = w.part_ml + at;
        }
        // of a part, L below zero: O is the sum of shares
        if (c == 0 && ml) *ml = make_float2(M, Path::shares && slot >= 0 ? -L : L);
    }
    return z != 0.0f;
}

// A stretch of 256 sequences, four to a lane; every wave has it for itself, so
// that finding one's place on the line takes no barrier.
constexpr int STRETCH = 256;
struct Stretch {
    int c0;                          // the first
    uint32_t end;                    // units of a pair up to the last one's end
    int len[4];                      // the lane's: tokens, units, units before
    uint32_t units[4], before[4];
};

__device__ __forceinline__ Stretch scan_lens(const ornk_kv_pages &p, const ornk_attend_args &a,
                                             const AttendWs &w, int c0, uint32_t before, int lane)
{
    Stretch s;
    s.c0 = c0;
    const int b0 = c0 + 4 * lane;
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = a.lens[min(b0 + i, a.n_seqs - 1)];
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s.len[i] = b0 + i < a.n_seqs ? kv_len(p, at[i], b0 + i, a.max_len) : 0;
        s.units[i] = (uint32_t)((s.len[i] + (1ll << w.unit_log2) - 1) >> w.unit_log2);
        s.before[i] = sum;
        sum += s.units[i];
    }
    const uint32_t x = wave_scan(sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) s.before[i] += before + x - sum;
    s.end = before + __builtin_amdgcn_readlane(x, 63);
    return s;
}

struct AttendCall {
    ornk_kv_pages p;
    ornk_attend_args a;
    AttendWs w;
};

// The segments of this group's stretch of the line, in order.
template <class F>
__device__ __forceinline__ void walk(const AttendCall &call, int tid, F segment)
{
    const ornk_kv_pages &p = call.p;
    const ornk_attend_args &a = call.a;
    const AttendWs &w = call.w;
    const int G = a.heads / p.kv, HT = (G + 15) / 16;
    const uint32_t per = p.kv * HT;  // pairs of a sequence
    const int lane = tid & 63;
    Stretch st;
    for (int c = 0; c == 0 || c < a.n_seqs; c += STRETCH) {
        st = scan_lens(p, a, w, c, c ? st.end : 0, lane);
        if (blockIdx.x == 0 && tid < 64) {
            const int b = c + 4 * tid;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (b + i < a.n_seqs) w.cum[b + i] = st.before[i];
            if (tid == 0) w.cum[min(c + STRETCH, a.n_seqs)] = st.end;
        }
    }
    const uint32_t T = st.end * per;
    const uint32_t lo = line_at(T, w.w_log2, blockIdx.x), hi = line_at(T, w.w_log2, blockIdx.x + 1);
    if (st.c0 && lo < hi) st = scan_lens(p, a, w, 0, 0, lane);
    const uint32_t whole = line_whole(T, w.w_log2, w.whole);
    for (uint32_t u = lo; u < hi;) {
        while (u >= st.end * per) st = scan_lens(p, a, w, st.c0 + STRETCH, st.end, lane);
        int b = -1, len = 0;  // u's sequence, in its lane
        uint32_t units = 0, start = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (u - st.before[i] * per < st.units[i] * per) {  // (wraps where u is before it)
                b = st.c0 + 4 * lane + i;
                len = st.len[i];
                units = st.units[i];
                start = st.before[i] * per;
            }
        const int from = __ffsll((unsigned long long)__ballot(b >= 0)) - 1;
        Seg sg;
        sg.b = __builtin_amdgcn_readlane(b, from);
        sg.len = __builtin_amdgcn_readlane(len, from);
        const uint32_t n = __builtin_amdgcn_readlane(units, from);
        const uint32_t off = u - __builtin_amdgcn_readlane(start, from);
        // off / n of integers below 2^22: fp32's quotient is at most one off
        uint32_t pair = (uint32_t)((float)off / (float)n);
        if (pair * n > off) --pair;
        else if (off - pair * n >= n) ++pair;
        uint32_t k = off - pair * n, cnt = min(n - k, hi - u);
        if (n <= whole) {  // a bound within it moves to its nearer end
            if (k && 2 * k >= n) {
                u += n - k;
                continue;
            }
            u -= k;
            if (hi - u < n && 2 * (hi - u) < n) break;
            k = 0, cnt = n;
        }
        const int tile = HT == 1 ? 0 : pair % HT, j = 16 * tile;
        sg.h = HT == 1 ? pair : pair / HT;
        sg.j0 = sg.h * G + j;
        sg.rows = min(16, G - j);
        sg.k0 = k << w.unit_log2;
        sg.k1 = (int)min((long long)sg.len, (long long)(k + cnt) << w.unit_log2);
        sg.score = ((size_t)sg.b * a.heads + sg.j0) * w.s_len;
        const int slot = cnt == n ? -1 : 2 * (int)blockIdx.x + (k ? 0 : 1);
        segment(sg, slot);
        u += cnt;
    }
}

template <int TYPE, int HD, class Path>
__global__ void __launch_bounds__(64 * WAVES, (1 << groups_log2(TYPE, HD))) k_kv_attend(AttendCall call)
{
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ uint32_t odd[MAX_SEGMENTS / 32 + 1];  // a bit each; whether there is one
    for (int i = threadIdx.x; i <= MAX_SEGMENTS / 32; i += 64 * WAVES) odd[i] = 0;
    uint32_t at = 0;
    walk(call, threadIdx.x, [&](const Seg &sg, int slot) {
        if (attend_segment<TYPE, HD, Path>(call.p, call.a, call.w, sg, lds, slot, threadIdx.x)) {
            atomicOr(&odd[at / 32], 1u << at % 32);
            odd[MAX_SEGMENTS / 32] = 1;
        }
        ++at;
    });
    // sequences without tokens: zeros
    const ornk_attend_args &a = call.a;
    for (int b = blockIdx.x; b < a.n_seqs; b += gridDim.x) {
        if (a.lens[b] > 0 && a.max_len > 0) continue;
        float *out = a.out + (size_t)b * a.heads * call.p.hd;
        for (size_t i = threadIdx.x; i < (size_t)a.heads * call.p.hd; i += 64 * WAVES) out[i] = 0.0f;
    }
    __syncthreads();
    if (!odd[MAX_SEGMENTS / 32]) return;
    // Segments whose sums were not finite.  Nothing that the first walk has formed is
    // held in registers for them (5 x 2047 tokens of 12 kv heads of 64 in fp32: 19.2
    // instead of 17.4 us): the call is read anew.
    auto args = __builtin_amdgcn_kernarg_segment_ptr();
    int tid = threadIdx.x;
    asm volatile("" : "+s"(args), "+v"(tid));
    const AttendCall again = *(const AttendCall *)args;
    at = 0;
    walk(again, tid, [&](const Seg &sg, int slot) {
        if (odd[at / 32] >> at % 32 & 1)
            attend_segment<TYPE, HD, Shares<TYPE, HD, Path::vec, Path::full>>(again.p, again.a, again.w, sg, lds,
                                                                              slot, tid);
        ++at;
    });
}

// The n parts of a pair (below 2: nothing is left to do), from group w0 on.
struct PairParts {
    uint32_t n, w0;
    __device__ __forceinline__ size_t slot(uint32_t i) const { return 2 * (w0 + i) + (i ? 0 : 1); }
};
__device__ __forceinline__ PairParts parts_of(const AttendWs &w, uint32_t per, int n_seqs, int b, int pair)
{
    const uint32_t before = w.cum[b], n = w.cum[b + 1] - before, T = w.cum[n_seqs] * per;
    const uint32_t s = before * per + pair * n;
    PairParts r = {1, 0};
    if (n <= line_whole(T, w.w_log2, w.whole)) return r;
    r.w0 = line_group(T, w.w_log2, s);
    r.n = line_group(T, w.w_log2, s + n - 1) - r.w0 + 1;
    return r;
}

// What is left after the groups, in one launch.  Work groups blockIdx.x < jx:
// the parts of a pair put together, JC float4s of its rows by JS shares of the
// parts.  The others, where the weights are asked for: what 4 FT tokens got,
// summed over a kv head's query heads; they put the parts' maxima and sums
// together for themselves.
constexpr int JC = 32, JS = 8, FT = JC * JS;

__device__ __forceinline__ void join_pair(const ornk_kv_pages &p, const ornk_attend_args &a, const AttendWs &w)
{
    __shared__ float sm[JS][JC], sl[JS][JC];
    __shared__ v4f so[JS][JC];
    const int b = blockIdx.z, pair = blockIdx.y, G = a.heads / p.kv, HT = (G + 15) / 16, hd = p.hd;
    const PairParts seg = parts_of(w, p.kv * HT, a.n_seqs, b, pair);
    if (seg.n < 2) return;
    const int j = 16 * (pair % HT), rows = min(16, G - j), j0 = pair / HT * G + j;
    const int x = threadIdx.x % JC, sub = threadIdx.x / JC, at = blockIdx.x * JC + x;
    const int row = at / (w.row / 4), c = at % (w.row / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float m2, float l2, v4f o2) {
        const float mn = fmaxf(m, m2), f = weight_from(m, mn), f2 = weight_from(m2, mn);
        m = mn;
        l = l * f + l2 * f2;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * f + o2[e] * f2;
    };
    if (row < rows)
#pragma unroll 4
        for (uint32_t i = sub; i < seg.n; i += JS) {
            const size_t slot = seg.slot(i) * 16 + row;
            const float2 ml = w.part_ml[slot];
            const v4f part = *reinterpret_cast<const v4f *>(w.part_o + slot * w.row + c);
            add(ml.x, fabsf(ml.y), ml.y < 0.0f ? part * -ml.y : part);
        }
    sm[sub][x] = m;
    sl[sub][x] = l;
    so[sub][x] = o;
    __syncthreads();
    if (sub || row >= rows) return;
    for (int i = 1; i < JS; ++i) add(sm[i][x], sl[i][x], so[i][x]);
    o *= l != 0.0f ? 1.0f / l : 0.0f;
    if (l == 0.0f) {
        o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};  // no weight, also of an infinity
    } else if (o[0] * 0.0f + o[1] * 0.0f + o[2] * 0.0f + o[3] * 0.0f != 0.0f) {
        // not finite, or past the largest number on the way: every part by its share
        m = -INFINITY, l = 0.0f;
        for (uint32_t i = 0; i < seg.n; ++i) m = fmaxf(m, w.part_ml[seg.slot(i) * 16 + row].x);
        for (uint32_t i = 0; i < seg.n; ++i) {
            const float2 ml = w.part_ml[seg.slot(i) * 16 + row];
            l += fabsf(ml.y) * weight_from(ml.x, m);
        }
        o = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t i = 0; i < seg.n; ++i) {
            const size_t slot = seg.slot(i) * 16 + row;
            const float2 ml = w.part_ml[slot];
            const float share = (ml.y < 0.0f ? -ml.y : 1.0f) * weight_from(ml.x, m) / l;
            o += *reinterpret_cast<const v4f *>(w.part_o + slot * w.row + c) * share;
        }
    }
    float *out = a.out + ((size_t)b * a.heads + j0 + row) * hd + c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < hd) out[e] = o[e] * p.v_scale;
}

__device__ __forceinline__ void sum_weights(const ornk_kv_pages &p, const ornk_attend_args &a,
                                            const AttendWs &w, int chunk)
{
    __shared__ float2 mi[16];  // of a tile's query heads: maximum, 1 / sum
    const int b = blockIdx.z, G = a.heads / p.kv, HT = (G + 15) / 16, h = blockIdx.y / HT;
    const int len = min(max(a.lens[b], 0), a.max_len);
    const long long t0 = (long long)chunk * FT * 4, t = t0 + threadIdx.x * 4;
    if (blockIdx.y % HT || t0 >= len) return;
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int tile = 0; tile < HT; ++tile) {
        const size_t j0 = (size_t)b * a.heads + h * G + 16 * tile;
        const int rows = min(16, G - 16 * tile), row = threadIdx.x / 16, share = threadIdx.x % 16;
        const PairParts seg = parts_of(w, p.kv * HT, a.n_seqs, b, h * HT + tile);
        float m = -INFINITY, l = 0.0f;
        auto add = [&](float m2, float l2) {
            const float mn = fmaxf(m, m2);
            l = l * weight_from(m, mn) + l2 * weight_from(m2, mn);
            m = mn;
        };
        if (row < rows) {
            if (seg.n < 2) {
                const float2 ml = w.ml[j0 + row];
                m = ml.x, l = share ? 0.0f : ml.y;
            } else {
#pragma unroll 4
                for (uint32_t i = share; i < seg.n; i += 16) {
                    const float2 ml = w.part_ml[seg.slot(i) * 16 + row];
                    add(ml.x, fabsf(ml.y));
                }
            }
        }
#pragma unroll
        for (int d = 8; d; d >>= 1) add(__shfl_xor(m, d, 16), __shfl_xor(l, d, 16));
        __syncthreads();  // the last tile's are consumed
        if (share == 0) mi[row] = make_float2(m, 1.0f / l);
        __syncthreads();
        if (t >= len) continue;
#pragma unroll 4
        for (int g = 0; g < rows; ++g) {
            const v4f s = *reinterpret_cast<const v4f *>(w.s + (j0 + g) * w.s_len + t);
            const float2 ml = mi[g];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += s[e] == -INFINITY ? 0.0f : exp2_(s[e] - ml.x) * ml.y;
        }
    }
    if (t >= len) return;
    const size_t i = ((size_t)b * p.kv + h) * a.score_stride + t;
    const int old = a.score_in ? max(len - a.score_new, 0) : 0;  // tokens that have a score
    if (a.score_stride % 4 == 0 && t + 4 <= len) {
        if (a.score_in) {
            const v4f x = *reinterpret_cast<const v4f *>(a.score_in + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = t + e < old ? fmaf(a.decay, x[e], sum[e]) : sum[e];
        }
        *reinterpret_cast<v4f *>(a.score_out + i) = sum;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (t + e < len) a.score_out[i + e] = t + e < old ? fmaf(a.decay, a.score_in[i + e], sum[e]) : sum[e];
}

__global__ void __launch_bounds__(FT) k_kv_finish(ornk_kv_pages p, ornk_attend_args a, AttendWs w, int jx)
{
    if ((int)blockIdx.x < jx) join_pair(p, a, w);
    else sum_weights(p, a, w, blockIdx.x - jx);
}

size_t attend_ws(const ornk_kv_pages *p, const ornk_attend_args *a, AttendWs *w)
{
    size_t off = 0;
    uint8_t *base = static_cast<uint8_t *>(a->ws);
    auto take = [&](size_t n) {
        uint8_t *at = base + off;
        off += (n + 255) & ~(size_t)255;
        return at;
    };
    const int HD = p->hd <= 64 ? 64 : p->hd <= 128 ? 128 : 256;
    w->w_log2 = CUS_LOG2 + groups_log2(p->type, HD);
    const int G = a->heads / p->kv, W = 1 << w->w_log2;
    w->row = (p->hd + 3) & ~3;
    w->unit_log2 = unit_log2(p->type, HD);
    const size_t pairs = (size_t)a->n_seqs * p->kv * ((G + 15) / 16);
    while (w->unit_log2 < 31 && pairs * (((size_t)a->max_len >> w->unit_log2) + 1) >> LINE_LOG2) ++w->unit_log2;
    const size_t longest = ((size_t)a->max_len + ((size_t)1 << w->unit_log2) - 1) >> w->unit_log2;
    w->whole = longest <= 2 || (longest <= 8 && pairs >= (size_t)W / 2) ? (uint32_t)longest : 1;
    w->cum = reinterpret_cast<uint32_t *>(take(((size_t)a->n_seqs + 1) * 4));
    w->part_ml = reinterpret_cast<float2 *>(take((size_t)2 * W * 16 * 8));
    w->part_o = reinterpret_cast<float *>(take((size_t)2 * W * 16 * w->row * 4));
    w->ml = nullptr;
    w->s = nullptr;
    w->s_len = 0;
    if (a->score_out) {
        const size_t rows = (size_t)a->n_seqs * a->heads;
        w->s_len = ((size_t)a->max_len + 63) / 64 * 64;  // whole tiles
        w->ml = reinterpret_cast<float2 *>(take(rows * 8));
        w->s = reinterpret_cast<float *>(take(rows * w->s_len * 4));
    }
    return off;
}

template <int TYPE, int HD, class Path>
int launch_hd(const ornk_kv_pages *p, const ornk_attend_args *a, const AttendWs &w, hipStream_t s)
{
    // the queries as the path takes them, then O of the waves; at most 64 KB
    const int G = a->heads / p->kv, rows = G < 16 ? G : 16;
    size_t lds = (size_t)WAVES * rows * HD * 4;
    if (lds < Path::Q_BYTES) lds = Path::Q_BYTES;
    if (lds < Exact<TYPE, HD, true, true>::Q_BYTES) lds = Exact<TYPE, HD, true, true>::Q_BYTES;
    const AttendCall call = {*p, *a, w};
    hipLaunchKernelGGL((k_kv_attend<TYPE, HD, Path>), dim3(1 << w.w_log2), dim3(64 * WAVES), lds, s, call);
    return hipGetLastError();
}

template <int TYPE, int HD, bool FULL>
int launch_full(const ornk_kv_pages *p, const ornk_attend_args *a, const AttendWs &w, hipStream_t s)
{
    if constexpr (TYPE == ORN_KV_F32) return launch_hd<TYPE, HD, Exact<TYPE, HD, true, FULL>>(p, a, w, s);
    else return launch_hd<TYPE, HD, Parts<TYPE, HD, FULL>>(p, a, w, s);
}

template <int TYPE, int HD>
int launch_type(const ornk_kv_pages *p, const ornk_attend_args *a, const AttendWs &w, hipStream_t s)
{
    return p->hd == HD ? launch_full<TYPE, HD, true>(p, a, w, s)
           : p->hd * elem_size<TYPE> % 16 == 0
               ? launch_full<TYPE, HD, false>(p, a, w, s)
               : launch_hd<TYPE, HD, Exact<TYPE, HD, false, false>>(p, a, w, s);
}

template <int TYPE>
int launch_type(const ornk_kv_pages *p, const ornk_attend_args *a, const AttendWs &w, hipStream_t s)
{
    return p->hd <= 64    ? launch_type<TYPE, 64>(p, a, w, s)
           : p->hd <= 128 ? launch_type<TYPE, 128>(p, a, w, s)
                          : launch_type<TYPE, 256>(p, a, w, s);
}

}  // namespace

extern "C" size_t ornk_kv_attend_ws(const ornk_kv_pages *p, const ornk_attend_args *a)
{
    AttendWs w;
    return attend_ws(p, a, &w);
}

extern "C" int ornk_kv_attend(const ornk_kv_pages *p, const ornk_attend_args *a, hipStream_t s)
{
    AttendWs w;
    attend_ws(p, a, &w);
    int rc = p->type == ORN_KV_F32    ? launch_type<ORN_KV_F32>(p, a, w, s)
             : p->type == ORN_KV_F16  ? launch_type<ORN_KV_F16>(p, a, w, s)
             : p->type == ORN_KV_BF16 ? launch_type<ORN_KV_BF16>(p, a, w, s)
                                      : launch_type<ORN_KV_E4M3>(p, a, w, s);
    if (rc != hipSuccess) return rc;
    const int G = a->heads / p->kv, HT = (G + 15) / 16;
    const int jx = a->max_len > (long long)w.whole << w.unit_log2  // else no pair is cut
                       ? ((G < 16 ? G : 16) * (w.row / 4) + JC - 1) / JC : 0;
    const int sx = a->score_out ? (int)(((long long)a->max_len + 4 * FT - 1) / (4 * FT)) : 0;
    if (jx + sx)
        hipLaunchKernelGGL(k_kv_finish, dim3(jx + sx, p->kv * HT, a->n_seqs), dim3(FT), 0, s, *p, *a, w, jx);
    return hipGetLastError();
}
