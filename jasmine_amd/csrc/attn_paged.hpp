// Attention of a ragged batch's rows over the paged cache: decode steps and chunks of prompts.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = 2^(scale log2(e) q . k_t - m) over the keys t that the row
// sees: one pass over the keys with the running maximum m and sum, in fp32.  The G query heads
// of a key head are rows like its tokens are: row r of a (sequence, key head) is token r / G,
// head r % G, and a tile is M such rows, so grouped heads read the cache once.
//
// Both kernels compute S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_bf16.  A lane's scores
// belong to its own row (lane % 16) and to keys {4 g + j, 16 + 4 g + j} of 32 (g = lane / 16, j < 4),
// which is the B operand of the second product if V is read in that order of keys, so P stays in
// the lane that made it.  V^T's rows may be any d: row r16 of product i is d = EV r16 + i, so a lane
// that reads EV neighbouring d of its eight keys holds EV operands, transposed in registers.
//
// fp32 rows: q and p as three bf16 parts each (exact, split.hpp), and fp32 cache values too, so
// that 3 or 6 products make fp32 accuracy.  8-bit codes are bf16 numbers exactly; a key's scale
// multiplies its scores, a value's scale times 2^16 its weight (so that the weight's lower parts are
// bf16 numbers too, whose last bit is 2^-133, where scales go down to 2^-126).  bf16 rows: p as one bf16 number where the sum
// of the weights can be taken of what was rounded (by a product with ones: a row that one key
// dominates then loses nothing), and as two where it cannot (scaled weights) or where the products
// are for nothing (few rows): one part alone left results 1.5 times as far from 64 bits as their own
// rounding does.
//
// What the products cannot give (infinities, NaN, sums past fp32, values that masked keys hold: a
// weight of 0 times NaN) ends in a result that is not finite; such a row is computed again by
// paged_row in plain fp32, which looks at no key that the row does not see.
#pragma once
#include "attn_paged_plan.hpp"
#include "paged.hpp"
#include "split.hpp"

#include <cfloat>

namespace jas {

struct PagedAttnArgs {
    const void *q;
    void *o;
    PagedView kv;
    BatchView bt;
    int H, G, max_len, causal;  // G: query heads per key head
    FastDiv by_group;
    long q_st, q_sh, o_st, o_sh;
    float scale_log2;
    int q_vec, o_vec;           // rows of Q, O start on 16 bytes
    int tiles, nsplit, chunk;   // grid: tiles x nsplit x key heads; keys of a split, at least
    int sorted, cus;            // tiles in order of falling length; compute units
    float *part;                // nsplit > 1: rows of D means, then exponent base and sum
};

// One call's kernels for head dim 32, 64, 128
void paged_launch_32(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s);
void paged_launch_64(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s);
void paged_launch_128(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s);

template <int CK>
constexpr int cache_bytes = CK == CK_F32 ? 4 : CK == CK_BF16 ? 2 : 1;

// 2^x on the hardware's unit; results below 2^-126 are zero, which no sum that holds 1 misses
__device__ __forceinline__ float paged_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float paged_max_rows(float v)  // over lanes l, l ^ 16, l ^ 32, l ^ 48
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float paged_sum_rows(float v)
{
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A sequence of the batch: its rows, and its length with them
struct PagedSeq {
    int row0, rows, len;
};

// Tile x of the grid: sequence b owns tiles from floor(cu[b] G / M) + b on, at least as many as
// its rows fill, so the thread that holds b knows it from cu[b] and cu[b + 1] alone: one round of
// loads, no running sum.  Returns x's tile number in b, or -1.  By the whole workgroup.
template <int M>
__device__ __forceinline__ int paged_tile(const PagedAttnArgs &p, int x, int &b, PagedSeq &sq)
{
    __shared__ int s_b, s_seq[4];
    if (threadIdx.x == 0) s_b = -1, s_seq[3] = -1;
    __syncthreads();
    int own = -2, row0 = 0, rows = 0, len = 0, at = 0;
    for (int j = threadIdx.x; j < p.bt.B; j += 256) {
        const int c0 = max(0, min(p.bt.cu[j], p.bt.n)), c1 = max(c0, min(p.bt.cu[j + 1], p.bt.n)), n = p.bt.lens[j];
        const int first = (int)((long)c0 * p.G / M + j);
        if (first <= x && (j + 1 == p.bt.B || (int)((long)c1 * p.G / M + j + 1) > x))
            own = j, row0 = c0, rows = c1 - c0, len = n, at = x - first;
    }
    if (own >= 0) s_b = own;  // (one thread's, where cu does not fall)
    __syncthreads();
    if (own == s_b) s_seq[0] = row0, s_seq[1] = rows, s_seq[2] = max(0, min(len, min(p.kv.cap, p.max_len))), s_seq[3] = at;
    __syncthreads();
    b = max(0, s_b);
    sq.row0 = s_seq[0], sq.rows = s_seq[1], sq.len = s_seq[2];
    return s_seq[3];
}

// The same in order of falling length, for launches whose workgroups own whole sequences of keys (B
// <= 256): each thread adds the tiles of the sequences before its own.  Workgroups start in the order
// of their ids; where two fit on a unit, i and i + cus share one, so the second cus of them are
// taken from the light end.  24 sequences of up to 2048 keys, chunks of up to 256
// beside single tokens, bf16: 96 us unsorted, 77 sorted; 4 chunks of up to 512 over up to 4096 keys, bf16:
// 137, 126 (121 since the exponents' base is a row's own maximum).
template <int M>
__device__ __forceinline__ int paged_tile_sorted(const PagedAttnArgs &p, int x, int &b, PagedSeq &sq)
{
    __shared__ int s_tiles[256], s_len[256], s_seq[5];
    const int j = threadIdx.x;
    int row0 = 0, rows = 0, len = 0;
    if (j < p.bt.B) {
        row0 = max(0, min(p.bt.cu[j], p.bt.n));
        rows = max(0, min(p.bt.cu[j + 1], p.bt.n) - row0);
        len = max(0, min(p.bt.lens[j], min(p.kv.cap, p.max_len)));
    }
    const int tiles = (int)(((long)rows * p.G + M - 1) / M);
    s_tiles[j] = tiles, s_len[j] = len;
    if (j == 0) s_seq[3] = -1, s_seq[4] = 0;
    __syncthreads();
    int first = 0, total = 0;
    for (int k = 0; k < p.bt.B; ++k) {
        const int t = s_tiles[k], n = s_len[k];
        total += t;
        first += n > len || (n == len && k < j) ? t : 0;
    }
    const int lo = p.cus / p.kv.n_kv, hi = min(2 * lo, total);  // tiles of the first and second round
    if (x >= lo && x < hi) x = lo + hi - 1 - x;
    if (x >= first && x < first + tiles) s_seq[0] = row0, s_seq[1] = rows, s_seq[2] = len, s_seq[3] = x - first, s_seq[4] = j;
    __syncthreads();
    sq.row0 = s_seq[0], sq.rows = s_seq[1], sq.len = s_seq[2], b = s_seq[4];
    return s_seq[3];
}

// A workgroup's key head, tile and split.  Key heads are the fastest: where they are a multiple of 8,
// their tiles share one XCD's L2.  An XCD hands its workgroups to its shader engines in turn, so
// nsplit is odd (paged_plan): with an even one every sequence's last splits, which shorter sequences
// leave empty, would fall on the same engines.
__device__ __forceinline__ void paged_block(const PagedAttnArgs &p, int &hk, int &x, int &split)
{
    const int id = blockIdx.x, rest = id / p.kv.n_kv;
    hk = id % p.kv.n_kv, split = rest % p.nsplit, x = rest / p.nsplit;
}

// Keys [k_lo, k_hi) of a split: p.chunk of them, or as many as nsplit splits need to cover kend
__device__ __forceinline__ void paged_split(const PagedAttnArgs &p, int kend, int split, int &k_lo, int &k_hi)
{
    const int per = max(p.chunk, ((kend + p.nsplit - 1) / p.nsplit + 127) / 128 * 128);
    k_lo = (int)min((long)kend, (long)split * per);
    k_hi = (int)min((long)kend, (long)k_lo + per);
}

// Where key t of sequence b lies: the table's entry for its page, and the slot
__device__ __forceinline__ int paged_entry(const PagedAttnArgs &p, int b, int t, int &slot)
{
    const int q = (int)p.kv.by_page.div((uint32_t)t);
    slot = t - q * p.kv.page_size;
    return p.kv.table[(long)b * p.kv.table_stride + q];
}

template <int CK>
__device__ __forceinline__ float cache_value(const void *pool, long at)
{
    if constexpr (CK == CK_F32) return ((const float *)pool)[at];
    else if constexpr (CK == CK_BF16) return bf16_to_f32(((const uint16_t *)pool)[at]);
    else if constexpr (CK == CK_I8) return (float)((const int8_t *)pool)[at];
    else return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)pool)[at], 0);
}

// One query row in fp32 arithmetic by one wave: keys [k_lo, k_hi) of sequence b, head hk; q: the
// row's D values.  Every lane holds the maximum m (exponent units) and the sum l of the weights;
// out: elements lane + 64 e of the weighted mean of the values.  A mean of numbers near the end
// of fp32 is one itself though their sum is not: acc2 adds them times 2^-32.
template <int D, int CK, typename T>
__device__ __forceinline__ void paged_row(const PagedAttnArgs &p, int b, int hk, const T *q, int k_lo, int k_hi,
                                                    float &m, float &l, float (&out)[(D + 63) / 64])
{
    const int lane = threadIdx.x & 63;
    constexpr int E = (D + 63) / 64;
    float acc[E], acc2[E];
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc2[e] = 0.f;
    for (int k0 = k_lo; k0 < k_hi; k0 += 64) {
        const int t = k0 + lane;
        int slot = 0, page = -1;
        if (t < k_hi) page = paged_entry(p, b, t, slot);
        const bool sees = page >= 0 && page < p.kv.n_pages;
        const long at = (long)page * p.kv.page_stride + hk * p.kv.head_stride + slot * p.kv.tok_stride;
        const long sc = ((long)page * p.kv.n_kv + hk) * p.kv.page_size + slot;
        float s = -INFINITY, vs = 1.f;
        if (sees) {
            float d = 0.f;
            for (int e = 0; e < D; ++e) {
                float x;
                if constexpr (sizeof(T) == 4) x = q[e];
                else x = bf16_to_f32(q[e]);
                d = __builtin_fmaf(x, cache_value<CK>(p.kv.k, at + e), d);
            }
            if (CK >= CK_I8) d *= p.kv.ks[sc], vs = p.kv.vs[sc];
            s = d * p.scale_log2;
        }
        const float mx = fmaxf(m, wave_max(s)), base = mx == -INFINITY ? 0.f : mx;
        const float corr = paged_exp2(m - base), pv = sees ? paged_exp2(s - base) : 0.f;
        l = l * corr + wave_sum(pv);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= corr, acc2[e] *= corr;
        const unsigned long long seen = __builtin_amdgcn_ballot_w64(sees);
        for (int k = 0; k < 64; ++k) {
            if (!(seen >> k & 1)) continue;
            const float pk = __shfl(pv, k, WAVE) * __shfl(vs, k, WAVE);
            const long vat = __shfl(at, k, WAVE);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane + 64 * e < D) {
                    const float v = cache_value<CK>(p.kv.v, vat + lane + 64 * e);
                    acc[e] = __builtin_fmaf(pk, v, acc[e]);
                    acc2[e] = __builtin_fmaf(pk, v * 0x1p-32f, acc2[e]);
                }
        }
        m = mx;
    }
    const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = fabsf(acc[e]) <= FLT_MAX ? acc[e] * inv : acc2[e] * inv * 0x1p32f;
}

template <typename T>
__device__ __forceinline__ void paged_put(T *o, float v)
{
    if constexpr (sizeof(T) == 4) *o = v;
    else *o = __builtin_bit_cast(uint16_t, (__bf16)v);
}

// A row of a tile: its token row of Q and O, its head, and the keys below `end` that it sees
struct PagedRow {
    long tok;
    int h, end;
};
__device__ __forceinline__ PagedRow paged_row_of(const PagedAttnArgs &p, const PagedSeq &sq, int hk, int r)
{
    const int i = (int)p.by_group.div((uint32_t)r);
    PagedRow w;
    w.tok = sq.row0 + i;
    w.h = hk * p.G + r - i * p.G;
    w.end = p.causal ? max(0, min(sq.len, sq.len - sq.rows + i + 1)) : sq.len;
    return w;
}

// Computes the rows of a tile again whose bit in bad[] is set: results or partial results
template <int D, int CK, typename T>
__device__ __forceinline__ void paged_again(const PagedAttnArgs &p, int b, int hk, const PagedSeq &sq, int r0, int rows,
                                                      const unsigned *bad, int k_lo, int k_hi, float *part)
{
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int r = w; r < rows; r += 4) {
        if (!(bad[r / 32] >> (r % 32) & 1)) continue;
        const PagedRow row = paged_row_of(p, sq, hk, r0 + r);
        float m, l, out[(D + 63) / 64];
        paged_row<D, CK, T>(p, b, hk, (const T *)p.q + row.tok * p.q_st + row.h * p.q_sh, k_lo, min(k_hi, row.end), m, l, out);
        for (int e = 0; e < (D + 63) / 64; ++e) {
            const int d = lane + 64 * e;
            if (d >= D) continue;
            if (part) part[(long)r * (D + 4) + d] = out[e];
            else paged_put((T *)p.o + row.tok * p.o_st + row.h * p.o_sh + d, out[e]);
        }
        if (part && lane == 0) part[(long)r * (D + 4) + D] = m, part[(long)r * (D + 4) + D + 1] = l;
    }
}

// ---------------------------------------------------------------- operands
// Raw registers of 32 d of a key row, in the order of K's operand: lane (row r16, group g) slot
// j holds d = 32 c + 8 g + j (bf16), 32 c + 4 g + j and 32 c + 16 + 4 g + j - 4 (fp32), and with codes
// the 64 d of two steps lie 16 a lane: 64 (c / 2) + 16 g + 8 (c % 2) + j (D = 32: as bf16).
template <bool NT, typename V>
__device__ __forceinline__ V cache_load(const void *p)
{
    return NT ? __builtin_nontemporal_load((const V *)p) : *(const V *)p;
}
template <int D, int CK>
struct KOperand {
    static constexpr int CD = D / 32, RW = CK == CK_F32 ? 8 : CK == CK_BF16 ? 4 : 2;
    static __device__ __forceinline__ int d_of(int c, int g, int j)
    {
        if (CK == CK_F32) return 32 * c + 4 * g + (j < 4 ? j : 12 + j);
        if (CK == CK_BF16 || D == 32) return 32 * c + 8 * g + j;
        return 64 * (c / 2) + 16 * g + 8 * (c % 2) + j;
    }
    // steps c0 .. c0 + KC - 1 of a key (row: its first element); NT: a stream that is read once
    template <int KC, bool NT = false>
    static __device__ __forceinline__ void load(const void *row, int g, int c0, uint32_t (&r)[KC][RW])
    {
        const char *p = (const char *)row;
        if constexpr (CK == CK_F32) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 a = cache_load<NT, u32x4>(p + 128 * (c0 + c) + 16 * g), b = cache_load<NT, u32x4>(p + 128 * (c0 + c) + 16 * g + 64);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[c][e] = a[e], r[c][4 + e] = b[e];
            }
        } else if constexpr (CK == CK_BF16) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const u32x4 a = cache_load<NT, u32x4>(p + 64 * (c0 + c) + 16 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[c][e] = a[e];
            }
        } else if constexpr (D == 32) {
            const u32x2 a = cache_load<NT, u32x2>(p + 8 * g);
            r[0][0] = a[0], r[0][1] = a[1];
        } else {
            static_assert(KC % 2 == 0, "pairs of steps lie together");
#pragma unroll
            for (int c = 0; c < KC; c += 2) {
                const u32x4 a = cache_load<NT, u32x4>(p + 32 * (c0 + c) + 16 * g);
                r[c][0] = a[0], r[c][1] = a[1], r[c + 1][0] = a[2], r[c + 1][1] = a[3];
            }
        }
    }
};

// Codes of a word, low or high two, as bf16 numbers
template <int CK>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w, bool hi)
{
    if constexpr (CK == CK_F8) {
        return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    } else {
        const int sh = hi ? 16 : 0;
        const float a = (float)(int8_t)(w >> sh), b = (float)(int8_t)(w >> (sh + 8));
        // (bf16 numbers in fp32: their upper halves)
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
}

// Eight values of K's raw registers as operand planes (one, or three of 2^16 times fp32 values)
template <int CK, int RW, int NK>
__device__ __forceinline__ void k_planes(const uint32_t (&r)[RW], u32x4 (&pl)[NK])
{
    if constexpr (CK == CK_F32) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(r[e]);
        split8<true>(x, pl[0], pl[1], pl[2]);
    } else if constexpr (CK == CK_BF16) {
        pl[0] = u32x4{r[0], r[1], r[2], r[3]};
    } else {
        pl[0] = u32x4{codes_bf16<CK>(r[0], false), codes_bf16<CK>(r[0], true), codes_bf16<CK>(r[1], false), codes_bf16<CK>(r[1], true)};
    }
}

// EV neighbouring d of one key's value row: raw words
template <int CK, int EV>
struct VOperand {
    static constexpr int BYTES = EV * cache_bytes<CK>, RW = BYTES < 4 ? 1 : BYTES / 4;
    template <bool NT = false>
    static __device__ __forceinline__ void load(const void *p, uint32_t (&r)[RW])
    {
        if constexpr (BYTES == 2) r[0] = cache_load<NT, uint16_t>(p);
        else if constexpr (BYTES == 4) r[0] = cache_load<NT, uint32_t>(p);
        else if constexpr (BYTES == 8) {
            const u32x2 a = cache_load<NT, u32x2>(p);
            r[0] = a[0], r[1] = a[1];
        } else {
#pragma unroll
            for (int k = 0; k < RW; k += 4) {
                const u32x4 a = cache_load<NT, u32x4>((const char *)p + 4 * k);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[k + e] = a[e];
            }
        }
    }
};

// Element i of eight keys' raw registers as operand planes
template <int CK, int RW, int NK>
__device__ __forceinline__ void v_planes(const uint32_t (&r)[8][RW], int i, u32x4 (&pl)[NK])
{
    if constexpr (CK == CK_F32) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(r[j][i]);
        split8<true>(x, pl[0], pl[1], pl[2]);
    } else {
        const uint32_t sel = i % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t a, b;
            if constexpr (CK == CK_BF16) a = r[2 * k][i / 2], b = r[2 * k + 1][i / 2];
            else a = codes_bf16<CK>(r[2 * k][i / 4], i % 4 >= 2), b = codes_bf16<CK>(r[2 * k + 1][i / 4], i % 4 >= 2);
            pl[0][k] = __builtin_amdgcn_perm(b, a, sel);
        }
    }
}

__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// acc += a b over 32 k: NA planes of a, NB of b, small products first
template <int NA, int NB>
__device__ __forceinline__ floatx4 mfma_planes(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], floatx4 acc)
{
    if constexpr (NA == 3 && NB == 3) return mfma_split(a, b, acc);
    else {
        static_assert(NA == 1, "split operands meet split ones, or stand on the right");
#pragma unroll
        for (int k = NB - 1; k >= 0; --k) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[k], acc, 0, 0, 0);
        return acc;
    }
}

// Eight values of a lane's P operand as planes
template <int NP>
__device__ __forceinline__ void p_planes(const float (&e)[8], bf16x8 (&pf)[NP])
{
    if constexpr (NP == 3) {
        u32x4 a, b, c;
        split8(e, a, b, c);
        pf[0] = as_bf16x8(a), pf[1] = as_bf16x8(b), pf[2] = as_bf16x8(c);
    } else {
        float r[8];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const __bf16 h = (__bf16)(k ? r[j] : e[j]);
                pf[k][j] = h;
                r[j] = e[j] - (float)h;  // exact
            }
        }
    }
}

// Q's operand for one row: eight values a step in K's order of d (a row that is none: zeros)
template <int D, int CK, typename T, int NP>
__device__ __forceinline__ void q_planes(const T *q, bool there, int g, bool vec, bf16x8 (&qf)[D / 32][NP])
{
    using KO = KOperand<D, CK>;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (there) {
            if constexpr (sizeof(T) == 4) {
                const T *a = q + KO::d_of(c, g, 0), *b = q + KO::d_of(c, g, 4);
                if (vec) {
                    const floatx4 u = *(const floatx4 *)a, v = *(const floatx4 *)b;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = u[j], x[4 + j] = v[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
                }
            } else {
                const T *a = q + KO::d_of(c, g, 0);  // (eight neighbours: bf16 rows meet no fp32 cache)
                if (vec) {
                    const u32x4 u = *(const u32x4 *)a;
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[2 * j] = __uint_as_float(u[j] << 16), x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = bf16_to_f32(a[j]);
                }
            }
        }
        if constexpr (NP == 3) {
            u32x4 h, m, l;
            split8<true>(x, h, m, l);
            qf[c][0] = as_bf16x8(h), qf[c][1] = as_bf16x8(m), qf[c][2] = as_bf16x8(l);
        } else {
            p_planes<1>(x, qf[c]);
        }
    }
}

// ---------------------------------------------------------------- few rows: decode steps
// One workgroup: a tile of 16 rows and one split of its keys; the four waves take tiles of 32 keys in
// turn and keep a softmax each, joined at the end.  Nothing goes through LDS on the way: K and V
// are read from memory in operand order (each 16-lane group reads whole value rows, 64-byte
// pieces of key rows), V is transposed by v_perm in the lane that read it.
// Bound by memory: 32 sequences of 1024 to 4096 keys, 8 heads of 128, bf16: 342 MB in 71.5 us with the
// merge, 4.8 TB/s (a copy of 1 GiB: 5.1); 3 of up to 65536 in int8: 327 MB in 73; one of 1000 in fp32: 10 us,
// two launches and a chain of dependent loads.
// Waves a SIMD: loads in flight hide the memory's latency, as many as registers hold (fp32 rows keep
// three planes of Q, fp32 caches twice the raw words)
template <int D, int CK, typename T>
constexpr int stream_waves = D == 128 ? (sizeof(T) == 2 ? 3 : CK == CK_F32 ? 1 : 2) : CK == CK_F32 ? 2 : 3;

template <int D, int CK, typename T>
__global__ void __launch_bounds__(256, (stream_waves<D, CK, T>)) paged_stream_kernel(const PagedAttnArgs p)
{
    constexpr int M = 16, CD = D / 32, EV = D / 16, NP = sizeof(T) == 4 ? 3 : 1, NK = CK == CK_F32 ? 3 : 1;
    constexpr int PP = sizeof(T) == 4 ? 3 : 2;  // planes of P
    using KO = KOperand<D, CK>;
    using VO = VOperand<CK, EV>;
    constexpr int ES = cache_bytes<CK>, LD = D + 4;
    constexpr bool EIGHT = CK >= CK_I8;
    __shared__ float s_o[4][M][LD];
    __shared__ float s_m[4][M], s_l[4][M];
    __shared__ unsigned s_bad[1];
    __shared__ long s_off[4][32];
    __shared__ float s_sc[4][2][32];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int hk, x, split;
    paged_block(p, hk, x, split);
    int b;
    PagedSeq sq;
    const int tile = paged_tile<M>(p, x, b, sq);
    const int r0 = tile * M, rows = min(M, sq.rows * p.G - r0);
    if (tile < 0 || rows <= 0) return;
    const PagedRow row = paged_row_of(p, sq, hk, r0 + min(r16, rows - 1));
    const int kend = paged_row_of(p, sq, hk, r0 + rows - 1).end;  // (the last row of a tile sees most)
    const int kmin = paged_row_of(p, sq, hk, r0).end;
    int k_lo, k_hi;
    paged_split(p, kend, split, k_lo, k_hi);
    float *part = p.nsplit > 1 ? p.part + (((long)x * p.kv.n_kv + hk) * p.nsplit + split) * M * LD : nullptr;
    if (part && k_lo >= k_hi) {  // a split that this sequence does not need
        if ((int)threadIdx.x < rows) part[(long)threadIdx.x * LD + D] = -INFINITY, part[(long)threadIdx.x * LD + D + 1] = 0.f;
        return;
    }
    if (threadIdx.x == 0) s_bad[0] = 0;

    bf16x8 qf[CD][NP];
    q_planes<D, CK, T, NP>((const T *)p.q + row.tok * p.q_st + row.h * p.q_sh, r16 < rows, g, p.q_vec, qf);

    const char *kpool = (const char *)p.kv.k + hk * p.kv.head_stride * ES;
    const char *vpool = (const char *)p.kv.v + hk * p.kv.head_stride * ES + r16 * EV * ES;
    // The next tile's entries of the table, one key a lane (past the end: the last key's, unused).
    // Every load of the loop is made on every pass, so that each wait counts exactly the loads
    // that it needs; keys that are none read page 0, slot 0, over and over the same row.
    const int key_of = lane & 31;
    int page = 0, slot = 0;
    bool in = false;
    auto entry = [&](int t0) {
        in = t0 + key_of < k_hi;
        page = paged_entry(p, b, max(0, min(t0 + key_of, k_hi - 1)), slot);
    };
    unsigned valid = 0;  // keys of the tile in flight that have a page
    float ks = 0.f, vs = 0.f;
    auto place = [&]() {
        in = in & (page >= 0) & (page < p.kv.n_pages);
        valid = (unsigned)__builtin_amdgcn_ballot_w64(in);
        const long pg = in ? page : 0, sl = in ? slot : 0;
        s_off[w][lane & 31] = (pg * p.kv.page_stride + sl * p.kv.tok_stride) * ES;  // (both halves alike)
        if (EIGHT) {
            const long sc = (pg * p.kv.n_kv + hk) * p.kv.page_size + sl;
            ks = p.kv.ks[sc], vs = p.kv.vs[sc];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    uint32_t kr[2][CD][KO::RW], vr[8][VO::RW];
    auto kload = [&]() {
#pragma unroll
        for (int a = 0; a < 2; ++a) KO::template load<CD, true>(kpool + s_off[w][16 * a + r16], g, 0, kr[a]);
    };
    auto vload = [&]() {
#pragma unroll
        for (int j = 0; j < 8; ++j) VO::template load<true>(vpool + s_off[w][4 * g + j + (j < 4 ? 0 : 12)], vr[j]);
    };

    floatx4 oacc[EV];
    float m = -INFINITY, l = 0.f;  // this lane's row; l over its own keys
#pragma unroll
    for (int i = 0; i < EV; ++i) oacc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    const float sl2 = p.scale_log2 * (NP == 3 ? SPLIT_UNSCALE : 1.f) * (NK == 3 ? SPLIT_UNSCALE : 1.f);

    int t0 = k_lo + 32 * w;
    if (t0 < k_hi) {
        entry(t0);
        place();
        entry(t0 + 128);
        __builtin_amdgcn_sched_barrier(0);  // (the same order as in the loop)
        kload();
        __builtin_amdgcn_sched_barrier(0);
        vload();
        __builtin_amdgcn_sched_barrier(0);
    }
    for (; t0 < k_hi; t0 += 128) {
        const unsigned now = valid;
        floatx4 s[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            s[a] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < CD; ++c) {
                u32x4 pl[NK];
                k_planes<CK>(kr[a][c], pl);
                bf16x8 kf[NK];
#pragma unroll
                for (int k = 0; k < NK; ++k) kf[k] = as_bf16x8(pl[k]);
                s[a] = mfma_planes(kf, qf[c], s[a]);
            }
        }
        float vsc[8];
        if (EIGHT) {
            s_sc[w][0][lane & 31] = ks, s_sc[w][1][lane & 31] = vs * SPLIT_SCALE;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const floatx4 f = *(const floatx4 *)&s_sc[w][0][16 * a + 4 * g], v = *(const floatx4 *)&s_sc[w][1][16 * a + 4 * g];
                s[a] *= f;
#pragma unroll
                for (int r = 0; r < 4; ++r) vsc[4 * a + r] = v[r];
            }
        }
        place();          // the next tile's offsets (this tile's V is still in flight)
        entry(t0 + 256);  // (loads end in the order of their issue: before K, or the next place() waits for V)
        __builtin_amdgcn_sched_barrier(0);
        kload();
        __builtin_amdgcn_sched_barrier(0);
        // values of keys without a page, or past the end, are none
        if (now != 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool there = now >> (4 * g + j + (j < 4 ? 0 : 12)) & 1;
#pragma unroll
                for (int e = 0; e < VO::RW; ++e) vr[j][e] = there ? vr[j][e] : 0u;
                if (EIGHT) vsc[j] = there ? vsc[j] : 0.f;
            }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) s[a] *= sl2;
        if (now != 0xffffffffu || t0 + 32 > kmin) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int k = 16 * a + 4 * g + r;
                    s[a][r] = (now >> k & 1) && t0 + k < row.end ? s[a][r] : -INFINITY;
                }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = fmaxf(m, paged_max_rows(mx));
        if (__builtin_amdgcn_ballot_w64(mx > m)) {
            const float corr = m == -INFINITY ? 0.f : paged_exp2(m - mx);
            l *= corr;
#pragma unroll
            for (int i = 0; i < EV; ++i) oacc[i] *= corr;
            m = mx;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float e[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = paged_exp2(s[0][r] - base), e[4 + r] = paged_exp2(s[1][r] - base);
        l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        if (EIGHT)
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] *= vsc[j];
        bf16x8 pf[PP];
        p_planes<PP>(e, pf);
#pragma unroll
        for (int i = 0; i < EV; ++i) {
            u32x4 pl[NK];
            v_planes<CK>(vr, i, pl);
            bf16x8 vf[NK];
#pragma unroll
            for (int k = 0; k < NK; ++k) vf[k] = as_bf16x8(pl[k]);
            oacc[i] = mfma_planes(vf, pf, oacc[i]);
        }
        vload();
    }
    // join the waves: means, so that sums near the end of fp32 stay in it
    l = paged_sum_rows(l);
    if (g == 0) s_m[w][r16] = m, s_l[w][r16] = l;
    __syncthreads();
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) mm = fmaxf(mm, s_m[k][r16]);
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int k = 0; k < 4; ++k) ll += s_l[k][r16] * paged_exp2(s_m[k][r16] - base);
    const float f = (ll != 0.f ? paged_exp2(m - base) / ll : 0.f) * (NK == 3 || EIGHT ? SPLIT_UNSCALE : 1.f);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < EV; ++i) s_o[w][r16][(4 * g + r) * EV + i] = oacc[i][r] * f;
    __syncthreads();
    float v[M * D / 256];
#pragma unroll
    for (int k = 0; k < M * D / 256; ++k) {
        const int r = (threadIdx.x + 256 * k) / D, d = threadIdx.x % D;
        v[k] = (s_o[0][r][d] + s_o[1][r][d]) + (s_o[2][r][d] + s_o[3][r][d]);
        if (r < rows && !(fabsf(v[k]) <= FLT_MAX)) atomicOr(&s_bad[0], 1u << r);
    }
    __syncthreads();
    const unsigned bad = s_bad[0];
#pragma unroll
    for (int k = 0; k < M * D / 256; ++k) {
        const int r = (threadIdx.x + 256 * k) / D, d = threadIdx.x % D;
        if (r >= rows || (bad >> r & 1)) continue;
        if (part) part[(long)r * LD + d] = v[k];
        else {
            const PagedRow o = paged_row_of(p, sq, hk, r0 + r);
            paged_put((T *)p.o + o.tok * p.o_st + o.h * p.o_sh + d, v[k]);
        }
    }
    if (part && w == 0 && g == 0 && r16 < rows && !(bad >> r16 & 1)) part[(long)r16 * LD + D] = mm, part[(long)r16 * LD + D + 1] = ll;
    if (bad) paged_again<D, CK, T>(p, b, hk, sq, r0, rows, s_bad, k_lo, k_hi, part);
}

// ---------------------------------------------------------------- many rows: chunks
// One workgroup: a tile of 64 NQ rows, 16 NQ a wave, and one split of its keys.  Tiles of BK keys go
// through LDS in operand order (one ds_read_b128 a fragment, no bank conflict on either side): read
// from their pages a tile ahead, widened or split once, V transposed by the lanes that stage it.
// Where operands are single bf16 planes two buffers of LDS need one barrier a tile; three planes
// take one buffer and two barriers.
// 32 rows a wave read a fragment from LDS for twice the products that 16 do.  With 16 and eight waves, which
// share out the staging, 4 chunks of up to 512 over up to 4096 keys take 181 us over int8 and 132 over bf16,
// with 32 and four 171 and 126; with 32 and eight, tiles of 256 rows are too few to even out: 260.  Scales of
// values are read from LDS where they are used: held in registers (two fragments in flight): 258.
// Those chunks over bf16 are 73.6 GFLOP in 121 us, alone and back to back: 609 TFLOP/s, where a large bf16
// product of a library reaches 1208; over int8 168, e4m3 161.  A unit is held for 0.77 of the kernel (two
// tiles of unequal length each); of that time the matrix cores are busy 0.32 and the vector ALU (softmax,
// staging) 0.36.  Neither is full: a wave's products and its softmax take turns, and the one other
// wave of its SIMD does not fill the gaps (0.29 of a wave's cycles wait for memory, LDS or the barrier, 0.32 to
// issue).  Two groups of waves that share a tile's keys (142 us), keys split so that tiles are equal (158), two sets of
// registers for the staged rows (no change) and longer rings (they spill: 151) were slower.
template <int D, int CK, typename T, int NQ>
__global__ void __launch_bounds__(256, 2) paged_tile_kernel(const PagedAttnArgs p)
{
    constexpr int NP = sizeof(T) == 4 ? 3 : 1, NK = CK == CK_F32 ? 3 : 1, NB = NK == 3 ? 1 : 2;
    constexpr int BK = NK == 3 && D == 128 ? 32 : 64, NW = 4, M = 16 * NQ * NW;
    constexpr int CD = D / 32, NC = D / 16, NJ = BK / 16, NM = BK / 32;
    constexpr int EV = D == 128 ? 4 : 2, NH = D / (16 * EV), NU = NM * NH;  // V: units of 32 keys x 16 EV d
    constexpr int KC = CD * NJ / NW;  // K: a wave stages KC steps of 16 keys
    using KO = KOperand<D, CK>;
    using VO = VOperand<CK, EV>;
    constexpr int ES = cache_bytes<CK>, LD = D + 4, RING = NK == 3 ? 2 : 4;  // (as many as registers leave room for)
    constexpr bool EIGHT = CK >= CK_I8, ONES = NP == 1 && !EIGHT;  // row sums as P^T times ones
    constexpr int PP = NP == 3 ? 3 : EIGHT ? 2 : 1;                // planes of P
    static_assert(NW % NJ == 0 && KC > 0, "a block of 16 keys is staged by NW / NJ waves");
    __shared__ u32x4 Ks[NB][NK][NJ * CD * 64];
    __shared__ u32x4 Vs[NB][NK][NC * NM * 64];
    __shared__ long s_off[2][64];
    __shared__ unsigned long long s_valid[2];
    __shared__ float s_sc[2][2][64];
    __shared__ unsigned s_bad[4];
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int hk, x, split;
    paged_block(p, hk, x, split);
    int b;
    PagedSeq sq;
    const int tile = p.sorted ? paged_tile_sorted<M>(p, x, b, sq) : paged_tile<M>(p, x, b, sq);
    const int r0 = tile * M, rows = min(M, sq.rows * p.G - r0);
    if (tile < 0 || rows <= 0) return;
    const int kend = paged_row_of(p, sq, hk, r0 + rows - 1).end;  // (the last row of a tile sees most)
    int k_lo, k_hi;
    paged_split(p, kend, split, k_lo, k_hi);
    float *part = p.nsplit > 1 ? p.part + (((long)x * p.kv.n_kv + hk) * p.nsplit + split) * M * LD : nullptr;
    if (part && k_lo >= k_hi) {  // a split that this sequence does not need
        if (tid < rows) part[(long)tid * LD + D] = -INFINITY, part[(long)tid * LD + D + 1] = 0.f;
        return;
    }
    if (tid < 4) s_bad[tid] = 0;

    // this wave's rows: 16 a block, and what its first and last see
    const int wr = w * 16 * NQ;
    const int wave_end = wr < rows ? min(k_hi, paged_row_of(p, sq, hk, r0 + min(wr + 16 * NQ, rows) - 1).end) : 0;
    bf16x8 qf[NQ][CD][NP];
    int end[NQ], first_end[NQ];
#pragma unroll
    for (int a = 0; a < NQ; ++a) {
        const int r = wr + 16 * a + r16;
        const PagedRow row = paged_row_of(p, sq, hk, r0 + min(r, rows - 1));
        end[a] = row.end;
        first_end[a] = paged_row_of(p, sq, hk, r0 + min(wr + 16 * a, rows - 1)).end;
        q_planes<D, CK, T, NP>((const T *)p.q + row.tok * p.q_st + row.h * p.q_sh, r < rows, g, p.q_vec, qf[a]);
    }

    const char *kpool = (const char *)p.kv.k + hk * p.kv.head_stride * ES;
    const char *vpool = (const char *)p.kv.v + hk * p.kv.head_stride * ES + r16 * EV * ES;
    const int kj = w % NJ, kc = w / NJ * KC;  // this wave's block of keys, and its first step
    // the tile two ahead: its entries of the table (wave 0, one key a lane); one ahead: its places
    int page = 0, slot = 0;
    bool in = false;
    float ks = 0.f, vs = 0.f;
    auto entry = [&](int t0) {
        if (w == 0) {  // (past the end: the last key's, unused)
            in = lane < BK && t0 + lane < k_hi;
            page = paged_entry(p, b, max(0, min(t0 + lane, k_hi - 1)), slot);
        }
    };
    auto place = [&](int at) {
        if (w == 0) {
            in = in & (page >= 0) & (page < p.kv.n_pages);
            const unsigned long long valid = __builtin_amdgcn_ballot_w64(in);
            const long pg = in ? page : 0, sl = in ? slot : 0;
            s_off[at][lane] = (pg * p.kv.page_stride + sl * p.kv.tok_stride) * ES;
            if (lane == 0) s_valid[at] = valid;
            if (EIGHT) {
                const long sc = (pg * p.kv.n_kv + hk) * p.kv.page_size + sl;
                ks = p.kv.ks[sc], vs = p.kv.vs[sc];
            }
        }
    };
    uint32_t kr[KC][KO::RW], vr[(NU + NW - 1) / NW][8][VO::RW];
    auto gload = [&](int at) {
        KO::template load<KC>(kpool + s_off[at][16 * kj + r16], g, kc, kr);
#pragma unroll
        for (int q = 0; q < (NU + NW - 1) / NW; ++q) {
            const int u = w + NW * q;
            if (NU % NW != 0 && u >= NU) continue;
            const int mm = u / NH, h = u % NH;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                VO::load(vpool + h * 16 * EV * ES + s_off[at][32 * mm + 4 * g + j + (j < 4 ? 0 : 12)], vr[q][j]);
        }
    };
    auto lstore = [&](int buf, int at, unsigned long long valid) {
        if (EIGHT && w == 0) s_sc[at][0][lane] = ks, s_sc[at][1][lane] = (valid >> lane & 1) ? vs * SPLIT_SCALE : 0.f;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            u32x4 pl[NK];
            k_planes<CK>(kr[c], pl);
            const int u = kj * CD + kc + c;
#pragma unroll
            for (int k = 0; k < NK; ++k) Ks[buf][k][u * 64 + lane] = pl[k];
        }
#pragma unroll
        for (int q = 0; q < (NU + NW - 1) / NW; ++q) {
            const int u = w + NW * q;
            if (NU % NW != 0 && u >= NU) continue;
            const int mm = u / NH, h = u % NH;
            if (valid != (BK == 64 ? ~0ull : 0xffffffffull)) {  // values of keys without a page, or past the end, are none
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool in = valid >> (32 * mm + 4 * g + j + (j < 4 ? 0 : 12)) & 1;
#pragma unroll
                    for (int e = 0; e < VO::RW; ++e) vr[q][j][e] = in ? vr[q][j][e] : 0u;
                }
            }
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                u32x4 pl[NK];
                v_planes<CK>(vr[q], i, pl);
#pragma unroll
                for (int k = 0; k < NK; ++k) Vs[buf][k][((h * EV + i) * NM + mm) * 64 + lane] = pl[k];
            }
        }
    };

    floatx4 oacc[NC][NQ], lacc[NQ];
    float l[NQ], mb[NQ], m_lane[NQ];  // row sums, exponent base, this lane's running maximum relative to it
#pragma unroll
    for (int a = 0; a < NQ; ++a) {
        l[a] = 0.f, mb[a] = 0.f, m_lane[a] = -INFINITY, lacc[a] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) oacc[c][a] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    // Scores are masked before they are scaled (after it, the same work took 44.4 us for 38.3 of attn_chunk_f32), so
    // a masked score is what the scale makes -inf: of the other sign under a negative one, and 2^-126 stands
    // for 0, which leaves scores of up to 2^60 their weight of 1.
    const float scaled = p.scale_log2 * (NP == 3 ? SPLIT_UNSCALE : 1.f) * (NK == 3 ? SPLIT_UNSCALE : 1.f);
    const float sl2 = scaled == 0.f ? 0x1p-126f : scaled, none = sl2 < 0.f ? INFINITY : -INFINITY;
    const bf16x8 ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};

    if (k_lo < k_hi) {
        entry(k_lo);
        place(0);
        __syncthreads();
        gload(0);
        entry(k_lo + BK);
    }
    for (int kv0 = k_lo, it = 0; kv0 < k_hi; kv0 += BK, ++it) {
        const int at = it & 1, buf = NB == 2 ? at : 0;
        if (NB == 1) __syncthreads();  // every wave is done with the previous tile
        const unsigned long long valid = s_valid[at];
        lstore(buf, at, valid);
        place(at ^ 1);  // (past the last tile: no key has a page, and page 0 is read)
        entry(kv0 + 2 * BK);
        __syncthreads();
        gload(at ^ 1);
        if (kv0 >= wave_end) continue;  // nothing that a row of this wave sees
        // Fragments of K, then of V, pass through a ring of registers, RING - 1 of them in flight: a
        // read takes about 200 cycles with four waves at it, the products of one fragment 16 to
        // 96.  (The fences keep the compiler from moving a read down to its use.)
        bf16x8 ring[RING][NK];
        auto fetch_k = [&](int f) {  // step f: 32 d, 16 keys
#pragma unroll
            for (int k = 0; k < NK; ++k) ring[f % RING][k] = as_bf16x8(Ks[buf][k][(f % NJ * CD + f / NJ) * 64 + lane]);
        };
        auto fetch_v = [&](int f) {  // step f: 32 keys, 16 d
#pragma unroll
            for (int k = 0; k < NK; ++k) ring[f % RING][k] = as_bf16x8(Vs[buf][k][(f % NC * NM + f / NC) * 64 + lane]);
        };
        floatx4 s[NJ][NQ];
#pragma unroll
        for (int f = 0; f < RING - 1; ++f) fetch_k(f);
#pragma unroll
        for (int f = 0; f < NJ * CD; ++f) {
            if (f + RING - 1 < NJ * CD) fetch_k(f + RING - 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int a = 0; a < NQ; ++a)
                s[f % NJ][a] = mfma_planes(ring[f % RING], qf[a][f / NJ], f < NJ ? floatx4{0.f, 0.f, 0.f, 0.f} : s[f % NJ][a]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int f = 0; f < RING - 1; ++f) fetch_v(f);
        if (EIGHT) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const floatx4 f = *(const floatx4 *)&s_sc[at][0][16 * j + 4 * g];
#pragma unroll
                for (int a = 0; a < NQ; ++a) s[j][a] *= f;
            }
        }
        bf16x8 pf[NM][NQ][PP];
#pragma unroll
        for (int a = 0; a < NQ; ++a) {
            if (valid != (BK == 64 ? ~0ull : 0xffffffffull) || kv0 + BK > first_end[a]) {
                const unsigned long long see = valid >> (4 * g);
                const int lim = end[a] - kv0 - 4 * g;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[j][a][r] = (see >> (16 * j + r) & 1) && 16 * j + r < lim ? s[j][a][r] : none;
            }
            // exponent units relative to the base: p = 2^s below
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[j][a][r] = __builtin_fmaf(s[j][a][r], sl2, -mb[a]);
            // The base is the row's maximum over the first tile in which it sees a key, and moves only when its
            // running maximum passes mb + 8: p stays below 2^8 and the largest at or above 1, numerator and
            // sum share the base, and the result is unchanged.  Each lane tests its own maximum; the row's is
            // formed only when one trips.
            const float m_prev = m_lane[a];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                m_lane[a] = fmaxf(fmaxf(m_lane[a], fmaxf(s[j][a][0], s[j][a][1])), fmaxf(s[j][a][2], s[j][a][3]));
            if (__builtin_amdgcn_ballot_w64(m_lane[a] > 8.f || (m_prev == -INFINITY && m_lane[a] != -INFINITY))) {
                const float row_prev = paged_max_rows(m_prev), row = paged_max_rows(m_lane[a]);
                if (row > 8.f || (row_prev == -INFINITY && row != -INFINITY)) {
                    // nothing accumulated yet (row_prev = -inf): factor 0, not a 2^-row that overflows
                    const float corr = row_prev == -INFINITY ? 0.f : paged_exp2(-row);
                    mb[a] += row;
                    m_lane[a] -= row;
                    l[a] *= corr, lacc[a] *= corr;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) s[j][a] -= row;
#pragma unroll
                    for (int c = 0; c < NC; ++c) oacc[c][a] *= corr;
                }
            }
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                float e[8];
#pragma unroll
                for (int r = 0; r < 4; ++r) e[r] = paged_exp2(s[2 * m][a][r]), e[4 + r] = paged_exp2(s[2 * m + 1][a][r]);
                if (!ONES) l[a] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
                if (EIGHT) {
                    const floatx4 v0 = *(const floatx4 *)&s_sc[at][1][32 * m + 4 * g], v1 = *(const floatx4 *)&s_sc[at][1][32 * m + 16 + 4 * g];
#pragma unroll
                    for (int r = 0; r < 4; ++r) e[r] *= v0[r], e[4 + r] *= v1[r];
                }
                p_planes<PP>(e, pf[m][a]);
                if (ONES) lacc[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[m][a][0], lacc[a], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < NC * NM; ++f) {
            if (f + RING - 1 < NC * NM) fetch_v(f + RING - 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int a = 0; a < NQ; ++a) oacc[f % NC][a] = mfma_planes(ring[f % RING], pf[f / NC][a], oacc[f % NC][a]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

#pragma unroll
    for (int a = 0; a < NQ; ++a) {
        const int r = wr + 16 * a + r16;
        const float ll = ONES ? lacc[a][0] : paged_sum_rows(l[a]);
        const float inv = (ll != 0.f ? 1.0f / ll : 0.f) * (NK == 3 || EIGHT ? SPLIT_UNSCALE : 1.f);
        bool bad = !(ll <= FLT_MAX);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            oacc[c][a] *= inv;
#pragma unroll
            for (int k = 0; k < 4; ++k) bad |= !(fabsf(oacc[c][a][k]) <= FLT_MAX);
        }
        const unsigned long long any = __builtin_amdgcn_ballot_w64(bad);
        const unsigned bits = (unsigned)((any | any >> 16 | any >> 32 | any >> 48) & 0xffff);  // one a row
        if (lane == 0 && bits) atomicOr(&s_bad[(wr + 16 * a) / 32], bits << ((wr + 16 * a) % 32));
        if (r >= rows || (bits >> r16 & 1)) continue;
        const PagedRow row = paged_row_of(p, sq, hk, r0 + r);
        T *o = (T *)p.o + row.tok * p.o_st + row.h * p.o_sh;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = h * 16 * EV + (4 * g + k) * EV;  // EV neighbours
                float v[EV];
#pragma unroll
                for (int i = 0; i < EV; ++i) v[i] = oacc[h * EV + i][a][k];
                if (part) {
#pragma unroll
                    for (int i = 0; i < EV; ++i) part[(long)r * LD + d + i] = v[i];
                } else if (p.o_vec) {
                    if constexpr (sizeof(T) == 4) {
                        if constexpr (EV == 4) *(floatx4 *)(o + d) = floatx4{v[0], v[1], v[2], v[3]};
                        else *(u32x2 *)(o + d) = u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])};
                    } else {
                        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
                        const uint32_t t = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[0], (__bf16)v[1]});
                        if constexpr (EV == 4) *(u32x2 *)(o + d) = u32x2{t, __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2], (__bf16)v[3]})};
                        else *(uint32_t *)(o + d) = t;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < EV; ++i) paged_put(o + d + i, v[i]);
                }
            }
        if (part && g == 0) part[(long)r * LD + D] = ll != 0.f ? mb[a] : -INFINITY, part[(long)r * LD + D + 1] = ll;
    }
    __syncthreads();
    if (s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3]) paged_again<D, CK, T>(p, b, hk, sq, r0, rows, s_bad, k_lo, k_hi, part);
}

// Joins the splits of a tile's rows, one wave a row: lane i weighs split i (nsplit <= 64), then the
// wave adds the means of the splits that saw a key, sixteen in flight (one of no weight too: 0 times NaN).  (6 us of the 71.5 above; 9 of
// int8's 73, whose rows have 63 splits.)
template <int D, typename T>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnArgs p, int M)
{
    constexpr int LD = D + 4, E = (D + 63) / 64;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = blockIdx.x % (M / 4), rest = blockIdx.x / (M / 4), hk = rest % p.kv.n_kv, x = rest / p.kv.n_kv;
    int b;
    PagedSeq sq;
    const int tile = M == 16 ? paged_tile<16>(p, x, b, sq) : M == 64 ? paged_tile<64>(p, x, b, sq) : paged_tile<128>(p, x, b, sq);
    const int r = quarter * 4 + w;
    if (tile < 0 || r >= sq.rows * p.G - tile * M) return;
    const float *part = p.part + (((long)x * p.kv.n_kv + hk) * p.nsplit * M + r) * LD;
    const long step = (long)M * LD;  // from a split to the next
    const bool in = lane < p.nsplit;
    const float m = in ? part[lane * step + D] : -INFINITY, l = in ? part[lane * step + D + 1] : 0.f;
    const float mm = wave_max(m), base = mm == -INFINITY ? 0.f : mm;
    float wt = l != 0.f ? paged_exp2(m - base) * l : 0.f;
    const float ll = wave_sum(wt);
    wt *= ll != 0.f ? 1.0f / ll : 0.f;
    unsigned long long left = __builtin_amdgcn_ballot_w64(l != 0.f);  // (a NaN sum too)
    const int d = lane * E;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    while (left) {
        float f[16], q[16][E];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int s = left ? __builtin_ctzll(left) : 0;
            f[k] = left ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wt), s)) : 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) q[k][e] = left && d < D ? part[s * step + d + e] : 0.f;
            left &= left - 1;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = __builtin_fmaf(f[k], q[k][e], v[e]);
    }
    if (d >= D) return;
    const PagedRow o = paged_row_of(p, sq, hk, tile * M + r);
#pragma unroll
    for (int e = 0; e < E; ++e) paged_put((T *)p.o + o.tok * p.o_st + o.h * p.o_sh + d + e, v[e]);
}

template <int D, int CK, typename T>
void paged_launch_as(const PagedAttnArgs &p, int rows, hipStream_t s)
{
    const dim3 grid((unsigned)p.tiles * p.nsplit * p.kv.n_kv), block(256);
    if (rows == 16) hipLaunchKernelGGL((paged_stream_kernel<D, CK, T>), grid, block, 0, s, p);
    else if (rows == 64) hipLaunchKernelGGL((paged_tile_kernel<D, CK, T, 1>), grid, block, 0, s, p);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((paged_tile_kernel<D, CK, T, 2>), grid, block, 0, s, p);
    if (p.nsplit > 1) hipLaunchKernelGGL((paged_merge_kernel<D, T>), dim3((unsigned)p.tiles * p.kv.n_kv * (rows / 4)), block, 0, s, p, rows);
}

template <int D>
void paged_launch(const PagedAttnArgs &p, int rows, int cache, int dtype, hipStream_t s)
{
    if (dtype == JAS_F32) {
        if (cache == JAS_F32) paged_launch_as<D, CK_F32, float>(p, rows, s);
        else if (cache == JAS_BF16) paged_launch_as<D, CK_BF16, float>(p, rows, s);
        else if (cache == JAS_I8) paged_launch_as<D, CK_I8, float>(p, rows, s);
        else paged_launch_as<D, CK_F8, float>(p, rows, s);
    } else {
        if (cache == JAS_BF16) paged_launch_as<D, CK_BF16, uint16_t>(p, rows, s);
        else if (cache == JAS_I8) paged_launch_as<D, CK_I8, uint16_t>(p, rows, s);
        else paged_launch_as<D, CK_F8, uint16_t>(p, rows, s);
    }
}

} // namespace jas
