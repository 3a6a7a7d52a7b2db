// Attention over the paged MXFP4 cache.
#include "qw_kv.h"
#include <algorithm>

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

struct qw_attn_args {
    const uint8_t* pages;
    const int32_t* row_start;
    const int32_t* lengths;
    const int32_t* table;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    float* part;           // [parts][rows][q_heads][D] sums, then [parts][rows][q_heads][2] what the weights' exponents are less (`top`) and the sum of weights
    qw_kv_geometry geo;
    uint32_t page_count, kv_heads, ld_table, max_rows, max_length, rows, q_heads, shared, ld_q, ld_out, window, parts, tiles;
    float scale2, digit, digit_rest;   // scale * log2(e) as fp32 rounds it; what a digit of a score is then, scale / scale2, in two parts
};

// A sequence's rows and tokens, cut to what the host allows; the position of its first row.
struct qw_attn_seq {
    uint32_t row0, n, length;
    int32_t pos0;
};
__device__ __forceinline__ qw_attn_seq qw_attn_sequence(const qw_attn_args& a, uint32_t seq) {
    qw_attn_seq s;
    const int32_t from = a.row_start ? a.row_start[seq] : (int32_t)seq, to = a.row_start ? a.row_start[seq + 1u] : (int32_t)seq + 1;
    s.row0 = (uint32_t)max(0, min(from, (int32_t)a.rows));
    const int32_t n = max(0, min(to, (int32_t)a.rows) - (int32_t)s.row0);
    s.n = min((uint32_t)n, a.max_rows);
    s.length = (uint32_t)max(0, min(a.lengths[seq], (int32_t)a.max_length));
    s.pos0 = (int32_t)s.length - n;
    return s;
}

// The tokens that the columns c0 .. c1 of a sequence see together, from a step's border on, and this part's share of the steps.
struct qw_attn_range {
    int32_t pos_a, pos_b;        // positions of the first and the last column's rows; negative: sees nothing
    uint32_t low_a, low_b;       // the first tokens that these see
    uint32_t first, from, to;    // first token of the steps, this part's steps
};
__device__ __forceinline__ uint32_t qw_attn_low(const qw_attn_args& a, int32_t pos) {
    return a.window && pos + 1 > (int32_t)a.window ? (uint32_t)(pos + 1 - (int32_t)a.window) : 0u;
}
template <uint32_t T>
__device__ __forceinline__ qw_attn_range qw_attn_tokens(const qw_attn_args& a, const qw_attn_seq& s, uint32_t c0, uint32_t c1, uint32_t part) {
    qw_attn_range r;
    r.pos_a = s.pos0 + (int32_t)(c0 / a.shared), r.pos_b = s.pos0 + (int32_t)(c1 / a.shared);
    r.low_a = qw_attn_low(a, r.pos_a), r.low_b = qw_attn_low(a, r.pos_b);
    r.first = r.low_a & ~(T - 1u);
    const uint32_t end = r.pos_b < 0 ? r.first : (uint32_t)r.pos_b + 1u;   // pos_b < 0: low_a is 0
    const uint32_t steps = (end - r.first + T - 1u) / T, each = (steps + a.parts - 1u) / a.parts;
    r.from = min(part * each, steps), r.to = min(r.from + each, steps);
    return r;
}
// Steps begin and end on borders of their own: the tokens of a step that the columns do not see, in front of their window or behind the last, get a harmless scale, so that what
// is in their places decides nothing, the form neither.  One byte of each of the four tokens from `t` on, set where it is among low .. stop - 1.
__device__ __forceinline__ uint32_t qw_attn_there(uint32_t t, uint32_t low, uint32_t stop) {
    const uint32_t behind = t + 4u <= stop ? ~0u : t >= stop ? 0u : (1u << (8u * (stop - t))) - 1u;
    return behind & (t >= low ? ~0u : t + 4u <= low ? 0u : ~0u << (8u * (low - t)));
}
__device__ __forceinline__ uint32_t qw_attn_seen(uint32_t scales, uint32_t there) { return (scales & there) | (0x7F7F7F7Fu & ~there); }

// What a lane carries of a step of 32 tokens, 16 h .. 16 h + 15 in half h.  Keys: rows of an operand of each half, lane (i, g) has elements of its token i; values:
// lane (i, g) has eight elements of the tokens 4 g .. 4 g + 3 of both halves.  A score of half h, accumulator row 4 g + r, is then token 16 h + 4 g + r: the weights
// are in place as an operand against the values, and every load takes whole lines.
template <int D>
struct qw_attn_step {
    static constexpr uint32_t SETS = D == 256 ? 2 : 1, WORDS = D == 64 ? 2 : 4;
    uint32_t k[2][SETS][WORDS];
    uint32_t k_scale[2][SETS];
    u4_t v[SETS][2];
    uint32_t v_scale[SETS][2];
};
// Where a lane's pieces are in a page, from a half's first token on.
template <int D>
struct qw_attn_place {
    uint32_t k, k_scale, v, v_scale;
    __device__ __forceinline__ void set(const qw_attn_args& a, uint32_t i, uint32_t g) {
        const uint32_t word = D == 64 ? i & 7u : i;
        k = i * (D / 2u) + g * (4u * qw_attn_step<D>::WORDS);
        k_scale = a.geo.k_scales + i * (D / 32u) + (D == 64 ? g >> 1 : g);
        v = a.geo.v_codes + ((g >> 1) * (D / 8u) + word) * 32u + (g & 1u) * 16u;
        v_scale = a.geo.v_scales + ((g >> 1) * (D / 32u) + (word >> 2)) * 8u + (g & 1u) * 4u;
    }
};
template <bool ONCE, typename T>
__device__ __forceinline__ T qw_attn_codes(const T* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
}
// The 32 tokens from t0 on, of one page or (SMALL: pages of 16) two, of which low .. stop - 1 are seen: a half without one of them is read from the page of the nearest, and
// masked, so that the table's entries around them are not looked at.  The pages are the same for all lanes: scalar loads and addresses.  ONCE: of a sequence one
// workgroup reads these codes, they are marked as read once (64 tokens behind 8192 each 99 us, 105 unmarked; sequences that share pages lose nothing by it: all 8192
// tokens shared 68 us either way).
template <int D, bool SMALL, bool ONCE>
__device__ __forceinline__ void qw_attn_load(const qw_attn_args& a, const uint8_t* head, uint32_t stride, const int32_t* table, uint32_t t0, uint32_t low, uint32_t stop,
                                             const qw_attn_place<D>& at, qw_attn_step<D>& s) {
    constexpr uint32_t SETS = qw_attn_step<D>::SETS, WORDS = qw_attn_step<D>::WORDS;
    const uint32_t page0 = (uint32_t)table[(SMALL ? max(t0, low) : t0) >> a.geo.page_log2];
    const uint8_t* piece[2];
    uint32_t in[2] = {t0 & ((1u << a.geo.page_log2) - 1u), 0u};
    piece[0] = head + (uint64_t)(page0 < a.page_count ? page0 : 0u) * stride;
    if constexpr (SMALL) {
        const uint32_t page1 = (uint32_t)table[min(t0 + 16u, stop - 1u) >> 4];
        piece[1] = head + (uint64_t)(page1 < a.page_count ? page1 : 0u) * stride;
    } else {
        piece[1] = piece[0];
        in[1] = in[0] + 16u;
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint8_t* const codes = piece[h] + in[h] * (D / 2u);
        const uint8_t* const scales = piece[h] + in[h] * (D / 32u);
#pragma unroll
        for (uint32_t c = 0; c < SETS; ++c) {
            typedef uint32_t words_t __attribute__((ext_vector_type(WORDS)));
            const words_t k = qw_attn_codes<ONCE>((const words_t*)(codes + at.k + c * 64u));
            __builtin_memcpy(s.k[h][c], &k, 4 * WORDS);
            s.k_scale[h][c] = qw_attn_codes<ONCE>(scales + at.k_scale + 4u * c);
            s.v[c][h] = qw_attn_codes<ONCE>((const u4_t*)(codes + at.v + c * 512u));
            s.v_scale[c][h] = qw_attn_codes<ONCE>((const uint32_t*)(scales + at.v_scale + c * 32u));
        }
    }
}
template <int D>
__device__ __forceinline__ void qw_attn_cut(uint32_t t0, uint32_t low, uint32_t stop, uint32_t i, uint32_t g, qw_attn_step<D>& s) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t key = t0 + 16u * h + i, there = qw_attn_there(t0 + 16u * h + 4u * g, low, stop);
#pragma unroll
        for (uint32_t c = 0; c < qw_attn_step<D>::SETS; ++c) {
            if (key < low || key >= stop) s.k_scale[h][c] = 127u;
            s.v_scale[c][h] = qw_attn_seen(s.v_scale[c][h], there);
        }
    }
}

// Eight codes of a word as f16 or bf16 operands under the power of two `scale`.
template <int DT>
__device__ __forceinline__ u4_t qw_attn_operand(uint32_t w, float scale) {
    u4_t o;
    if constexpr (DT == QWHIP_F16) {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
    } else {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    }
    return o;
}
template <int DT, int J>   // elements 2 J and 2 J + 1
__device__ __forceinline__ uint32_t qw_attn_pair(uint32_t w, float scale) {
    if constexpr (DT == QWHIP_F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, J));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, J));
}
template <int N, typename F>   // f of 0 .. N - 1 as constants
__device__ __forceinline__ void qw_attn_pairs(F f) {
    if constexpr (N > 0) {
        qw_attn_pairs<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
template <int DT>
__device__ __forceinline__ f4_t qw_attn_mfma(u4_t a, u4_t b, f4_t c) {
    if constexpr (DT == QWHIP_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
// Two floats as bf16, the first in the low half.
__device__ __forceinline__ uint32_t qw_attn_bf16x2(float a, float b) { return (uint32_t)qw_f32_to_bf16(a) | ((uint32_t)qw_f32_to_bf16(b) << 16); }

// Eight f16 numbers as two bf16 numbers each, whose sum they are: eight bits and the last three (an infinity's or a NaN's rest is zero).
__device__ __forceinline__ void qw_attn_split(u4_t q, u4_t& hi, u4_t& lo) {
    const h8_t x = __builtin_bit_cast(h8_t, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x0 = (float)x[2 * e], x1 = (float)x[2 * e + 1];
        const uint32_t h0 = __float_as_uint(x0) & 0xFFFF0000u, h1 = __float_as_uint(x1) & 0xFFFF0000u;
        const float l0 = (h0 & 0x7F800000u) == 0x7F800000u ? 0.0f : x0 - __uint_as_float(h0), l1 = (h1 & 0x7F800000u) == 0x7F800000u ? 0.0f : x1 - __uint_as_float(h1);
        hi[e] = (h0 >> 16) | h1;
        lo[e] = (__float_as_uint(l0) >> 16) | (__float_as_uint(l1) & 0xFFFF0000u);
    }
}
// Floats of an output row: 1, 2, 4 or 8.
template <int DT, uint32_t E>
__device__ __forceinline__ void qw_attn_store(uint16_t* y, const float* o) {
    typedef uint16_t v_t __attribute__((ext_vector_type(E)));
    v_t v;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) v[e] = DT == QWHIP_F16 ? __builtin_bit_cast(uint16_t, (h1_t)o[e]) : qw_f32_to_bf16(o[e]);
    *(v_t*)y = v;
}
// f16 holds the elements under a scale byte as normal numbers, exactly, from 2^-13 to 2^13 (and the zeros of a block of zeros: byte 0, whose other elements are
// under 2^-124 and count as zero); bf16 up to 2^125.
constexpr uint32_t QW_ATTN_F16_LEAST = 114, QW_ATTN_F16_MOST = 140, QW_ATTN_BF16_MOST = 252;
template <int DT>
__device__ __forceinline__ uint32_t qw_attn_far(uint32_t byte) {   // 1 or 0: added up without branches
    if constexpr (DT == QWHIP_F16) return (uint32_t)(byte - QW_ATTN_F16_LEAST > QW_ATTN_F16_MOST - QW_ATTN_F16_LEAST) & (uint32_t)(byte != 0u);
    else return (uint32_t)(byte > QW_ATTN_BF16_MOST);
}
// The same for eight bytes, four at a time: not zero for one that is over 140, or 1 .. 113.
__device__ __forceinline__ uint32_t qw_attn_far8(u2_t scales) {
    uint32_t bad = 0;
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e) {
        const uint32_t b = scales[e], low = b & 0x7F7F7F7Fu;
        const uint32_t over = b & (low + 0x73737373u);                                          // top bits: 128 + at least 13
        const uint32_t under = ~b & ~(low + 0x0E0E0E0Eu) & (low + 0x7F7F7F7Fu);                  // no top bit, under 114, not zero
        bad |= (over | under) & 0x80808080u;
    }
    return bad;
}
// Byte e of eight as the scale of a conversion, which reads the exponent field alone.
__device__ __forceinline__ float qw_attn_unit(u2_t scales, uint32_t e) {
    const uint32_t w = scales[e >> 2];
    return __uint_as_float((e & 3u) == 3u ? w >> 1 : w << (23u - 8u * (e & 3u)));
}

// A weight is 2 to the power of its scaled score (in binary digits) less `top`: the column's maximum less QW_ATTN_UNDER when it was last taken.  A maximum that grows is taken
// again only where a weight would pass 2^QW_ATTN_ROOM, so that sums and accumulators are hardly ever scaled.  f16 holds up to 2^15.999, 11 bits from 2^-14 on and steps
// of 2^-24 below: weights from 2^-26 of the largest on have all their bits, n smaller ones are off by n 2^-37 of it.  (Weights of at most one would be lost to the values
// from 2^-25 on, and stay in the sum.)  Room for a growth of 3.9 digits costs 0 .. 1.5 % over room for 8, 3 digits 2 .. 3 % (a prompt of 4096 rows 195.6, 194.4,
// 199.3 us).  The wide form's bf16 numbers have fp32's range, and its values may be near
// the end of it: its weights are at most one, so that no sum leaves the range sooner than in the softmax as it is written.
constexpr float QW_ATTN_UNDER = 12.0f, QW_ATTN_ROOM = 15.9f, QW_ATTN_ROOM_WIDE = 0.0f;

// A weight's exponent is one multiply-add of the product q.k, which is not rounded in between, but `top` comes from a rounded score: all weights of a column are off by the
// power of that rounding.  It cancels, but from 2^23 binary digits on it takes weights out of any range.  A range with such a column, from 2^17 on (under it
// the rounding is within the tenth of a digit that the room leaves), is done in the wide form, which rounds a score before it takes `top` off: the largest weight is one
// whatever the score.  (Both ways in a step cost every call one percent.)
constexpr float QW_ATTN_FAR_SCORE = 0x1p17f;
__device__ __forceinline__ uint32_t qw_attn_far_score(float top) { return fabsf(top) >= QW_ATTN_FAR_SCORE && top != -__builtin_inff() ? 1u : 0u; }

// What a row's sums are multiplied by, and the logarithm of its sum.  Maxima are of scaled scores: one under fp32's range is -inf and none at all, and a row
// without a score over -inf has neither; one over the range is an infinity under which nothing has a finite weight: NaN.  The sum's exponent goes to the maximum
// first, so that the logarithm of what is left has all of its bits, and the digits become a logarithm by what the scale's own rounding made of them: one rounding of fp32
// in all, and 2^-20 for the weights' exponents.
__device__ __forceinline__ float qw_attn_inverse(float best, float total) { return best == -__builtin_inff() && total == 0.0f ? 0.0f : 1.0f / total; }
__device__ __forceinline__ float qw_attn_log(const qw_attn_args& a, float best, float total) {
    if (best == -__builtin_inff() && total == 0.0f) return -__builtin_inff();
    const float exponent = (float)__builtin_amdgcn_frexp_expf(total), s = best + exponent, b = s - best, rest = (best - (s - b)) + (exponent - b);   // s + rest: the sum
    const float less = (rest + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(total))) * a.digit;
    return __builtin_fmaf(s, a.digit, __builtin_fmaf(s, a.digit_rest, less));
}

// E elements from `at` on of a row and head: into the output where the range is the whole, else with the range's maximum and sum into the workspace.
template <int DT, int D, uint32_t E>
__device__ __forceinline__ void qw_attn_write(const qw_attn_args& a, uint32_t part, uint32_t row, uint32_t head, uint32_t at, float* o, float best, float total, bool first) {
    const uint64_t item = (uint64_t)row * a.q_heads + head;
    if (a.parts > 1u) {
        const uint64_t items = (uint64_t)a.rows * a.q_heads, place = part * items + item;
        if (first) *(f2_t*)(a.part + a.parts * items * D + place * 2u) = f2_t{best, total};
#pragma unroll
        for (uint32_t e = 0; e < E; e += 4u) *(f4_t*)(a.part + place * D + at + e) = f4_t{o[e], o[e + 1], o[e + 2], o[e + 3]};
        return;
    }
    const float inv = qw_attn_inverse(best, total);
    uint16_t* const y = a.out + (uint64_t)row * a.ld_out + head * D + at;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) o[e] *= inv;
#pragma unroll
    for (uint32_t e = 0; e < E; e += E < 8u ? E : 8u) qw_attn_store<DT, (E < 8u ? E : 8u)>(y + e, o + e);
    if (a.lse && first) a.lse[item] = qw_attn_log(a, best, total);
}

// ------------------------------------------------------------------------------------------------
// Streaming: four waves share 16 columns (query rows of a group of heads) and a range of tokens, a step of 32 tokens of its own each, the next step's codes on their
// way; all stays in registers.  S^T = K q^T by two operands of 16 tokens; the running maximum of a column over the lanes of the wave; O^T += V^T P^T.  Elements become
// f16 (keys of bf16 queries: bf16) on the way into the matrix unit.  Where a scale leaves f16's range, a block is broken or a score is far from zero, which the waves notice at the end of
// their range, the range is done once more in the wide form: keys and values in bf16, which holds them all, f16 queries and the weights as two bf16 numbers each, a broken
// block of values for the rows alone that see its token.
// One workgroup a range is bound by the bytes: a token of 64 sequences of up to 8192, 40 heads of 128 over 8: 73 us = 5.6 TB/s of codes and scales (a read of 4 GiB
// 6.15); behind 131077: 30 us (26 = 5.5 TB/s and the join); behind 4096: 8.7 us, latency of two launches.  Several, which read the same tokens from the L2, by the
// vector unit (200 instructions a wave and step, 96 of them turn elements): 8 rows of 16 windows of 1000 tokens, heads of 256: 17.2 us.
// Steps on the 64: one wave's registers for both forms 117 us; 128 registers 100; four scale bytes at a time 93; pages by scalar loads, the tail's care in the last step
// alone, two register sets in turn 85; loads of whole lines, codes as streamed loads 78; three workgroups a unit, not four: 168 registers, so that the
// loads of a step stay ahead of it 73 (three steps ahead 75, four 77).  The four waves' sums meet in LDS at the end.
// ------------------------------------------------------------------------------------------------
template <int D>
struct qw_attn_shared {
    float sums[4][16][D + 4];
    float stats[4][16][2];
};

__device__ __forceinline__ float qw_attn_max_rows(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// The columns c0 .. c0 + 15 over the tokens begin .. end - 1 (begin a multiple of 32).  Whether the range has to be done in the wide form (the same answer in every
// wave); otherwise its results are written.  All of a workgroup call it.
template <int DT, int D, bool SMALL, bool ONCE, bool WIDE>
__device__ __forceinline__ bool qw_attn_stream(const qw_attn_args& a, const qw_attn_seq& s, uint32_t seq, uint32_t head, uint32_t part, uint32_t c0, uint32_t begin, uint32_t end,
                                               qw_attn_shared<D>& sh) {
    constexpr uint32_t SETS = qw_attn_step<D>::SETS, WORDS = qw_attn_step<D>::WORDS, ROWS = D / 16u;   // ROWS: accumulators, and elements of a column that a thread stores
    constexpr int VT = WIDE ? QWHIP_BF16 : QWHIP_F16;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), i = lane & 15u, g = lane >> 4;
    const uint32_t count = s.n * a.shared;
    qw_attn_range t = qw_attn_tokens<32>(a, s, c0, min(c0 + 15u, count - 1u), 0u);
    t.first = max(t.first, begin), t.from = 0u;
    t.to = t.pos_b < 0 || t.first >= end ? 0u : (min(end, (uint32_t)t.pos_b + 1u) + 31u - min(t.first, (uint32_t)t.pos_b + 1u)) / 32u;
    const uint32_t stop = (uint32_t)t.pos_b + 1u;   // behind what they see; read only where there are steps
    // this lane's column
    const uint32_t col = min(c0 + i, count - 1u), row = col / a.shared, member = col - row * a.shared;
    const int32_t pos = s.pos0 + (int32_t)row, low = (int32_t)qw_attn_low(a, pos);

    u4_t q[SETS][WORDS];
    {
        const uint16_t* const x = a.q + (uint64_t)(s.row0 + row) * a.ld_q + (head * a.shared + member) * D;
#pragma unroll
        for (uint32_t c = 0; c < SETS; ++c)
#pragma unroll
            for (uint32_t j = 0; j < WORDS; ++j) q[c][j] = *(const u4_t*)(x + c * 128u + g * (8u * WORDS) + 8u * j);
    }
    f4_t acc[ROWS];
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j) acc[j] = f4_t{0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), sum = 0.0f;   // top: what the weights' exponents are less
    uint32_t far = 0, far_k = 0;
    const uint8_t* const pages = a.pages + (uint64_t)head * a.geo.piece;
    const uint32_t stride = a.kv_heads * a.geo.piece;
    const int32_t* const table = a.table + (uint64_t)seq * a.ld_table;
    qw_attn_place<D> place;
    place.set(a, i, g);

    auto one = [&](uint32_t t0, qw_attn_step<D>& now) {
        if (t0 < t.low_a || t0 + 32u > stop) qw_attn_cut<D>(t0, t.low_a, stop, i, g, now);
        if constexpr (!WIDE) {
#pragma unroll
            for (uint32_t c = 0; c < SETS; ++c) {
                far |= qw_attn_far8(u2_t{now.v_scale[c][0], now.v_scale[c][1]});
                if constexpr (DT == QWHIP_F16) far |= qw_attn_far<DT>(now.k_scale[0][c]) | qw_attn_far<DT>(now.k_scale[1][c]);
                else far_k = max(far_k, max(now.k_scale[0][c], now.k_scale[1][c]));
            }
        }
        f4_t x[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t c = 0; c < SETS; ++c) {
                const bool nan = WIDE && now.k_scale[h][c] > QW_ATTN_BF16_MOST;
                const float unit = __uint_as_float((nan ? 127u : now.k_scale[h][c]) << 23);
#pragma unroll
                for (uint32_t j = 0; j < WORDS; ++j) {
                    u4_t k = qw_attn_operand<WIDE ? QWHIP_BF16 : DT>(now.k[h][c][j], unit);
                    if (nan) k = u4_t{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
                    if constexpr (WIDE && DT == QWHIP_F16) {
                        u4_t hi, lo, y = q[c][j];
                        asm volatile("" : "+v"(y));   // split anew every time: the parts would take as many registers again
                        qw_attn_split(y, hi, lo);
                        x[h] = qw_attn_mfma<QWHIP_BF16>(k, hi, qw_attn_mfma<QWHIP_BF16>(k, lo, x[h]));
                    } else {
                        x[h] = qw_attn_mfma<DT>(k, q[c][j], x[h]);
                    }
                }
            }
        // masks where a column does not see the whole step
        uint32_t seen = 0xFFu;
        if ((int32_t)(t0 + 31u) > t.pos_a || t0 < t.low_b) {
            seen = 0u;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const int32_t at = (int32_t)(t0 + 16u * (e >> 2) + 4u * g + (e & 3u));
                const bool in = at <= pos && at >= low;
                seen |= in ? 1u << e : 0u;
                if (!in) x[e >> 2][e & 3u] = -__builtin_inff();
            }
        }
        const float most = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3]))) * a.scale2;
        // where no weight is too large lanes need not meet (the first score always is)
        if (__ballot(most - top > (WIDE ? QW_ATTN_ROOM_WIDE : QW_ATTN_ROOM)) != 0ull) {
            const float all = qw_attn_max_rows(most), larger = all - top > (WIDE ? QW_ATTN_ROOM_WIDE : QW_ATTN_ROOM) ? all - (WIDE ? 0.0f : QW_ATTN_UNDER) : top;
            const float fade = __builtin_amdgcn_exp2f(top - (larger == -__builtin_inff() ? 0.0f : larger));
            sum *= fade;
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j) acc[j] = acc[j] * fade;
            top = larger;
            if constexpr (!WIDE) far |= qw_attn_far_score(top);
        }
        const float shift = top == -__builtin_inff() ? 0.0f : top;
        float p[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(WIDE ? x[e >> 2][e & 3u] * a.scale2 - shift : __builtin_fmaf(x[e >> 2][e & 3u], a.scale2, -shift));
        sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        u4_t hi, lo, in;   // the weights; wide: as two bf16 numbers, and whether their tokens are seen
        if constexpr (!WIDE) {
            h8_t w;
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = (h1_t)p[e];
            hi = __builtin_bit_cast(u4_t, w);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = qw_attn_bf16x2(p[2 * e], p[2 * e + 1]);
                lo[e] = qw_attn_bf16x2(p[2 * e] - __uint_as_float(hi[e] << 16), p[2 * e + 1] - __uint_as_float(hi[e] & 0xFFFF0000u));
                in[e] = ((seen >> (2 * e)) & 1u ? 0x3F80u : 0u) | ((seen >> (2 * e)) & 2u ? 0x3F800000u : 0u);
            }
        }
#pragma unroll
        for (uint32_t c = 0; c < SETS; ++c) {
            float unit[8];
            uint32_t word[8];
            u4_t broken = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                unit[e] = qw_attn_unit(u2_t{now.v_scale[c][0], now.v_scale[c][1]}, e);
                word[e] = D == 64 ? now.v[c][e >> 2][e & 3u] >> (16u * (i >> 3)) : now.v[c][e >> 2][e & 3u];
                if constexpr (WIDE) {
                    const bool nan = ((__float_as_uint(unit[e]) >> 23) & 0xFFu) > QW_ATTN_BF16_MOST;
                    unit[e] = nan ? 1.0f : unit[e];
                    word[e] = nan ? 0u : word[e];
                    broken[e >> 1] |= nan ? 0x3F80u << (16u * (e & 1u)) : 0u;
                }
            }
            f4_t bad = {0.f, 0.f, 0.f, 0.f};
            if constexpr (WIDE) bad = qw_attn_mfma<QWHIP_BF16>(broken, in, bad);   // an accumulator's row is in one block in all of a set's
            qw_attn_pairs<D == 64 ? 2 : 4>([&](auto pair) {
                constexpr int j = decltype(pair)::value;
                uint32_t v[8];
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) v[e] = qw_attn_pair<VT, j>(word[e], unit[e]);
                u4_t even, odd;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    even[e] = __builtin_amdgcn_perm(v[2 * e + 1], v[2 * e], 0x05040100u);
                    odd[e] = __builtin_amdgcn_perm(v[2 * e + 1], v[2 * e], 0x07060302u);
                }
#pragma unroll
                for (uint32_t o = 0; o < 2; ++o) {
                    f4_t& u = acc[8 * c + 2 * j + o];
                    if constexpr (WIDE) u = qw_attn_mfma<VT>(o ? odd : even, lo, u);
                    u = qw_attn_mfma<VT>(o ? odd : even, hi, u);
                    if constexpr (WIDE) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (bad[r] > 0.0f) u[r] = __builtin_nanf("");
                    }
                }
            });
        }
    };
    if (wave < t.to) {
        // wave w has the steps w, w + 4, ..
        auto load = [&](uint32_t step, qw_attn_step<D>& f) { qw_attn_load<D, SMALL, ONCE>(a, pages, stride, table, t.first + 32u * min(step, t.to - 1u), t.low_a, stop, place, f); };
        qw_attn_step<D> f[WIDE ? 1 : 2];
        if constexpr (WIDE) {
            for (uint32_t step = wave; step < t.to; step += 4u) {
                load(step, f[0]);
                one(t.first + 32u * step, f[0]);
            }
        } else {
            load(wave, f[0]);
            for (uint32_t step = wave; step < t.to; step += 8u) {
                load(step + 4u, f[1]);
                one(t.first + 32u * step, f[0]);
                load(step + 8u, f[0]);
                if (step + 4u < t.to) one(t.first + 32u * (step + 4u), f[1]);
            }
        }
    }
    if constexpr (!WIDE) {
        far |= qw_attn_far<QWHIP_BF16>(far_k);
        if (__syncthreads_or((int)far)) return true;
    } else {
        __syncthreads();   // what an earlier range left in LDS has been read
    }

    // the four waves' columns, then the columns' rows
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (g == 0u) sh.stats[wave][i][0] = top, sh.stats[wave][i][1] = sum;
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t m = 4u * g + r;   // the accumulator's row
            sh.sums[wave][i][D == 64 ? 8u * (m & 7u) + 4u * (m >> 3) + j : 128u * (j >> 3) + 8u * m + (j & 7u)] = acc[j][r];
        }
    __syncthreads();
    const uint32_t mine = tid >> 4, at = (tid & 15u) * ROWS;   // 16 threads a column, ROWS elements each
    if (c0 + mine >= count) return false;
    const uint32_t my_row = (c0 + mine) / a.shared, my_head = head * a.shared + (c0 + mine) - my_row * a.shared;
    float best = -__builtin_inff(), total = 0.0f, o[ROWS] = {};
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) best = fmaxf(best, sh.stats[w][mine][0]);
    const float shift = best == -__builtin_inff() ? 0.0f : best;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(sh.stats[w][mine][0] - shift);
        total += f * sh.stats[w][mine][1];
#pragma unroll
        for (uint32_t e = 0; e < ROWS; ++e) o[e] += f * sh.sums[w][mine][at + e];
    }
    qw_attn_write<DT, D, ROWS>(a, part, s.row0 + my_row, my_head, at, o, best, total, at == 0u);
    return false;
}

template <int DT, int D, bool SMALL, bool ONCE>
__global__ __launch_bounds__(256, D == 256 ? 2 : D == 128 ? 3 : 4) void qw_attn_stream_kernel(const qw_attn_args a) {
    __shared__ qw_attn_shared<D> sh;
    const uint32_t part = blockIdx.x % a.parts, rest = blockIdx.x / a.parts, head = rest % a.kv_heads, tile = a.tiles - 1u - rest / a.kv_heads, seq = blockIdx.y;   // the last rows see the most: first
    const qw_attn_seq s = qw_attn_sequence(a, seq);
    if (tile * 16u >= s.n * a.shared) return;
    const qw_attn_range t = qw_attn_tokens<32>(a, s, tile * 16u, min(tile * 16u + 15u, s.n * a.shared - 1u), part);
    const uint32_t begin = t.first + 32u * t.from, end = t.first + 32u * t.to;
    if (qw_attn_stream<DT, D, SMALL, ONCE, false>(a, s, seq, head, part, tile * 16u, begin, end, sh))
        qw_attn_stream<DT, D, SMALL, false, true>(a, s, seq, head, part, tile * 16u, begin, end, sh);
}

// ------------------------------------------------------------------------------------------------
// Many rows, heads of 64 and 128: four waves of 32 columns each share tiles of 64 tokens.  A tile's codes are on their way while the tile before it is contracted;
// the threads then turn them into f16 (keys of bf16 queries: bf16) and leave them in LDS as the operands that the waves read, lane by lane: a conversion serves all
// columns of the workgroup.
//   keys     operand of 32 tokens x 16 elements, lane (r, h) elements 8 h .. of token 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4: an accumulator's
//            scores are then eight tokens in a row, twice, the operand of the weights
//   values   operand of 32 elements x 16 tokens, lane (r, h) tokens 8 h .. of element 8 (r % W) + j, W = D / 8 words, r / W picking j in its tile
// A step: the weights of its tile out of its scores, the next tile turned into LDS, a meeting; its values under its weights and the next tile's scores, 32 matrix
// instructions in a row whose operands come from LDS eight ahead.  One meeting does: what a wave that is ahead turns goes into the half of LDS that all have left
// behind them at the meeting before.  Bound by the vector unit beside the matrix unit (heads of 128: 297 vector instructions a wave and step against 32 matrix ones
// of 32 cycles, which keep that unit busy for 39 % of the cycles; the two workgroups of a compute unit overlap little, and four waves that multiply read LDS at its
// full rate): 4096 rows of a prompt, 40 heads of 128, bf16: 195 .. 201 us by card = 880 TFLOP/s (the library's product of 8192 x 8192 bf16 matrices: 1230); six
// ragged chunks of up to 700 rows behind up to 6001 tokens, 24 heads of 64, whose scores cost as much for half the products, in three parts: 157 .. 165 us = 480
// TFLOP/s.  Steps on the prompt: 16 columns a wave in the streaming kernel 510 us; tiles through LDS 253; scores a tile ahead 215; operands eight reads ahead 208, a
// wave's priority around them 204; scale bytes four at a time 201; pages and addresses on the scalar unit, one meeting a step 196.  Eight waves a workgroup turn a
// tile for twice the columns, but meet more of each other (245); two groups of waves half a step apart leave a SIMD's vector unit to one wave at a time (252);
// without the wide form behind it the kernel would take 5 % less.
// ------------------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ f16_t qw_attn_mfma32(u4_t a, u4_t b, f16_t c) {
    if constexpr (DT == QWHIP_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

constexpr uint32_t QW_ATTN_WAVES = 4, QW_ATTN_COLUMNS = 32 * QW_ATTN_WAVES;
template <int D>
struct qw_attn_tile {
    static constexpr uint32_t T = 64, THREADS = QW_ATTN_WAVES * 64, W = D / 8, JT = 256 / D;
    static constexpr uint32_t KW = T * W / THREADS;        // words of a token that a thread turns
    static constexpr uint32_t VS = T * D / 16 / THREADS;   // pairs of elements of eight tokens' words
    static constexpr uint32_t K_BYTES = T * D * 2;
};
template <int D>
struct qw_attn_fetch {
    uint32_t k[qw_attn_tile<D>::KW], k_scale;
    u4_t v[2];
    u2_t v_scale;
};

template <int DT, int D, bool BIG>
__global__ __launch_bounds__(256, D == 128 ? 2 : 3) void qw_attn_tile_kernel(const qw_attn_args a) {
    typedef qw_attn_tile<D> L;
    constexpr uint32_t T = L::T, W = L::W, JT = L::JT, NT = D / 32, KS = D / 16, HALVES = T / 32;
    __shared__ union __attribute__((aligned(16))) {
        struct {
            uint8_t k[2][L::K_BYTES], v[2][L::K_BYTES];
        } tile;
        qw_attn_shared<D> stream;
    } sh;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), r = lane & 31u, hf = lane >> 5;
    const uint32_t head = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads, part = rest % a.parts, tile = a.tiles - 1u - rest / a.parts, seq = blockIdx.y;
    const qw_attn_seq s = qw_attn_sequence(a, seq);
    const uint32_t count = s.n * a.shared, c0 = tile * QW_ATTN_COLUMNS;
    if (c0 >= count) return;
    const qw_attn_range rg = qw_attn_tokens<T>(a, s, c0, min(c0 + QW_ATTN_COLUMNS - 1u, count - 1u), part);
    // this lane's column
    const uint32_t w0 = c0 + wave * 32u, col = min(w0 + r, count - 1u), row = col / a.shared, member = col - row * a.shared;
    const int32_t pos = s.pos0 + (int32_t)row, low = (int32_t)qw_attn_low(a, pos);
    const qw_attn_range mine = qw_attn_tokens<T>(a, s, min(w0, count - 1u), min(w0 + 31u, count - 1u), 0u);   // what the wave's columns see
    const bool busy = w0 < count;
    uint32_t far = 0;

    u4_t q[KS];
    {
        const uint16_t* const x = a.q + (uint64_t)(s.row0 + row) * a.ld_q + (head * a.shared + member) * D;
#pragma unroll
        for (uint32_t j = 0; j < KS; ++j) q[j] = *(const u4_t*)(x + 16u * j + 8u * hf);
    }
    f16_t acc[NT];
#pragma unroll
    for (uint32_t j = 0; j < NT; ++j) acc[j] = f16_t{};
    float top = -__builtin_inff(), sum = 0.0f;   // top: what the weights' exponents are less

    // what this thread turns: token kt, words kw .. of the keys; eight tokens vt .., word vw, pairs vs .. of the values
    const uint32_t kt = tid % T, kw = tid / T * L::KW, vw = tid % W, vt = tid / W % (T / 8u) * 8u, vs = tid / W / (T / 8u) * L::VS;
    // A tile lies in one page, the same for all threads (BIG: scalar loads and addresses), or in several small ones.
    const uint32_t stop = (uint32_t)rg.pos_b + 1u, first_page = rg.low_a >> a.geo.page_log2, last_page = (stop - 1u) >> a.geo.page_log2;   // read only where there are steps
    const uint32_t inside = (1u << a.geo.page_log2) - 1u, last = max(rg.to, 1u) - 1u;
    const uint32_t kin = BIG ? kt : kt & inside, vin = BIG ? vt : vt & inside, kpage = BIG ? 0u : kt >> a.geo.page_log2, vpage = BIG ? 0u : vt >> a.geo.page_log2;
    const uint32_t k_at = kin * (D / 2u) + kw * 4u, ks_at = a.geo.k_scales + kin * (D / 32u) + kw / 4u;
    const uint32_t v_at = a.geo.v_codes + ((vin >> 3) * W + vw) * 32u, vs_at = a.geo.v_scales + ((vin >> 3) * (D / 32u) + vw / 4u) * 8u;
    const uint8_t* const pages = a.pages + (uint64_t)head * a.geo.piece;
    const uint32_t stride = a.kv_heads * a.geo.piece;
    const int32_t* const table = a.table + (uint64_t)seq * a.ld_table;
    auto tile_of = [&](uint32_t step) { return rg.first + min(step, last) * T; };   // first token; behind the last tile the last one's
    // whether only some of a tile's tokens are seen; whole ones begin at whole .. whole + wholes
    const uint32_t whole = stop - rg.low_a >= T ? rg.low_a : ~0u, wholes = stop - rg.low_a >= T ? stop - T - rg.low_a : 0u;
    auto part_of = [&](uint32_t t0) { return t0 - whole > wholes; };
    auto page_at = [&](uint32_t t0, uint32_t more) {
        const uint32_t p = (t0 >> a.geo.page_log2) + more;   // a part of a tile in front of the first token that is seen, or behind the last, is read from theirs, and masked
        return (uint32_t)table[BIG ? p : min(max(p, first_page), last_page)];
    };
    auto base_of = [&](uint32_t page) { return pages + (uint64_t)(page < a.page_count ? page : 0u) * stride; };
    auto fetch_k = [&](uint32_t t0, uint32_t page, qw_attn_fetch<D>& f) {
        const uint8_t* const b = base_of(page);
        const uint32_t in = BIG ? t0 & inside : 0u;
        __builtin_memcpy(f.k, __builtin_assume_aligned(b + in * (D / 2u) + k_at, 4 * L::KW), 4 * L::KW);
        f.k_scale = (b + in * (D / 32u))[ks_at];
    };
    auto fetch_v = [&](uint32_t t0, uint32_t page, qw_attn_fetch<D>& f) {
        const uint8_t* const b = base_of(page);
        const uint32_t in = BIG ? t0 & inside : 0u;
        const uint8_t* const w = b + in * (D / 2u) + v_at;
        f.v[0] = *(const u4_t*)w;
        f.v[1] = *(const u4_t*)(w + 16);
        f.v_scale = *(const u2_t*)(b + in * (D / 32u) + vs_at);
    };
    auto turn_k = [&](const qw_attn_fetch<D>& f, uint32_t t0, uint32_t slot) {
        uint32_t byte = f.k_scale;
        if (part_of(t0)) byte = t0 + kt < rg.low_a || t0 + kt >= stop ? 127u : byte;
        far |= qw_attn_far<DT>(byte);
        const float unit = __uint_as_float(byte << 23);
        const uint32_t t = kt & 31u, at = (t & 16u) | ((t & 4u) << 1) | ((t & 8u) >> 1) | (t & 3u);
#pragma unroll
        for (uint32_t i = 0; i < L::KW; ++i) {
            const uint32_t w = kw + i;
            *(u4_t*)(sh.tile.k[slot] + ((((kt >> 5) * KS + (w >> 1)) * 64u) + (w & 1u) * 32u + at) * 16u) = qw_attn_operand<DT>(f.k[i], unit);
        }
    };
    auto turn_v = [&](const qw_attn_fetch<D>& f, uint32_t t0, uint32_t slot) {
        u2_t scales = f.v_scale;
        if (part_of(t0))
            scales = u2_t{qw_attn_seen(scales[0], qw_attn_there(t0 + vt, rg.low_a, stop)), qw_attn_seen(scales[1], qw_attn_there(t0 + vt + 4u, rg.low_a, stop))};
        far |= qw_attn_far8(scales);
#pragma unroll
        for (uint32_t i = 0; i < L::VS; ++i) {
            const uint32_t pair = vs + i;
            uint32_t x[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                x[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(f.v[e >> 2][e & 3u] >> (8u * pair), qw_attn_unit(scales, e), 0));
            u4_t even, odd;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                even[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x05040100u);
                odd[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);
            }
#pragma unroll
            for (uint32_t o = 0; o < 2; ++o) {
                const uint32_t j = 2u * pair + o;
                *(u4_t*)(sh.tile.v[slot] + (((j / JT) * (T / 16u) + (vt >> 4)) * 64u + ((vt >> 3) & 1u) * 32u + vw + W * (j % JT)) * 16u) = o ? odd : even;
            }
        }
    };

    // a wave's scores of the next tile and its weights of this one
    f16_t x[HALVES];
    h8_t p[2 * HALVES];
    auto sees = [&](uint32_t step) { return step < rg.to && busy && (int32_t)(rg.first + step * T) <= mine.pos_b && rg.first + (step + 1u) * T > mine.low_a; };
    // The matrix unit's part of a step: this tile's values under its weights (`out`), the next tile's scores.  Operands come from LDS AHEAD of their use.
    auto products = [&](uint32_t step, auto out) {
        constexpr int OUTS = decltype(out)::value ? 2 * HALVES * NT : 0, ALL = OUTS + KS * HALVES, AHEAD = 8;
        const uint8_t* const values = sh.tile.v[step & 1u] + lane * 16u;
        const uint8_t* const keys = sh.tile.k[(step + 1u) & 1u] + lane * 16u;
        u4_t y[AHEAD];
        auto load = [&](int n) {
            y[n % AHEAD] = n < OUTS ? *(const u4_t*)(values + ((n % NT) * (T / 16u) + n / NT) * 1024u)
                                    : *(const u4_t*)(keys + ((n - OUTS) % HALVES * KS + (n - OUTS) / HALVES) * 1024u);
        };
#pragma unroll
        for (uint32_t h = 0; h < HALVES; ++h) x[h] = f16_t{};
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) load(n);
#pragma unroll
        for (int n = 0; n < ALL; ++n) {
            if (n < OUTS) acc[n % NT] = qw_attn_mfma32<QWHIP_F16>(y[n % AHEAD], __builtin_bit_cast(u4_t, p[n / NT]), acc[n % NT]);
            else x[(n - OUTS) % HALVES] = qw_attn_mfma32<DT>(y[n % AHEAD], q[(n - OUTS) / HALVES], x[(n - OUTS) % HALVES]);
            if (n + AHEAD < ALL) load(n + AHEAD);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);   // reads of LDS, then one for each matrix instruction
#pragma unroll
        for (int n = 0; n < ALL - AHEAD; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
    };
    // masks, the running maximum, exponentials, their sum
    auto weights = [&](uint32_t step) {
        const uint32_t t0 = rg.first + step * T;
        if ((int32_t)(t0 + T - 1u) > mine.pos_a || t0 < mine.low_b) {
#pragma unroll
            for (uint32_t h = 0; h < HALVES; ++h)
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e) {
                    const int32_t t = (int32_t)(t0 + 32u * h + 16u * (e >> 3) + 8u * hf + (e & 7u));
                    if (t > pos || t < low) x[h][e] = -__builtin_inff();
                }
        }
        float most = x[0][0];
#pragma unroll
        for (uint32_t h = 0; h < HALVES; ++h)
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) most = fmaxf(most, x[h][e]);
        most *= a.scale2;
        // where no weight is too large lanes need not meet (the first score always is)
        if (__ballot(most - top > QW_ATTN_ROOM) != 0ull) {
            const float all = fmaxf(most, __shfl_xor(most, 32, 64)), larger = all - top > QW_ATTN_ROOM ? all - QW_ATTN_UNDER : top;
            const float fade = __builtin_amdgcn_exp2f(top - (larger == -__builtin_inff() ? 0.0f : larger));
            sum *= fade;
#pragma unroll
            for (uint32_t j = 0; j < NT; ++j) acc[j] = acc[j] * fade;
            top = larger;
            far |= qw_attn_far_score(top);
        }
        const float shift = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (uint32_t h = 0; h < HALVES; ++h) {
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) x[h][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[h][e], a.scale2, -shift));
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) p[2 * h + (e >> 3)][e & 7u] = (h1_t)x[h][e];
            sum += (((x[h][0] + x[h][1]) + (x[h][2] + x[h][3])) + ((x[h][4] + x[h][5]) + (x[h][6] + x[h][7]))) +
                   (((x[h][8] + x[h][9]) + (x[h][10] + x[h][11])) + ((x[h][12] + x[h][13]) + (x[h][14] + x[h][15])));
        }
    };
    // LDS is written and read in order, loads from memory go on
#define QW_ATTN_MEET() asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory")

    if (rg.from < rg.to) {
        qw_attn_fetch<D> f;
        // a turn leaves the values of `step` and the keys of step + 1 in LDS
        {
            const uint32_t t0 = tile_of(rg.from);
            fetch_k(t0, page_at(t0, kpage), f);
            turn_k(f, t0, rg.from & 1u);
        }
        fetch_k(tile_of(rg.from + 1u), page_at(tile_of(rg.from + 1u), kpage), f);
        fetch_v(tile_of(rg.from), page_at(tile_of(rg.from), vpage), f);
        uint32_t next_k = page_at(tile_of(rg.from + 2u), kpage), next_v = page_at(tile_of(rg.from + 1u), vpage);
        QW_ATTN_MEET();
        if (sees(rg.from)) products(rg.from - 1u, std::false_type{});
        for (uint32_t step = rg.from; step < rg.to; ++step) {
            const bool now = sees(step);
            if (now) {
                weights(step);
            } else {
#pragma unroll
                for (uint32_t m = 0; m < 2 * HALVES; ++m) p[m] = h8_t{};
            }
            turn_k(f, tile_of(step + 1u), (step + 1u) & 1u);
            turn_v(f, tile_of(step), step & 1u);
            fetch_k(tile_of(step + 2u), next_k, f);
            fetch_v(tile_of(step + 1u), next_v, f);
            next_k = page_at(tile_of(step + 3u), kpage), next_v = page_at(tile_of(step + 2u), vpage);
            QW_ATTN_MEET();
            __builtin_amdgcn_s_setprio(1);
            if (now || sees(step + 1u)) products(step, std::true_type{});   // one of the two may be idle work at either end of the range
            __builtin_amdgcn_s_setprio(0);
        }
    }
#undef QW_ATTN_MEET
    if (__syncthreads_or((int)far)) {
        const uint32_t begin = rg.first + rg.from * T, end = rg.first + rg.to * T;
        if (a.geo.page_log2 == 4u)
            for (uint32_t c = c0; c < min(c0 + QW_ATTN_COLUMNS, count); c += 16u) qw_attn_stream<DT, D, true, false, true>(a, s, seq, head, part, c, begin, end, sh.stream);
        else
            for (uint32_t c = c0; c < min(c0 + QW_ATTN_COLUMNS, count); c += 16u) qw_attn_stream<DT, D, false, false, true>(a, s, seq, head, part, c, begin, end, sh.stream);
        return;
    }

    if (w0 + r >= count) return;
    sum += __shfl_xor(sum, 32, 64);   // lanes r and r + 32 are the same column: both are here
    // accumulator row m of tile j: element 8 (m % W) + JT j + m / W; a lane has whole words
    constexpr uint32_t HALF = W / 2u;
#pragma unroll
    for (uint32_t e = 0; e < HALF; ++e) {
        float o[8];
#pragma unroll
        for (uint32_t j = 0; j < NT; ++j)
#pragma unroll
            for (uint32_t k = 0; k < JT; ++k) o[JT * j + k] = acc[j][e + HALF * k];
        qw_attn_write<DT, D, 8>(a, part, s.row0 + row, head * a.shared + member, 8u * (8u * (e >> 2) + 4u * hf + (e & 3u)), o, top, sum, e == 0u && hf == 0u);
    }
}

// The parts of a row and head, joined in their order: few parts by D / 4 threads, more by a workgroup, whose threads take every (1024 / D)th part and meet in LDS.
constexpr uint32_t QW_ATTN_MOST_PARTS = 256, QW_ATTN_FEW_PARTS = 4;
template <int DT, int D, bool FEW>
__global__ __launch_bounds__(256) void qw_attn_join_kernel(const qw_attn_args a) {
    constexpr uint32_t LANES = D / 4u, GROUPS = 256u / LANES;
    __shared__ float weight[QW_ATTN_MOST_PARTS], fold[2][4];
    __shared__ f4_t sums[FEW ? 1 : GROUPS][LANES];
    const uint32_t tid = threadIdx.x, lane = tid % LANES, group = tid / LANES, at = FEW ? blockIdx.x * GROUPS + group : blockIdx.x, seq = blockIdx.y;
    const qw_attn_seq s = qw_attn_sequence(a, seq);
    const uint32_t row = at / a.q_heads;
    if (row >= s.n) return;
    const uint64_t items = (uint64_t)a.rows * a.q_heads, item = (uint64_t)s.row0 * a.q_heads + at;
    const float* const stats = a.part + a.parts * items * D + item * 2u;
    const float* const x = a.part + item * D + lane * 4u;
    float best = -__builtin_inff(), total = 0.0f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    if constexpr (FEW) {
        f2_t st[QW_ATTN_FEW_PARTS];
        f4_t y[QW_ATTN_FEW_PARTS];
#pragma unroll
        for (uint32_t p = 0; p < QW_ATTN_FEW_PARTS; ++p) {
            const uint32_t from = min(p, a.parts - 1u);
            st[p] = *(const f2_t*)(stats + from * items * 2u);
            y[p] = *(const f4_t*)(x + from * items * D);
        }
#pragma unroll
        for (uint32_t p = 0; p < QW_ATTN_FEW_PARTS; ++p) best = fmaxf(best, st[p][0]);
        const float shift = best == -__builtin_inff() ? 0.0f : best;
#pragma unroll
        for (uint32_t p = 0; p < QW_ATTN_FEW_PARTS; ++p) {
            if (p >= a.parts) break;
            const float f = __builtin_amdgcn_exp2f(st[p][0] - shift);
            total += f * st[p][1];
            o += f * y[p];
        }
    } else {
        const f2_t st = tid < a.parts ? *(const f2_t*)(stats + tid * items * 2u) : f2_t{-__builtin_inff(), 0.0f};
        best = st[0];
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor(best, off, 64));
        if ((tid & 63u) == 0u) fold[0][tid >> 6] = best;
        __syncthreads();
        best = fmaxf(fmaxf(fold[0][0], fold[0][1]), fmaxf(fold[0][2], fold[0][3]));
        const float f = __builtin_amdgcn_exp2f(st[0] - (best == -__builtin_inff() ? 0.0f : best));
        weight[tid] = f;
        total = f * st[1];
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
        if ((tid & 63u) == 0u) fold[1][tid >> 6] = total;
        __syncthreads();
        total = (fold[1][0] + fold[1][1]) + (fold[1][2] + fold[1][3]);
#pragma unroll 4
        for (uint32_t p = group; p < a.parts; p += GROUPS) o += weight[p] * *(const f4_t*)(x + p * items * D);
        sums[group][lane] = o;
        __syncthreads();
        if (group != 0u) return;
#pragma unroll
        for (uint32_t k = 1; k < GROUPS; ++k) o += sums[k][lane];
    }
    const float inv = qw_attn_inverse(best, total);
    float y[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    qw_attn_store<DT, 4>(a.out + (uint64_t)(s.row0 + row) * a.ld_out + (at - row * a.q_heads) * D + lane * 4u, y);
    if (a.lse && tid % LANES == 0u) a.lse[item] = qw_attn_log(a, best, total);
}

constexpr uint32_t QW_ATTN_MOST_TILES = 1u << 22;   // of 256 threads, a launch holds under 2^32
// The kernel of a call and how many parts its rows are split into, from the shapes and the host's bounds.
// The streaming kernel turns a token's elements anew for every 16 columns (rows x heads of a group), but has more and shorter workgroups: the tile kernel is for
// many columns over many tokens, from 256 columns and 2^20 tokens over all its tiles.  Stream / tile, each with the better number of parts, us: heads of 128, 8 rows of
// 40 columns behind 4096 tokens, one sequence 12 / 15, 64 of them 78 / 122; 512 rows of a prompt 16 / 21, 1024 33 / 36, 2048 89 / 70, 4096 283 / 217; 256 rows behind
// 16384 142 / 120, 512 259 / 205, behind 4096 70 / 68; heads of 64, 1024 rows 17 / 24, behind 16384 221 / 152, 4096 rows 126 / 93.  With heads of 256, whose tiles leave
// a compute unit one workgroup, it was the slower one but for 4096 rows of a prompt (271 / 260; 1024 37 / 52; 8 rows in 16 windows of 1000 18 / 25), so it has none.
// Parts give a launch workgroups enough, but a part has to be worth its share of the join (3 .. 5 us) and of the partial results, which are written and read once more.
// Streaming: powers of two, so that one part of all heads and tiles meets in one XCD's L2 (8 sequences of 8 rows behind 4096 in 1 / 2 / 3 / 4 / 5 / 8 parts 24 / 23 / 24 /
// 20 / 23 / 24 us).  A workgroup a range: up to 16 parts two workgroups a compute unit, more for one, of at least 128 tokens (a token behind 131077 in 16 / 32 / 48: 47 / 30 /
// 33; 4 sequences of up to 32768 in 4 / 8 / 16 / 32: 46 / 29 / 26 / 29; 24 of up to 8192 in 1 / 2 / 4 / 8: 44 / 38 / 35 / 36, 64 of them 74 / 77 / 77 / 84; behind 500 in 1 / 4:
// 7.2 / 8.9).  Several, bound by the vector unit: up to 256 workgroups, or 1024 of at least 1024 tokens (16 rows behind 32768, 40 workgroups, in 8 / 16 / 32 / 48: 40 / 33 / 32 /
// 37; 8 rows behind 4096, 24, in 4 / 8 / 16: 13.0 / 11.4 / 12.5; up to 342 workgroups instead took 10 % longer over 68 shapes that they change: 16 rows behind 1500 in 4 /
// 8: 11.1 / 12.4, 64 in 1 / 2: 12.2 / 15.3, 20 sequences of 8 rows and heads of 256 in a window of 1000 in 1 / 2: 18.1 / 23.0).
// Tiles: as many as run at once, else two rounds of them (heads of 64: three), of at least 1536 tokens (heads of 128, two a unit: 160 tiles in 2 / 3 / 4 parts 276 /
// 207 / 246, two chunks of 512 rows, 320, in 1 / 3 / 4: 242 / 199 / 206, eight of up to 256, 640, in 1 / 2: 142 / 152; heads of 64, three a unit: 192 in 3 / 4 / 6: 190 /
// 154 / 186; six ragged chunks, 680, in 1 / 2 / 3: 178 / 161 / 152).
struct qw_attn_plan {
    bool stream;
    uint64_t tiles;   // of a sequence and a head
    uint32_t parts;
};
static qw_attn_plan qw_attn_choose(const qwhip_kv_cache* c, const qwhip_kv_batch* b, uint32_t rows, uint32_t q_heads, uint32_t window) {
    const uint32_t shared = q_heads / c->kv_heads;
    const uint64_t columns = (uint64_t)(b->max_rows < rows ? b->max_rows : rows) * shared;
    const uint32_t longest = window && window < b->max_length && b->max_rows < b->max_length - window ? window + b->max_rows : b->max_length;
    // workgroups of `width` columns over all sequences, of which ragged ones have fewer than the bound says
    auto workgroups = [&](uint64_t tiles, uint32_t width) {
        const uint64_t most = tiles * b->seqs, some = (uint64_t)rows * shared / width + b->seqs;
        return (most < some ? most : some) * c->kv_heads;
    };
    qw_attn_plan p;
    p.tiles = (columns + QW_ATTN_COLUMNS - 1u) / QW_ATTN_COLUMNS;
    uint64_t all = workgroups(p.tiles, QW_ATTN_COLUMNS), parts = 1u;
    p.stream = c->head_dim == 256u || columns < 256u || all * longest < 1u << 20;
    if (p.stream) {
        p.tiles = (columns + 15u) / 16u;
        all = workgroups(p.tiles, 16u);
        if (longest > (c->head_dim == 256u ? 512u : 1024u)) {
            auto up = [](uint64_t n, uint64_t d) {   // the power of two at or over n / d
                uint64_t two = 1u;
                while (two * d < n) two *= 2u;
                return two;
            };
            auto down = [](uint64_t n, uint64_t d) {   // at or under it, one at least
                uint64_t two = 1u;
                while (two * 2u * d <= n) two *= 2u;
                return two;
            };
            if (p.tiles == 1u) parts = up(512u, all) <= 16u ? up(512u, all) : std::max<uint64_t>(16u, up(256u, all));
            else parts = down(256u, all);
            parts = std::min(parts, down(longest, 128u));
            if (p.tiles > 1u) parts = std::max(parts, std::min(up(1024u, all), down(longest, 1024u)));
        }
    } else {
        const uint64_t units = c->head_dim == 128u ? 512u : 768u, rounds = c->head_dim == 128u ? 2u : 3u;
        parts = std::min<uint64_t>(all * 2u <= units ? units / all : rounds * units / all, longest / 1536u);
    }
    p.parts = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(parts, 1u), QW_ATTN_MOST_PARTS);
    return p;
}
static uint64_t qw_attn_part_bytes(uint32_t rows, uint32_t q_heads, uint32_t d) { return (uint64_t)rows * q_heads * (d + 2u) * 4u; }

static qwhip_status qw_attn_check(const qwhip_kv_cache* cache, const qwhip_kv_batch* b, uint32_t q_heads, uint32_t rows) {
    const qwhip_status st = qwhip_kv_cache_validate(cache);
    if (st != QWHIP_OK) return st;
    QWHIP_REQUIRE(b);
    if (q_heads == 0 || q_heads > 65535u || q_heads % cache->kv_heads != 0)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u query heads over %u heads of the cache", q_heads, cache->kv_heads);
    if (b->seqs > 65535u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u sequences do not fit one launch", b->seqs);
    if (rows > 0x7FFFFFFFu || b->max_rows > 0x7FFFFFFFu) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows, %u of a sequence", rows, b->max_rows);
    if (b->max_length > 0x7FFFFFFFu || b->max_length > (uint64_t)b->ld_table * cache->page_size)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "sequences of %u tokens in tables of %u pages of %u", b->max_length, b->ld_table, cache->page_size);
    if (!b->row_start && (b->seqs != rows || b->max_rows == 0)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "without row_start %u sequences have %u rows", b->seqs, rows);
    return QWHIP_OK;
}

extern "C" uint64_t qwhip_kv_attention_workspace_bytes(const qwhip_kv_cache* cache, const qwhip_kv_batch* b, uint32_t q_heads, uint32_t rows, uint32_t window) {
    if (qw_attn_check(cache, b, q_heads, rows) != QWHIP_OK || rows == 0 || b->seqs == 0 || b->max_rows == 0) return 0;
    const uint32_t parts = qw_attn_choose(cache, b, rows, q_heads, window).parts;
    return parts > 1u ? parts * qw_attn_part_bytes(rows, q_heads, cache->head_dim) : 0u;
}

template <int DT, int D>
static void qw_launch_attn(qwhip_stream_t s, const qw_attn_args& a, bool stream, uint32_t seqs) {
    const dim3 grid(a.parts * a.kv_heads * a.tiles, seqs);
    if (stream) {
        const bool small = a.geo.page_log2 == 4u;
        if (a.tiles == 1u && small) hipLaunchKernelGGL((qw_attn_stream_kernel<DT, D, true, true>), grid, dim3(256), 0, s->stream, a);
        else if (a.tiles == 1u) hipLaunchKernelGGL((qw_attn_stream_kernel<DT, D, false, true>), grid, dim3(256), 0, s->stream, a);
        else if (small) hipLaunchKernelGGL((qw_attn_stream_kernel<DT, D, true, false>), grid, dim3(256), 0, s->stream, a);
        else hipLaunchKernelGGL((qw_attn_stream_kernel<DT, D, false, false>), grid, dim3(256), 0, s->stream, a);
    } else if constexpr (D != 256) {
        if ((1u << a.geo.page_log2) >= qw_attn_tile<D>::T) hipLaunchKernelGGL((qw_attn_tile_kernel<DT, D, true>), grid, dim3(256), 0, s->stream, a);
        else hipLaunchKernelGGL((qw_attn_tile_kernel<DT, D, false>), grid, dim3(256), 0, s->stream, a);
    }
    const uint32_t items = a.max_rows * a.q_heads;
    if (a.parts > QW_ATTN_FEW_PARTS) hipLaunchKernelGGL((qw_attn_join_kernel<DT, D, false>), dim3(items, seqs), dim3(256), 0, s->stream, a);
    else if (a.parts > 1u) hipLaunchKernelGGL((qw_attn_join_kernel<DT, D, true>), dim3(qwhip_cdiv(items, 1024u / D), seqs), dim3(256), 0, s->stream, a);
}

extern "C" qwhip_status qwhip_kv_attention_mxfp4(qwhip_stream_t s, const qwhip_kv_cache* cache, const qwhip_kv_batch* batch, const void* q, uint32_t dtype,
                                                 uint32_t q_heads, uint32_t ld_q, uint32_t rows, float scale, uint32_t window, void* out, uint32_t ld_out, float* lse,
                                                 void* workspace, uint64_t workspace_bytes) {
    QWHIP_REQUIRE(s);
    const qwhip_status st = qw_attn_check(cache, batch, q_heads, rows);
    if (st != QWHIP_OK) return st;
    const uint32_t d = cache->head_dim;
    if (dtype != QWHIP_F16 && dtype != QWHIP_BF16) return qwhip_fail(QWHIP_E_BAD_SHAPE, "queries must be f16 or bf16, got dtype %u", dtype);
    if (!(scale > 0.0f) || scale >= 0x1p127f) return qwhip_fail(QWHIP_E_BAD_SHAPE, "scale must be positive, under 2^127");
    if (ld_q == 0) ld_q = q_heads * d;
    if (ld_out == 0) ld_out = q_heads * d;
    if (ld_q < q_heads * d || ld_out < q_heads * d || ld_q % 8u != 0 || ld_out % 8u != 0)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "row pitches %u, %u must be multiples of 8 elements, at least %u", ld_q, ld_out, q_heads * d);
    if (workspace_bytes && ((uintptr_t)workspace & 15u)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "the workspace must be 16-byte aligned");
    if (rows == 0 || batch->seqs == 0 || batch->max_rows == 0) return QWHIP_OK;
    QWHIP_REQUIRE(q);
    QWHIP_REQUIRE(out);
    QWHIP_REQUIRE(batch->lengths);
    if (batch->max_length) QWHIP_REQUIRE(batch->block_table);
    if (((uintptr_t)q | (uintptr_t)out) & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "queries and output must be 16-byte aligned");
    const uint32_t shared = q_heads / cache->kv_heads, max_rows = batch->max_rows < rows ? batch->max_rows : rows;
    const qw_attn_plan plan = qw_attn_choose(cache, batch, rows, q_heads, window);
    if (plan.tiles * cache->kv_heads * plan.parts > QW_ATTN_MOST_TILES) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows of a sequence do not fit one launch", max_rows);
    QW_ON_DEVICE_OF(s);
    qw_attn_args a = {};
    a.pages = (const uint8_t*)cache->pages;
    a.row_start = batch->row_start, a.lengths = batch->lengths, a.table = batch->block_table;
    a.q = (const uint16_t*)q, a.out = (uint16_t*)out, a.lse = lse, a.part = (float*)workspace;
    a.geo = qw_kv_geometry_of(cache);
    a.page_count = cache->page_count, a.kv_heads = cache->kv_heads, a.ld_table = batch->ld_table, a.max_rows = max_rows, a.max_length = batch->max_length;
    a.rows = rows, a.q_heads = q_heads, a.shared = shared, a.ld_q = ld_q, a.ld_out = ld_out, a.window = window > 0x7FFFFFFFu ? 0u : window;
    a.tiles = (uint32_t)plan.tiles;
    a.scale2 = scale * 1.4426950408889634f;
    a.digit = (float)((double)scale / a.scale2), a.digit_rest = (float)((double)scale / a.scale2 - a.digit);
    a.parts = 1;
    if (workspace) {
        a.parts = plan.parts;
        const uint64_t fit = workspace_bytes / qw_attn_part_bytes(rows, q_heads, d);
        if (fit < a.parts) a.parts = fit > 1u ? (uint32_t)fit : 1u;
    }
#define QW_ATTN(DT)                                                          \
    do {                                                                     \
        if (d == 64u) qw_launch_attn<DT, 64>(s, a, plan.stream, batch->seqs);             \
        else if (d == 128u) qw_launch_attn<DT, 128>(s, a, plan.stream, batch->seqs);      \
        else qw_launch_attn<DT, 256>(s, a, plan.stream, batch->seqs);                     \
    } while (0)
    if (dtype == QWHIP_F16) QW_ATTN(QWHIP_F16);
    else QW_ATTN(QWHIP_BF16);
#undef QW_ATTN
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
