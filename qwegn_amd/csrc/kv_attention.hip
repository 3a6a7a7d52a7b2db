// Attention over the paged MXFP4 cache.
#include "qw_kv.h"

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

struct qw_attn_args {
    const uint8_t* pages;
    const int32_t* row_start;
    const int32_t* lengths;
    const int32_t* table;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    float* part;           // [parts][rows][q_heads][D] sums, then [parts][rows][q_heads][2] maximum (of raw scores) and sum of weights
    qw_kv_geometry geo;
    uint32_t page_count, kv_heads, ld_table, max_rows, max_length, rows, q_heads, shared, ld_q, ld_out, window, parts, tiles;
    float scale, scale2;   // scale2 = scale * log2(e)
};

// A sequence's rows and tokens, cut to what the host allows.
struct qw_attn_seq {
    uint32_t row0, n, length;
};
__device__ __forceinline__ qw_attn_seq qw_attn_sequence(const qw_attn_args& a, uint32_t seq) {
    qw_attn_seq s;
    const int32_t from = a.row_start ? a.row_start[seq] : (int32_t)seq, to = a.row_start ? a.row_start[seq + 1u] : (int32_t)seq + 1;
    s.row0 = (uint32_t)max(0, min(from, (int32_t)a.rows));
    s.n = min((uint32_t)max(0, min(to, (int32_t)a.rows) - (int32_t)s.row0), a.max_rows);
    s.length = (uint32_t)max(0, min(a.lengths[seq], (int32_t)a.max_length));
    return s;
}

// What a lane carries of a step of 32 tokens.  Keys: rows of two 16-row operands, lane (i, g) has elements of token 8 (i / 4) + 4 a + i % 4; values: lane
// (i, g) has eight elements of each of the tokens 8 g .. 8 g + 7.  A score of operand a, accumulator row 4 g + r, is then token 8 g + 4 a + r: the weights
// are in place as an operand against the values.
template <int D>
struct qw_attn_step {
    static constexpr uint32_t SETS = D == 256 ? 2 : 1, WORDS = D == 64 ? 2 : 4;
    uint32_t k[2][SETS][WORDS];
    uint32_t k_scale[2][SETS];
    u4_t v[SETS][2];
    u2_t v_scale[SETS];
};
template <int D>
__device__ __forceinline__ void qw_attn_load(const qw_attn_args& a, const uint8_t* head, uint32_t stride_lo, const int32_t* table, uint32_t first_page, uint32_t t0,
                                             uint32_t length, uint32_t i, uint32_t g, qw_attn_step<D>& s) {
    constexpr uint32_t SETS = qw_attn_step<D>::SETS, WORDS = qw_attn_step<D>::WORDS;
    const uint32_t inside = (1u << a.geo.page_log2) - 1u, last = length - 1u;
    // a group of eight tokens behind the last one's is read in its place, and masked
    const uint32_t kt = min(t0 + 8u * (i >> 2), last & ~7u) + (i & 3u), vt = min(t0 + 8u * g, last & ~7u);
    const uint8_t* const kp = head + (uint64_t)(uint32_t)table[(kt >> a.geo.page_log2) - first_page] * stride_lo;
    const uint8_t* const vp = head + (uint64_t)(uint32_t)table[(vt >> a.geo.page_log2) - first_page] * stride_lo;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t t = (kt & inside) + 4u * h;
#pragma unroll
        for (uint32_t c = 0; c < SETS; ++c) {
            __builtin_memcpy(s.k[h][c], __builtin_assume_aligned(kp + t * (D / 2u) + c * 64u + g * (4u * WORDS), 4 * WORDS), 4 * WORDS);
            s.k_scale[h][c] = kp[a.geo.k_scales + t * (D / 32u) + (D == 64 ? g >> 1 : 4u * c + g)];
        }
    }
    const uint32_t t8 = (vt & inside) >> 3, word = D == 64 ? i & 7u : i;
#pragma unroll
    for (uint32_t c = 0; c < SETS; ++c) {
        const uint8_t* const w = vp + a.geo.v_codes + (t8 * (D / 8u) + 16u * c + word) * 32u;
        s.v[c][0] = *(const u4_t*)w;
        s.v[c][1] = *(const u4_t*)(w + 16);
        s.v_scale[c] = *(const u2_t*)(vp + a.geo.v_scales + (t8 * (D / 32u) + 4u * c + (word >> 2)) * 8u);
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
template <int DT>
__device__ __forceinline__ f4_t qw_attn_mfma(u4_t a, u4_t b, f4_t c) {
    if constexpr (DT == QWHIP_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
// Two floats as bf16, the first in the low half.
__device__ __forceinline__ uint32_t qw_attn_bf16x2(float a, float b) { return (uint32_t)qw_f32_to_bf16(a) | ((uint32_t)qw_f32_to_bf16(b) << 16); }

// f16 holds the elements under a scale byte exactly, as normal numbers, from 2^-13 to 2^13; bf16 up to 2^125.
constexpr uint32_t QW_ATTN_F16_LEAST = 114, QW_ATTN_F16_MOST = 140, QW_ATTN_BF16_MOST = 252;

template <int D>
__device__ __forceinline__ float qw_attn_xor_rows(float v, bool largest) {
    const float a = __shfl_xor(v, 16, 64);
    v = largest ? fmaxf(v, a) : v + a;
    const float b = __shfl_xor(v, 32, 64);
    return largest ? fmaxf(v, b) : v + b;
}

// ------------------------------------------------------------------------------------------------
// Four waves share a tile of 16 query rows (token and head of a group) and a range of tokens, a step of 32 tokens of its own each; all stays in registers.
// S^T = K q^T, two operands of 16 tokens; the running maximum of a column (a query row) over the lanes of the wave; O^T += V^T P^T.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t QW_ATTN_TABLE = 1024;   // page numbers of a range that wait in LDS

template <int DT, int D>
__global__ __launch_bounds__(256) void qw_attn_stream_kernel(const qw_attn_args a) {
    constexpr uint32_t SETS = qw_attn_step<D>::SETS, WORDS = qw_attn_step<D>::WORDS, ROWS = D / 16u, PITCH = D + 4u;   // ROWS: elements of a column's sum a lane has in one of 4
    __shared__ int32_t table[QW_ATTN_TABLE];
    __shared__ float sums[4][16][PITCH];
    __shared__ float stats[4][16][2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, i = lane & 15u, g = lane >> 4;
    const uint32_t part = blockIdx.x % a.parts, rest = blockIdx.x / a.parts, head = rest % a.kv_heads, tile = rest / a.kv_heads, seq = blockIdx.y;
    const qw_attn_seq s = qw_attn_sequence(a, seq);
    const uint32_t count = s.n * a.shared, c0 = tile * 16u;
    if (c0 >= count) return;
    // this lane's column
    const uint32_t col = min(c0 + i, count - 1u), row = col / a.shared, member = col - row * a.shared;
    const int32_t pos = (int32_t)(s.length - s.n + row);                                 // negative: sees nothing
    const int32_t low = a.window && pos + 1 > (int32_t)a.window ? pos + 1 - (int32_t)a.window : 0;
    // the tile's tokens: from its first row's first to its last row's last
    const uint32_t row_a = c0 / a.shared, row_b = min(c0 + 15u, count - 1u) / a.shared;
    const int32_t pos_a = (int32_t)(s.length - s.n + row_a), pos_b = (int32_t)(s.length - s.n + row_b);
    const uint32_t low_a = a.window && pos_a + 1 > (int32_t)a.window ? (uint32_t)(pos_a + 1 - (int32_t)a.window) : 0u;
    const uint32_t low_b = a.window && pos_b + 1 > (int32_t)a.window ? (uint32_t)(pos_b + 1 - (int32_t)a.window) : 0u;
    const uint32_t first = low_a & ~31u, end = pos_b < 0 ? first : (uint32_t)pos_b + 1u;   // pos_b < 0: low_a is 0
    const uint32_t steps = (end - first + 31u) / 32u, each = (steps + a.parts - 1u) / a.parts;
    const uint32_t from = min(part * each, steps), to = min(from + each, steps);

    u4_t qf[SETS][WORDS];
    {
        const uint16_t* const x = a.q + (uint64_t)(s.row0 + row) * a.ld_q + (head * a.shared + member) * D;
#pragma unroll
        for (uint32_t c = 0; c < SETS; ++c)
#pragma unroll
            for (uint32_t j = 0; j < WORDS; ++j) qf[c][j] = *(const u4_t*)(x + c * 128u + g * (8u * WORDS) + 8u * j);
    }
    f4_t acc[ROWS];
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j) acc[j] = f4_t{0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), sum = 0.0f;
    const uint8_t* const pages = a.pages + (uint64_t)head * a.geo.piece;
    const uint32_t stride = a.kv_heads * a.geo.piece;

    const uint32_t hold = ((QW_ATTN_TABLE - 1u) << a.geo.page_log2) >> 5;   // steps whose pages LDS holds, where they begin inside one too
    for (uint32_t base = from; base < to; base += hold) {
        const uint32_t stop = min(base + hold, to), first_page = (first + 32u * base) >> a.geo.page_log2;
        const uint32_t last_page = min(first + 32u * stop - 1u, s.length - 1u) >> a.geo.page_log2;
        __syncthreads();
        for (uint32_t p = tid; p <= last_page - first_page; p += 256u) {
            const int32_t page = a.table[(uint64_t)seq * a.ld_table + first_page + p];
            table[p] = (uint32_t)page < a.page_count ? page : 0;
        }
        __syncthreads();
        qw_attn_step<D> now, next;
        if (base + wave < stop) qw_attn_load<D>(a, pages, stride, table, first_page, first + 32u * (base + wave), s.length, i, g, now);
        for (uint32_t step = base + wave; step < stop; step += 4u) {
            const uint32_t t0 = first + 32u * step;
            if (step + 4u < stop) qw_attn_load<D>(a, pages, stride, table, first_page, t0 + 128u, s.length, i, g, next);
            uint32_t far_v = 0, far_k = 0;
#pragma unroll
            for (uint32_t c = 0; c < SETS; ++c) {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) far_v = max(far_v, ((now.v_scale[c][e >> 2] >> (8u * (e & 3u))) & 0xFFu) - QW_ATTN_F16_LEAST);
                far_k = max(far_k, max(now.k_scale[0][c], now.k_scale[1][c]) - (DT == QWHIP_F16 ? QW_ATTN_F16_LEAST : 0u));
                if constexpr (DT == QWHIP_F16) far_k = max(far_k, min(now.k_scale[0][c], now.k_scale[1][c]) - QW_ATTN_F16_LEAST);
            }
            const bool plain = __ballot(far_v > QW_ATTN_F16_MOST - QW_ATTN_F16_LEAST ||
                                        far_k > (DT == QWHIP_F16 ? QW_ATTN_F16_MOST - QW_ATTN_F16_LEAST : QW_ATTN_BF16_MOST)) == 0ull;
            f4_t score[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};
            if (plain) {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t c = 0; c < SETS; ++c) {
                        const float unit = __uint_as_float(now.k_scale[h][c] << 23);
#pragma unroll
                        for (uint32_t j = 0; j < WORDS; ++j) score[h] = qw_attn_mfma<DT>(qw_attn_operand<DT>(now.k[h][c][j], unit), qf[c][j], score[h]);
                    }
            } else {
                // keys in bf16, which holds every element; f16 queries as two bf16 numbers, which hold their eleven bits
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t c = 0; c < SETS; ++c) {
                        const uint32_t byte = now.k_scale[h][c];
                        const float unit = __uint_as_float((byte > QW_ATTN_BF16_MOST ? 127u : byte) << 23);
#pragma unroll
                        for (uint32_t j = 0; j < WORDS; ++j) {
                            u4_t k = qw_attn_operand<QWHIP_BF16>(now.k[h][c][j], unit);
                            if (byte > QW_ATTN_BF16_MOST) k = u4_t{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
                            if constexpr (DT == QWHIP_BF16) {
                                score[h] = qw_attn_mfma<QWHIP_BF16>(k, qf[c][j], score[h]);
                            } else {
                                u4_t hi, lo;
                                const h8_t x = __builtin_bit_cast(h8_t, qf[c][j]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float x0 = (float)x[2 * e], x1 = (float)x[2 * e + 1];
                                    const uint32_t h0 = __float_as_uint(x0) & 0xFFFF0000u, h1 = __float_as_uint(x1) & 0xFFFF0000u;
                                    hi[e] = (h0 >> 16) | h1;
                                    // an infinity's or a NaN's rest is zero
                                    const float l0 = (h0 & 0x7F800000u) == 0x7F800000u ? 0.0f : x0 - __uint_as_float(h0);
                                    const float l1 = (h1 & 0x7F800000u) == 0x7F800000u ? 0.0f : x1 - __uint_as_float(h1);
                                    lo[e] = (__float_as_uint(l0) >> 16) | (__float_as_uint(l1) & 0xFFFF0000u);
                                }
                                score[h] = qw_attn_mfma<QWHIP_BF16>(k, lo, score[h]);
                                score[h] = qw_attn_mfma<QWHIP_BF16>(k, hi, score[h]);
                            }
                        }
                    }
            }
            // masks where a column of the tile does not see the whole step
            uint32_t seen = 0xFFu;
            if ((int32_t)(t0 + 31u) > pos_a || t0 < low_b) {
                seen = 0;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    const int32_t t = (int32_t)(t0 + 8u * g + e);
                    const bool in = t <= pos && t >= low;
                    seen |= in ? 1u << e : 0u;
                    if (!in) score[e >> 2][e & 3u] = -__builtin_inff();
                }
            }
            float most = fmaxf(fmaxf(fmaxf(score[0][0], score[0][1]), fmaxf(score[0][2], score[0][3])), fmaxf(fmaxf(score[1][0], score[1][1]), fmaxf(score[1][2], score[1][3])));
            most = qw_attn_xor_rows<D>(most, true);
            const float larger = fmaxf(top, most), shift = larger == -__builtin_inff() ? 0.0f : larger * a.scale2;
            const float fade = __builtin_amdgcn_exp2f(top * a.scale2 - shift);
            float p[8];
            float add = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[e >> 2][e & 3u], a.scale2, -shift));
                add += p[e];
            }
            sum = sum * fade + add;
            top = larger;
#pragma unroll
            for (uint32_t j = 0; j < ROWS; ++j) acc[j] = acc[j] * fade;
            if (plain) {
                u4_t w;
                {
                    h8_t x;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = (h1_t)p[e];
                    w = __builtin_bit_cast(u4_t, x);
                }
#pragma unroll
                for (uint32_t c = 0; c < SETS; ++c) {
                    uint32_t x[8][4];   // [token][pair of elements]
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const float unit = __uint_as_float(((now.v_scale[c][e >> 2] >> (8u * (e & 3u))) & 0xFFu) << 23);
                        const uint32_t word = D == 64 ? now.v[c][e >> 2][e & 3u] >> (16u * (i >> 3)) : now.v[c][e >> 2][e & 3u];
                        const u4_t o = qw_attn_operand<QWHIP_F16>(word, unit);
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) x[e][j] = o[j];
                    }
#pragma unroll
                    for (uint32_t j = 0; j < (D == 64 ? 2u : 4u); ++j) {
                        u4_t even, odd;
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            even[e] = __builtin_amdgcn_perm(x[2 * e + 1][j], x[2 * e][j], 0x05040100u);
                            odd[e] = __builtin_amdgcn_perm(x[2 * e + 1][j], x[2 * e][j], 0x07060302u);
                        }
                        acc[8 * c + 2 * j] = qw_attn_mfma<QWHIP_F16>(even, w, acc[8 * c + 2 * j]);
                        acc[8 * c + 2 * j + 1] = qw_attn_mfma<QWHIP_F16>(odd, w, acc[8 * c + 2 * j + 1]);
                    }
                }
            } else {
                // weights as two bf16 numbers (sixteen bits), values in bf16; a NaN block counts where a row sees its token
                u4_t hi, lo, in;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = qw_attn_bf16x2(p[2 * e], p[2 * e + 1]);
                    lo[e] = qw_attn_bf16x2(p[2 * e] - __uint_as_float(hi[e] << 16), p[2 * e + 1] - __uint_as_float(hi[e] & 0xFFFF0000u));
                    in[e] = ((seen >> (2 * e)) & 1u ? 0x3F80u : 0u) | ((seen >> (2 * e + 1)) & 1u ? 0x3F800000u : 0u);
                }
#pragma unroll
                for (uint32_t c = 0; c < SETS; ++c) {
                    uint32_t x[8][4];
                    u4_t broken = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const uint32_t byte = (now.v_scale[c][e >> 2] >> (8u * (e & 3u))) & 0xFFu;
                        if (byte > QW_ATTN_BF16_MOST) broken[e >> 1] |= (e & 1u) ? 0x3F800000u : 0x3F80u;
                        uint32_t word = D == 64 ? now.v[c][e >> 2][e & 3u] >> (16u * (i >> 3)) : now.v[c][e >> 2][e & 3u];
                        if (byte > QW_ATTN_BF16_MOST) word = 0u;
                        const u4_t o = qw_attn_operand<QWHIP_BF16>(word, __uint_as_float((byte > QW_ATTN_BF16_MOST ? 127u : byte) << 23));
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) x[e][j] = o[j];
                    }
                    const f4_t bad = qw_attn_mfma<QWHIP_BF16>(broken, in, f4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (uint32_t j = 0; j < (D == 64 ? 2u : 4u); ++j) {
                        u4_t even, odd;
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            even[e] = __builtin_amdgcn_perm(x[2 * e + 1][j], x[2 * e][j], 0x05040100u);
                            odd[e] = __builtin_amdgcn_perm(x[2 * e + 1][j], x[2 * e][j], 0x07060302u);
                        }
                        f4_t& u = acc[8 * c + 2 * j];
                        f4_t& v = acc[8 * c + 2 * j + 1];
                        u = qw_attn_mfma<QWHIP_BF16>(even, hi, qw_attn_mfma<QWHIP_BF16>(even, lo, u));
                        v = qw_attn_mfma<QWHIP_BF16>(odd, hi, qw_attn_mfma<QWHIP_BF16>(odd, lo, v));
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (bad[r] > 0.0f) u[r] = v[r] = __builtin_nanf("");
                    }
                }
            }
            now = next;
        }
    }

    // the four waves' columns, then the tile's rows
    sum = qw_attn_xor_rows<D>(sum, false);
    if (g == 0u) stats[wave][i][0] = top, stats[wave][i][1] = sum;
#pragma unroll
    for (uint32_t j = 0; j < ROWS; ++j)
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t m = 4u * g + r;   // the accumulator's row
            sums[wave][i][D == 64 ? 8u * (m & 7u) + 4u * (m >> 3) + j : 128u * (j >> 3) + 8u * m + (j & 7u)] = acc[j][r];
        }
    __syncthreads();
    const uint32_t mine = tid >> 4, at = (tid & 15u) * ROWS;   // 16 threads a column, ROWS elements each
    if (c0 + mine >= count) return;
    const uint32_t my_row = (c0 + mine) / a.shared, my_head = head * a.shared + (c0 + mine) - my_row * a.shared;
    float best = -__builtin_inff(), total = 0.0f, o[ROWS] = {};
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) best = fmaxf(best, stats[w][mine][0]);
    const float shift = best == -__builtin_inff() ? 0.0f : best * a.scale2;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(stats[w][mine][0] * a.scale2 - shift);
        total += f * stats[w][mine][1];
#pragma unroll
        for (uint32_t e = 0; e < ROWS; ++e) o[e] += f * sums[w][mine][at + e];
    }
    const uint64_t item = (uint64_t)(s.row0 + my_row) * a.q_heads + my_head;
    if (a.parts > 1u) {
        const uint64_t items = (uint64_t)a.rows * a.q_heads, place = part * items + item;
        float* const st = a.part + a.parts * items * D + place * 2u;
        if (at == 0u) st[0] = best, st[1] = total;
#pragma unroll
        for (uint32_t e = 0; e < ROWS; e += 4u) *(f4_t*)(a.part + place * D + at + e) = f4_t{o[e], o[e + 1], o[e + 2], o[e + 3]};
        return;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* const y = a.out + (uint64_t)(s.row0 + my_row) * a.ld_out + my_head * D + at;
#pragma unroll
    for (uint32_t e = 0; e < ROWS; ++e) {
        const float x = o[e] * inv;
        y[e] = DT == QWHIP_F16 ? __builtin_bit_cast(uint16_t, (h1_t)x) : qw_f32_to_bf16(x);
    }
    if (a.lse && at == 0u) a.lse[item] = best == -__builtin_inff() && total == 0.0f ? -__builtin_inff() : best * a.scale + 0.6931471805599453f * __builtin_amdgcn_logf(total);
}

// The parts of a row, joined in their order: a wave a row and head.
template <int DT, int D>
__global__ __launch_bounds__(256) void qw_attn_join_kernel(const qw_attn_args a) {
    constexpr uint32_t E = D / 64u;
    const uint32_t lane = threadIdx.x & 63u, at = blockIdx.x * 4u + (threadIdx.x >> 6), seq = blockIdx.y;
    const qw_attn_seq s = qw_attn_sequence(a, seq);
    const uint32_t row = at / a.q_heads;
    if (row >= s.n) return;
    const uint64_t items = (uint64_t)a.rows * a.q_heads, item = (uint64_t)s.row0 * a.q_heads + at;
    const float* const stats = a.part + a.parts * items * D + item * 2u;
    float best = -__builtin_inff();
    for (uint32_t p = lane; p < a.parts; p += 64u) best = fmaxf(best, stats[p * items * 2u]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor(best, off, 64));
    const float shift = best == -__builtin_inff() ? 0.0f : best * a.scale2;
    float total = 0.0f, o[E] = {};
    for (uint32_t p = 0; p < a.parts; ++p) {
        const float f = __builtin_amdgcn_exp2f(stats[p * items * 2u] * a.scale2 - shift);
        total += f * stats[p * items * 2u + 1u];
        const float* const x = a.part + (p * items + item) * D + lane * E;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) o[e] += f * x[e];
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* const y = a.out + (uint64_t)(s.row0 + row) * a.ld_out + (at - row * a.q_heads) * D + lane * E;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        const float x = o[e] * inv;
        y[e] = DT == QWHIP_F16 ? __builtin_bit_cast(uint16_t, (h1_t)x) : qw_f32_to_bf16(x);
    }
    if (a.lse && lane == 0u) a.lse[item] = best == -__builtin_inff() && total == 0.0f ? -__builtin_inff() : best * a.scale + 0.6931471805599453f * __builtin_amdgcn_logf(total);
}

constexpr uint32_t QW_ATTN_MOST_TILES = 1u << 22;   // of 256 threads, a launch holds under 2^32
static uint64_t qw_attn_tiles(const qwhip_kv_batch* b, uint32_t rows, uint32_t shared) { return ((uint64_t)(b->max_rows < rows ? b->max_rows : rows) * shared + 15u) / 16u; }
// How many parts a call's rows are split into: workgroups for every compute unit four times over, at least two steps a wave.
static uint32_t qw_attn_parts(uint64_t tiles, const qwhip_kv_batch* b, uint32_t window) {
    if (tiles >= 1024u) return 1u;
    const uint32_t longest = window && window < b->max_length && b->max_rows < b->max_length - window ? window + b->max_rows : b->max_length;
    const uint32_t want = (uint32_t)((1024u + tiles - 1u) / tiles), most = (longest + 255u) / 256u;
    return want < most ? want : most ? most : 1u;
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
    const uint64_t tiles = qw_attn_tiles(b, rows, q_heads / cache->kv_heads) * cache->kv_heads * b->seqs;
    const uint32_t parts = qw_attn_parts(tiles, b, window);
    return parts > 1u ? parts * qw_attn_part_bytes(rows, q_heads, cache->head_dim) : 0u;
}

template <int DT, int D>
static void qw_launch_attn(qwhip_stream_t s, const qw_attn_args& a, uint32_t seqs) {
    hipLaunchKernelGGL((qw_attn_stream_kernel<DT, D>), dim3(a.parts * a.kv_heads * a.tiles, seqs), dim3(256), 0, s->stream, a);
    if (a.parts > 1u) hipLaunchKernelGGL((qw_attn_join_kernel<DT, D>), dim3(qwhip_cdiv(a.max_rows * a.q_heads, 4u), seqs), dim3(256), 0, s->stream, a);
}

extern "C" qwhip_status qwhip_kv_attention_mxfp4(qwhip_stream_t s, const qwhip_kv_cache* cache, const qwhip_kv_batch* batch, const void* q, uint32_t dtype,
                                                 uint32_t q_heads, uint32_t ld_q, uint32_t rows, float scale, uint32_t window, void* out, uint32_t ld_out, float* lse,
                                                 void* workspace, uint64_t workspace_bytes) {
    QWHIP_REQUIRE(s);
    const qwhip_status st = qw_attn_check(cache, batch, q_heads, rows);
    if (st != QWHIP_OK) return st;
    const uint32_t d = cache->head_dim;
    if (dtype != QWHIP_F16 && dtype != QWHIP_BF16) return qwhip_fail(QWHIP_E_BAD_SHAPE, "queries must be f16 or bf16, got dtype %u", dtype);
    if (!(scale > 0.0f) || scale > 3.0e38f) return qwhip_fail(QWHIP_E_BAD_SHAPE, "scale must be positive and finite");
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
    const uint64_t tiles = qw_attn_tiles(batch, rows, shared);
    if (tiles * cache->kv_heads > QW_ATTN_MOST_TILES) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows of a sequence do not fit one launch", max_rows);
    QW_ON_DEVICE_OF(s);
    qw_attn_args a = {};
    a.pages = (const uint8_t*)cache->pages;
    a.row_start = batch->row_start, a.lengths = batch->lengths, a.table = batch->block_table;
    a.q = (const uint16_t*)q, a.out = (uint16_t*)out, a.lse = lse, a.part = (float*)workspace;
    a.geo = qw_kv_geometry_of(cache);
    a.page_count = cache->page_count, a.kv_heads = cache->kv_heads, a.ld_table = batch->ld_table, a.max_rows = max_rows, a.max_length = batch->max_length;
    a.rows = rows, a.q_heads = q_heads, a.shared = shared, a.ld_q = ld_q, a.ld_out = ld_out, a.window = window > 0x7FFFFFFFu ? 0u : window;
    a.tiles = (uint32_t)tiles;
    a.scale = scale, a.scale2 = scale * 1.4426950408889634f;
    a.parts = 1;
    if (workspace) {
        a.parts = qw_attn_parts(tiles * cache->kv_heads * batch->seqs, batch, a.window);
        const uint64_t fit = workspace_bytes / qw_attn_part_bytes(rows, q_heads, d);
        if (fit < a.parts) a.parts = fit > 1u ? (uint32_t)fit : 1u;
    }
#define QW_ATTN(DT)                                                          \
    do {                                                                     \
        if (d == 64u) qw_launch_attn<DT, 64>(s, a, batch->seqs);             \
        else if (d == 128u) qw_launch_attn<DT, 128>(s, a, batch->seqs);      \
        else qw_launch_attn<DT, 256>(s, a, batch->seqs);                     \
    } while (0)
    if (dtype == QWHIP_F16) QW_ATTN(QWHIP_F16);
    else QW_ATTN(QWHIP_BF16);
#undef QW_ATTN
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
