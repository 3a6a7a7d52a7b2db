// Between the q|k|v projection and the attention: norms of queries and keys head by head, the positions' rotation, the 32-point transform, and
// the keys and values of the same rows into the paged MXFP4 cache.
#include "qw_kv.h"

extern "C" uint64_t qwhip_kv_page_bytes(uint32_t page_size, uint32_t kv_heads, uint32_t head_dim) {
    const bool page = page_size >= 16u && page_size <= 256u && (page_size & (page_size - 1u)) == 0;
    if (!page || kv_heads == 0 || kv_heads > 1024u || (head_dim != 64u && head_dim != 128u && head_dim != 256u)) return 0;
    return (uint64_t)page_size * kv_heads * (head_dim / 16u * 17u);
}

extern "C" qwhip_status qwhip_kv_cache_validate(const qwhip_kv_cache* c) {
    QWHIP_REQUIRE(c);
    const uint64_t page = qwhip_kv_page_bytes(c->page_size, c->kv_heads, c->head_dim);
    if (page == 0)
        return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "a cache needs pages of 16, 32, 64, 128 or 256 tokens, 1 .. 1024 heads of 64, 128 or 256 (page %u, heads %u, head %u)",
                          c->page_size, c->kv_heads, c->head_dim);
    if (c->page_count == 0 || (uint64_t)c->page_count * c->page_size >= (1ull << 31))
        return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "%u pages of %u tokens", c->page_count, c->page_size);
    QWHIP_REQUIRE(c->pages);
    if (c->bytes < page * c->page_count)
        return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "a cache of %u pages needs %llu bytes, has %llu", c->page_count, (unsigned long long)(page * c->page_count),
                          (unsigned long long)c->bytes);
    if ((uintptr_t)c->pages & 15u) return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "pages must be 16-byte aligned");
    return QWHIP_OK;
}

// ------------------------------------------------------------------------------------------------
// A head's elements lie eight to a lane: a quad of lanes holds a block of the transform and of the quantiser, 4 to 32 lanes a head.  Every operation is rounded by
// itself, in a fixed order (the sum is a tree): keys next to a border of the 4-bit grid fall on the side that the definition in fp32 says, from either door and at
// every number of rows. Bound by the bytes: 8192 rows of 40 + 8 heads of 128, bf16: 39 us = 5.3 TB/s (a copy of 4 GiB 4.8); the same rows with their values into the
// cache, all of them transformed, codes, scales and values written: 51 us = 4.9 TB/s; one row: the host's call (3.2 .. 3.6 us on the device).  Steps: the rotation's
// partners loaded and normed a second time 63 us; exchanged between lanes, gammas and table entries once a thread 41; a workgroup has queries, keys or values 39.
// Into the cache: a workgroup a row 76 us, whose values' four-byte words went out through eight L2s; eight rows a workgroup 69; the kinds apart, the transform's
// exchange on its additions 51.
// ------------------------------------------------------------------------------------------------
struct qw_heads_side {
    const void* x;
    void* out;             // the values' output for keys and values of the cache
    const h1_t* gamma;
    uint32_t heads, ld, ld_out;
};
struct qw_heads_args {
    qw_heads_side q, k, v;   // without the cache v has no heads
    const int32_t* position;
    const float* cos_sin;
    const int32_t* slots;
    uint8_t* pages;
    qw_kv_geometry geo;
    uint32_t rows, d, positions, rope, flags, slot_count;
    uint32_t across_log2;    // heads that a workgroup takes side by side
    uint32_t q_groups, k_groups;   // workgroups over a row's query heads, over its keys' (and values')
    float eps, inv_d;
};

// Lane l's value of lane l ^ N.
template <int N>
__device__ __forceinline__ float qw_xor_lane(float v) {
    if constexpr (N == 1) return QW_DPP_F32(v, 0xB1);                       // quad_perm [1,0,3,2]
    else if constexpr (N == 2) return QW_DPP_F32(v, 0x4E);                  // quad_perm [2,3,0,1]
    else if constexpr (N == 4) return QW_DPP_F32(QW_DPP_F32(v, 0x141), 0x1B);   // ^ 7, then ^ 3
    else if constexpr (N == 8) return QW_DPP_F32(QW_DPP_F32(v, 0x140), 0x141);  // ^ 15, then ^ 7
    else return __shfl_xor(v, N, 64);
}
template <int LANES>
__device__ __forceinline__ float qw_sum_lanes(float v) {
    if constexpr (LANES >= 32) v += qw_xor_lane<16>(v);
    if constexpr (LANES >= 16) v += qw_xor_lane<8>(v);
    if constexpr (LANES >= 8) v += qw_xor_lane<4>(v);
    v += qw_xor_lane<2>(v);
    v += qw_xor_lane<1>(v);
    return v;
}

// Eight elements as they are in memory.
template <int DT>
struct qw_raw8 {
    u4_t w[DT == QWHIP_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* x, uint64_t at) {
        if constexpr (DT == QWHIP_F32) w[0] = *(const u4_t*)((const float*)x + at), w[1] = *(const u4_t*)((const float*)x + at + 4);
        else w[0] = *(const u4_t*)((const uint16_t*)x + at);
    }
    __device__ __forceinline__ void floats(float* f) const { qw_load8_f32<DT>(w, 0, f); }
};

// What the head's normed elements are multiplied by.
__device__ __forceinline__ void qw_head_gamma8(const h1_t* gamma, uint32_t at, bool plus_one, float* g) {
    qw_load8_f32<QWHIP_F16>(gamma, at, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = plus_one ? 1.0f + g[i] : g[i];
}
// Eight elements of an output row, streamed.
template <int DT>
__device__ __forceinline__ void qw_head_store8(void* dst, uint64_t at, const float* f) {
    if constexpr (DT == QWHIP_BF16) {
        typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
        b8_t o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (__bf16)f[i];
        __builtin_nontemporal_store(__builtin_bit_cast(u4_t, o), (u4_t*)((uint16_t*)dst + at));
    } else {
        qw_stream8<DT>(dst, at, f);
    }
}

template <int DT, int ODT, int LANES, bool CACHE>
__global__ __launch_bounds__(256) void qw_heads_kernel(const qw_heads_args a) {
    const uint32_t lane = threadIdx.x & (LANES - 1), slot = threadIdx.x / LANES, across = 1u << a.across_log2;
    const uint32_t row = blockIdx.x * ((256u / LANES) >> a.across_log2) + (slot >> a.across_log2);
    if (row >= a.rows) return;   // whole heads leave
    uint32_t token = 0;
    if constexpr (CACHE) {
        token = (uint32_t)a.slots[row];
        if (token >= a.slot_count) return;
    }
    const uint32_t at = lane * 8u, half = a.rope / 2u;
    const bool there = at < a.d, turned = at < a.rope, pairs = (a.flags & QWHIP_HEAD_ROPE_PAIRS) != 0, second = !pairs && at >= half;
    const int other = (int)((threadIdx.x & 63u) + (turned ? second ? 0u - half / 8u : half / 8u : 0u)) * 4;   // the lane of the elements that a lane's turn with
    // queries, keys or values: a workgroup has one of them
    const uint32_t kind = blockIdx.y < a.q_groups ? 0u : !CACHE || blockIdx.y < a.q_groups + a.k_groups ? 1u : 2u;
    const qw_heads_side& side = kind == 0u ? a.q : kind == 1u ? a.k : a.v;
    const uint32_t groups = kind == 0u ? a.q_groups : a.k_groups, stride = groups * across;
    const bool value = CACHE && kind == 2u, rope = turned && !value;
    const uint64_t from = (uint64_t)row * side.ld + at;
    qw_raw8<DT> raw = {};
    auto load = [&](uint32_t head) {
        if (head < side.heads && there) raw.load(side.x, from + head * a.d);
    };
    uint32_t head = (blockIdx.y - (kind == 0u ? 0u : kind == 1u ? a.q_groups : a.q_groups + a.k_groups)) * across + (slot & (across - 1u));
    load(head);
    float c[8], s[8], gamma[8];
    if (rope) {
        const int32_t p = max(0, min(a.position[row], (int32_t)a.positions - 1));
        const float* const t = a.cos_sin + (uint64_t)p * a.rope + (pairs ? at / 2u : second ? at - half : at);
        if (pairs) {
            const f4_t x = *(const f4_t*)t, y = *(const f4_t*)(t + half);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = x[i], s[i] = y[i];
        } else {
            qw_load8_f32<QWHIP_F32>(t, 0, c);
            qw_load8_f32<QWHIP_F32>(t, half, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = second ? s[i] : -s[i];   // a c + b (-s) is a c - b s, bit for bit
        }
    }
    const bool plus_one = (a.flags & QWHIP_HEAD_GAMMA_PLUS_ONE) != 0;
    if (there && side.gamma) qw_head_gamma8(side.gamma, at, plus_one, gamma);
    for (; head < side.heads; head += stride) {
        float v[8];
        raw.floats(v);
        load(head + stride);   // the next head's elements on their way
        if (side.gamma) {
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = v[i] * v[i];
            float sum = ((q[0] + q[4]) + (q[2] + q[6])) + ((q[1] + q[5]) + (q[3] + q[7]));
            sum = qw_sum_lanes<LANES>(sum);
            const float r = 1.0f / sqrtf(sum * a.inv_d + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (v[i] * r) * gamma[i];
        }
        if (a.rope && !pairs && !value) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(other, __builtin_bit_cast(int, v[i])));
            if (rope) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * c[i] + o[i] * s[i];
            }
        } else if (rope) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = v[2 * i], x1 = v[2 * i + 1];
                v[2 * i] = x0 * c[i] - x1 * s[i];
                v[2 * i + 1] = x1 * c[i] + x0 * s[i];
            }
        }
        if (a.flags & (value ? QWHIP_HEAD_FWHT_V : QWHIP_HEAD_FWHT_QK)) qw_fwht32_quad(v, lane);
        if (CACHE && kind != 0u) {
            uint32_t w, byte;
            qw_mxfp4_code8(v, w, byte);
            if (!there) continue;
            uint8_t* const piece = a.pages + ((uint64_t)(token >> a.geo.page_log2) * a.k.heads + head) * a.geo.piece;
            const uint32_t t = token & ((1u << a.geo.page_log2) - 1u), block = lane / 4u, blocks = a.d / 32u;
            if (value) {
                *(uint32_t*)(piece + a.geo.v_codes + (((t / 8u) * (a.d / 8u) + lane) * 8u + t % 8u) * 4u) = w;
                if ((lane & 3u) == 0u) piece[a.geo.v_scales + ((t / 8u) * blocks + block) * 8u + t % 8u] = (uint8_t)byte;
            } else {
                *(uint32_t*)(piece + t * (a.d / 2u) + lane * 4u) = w;
                if ((lane & 3u) == 0u) piece[a.geo.k_scales + t * blocks + block] = (uint8_t)byte;
            }
            if (!side.out) continue;
            qw_e2m1_values8(w, qw_e8m0(byte), v);
        }
        if (there) qw_head_store8<ODT>(side.out, (uint64_t)row * side.ld_out + head * a.d + at, v);
    }
}

template <int DT, int ODT, bool CACHE>
static void qw_launch_heads(qwhip_stream_t s, qw_heads_args& a) {
    const uint32_t lanes = a.d <= 32u ? 4u : a.d <= 64u ? 8u : a.d <= 128u ? 16u : 32u, slots = 256u / lanes, most = a.q.heads > a.k.heads ? a.q.heads : a.k.heads;
    const uint32_t fewer = a.q.heads && a.q.heads < a.k.heads ? a.q.heads : a.k.heads ? a.k.heads : a.q.heads;
    a.inv_d = 1.0f / (float)a.d;
    // Few rows: every head on its own lanes.  Many: heads after each other, so that a row's table entries and the gammas are loaded once; into the cache eight rows
    // a workgroup, whose values' words of eight tokens meet in one L2.
    const bool many = a.rows >= 2048u;
    const uint32_t side_by_side = !many ? most : CACHE ? slots / 8u : fewer, each = !many ? 1u : CACHE ? 4u : most;
    a.across_log2 = 0;
    while ((1u << a.across_log2) < side_by_side && (1u << a.across_log2) < slots) ++a.across_log2;
    const uint32_t across = 1u << a.across_log2, down = slots >> a.across_log2, steps = (a.rows + down - 1u) / down;
    a.q_groups = (a.q.heads + across * each - 1u) / (across * each);
    a.k_groups = (a.k.heads + across * each - 1u) / (across * each);
    const dim3 grid(steps, a.q_groups + a.k_groups * (CACHE ? 2u : 1u)), block(256);
    if (lanes == 8u) hipLaunchKernelGGL((qw_heads_kernel<DT, ODT, 8, CACHE>), grid, block, 0, s->stream, a);
    else if (lanes == 16u) hipLaunchKernelGGL((qw_heads_kernel<DT, ODT, 16, CACHE>), grid, block, 0, s->stream, a);
    else if (lanes == 32u) hipLaunchKernelGGL((qw_heads_kernel<DT, ODT, 32, CACHE>), grid, block, 0, s->stream, a);
    else if constexpr (!CACHE) hipLaunchKernelGGL((qw_heads_kernel<DT, ODT, 4, CACHE>), grid, block, 0, s->stream, a);
}
template <int DT, bool CACHE>
static void qw_launch_heads_to(qwhip_stream_t s, uint32_t out_dtype, qw_heads_args& a) {
    if (out_dtype == QWHIP_F32) qw_launch_heads<DT, QWHIP_F32, CACHE>(s, a);
    else if (out_dtype == QWHIP_F16) qw_launch_heads<DT, QWHIP_F16, CACHE>(s, a);
    else qw_launch_heads<DT, QWHIP_BF16, CACHE>(s, a);
}
template <bool CACHE>
static void qw_launch_heads_from(qwhip_stream_t s, uint32_t dtype, uint32_t out_dtype, qw_heads_args& a) {
    if (dtype == QWHIP_F32) qw_launch_heads_to<QWHIP_F32, CACHE>(s, out_dtype, a);
    else if (dtype == QWHIP_F16) qw_launch_heads_to<QWHIP_F16, CACHE>(s, out_dtype, a);
    else qw_launch_heads_to<QWHIP_BF16, CACHE>(s, out_dtype, a);
}

constexpr uint32_t QW_HEADS_MOST_ROWS = (1u << 24) - 1u;   // a workgroup of 256 threads a row, under 2^32 of them

static bool qw_float_type(uint32_t t) { return t == QWHIP_F32 || t == QWHIP_F16 || t == QWHIP_BF16; }

// One side's rows; fills in the tight pitches.
static qwhip_status qw_heads_check(const char* what, uint32_t heads, uint32_t d, uint32_t dtype, const void* x, uint32_t* ld) {
    if (heads > 65535u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%s: %u heads", what, heads);
    if (heads == 0) return QWHIP_OK;
    if (*ld == 0) *ld = heads * d;
    const uint32_t whole = dtype == QWHIP_F32 ? 4u : 8u;   // elements of 16 bytes
    if (*ld < heads * d || *ld % whole != 0) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%s: row pitch %u must be a multiple of %u elements, at least %u", what, *ld, whole, heads * d);
    if (x == nullptr) return qwhip_fail(QWHIP_E_NULL, "%s is NULL", what);
    if ((uintptr_t)x & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%s must be 16-byte aligned", what);
    return QWHIP_OK;
}
static qwhip_status qw_head_rules_check(const qwhip_head_rules* r, uint32_t d) {
    if (r->flags > 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "head rules: flags %u", r->flags);
    if (((uintptr_t)r->cos_sin | (uintptr_t)r->q_gamma | (uintptr_t)r->k_gamma) & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "head rules need 16-byte aligned tables");
    if (r->q_gamma || r->k_gamma) {
        if (!(r->eps >= 0.0f) || r->eps > 3.4e38f) return qwhip_fail(QWHIP_E_BAD_SHAPE, "head rules: eps must be finite and not negative");
    }
    if (!r->cos_sin) return QWHIP_OK;
    if (!r->position) return qwhip_fail(QWHIP_E_NULL, "a rotation needs positions");
    if (r->rope_dims == 0 || r->rope_dims % 16u != 0 || r->rope_dims > d) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rotated elements of a head of %u", r->rope_dims, d);
    if (r->positions == 0 || r->positions > 0x7FFFFFFFu) return qwhip_fail(QWHIP_E_BAD_SHAPE, "a table of %u positions", r->positions);
    return QWHIP_OK;
}
static void qw_heads_take_rules(qw_heads_args& a, const qwhip_head_rules* r) {
    a.position = r->position;
    a.cos_sin = r->cos_sin;
    a.q.gamma = (const h1_t*)r->q_gamma;
    a.k.gamma = (const h1_t*)r->k_gamma;
    a.positions = r->positions;
    a.rope = r->cos_sin ? r->rope_dims : 0u;
    a.eps = r->eps;
    a.flags = r->flags;
}

extern "C" qwhip_status qwhip_head_norm_rope(qwhip_stream_t s, const qwhip_head_rules* rules, uint32_t rows, uint32_t head_dim, const void* q, uint32_t q_heads,
                                             uint32_t ld_q, const void* k, uint32_t k_heads, uint32_t ld_k, uint32_t dtype, void* q_out, uint32_t ld_q_out,
                                             void* k_out, uint32_t ld_k_out, uint32_t out_dtype) {
    QWHIP_REQUIRE(s);
    QWHIP_REQUIRE(rules);
    if (!qw_float_type(dtype) || !qw_float_type(out_dtype)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "heads must be f32, f16 or bf16, got dtypes %u and %u", dtype, out_dtype);
    if (head_dim == 0 || head_dim % 32u != 0 || head_dim > 256u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "a head of %u elements", head_dim);
    if (rows > QW_HEADS_MOST_ROWS) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows do not fit one launch", rows);
    qwhip_status st = qw_head_rules_check(rules, head_dim);
    if (st != QWHIP_OK) return st;
    if (rules->flags & QWHIP_HEAD_FWHT_V) return qwhip_fail(QWHIP_E_BAD_SHAPE, "there are no values to transform");
    if (rows == 0 || (q_heads == 0 && k_heads == 0)) return QWHIP_OK;
    if ((st = qw_heads_check("q", q_heads, head_dim, dtype, q, &ld_q)) != QWHIP_OK) return st;
    if ((st = qw_heads_check("k", k_heads, head_dim, dtype, k, &ld_k)) != QWHIP_OK) return st;
    if ((st = qw_heads_check("q_out", q_heads, head_dim, out_dtype, q_out, &ld_q_out)) != QWHIP_OK) return st;
    if ((st = qw_heads_check("k_out", k_heads, head_dim, out_dtype, k_out, &ld_k_out)) != QWHIP_OK) return st;
    if ((q_heads && q_out == q && (dtype != out_dtype || ld_q != ld_q_out)) || (k_heads && k_out == k && (dtype != out_dtype || ld_k != ld_k_out)))
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "in place types and row pitches are one");
    QW_ON_DEVICE_OF(s);
    qw_heads_args a = {};
    qw_heads_take_rules(a, rules);
    a.q.x = q, a.q.out = q_out, a.q.heads = q_heads, a.q.ld = ld_q, a.q.ld_out = ld_q_out;
    a.k.x = k, a.k.out = k_out, a.k.heads = k_heads, a.k.ld = ld_k, a.k.ld_out = ld_k_out;
    a.rows = rows;
    a.d = head_dim;
    qw_launch_heads_from<false>(s, dtype, out_dtype, a);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}

extern "C" qwhip_status qwhip_kv_append_mxfp4(qwhip_stream_t s, const qwhip_kv_cache* cache, const qwhip_head_rules* rules, uint32_t rows, const int32_t* slots,
                                              const void* k, uint32_t ld_k, const void* v, uint32_t ld_v, uint32_t dtype, const void* q, uint32_t q_heads, uint32_t ld_q,
                                              void* q_out, uint32_t ld_q_out, uint32_t out_dtype, void* k_values, void* v_values) {
    QWHIP_REQUIRE(s);
    qwhip_status st = qwhip_kv_cache_validate(cache);
    if (st != QWHIP_OK) return st;
    const uint32_t d = cache->head_dim, heads = cache->kv_heads;
    if (!qw_float_type(dtype)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "keys and values must be f32, f16 or bf16, got dtype %u", dtype);
    if ((q_heads || k_values || v_values) && !qw_float_type(out_dtype)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "outputs must be f32, f16 or bf16, got dtype %u", out_dtype);
    if (rows > QW_HEADS_MOST_ROWS) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows do not fit one launch", rows);
    if (rules && (st = qw_head_rules_check(rules, d)) != QWHIP_OK) return st;
    if (rows == 0) return QWHIP_OK;
    QWHIP_REQUIRE(slots);
    if ((st = qw_heads_check("k", heads, d, dtype, k, &ld_k)) != QWHIP_OK) return st;
    if ((st = qw_heads_check("v", heads, d, dtype, v, &ld_v)) != QWHIP_OK) return st;
    if ((st = qw_heads_check("q", q_heads, d, dtype, q, &ld_q)) != QWHIP_OK) return st;
    if ((st = qw_heads_check("q_out", q_heads, d, out_dtype, q_out, &ld_q_out)) != QWHIP_OK) return st;
    if (q_heads && q_out == q && (dtype != out_dtype || ld_q != ld_q_out)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "in place types and row pitches are one");
    if (((uintptr_t)k_values | (uintptr_t)v_values) & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "values must be 16-byte aligned");
    QW_ON_DEVICE_OF(s);
    qw_heads_args a = {};
    if (rules) qw_heads_take_rules(a, rules);
    const uint32_t tight = heads * d;
    a.q.x = q, a.q.out = q_out, a.q.heads = q_heads, a.q.ld = ld_q, a.q.ld_out = ld_q_out;
    a.k.x = k, a.k.out = k_values, a.k.heads = heads, a.k.ld = ld_k, a.k.ld_out = tight;
    a.v.x = v, a.v.out = v_values, a.v.heads = heads, a.v.ld = ld_v, a.v.ld_out = tight;
    a.slots = slots;
    a.pages = (uint8_t*)cache->pages;
    a.geo = qw_kv_geometry_of(cache);
    a.rows = rows;
    a.d = d;
    a.slot_count = cache->page_count * cache->page_size;
    qw_launch_heads_from<true>(s, dtype, q_heads || k_values || v_values ? out_dtype : QWHIP_F16, a);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
