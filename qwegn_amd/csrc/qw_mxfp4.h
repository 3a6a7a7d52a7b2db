// MXFP4, shared by its quantiser and its products: 32 elements of e2m1 (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3,
// 4, 6) under one power-of-two scale byte e8m0, 2^(byte - 127), 255 = NaN.
#pragma once
#include "qwhip_common.h"

typedef int i8_t __attribute__((ext_vector_type(8)));
typedef float f2_t __attribute__((ext_vector_type(2)));

// The device of a stream as the current one for the length of a door, the caller's one again behind it.
struct qw_device_scope {
    int before = -1;
    qwhip_status st = QWHIP_OK;
    explicit qw_device_scope(qwhip_stream_t s) {
        int now = -1;
        hipError_t e = hipGetDevice(&now);
        if (e == hipSuccess && now != s->dev->ordinal) {
            e = hipSetDevice(s->dev->ordinal);
            if (e == hipSuccess) before = now;
        }
        st = qwhip_hip_check(e, "hipSetDevice");
    }
    ~qw_device_scope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    qw_device_scope(const qw_device_scope&) = delete;
    qw_device_scope& operator=(const qw_device_scope&) = delete;
};
#define QW_ON_DEVICE_OF(s)          \
    qw_device_scope qw_scope_(s);   \
    if (qw_scope_.st != QWHIP_OK) return qw_scope_.st

static inline uint32_t qw_mxfp4_ld(const qwhip_mxfp4_view* v) { return v->ld ? v->ld : v->k; }

// 2^(byte - 127) as fp32: byte 0 is a subnormal, 255 a NaN.
__device__ __forceinline__ float qw_e8m0(uint32_t byte) {
    const uint32_t bits = byte == 0u ? 0x00400000u : byte << 23;
    return __uint_as_float(byte == 255u ? 0x7FC00000u : bits);
}

__device__ __forceinline__ uint32_t qw_quad_umax(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
}

// Eight values: 16-bit ones streamed past the caches (17408 x 5120 bf16 with values: 67.2 -> 65.5 us); a lane's 32 bytes of fp32 are two stores of
// half lines, which wait in the L2 for each other (dequant of 17408 x 5120: 138 us streamed, 78 this way; quantised with values 135 -> 134).
template <int DT>
__device__ __forceinline__ void qw_stream8(void* dst, uint64_t at, const float* f) {
    if constexpr (DT == QWHIP_F32) {
        qw_store8_f32((float*)dst + at, f);
    } else if constexpr (DT == QWHIP_F16) {
        h8_t o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (h1_t)f[i];
        __builtin_nontemporal_store(o, (h8_t*)((h1_t*)dst + at));
    } else {
        u4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = (uint32_t)qw_f32_to_bf16(f[2 * i]) | ((uint32_t)qw_f32_to_bf16(f[2 * i + 1]) << 16);
        __builtin_nontemporal_store(o, (u4_t*)((uint16_t*)dst + at));
    }
}

// Eight codes of one word, lowest element in the lowest nibble, as what they stand for under `unit`.
__device__ __forceinline__ void qw_e2m1_values8(uint32_t w, float unit, float* f) {
    const f2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    f[0] = a[0] * unit, f[1] = a[1] * unit, f[2] = b[0] * unit, f[3] = b[1] * unit;
    f[4] = c[0] * unit, f[5] = c[1] * unit, f[6] = d[0] * unit, f[7] = d[1] * unit;
}

// The quantiser's rule for eight values of a lane whose quad holds a block (the rule's words stand at the quantiser): their codes, lowest element in the
// lowest nibble, and the block's scale byte.  `v` is scaled.
__device__ __forceinline__ void qw_mxfp4_code8(float* v, uint32_t& w, uint32_t& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    const uint32_t field = qw_quad_umax(top) >> 23;
    const bool broken = field == 255u;
    byte = broken ? 255u : (field > 2u ? field - 2u : 0u);
    const float inverse = __uint_as_float((254u - byte) << 23);      // 2^(127 - byte), byte <= 252 where it is used
    w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = broken ? 0.0f : v[i] * inverse;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
}
