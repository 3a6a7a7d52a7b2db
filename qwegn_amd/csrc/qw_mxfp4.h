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
