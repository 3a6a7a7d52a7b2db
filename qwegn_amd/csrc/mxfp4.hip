// MXFP4 containers: the check of a view, the writer (weights at load time, activations in front of a product) and the reader.
#include "qw_mxfp4.h"

extern "C" qwhip_status qwhip_mxfp4_view_validate(const qwhip_mxfp4_view* v) {
    QWHIP_REQUIRE(v);
    if (v->n == 0 || v->k == 0 || v->k % 32u != 0)
        return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "MXFP4 needs rows and a multiple of 32 columns (n=%u k=%u)", v->n, v->k);
    const uint32_t ld = qw_mxfp4_ld(v);
    if (ld < v->k || ld % 32u != 0) return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "MXFP4 row pitch %u is not a multiple of 32 from k=%u on", ld, v->k);
    if (v->codes == nullptr || v->scales == nullptr) return qwhip_fail(QWHIP_E_NULL, "MXFP4 view has no codes or no scales");
    const uint64_t codes = (uint64_t)(v->n - 1u) * (ld / 2u) + v->k / 2u, scales = (uint64_t)(v->n - 1u) * (ld / 32u) + v->k / 32u;
    if (v->codes_bytes < codes || v->scales_bytes < scales)
        return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "MXFP4 planes hold %llu and %llu bytes, %llu and %llu needed", (unsigned long long)v->codes_bytes,
                          (unsigned long long)v->scales_bytes, (unsigned long long)codes, (unsigned long long)scales);
    if (((uintptr_t)v->codes & 15u) != 0) return qwhip_fail(QWHIP_E_BAD_WEIGHTS, "MXFP4 codes must be 16-byte aligned");
    return QWHIP_OK;
}

// ------------------------------------------------------------------------------------------------
// Writer.  Scale of a block: with a = max |v|, 2^(floor(log2 a) - 2) (2 = the exponent of e2m1's largest element), not under 2^-127;
// element: v / scale to the nearest e2m1 value, ties to the even code, what is over 6 to 6.  The exponent field of a is
// floor(log2 a) + 127 for a normal a, and a subnormal one ends in the clamp; v / scale is an exact product with a power of two.
// A block that holds an infinity or a NaN has no such scale: byte 255, codes 0, so that all of it reads as NaN.
//
// Four neighbouring lanes share a block, eight elements each: whole lines per load and store, the maximum by two exchanges inside the
// quad (as integers: magnitudes order like their bits, and infinities and NaN stay on top).  Bound by its bytes: 17408 x 5120 bf16 with
// the values, 404 MB, more than half of them written: 64 us = 6.3 TB/s (a copy of 4 GiB 4.7 .. 5.0, a fill 6.9); one row of 5120: 1.4 us on
// the device.
// ------------------------------------------------------------------------------------------------
template <int DT, bool STRIDED, bool VALUES>
__global__ __launch_bounds__(256) void qw_quantize_mxfp4_kernel(const void* __restrict__ src, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                 void* __restrict__ values, uint64_t pieces, uint32_t row_pieces, uint32_t ld) {
    const uint64_t p = (uint64_t)blockIdx.x * 256u + threadIdx.x;   // a piece: eight elements, a quad of them one block
    if (p >= pieces) return;                                         // pieces % 4 == 0: quads stay whole
    uint64_t from = p * 8u;
    if constexpr (STRIDED) {
        const uint64_t row = p / row_pieces;
        from = row * ld + (p - row * row_pieces) * 8u;
    }
    float v[8];
    qw_load8_f32<DT>(src, from, v);
    uint32_t w, byte;
    qw_mxfp4_code8(v, w, byte);
    codes[p] = w;
    if ((threadIdx.x & 3u) == 0u) scales[p >> 2] = (uint8_t)byte;
    if constexpr (VALUES) {
        qw_e2m1_values8(w, qw_e8m0(byte), v);
        qw_stream8<DT>(values, p * 8u, v);
    }
}

template <int DT>
static void qw_launch_quantize_mxfp4(qwhip_stream_t s, const void* src, uint32_t* codes, uint8_t* scales, void* values, uint64_t pieces, uint32_t row_pieces,
                                     uint32_t ld) {
    const dim3 grid((unsigned)((pieces + 255u) / 256u)), block(256);
    const bool strided = ld != row_pieces * 8u;
#define QW_QUANT(S, V) hipLaunchKernelGGL((qw_quantize_mxfp4_kernel<DT, S, V>), grid, block, 0, s->stream, src, codes, scales, values, pieces, row_pieces, ld)
    if (strided) {
        if (values) QW_QUANT(true, true);
        else QW_QUANT(true, false);
    } else {
        if (values) QW_QUANT(false, true);
        else QW_QUANT(false, false);
    }
#undef QW_QUANT
}

extern "C" qwhip_status qwhip_quantize_mxfp4(qwhip_stream_t s, const void* src, uint32_t src_dtype, uint32_t rows, uint32_t k, uint32_t ld, void* codes,
                                             void* scales, void* values) {
    QWHIP_REQUIRE(s);
    if (k == 0 || k % 32u != 0) return qwhip_fail(QWHIP_E_BAD_SHAPE, "MXFP4 needs a multiple of 32 columns, got %u", k);
    if (src_dtype != QWHIP_F32 && src_dtype != QWHIP_F16 && src_dtype != QWHIP_BF16)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "quantizer source must be f32, f16 or bf16, got dtype %u", src_dtype);
    if (ld == 0) ld = k;
    const uint32_t whole = src_dtype == QWHIP_F32 ? 4u : 8u;   // elements of 16 bytes
    if (ld < k || ld % whole != 0) return qwhip_fail(QWHIP_E_BAD_SHAPE, "row pitch %u must be a multiple of %u elements, at least k=%u", ld, whole, k);
    if (rows == 0) return QWHIP_OK;
    QWHIP_REQUIRE(src);
    QWHIP_REQUIRE(codes);
    QWHIP_REQUIRE(scales);
    if (((uintptr_t)src & 15u) || ((uintptr_t)codes & 15u) || ((uintptr_t)values & 15u))
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "quantizer needs a 16-byte aligned source, codes and values");
    const uint64_t pieces = (uint64_t)rows * (k / 8u);
    if (pieces > 0xFFFFFF00u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows of %u columns do not fit one launch", rows, k);
    QW_ON_DEVICE_OF(s);
    if (rows == 1) ld = k;
    if (src_dtype == QWHIP_F32) qw_launch_quantize_mxfp4<QWHIP_F32>(s, src, (uint32_t*)codes, (uint8_t*)scales, values, pieces, k / 8u, ld);
    else if (src_dtype == QWHIP_F16) qw_launch_quantize_mxfp4<QWHIP_F16>(s, src, (uint32_t*)codes, (uint8_t*)scales, values, pieces, k / 8u, ld);
    else qw_launch_quantize_mxfp4<QWHIP_BF16>(s, src, (uint32_t*)codes, (uint8_t*)scales, values, pieces, k / 8u, ld);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}

// ------------------------------------------------------------------------------------------------
// Reader: the values of a bank, [n, k] row-major.  Exact in bf16 and fp32; f16 rounds what its range does not hold.  A lane has eight elements of
// a quarter of a block: whole lines per load and store.  Bound by its bytes: 17408 x 5120 to f16 or bf16, 226 MB, 31.7 us = 7.1 TB/s, mostly
// writes; to fp32, 404 MB, 78 us = 5.2 TB/s.
// ------------------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void qw_dequant_mxfp4_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ out,
                                                                uint64_t pieces, uint32_t row_pieces, uint32_t ld) {
    const uint64_t p = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (p >= pieces) return;
    uint64_t at = p;
    if (ld != row_pieces * 8u) {
        const uint64_t row = p / row_pieces;
        at = row * (ld / 8u) + (p - row * row_pieces);
    }
    float f[8];
    qw_e2m1_values8(codes[at], qw_e8m0(scales[at >> 2]), f);
    qw_stream8<DT>(out, p * 8u, f);
}

extern "C" qwhip_status qwhip_dequant_mxfp4(qwhip_stream_t s, const qwhip_mxfp4_view* v, void* out, uint32_t out_dtype) {
    QWHIP_REQUIRE(s);
    const qwhip_status st = qwhip_mxfp4_view_validate(v);
    if (st != QWHIP_OK) return st;
    QWHIP_REQUIRE(out);
    if ((uintptr_t)out & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "dequant needs a 16-byte aligned output");
    if (out_dtype != QWHIP_F32 && out_dtype != QWHIP_F16 && out_dtype != QWHIP_BF16)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "dequant output must be f32, f16 or bf16, got dtype %u", out_dtype);
    const uint64_t pieces = (uint64_t)v->n * (v->k / 8u);
    if (pieces > 0xFFFFFF00u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows of %u columns do not fit one launch", v->n, v->k);
    QW_ON_DEVICE_OF(s);
    const dim3 grid((unsigned)((pieces + 255u) / 256u)), block(256);
    const uint32_t ld = v->n == 1 ? v->k : qw_mxfp4_ld(v);
#define QW_DEQUANT(DT) \
    hipLaunchKernelGGL(qw_dequant_mxfp4_kernel<DT>, grid, block, 0, s->stream, (const uint32_t*)v->codes, (const uint8_t*)v->scales, out, pieces, v->k / 8u, ld)
    if (out_dtype == QWHIP_F32) QW_DEQUANT(QWHIP_F32);
    else if (out_dtype == QWHIP_F16) QW_DEQUANT(QWHIP_F16);
    else QW_DEQUANT(QWHIP_BF16);
#undef QW_DEQUANT
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
