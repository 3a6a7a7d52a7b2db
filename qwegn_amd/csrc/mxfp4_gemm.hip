// Product of two MXFP4 operands, Y[m, n] = X[m, k] . W[n, k]^T, on the scaled fp4 matrix instruction.
#include "qw_mxfp4.h"

// ------------------------------------------------------------------------------------------------
// v_mfma_scale_f32_16x16x128_f8f6f4 contracts 128 columns of 16 rows of each operand: lane (i, g) = (lane & 15, lane >> 4) has the 16
// bytes of block g of row i and its scale byte, which are a block as the container stores it.  D: lane (i, g) has rows 4 g .. 4 g + 3 of
// the first operand in column i of the second.  Taken with W first, so that a lane holds four consecutive columns of Y.
// ------------------------------------------------------------------------------------------------
struct qw_mx_operand {
    const uint8_t* codes;
    const uint8_t* scales;
    uint32_t rows, ld32;   // ld32: blocks from row to row
};

__device__ __forceinline__ void qw_mx_load(const qw_mx_operand& o, uint32_t row, uint32_t block, uint32_t blocks, u4_t& q, uint32_t& s) {
    const uint64_t at = (uint64_t)min(row, o.rows - 1u) * o.ld32 + min(block, blocks - 1u);
    q = *(const u4_t*)(o.codes + at * 16u);
    s = o.scales[at];
    if (block >= blocks) q = u4_t{0, 0, 0, 0}, s = 0;   // behind the last column: zeros under a finite scale
}

__device__ __forceinline__ f4_t qw_mx_mfma(u4_t a, uint32_t sa, u4_t b, uint32_t sb, f4_t c) {
    const i8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

template <int DT>
__device__ __forceinline__ void qw_mx_store(void* y, uint64_t at, float v) {
    if constexpr (DT == QWHIP_F32) ((float*)y)[at] = v;
    else if constexpr (DT == QWHIP_F16) ((h1_t*)y)[at] = (h1_t)v;
    else ((uint16_t*)y)[at] = qw_f32_to_bf16(v);
}

// A wave: 32 x 32 of Y, operands straight from memory.
template <int DT>
__global__ __launch_bounds__(256) void qw_mx_gemm_plain_kernel(qw_mx_operand w, qw_mx_operand x, uint32_t blocks, void* __restrict__ y, uint32_t ldy) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, i = lane & 15u, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * 64u + (wave & 1u) * 32u, m0 = blockIdx.y * 64u + (wave >> 1) * 32u;
    f4_t acc[2][2] = {};
    for (uint32_t b = 0; b < blocks; b += 4u) {
        u4_t qw[2], qx[2];
        uint32_t sw[2], sx[2];
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t) {
            qw_mx_load(w, n0 + 16u * t + i, b + g, blocks, qw[t], sw[t]);
            qw_mx_load(x, m0 + 16u * t + i, b + g, blocks, qx[t], sx[t]);
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[a][c] = qw_mx_mfma(qw[a], sw[a], qx[c], sx[c], acc[a][c]);
    }
#pragma unroll
    for (uint32_t a = 0; a < 2; ++a)
#pragma unroll
        for (uint32_t c = 0; c < 2; ++c)
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t n = n0 + 16u * a + 4u * g + r, m = m0 + 16u * c + i;
                if (n < w.rows && m < x.rows) qw_mx_store<DT>(y, (uint64_t)m * ldy + n, acc[a][c][r]);
            }
}

extern "C" uint64_t qwhip_mxfp4_gemm_workspace_bytes(uint32_t m, uint32_t n, uint32_t k) {
    (void)m, (void)n, (void)k;
    return 0;
}

extern "C" qwhip_status qwhip_mxfp4_gemm(qwhip_stream_t s, const qwhip_mxfp4_view* w, const qwhip_mxfp4_view* x, void* y, uint32_t y_dtype, uint32_t ldy,
                                         void* workspace, uint64_t workspace_bytes) {
    QWHIP_REQUIRE(s);
    (void)workspace, (void)workspace_bytes;
    qwhip_status st = qwhip_mxfp4_view_validate(w);
    if (st != QWHIP_OK) return st;
    if (x != nullptr && x->n == 0 && x->k == w->k) return QWHIP_OK;   // no rows
    st = qwhip_mxfp4_view_validate(x);
    if (st != QWHIP_OK) return st;
    if (w->k != x->k) return qwhip_fail(QWHIP_E_BAD_SHAPE, "the operands have %u and %u columns", w->k, x->k);
    QWHIP_REQUIRE(y);
    if (y_dtype != QWHIP_F32 && y_dtype != QWHIP_F16 && y_dtype != QWHIP_BF16)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMM output must be f32, f16 or bf16, got dtype %u", y_dtype);
    if (ldy == 0) ldy = w->n;
    if (ldy < w->n) return qwhip_fail(QWHIP_E_BAD_SHAPE, "output row pitch %u is under n=%u", ldy, w->n);
    if ((uintptr_t)y & (y_dtype == QWHIP_F32 ? 3u : 1u)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMM output is not aligned to its elements");
    if ((uintptr_t)workspace & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMM workspace must be 16-byte aligned");
    if (x->n > 65535u * 64u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows do not fit one launch", x->n);
    QW_ON_DEVICE_OF(s);
    const qw_mx_operand ow = {(const uint8_t*)w->codes, (const uint8_t*)w->scales, w->n, qw_mxfp4_ld(w) / 32u};
    const qw_mx_operand ox = {(const uint8_t*)x->codes, (const uint8_t*)x->scales, x->n, qw_mxfp4_ld(x) / 32u};
    const dim3 grid(qwhip_cdiv(w->n, 64u), qwhip_cdiv(x->n, 64u)), block(256);
    if (y_dtype == QWHIP_F32) hipLaunchKernelGGL(qw_mx_gemm_plain_kernel<QWHIP_F32>, grid, block, 0, s->stream, ow, ox, w->k / 32u, y, ldy);
    else if (y_dtype == QWHIP_F16) hipLaunchKernelGGL(qw_mx_gemm_plain_kernel<QWHIP_F16>, grid, block, 0, s->stream, ow, ox, w->k / 32u, y, ldy);
    else hipLaunchKernelGGL(qw_mx_gemm_plain_kernel<QWHIP_BF16>, grid, block, 0, s->stream, ow, ox, w->k / 32u, y, ldy);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
