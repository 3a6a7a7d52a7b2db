// Decode / verify product of 1..16 rows of 16-bit activations with an MXFP4 weight matrix: y[m, n] = sum_k x[m, k] w[n, k].
#include "qw_mxfp4.h"

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));

// 4 x 4 transpose over the four 16-lane rows of a wavefront: lane row g's q[d] goes to lane row d's q[g].
__device__ __forceinline__ void qw_transpose_rows4(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile(
        "s_nop 1\n\tv_permlane32_swap_b32 %0, %2\n\tv_permlane32_swap_b32 %1, %3\n\ts_nop 1\n\t"
        "v_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3\n\ts_nop 1"
        : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
}

// Eight codes as f16 or bf16 operands, unscaled.
template <int DT>
__device__ __forceinline__ u4_t qw_e2m1_operand(uint32_t w) {
    u4_t o;
    if constexpr (DT == QWHIP_F16) {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3));
    } else {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
    }
    return o;
}

template <int DT>
__device__ __forceinline__ f4_t qw_mfma16(u4_t a, u4_t b) {
    const f4_t z = {0.f, 0.f, 0.f, 0.f};
    if constexpr (DT == QWHIP_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), z, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), z, 0, 0, 0);
}

// A workgroup: 16 weight rows, its waves every W-th group of four blocks.  Lane (i, g) loads block g of the four of weight row i; the
// transpose over the lane rows leaves it eight codes of each of the four blocks, so that one matrix instruction contracts one block of 16
// rows and the block's scale multiplies its fp32 sums.  The codes go in as 16-bit floats, exact.
template <int DT>
__global__ __launch_bounds__(1024) void qw_mx_gemv_plain_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t n, uint32_t blocks,
                                                                 uint32_t ld32, const uint16_t* __restrict__ x, uint32_t m, h1_t* __restrict__ y16,
                                                                 float* __restrict__ y32) {
    __shared__ f4_t part[16 * 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, i = lane & 15u, g = lane >> 4;
    const uint32_t row = min(blockIdx.x * 16u + i, n - 1u);
    const uint64_t base = (uint64_t)row * ld32;
    f4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t b = wave * 4u; b < blocks; b += waves * 4u) {
        const uint64_t at = base + min(b + g, blocks - 1u);
        u4_t q = *(const u4_t*)(codes + at * 16u);
        float s = qw_e8m0(scales[at]);
        if (b + g >= blocks) q = u4_t{0, 0, 0, 0}, s = 0.0f;
        uint32_t q0 = q[0], q1 = q[1], q2 = q[2], q3 = q[3];
        qw_transpose_rows4(q0, q1, q2, q3);
        const uint32_t own[4] = {q0, q1, q2, q3};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            u4_t xv = {0, 0, 0, 0};
            if (i < m && b + j < blocks) xv = *(const u4_t*)(x + ((uint64_t)i * blocks + b + j) * 32u + 8u * g);
            const f4_t d = qw_mfma16<DT>(xv, qw_e2m1_operand<DT>(own[j]));
            const float sj = __shfl(s, (int)(16u * j + i), 64);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(sj, d[r], acc[r]);
        }
    }
    part[wave * 64u + lane] = acc;
    __syncthreads();
    if (wave == 0u) {
        for (uint32_t w = 1; w < waves; ++w) acc += part[w * 64u + lane];
        const uint32_t col = blockIdx.x * 16u + i;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t t = 4u * g + r;
            if (col < n && t < m) {
                if (y16) y16[(uint64_t)t * n + col] = (h1_t)acc[r];
                if (y32) y32[(uint64_t)t * n + col] = acc[r];
            }
        }
    }
}

extern "C" qwhip_status qwhip_mxfp4_gemv(qwhip_stream_t s, const qwhip_mxfp4_view* w, const void* x, uint32_t x_dtype, uint32_t m, void* y16, float* y32) {
    QWHIP_REQUIRE(s);
    const qwhip_status st = qwhip_mxfp4_view_validate(w);
    if (st != QWHIP_OK) return st;
    if (x_dtype != QWHIP_F16 && x_dtype != QWHIP_BF16) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMV activations must be f16 or bf16, got dtype %u", x_dtype);
    if (m > 16) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMV takes 1..16 rows, got %u", m);
    if (m == 0) return QWHIP_OK;
    QWHIP_REQUIRE(x);
    if (!y16 && !y32) return qwhip_fail(QWHIP_E_NULL, "GEMV needs y16 or y32");
    if ((uintptr_t)x & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMV activations must be 16-byte aligned");
    if (((uintptr_t)y16 & 1u) || ((uintptr_t)y32 & 3u)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMV output is not aligned to its elements");
    QW_ON_DEVICE_OF(s);
    const uint32_t blocks = w->k / 32u, waves = min(16u, qwhip_cdiv(blocks, 4u));
    const dim3 grid(qwhip_cdiv(w->n, 16u)), block(64u * waves);
#define QW_GEMV(DT)                                                                                                                                  \
    hipLaunchKernelGGL(qw_mx_gemv_plain_kernel<DT>, grid, block, 0, s->stream, (const uint8_t*)w->codes, (const uint8_t*)w->scales, w->n, blocks,    \
                       qw_mxfp4_ld(w) / 32u, (const uint16_t*)x, m, (h1_t*)y16, y32)
    if (x_dtype == QWHIP_F16) QW_GEMV(QWHIP_F16);
    else QW_GEMV(QWHIP_BF16);
#undef QW_GEMV
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
