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

// Eight codes as f16 or bf16 operands, times the power of two `scale`.
template <int DT>
__device__ __forceinline__ u4_t qw_e2m1_operand(uint32_t w, float scale) {
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
__device__ __forceinline__ f4_t qw_mfma16(u4_t a, u4_t b, f4_t c) {
    if constexpr (DT == QWHIP_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

// A workgroup keeps x in LDS (all of it, or chunk after chunk) and takes tiles of 16 weight rows, a tile's columns dealt to `ways` waves in
// steps of 16 blocks (512 columns).  Lane (i, g) has blocks g, 4 + g, 8 + g, 12 + g of a step of weight row i and the step's 16 scales of
// that row, a step ahead of their use.
// The scaled elements are numbers of x's type where the scale is 2^-13 .. 2^13 (f16: normal numbers then) or at most 2^125 (bf16: 6 x 2^126 is
// past its range).  Where a wave's step has all of its scales there, a lane turns its block into four operands and the matrix unit contracts
// them with the same columns of x.  Otherwise the codes go in unscaled.  A transpose over the lane rows leaves a lane eight codes of each of
// four blocks; a matrix instruction then contracts one block, and the block's scale multiplies its fp32 sums.  (A block's instructions: 22 the
// first way, 54 the second.)
// Bound by the weights' bytes on long banks (151936 x 5120, one row: 74 .. 75 us = 5.5 TB/s; eight times the rows, 3.3 GB that no cache holds,
// 568 us = 5.8 TB/s), by start and end of the launch on shorter ones (17408 x 5120: 13.0 us = 3.6 TB/s from memory, 11.3 where the last-level
// cache has the bank).  x straight from memory instead of LDS, four of its lines for one of weights, took 14.7 and 114 us.  Eight f16 rows of
// 17408 columns pass x through LDS once for 32 weight rows: 21.2 us from memory, 17.5 from the cache (19.3 with every step unscaled).
constexpr uint32_t QW_MX_GEMV_STEP = 16, QW_MX_GEMV_AHEAD = 4, QW_MX_F16_LEAST = 114, QW_MX_F16_MOST = 140, QW_MX_BF16_MOST = 252;
struct qw_mx_gemv_load {   // what a lane carries of a step of weights
    u4_t q[4], sc;
};
template <bool TAIL>
__device__ __forceinline__ void qw_mx_gemv_fetch(uint32_t blocks, const uint8_t* crow, const uint8_t* srow, uint32_t b, uint32_t g, qw_mx_gemv_load& l) {
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t at = b + 4u * u + g;
        l.q[u] = *(const u4_t*)(crow + (TAIL ? min(at, blocks - 1u) : at) * 16u);
        if (TAIL && at >= blocks) l.q[u] = u4_t{0, 0, 0, 0};
    }
    if constexpr (!TAIL) {
        __builtin_memcpy(&l.sc, srow + b, 16);
    } else {
        l.sc = u4_t{0, 0, 0, 0};
        for (uint32_t k = 0; k < 16u && b + k < blocks; ++k) {
            const uint32_t v = (uint32_t)srow[b + k] << (8u * (k & 3u));
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) l.sc[u] |= (k >> 2) == u ? v : 0u;
        }
    }
}
// The scale of byte k of a word, times one, by the conversion itself (it reads the exponent field and knows both ends).
__device__ __forceinline__ float qw_mx_scale(uint32_t word, uint32_t shift) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(0x22u, __uint_as_float(((word >> shift) & 0xFFu) << 23), 0)[0];
}
// `xrow`: row i of x in LDS from the step's first column on.
template <int DT>
__device__ __forceinline__ void qw_mx_gemv_multiply(const qw_mx_gemv_load& l, const uint8_t* xrow, uint32_t g, f4_t (&acc)[2]) {
    uint32_t byte[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) byte[u] = (l.sc[u] >> (8u * g)) & 0xFFu;
    constexpr uint32_t LEAST = DT == QWHIP_F16 ? QW_MX_F16_LEAST : 0u, MOST = DT == QWHIP_F16 ? QW_MX_F16_MOST : QW_MX_BF16_MOST;
    uint32_t far = 0;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) far = max(far, byte[u] - LEAST);
    if (__ballot(far > MOST - LEAST) == 0ull) {
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const float s = __uint_as_float(byte[u] << 23);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)   // columns 8 j .. of the lane's own block
                acc[j & 1] = qw_mfma16<DT>(*(const u4_t*)(xrow + (4u * u + g) * 64u + 16u * j), qw_e2m1_operand<DT>(l.q[u][j], s), acc[j & 1]);
        }
        return;
    }
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
        uint32_t q0 = l.q[u][0], q1 = l.q[u][1], q2 = l.q[u][2], q3 = l.q[u][3];
        qw_transpose_rows4(q0, q1, q2, q3);
        const uint32_t own[4] = {q0, q1, q2, q3};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {   // columns 8 g .. of block j
            const f4_t d = qw_mfma16<DT>(*(const u4_t*)(xrow + (4u * u + j) * 64u + 16u * g), qw_e2m1_operand<DT>(own[j], 1.0f), f4_t{0.f, 0.f, 0.f, 0.f});
            const float s = qw_mx_scale(l.sc[u], 8u * j);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j & 1][r] = __builtin_fmaf(s, d[r], acc[j & 1][r]);
        }
    }
}

struct qw_mx_gemv_args {
    const uint8_t* codes;
    const uint8_t* scales;
    const uint16_t* x;
    h1_t* y16;
    float* y32;
    uint32_t n, blocks, ld32, m;
    uint32_t row_tiles, ways;   // waves of a workgroup: row_tiles tiles of 16 weight rows x ways ranges of the columns
    uint32_t chunk, chunks;     // steps of x that LDS holds at a time; how many times
    uint32_t group;             // rows of x that a workgroup takes, blockIdx.y its group
};

template <int DT, bool CHUNKED>
__global__ __launch_bounds__(1024) void qw_mx_gemv_kernel(const qw_mx_gemv_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t qw_gemv_lds[];
    const uint32_t tid = threadIdx.x, threads = blockDim.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), i = lane & 15u, g = lane >> 4;
    const uint32_t rt = wave / a.ways, way = wave - rt * a.ways, waves = a.row_tiles * a.ways;
    const uint32_t row_first = blockIdx.y * a.group, m = min(a.group, a.m - row_first);
    const uint16_t* const xg = a.x + (uint64_t)row_first * a.blocks * 32u;
    const uint32_t pitch = a.chunk * 1024u + 16u, buffer = m * pitch;   // rows 16 bytes on in the banks
    f4_t* const part = (f4_t*)(qw_gemv_lds + (CHUNKED ? 2u : 1u) * buffer);
    const uint8_t* const xlds = qw_gemv_lds + min(i, m - 1u) * pitch;   // rows behind the last one: sums that are not stored
    const uint32_t steps = (a.blocks + QW_MX_GEMV_STEP - 1u) / QW_MX_GEMV_STEP, tiles = (a.n + 15u) / 16u;

    // chunk ch of x: pieces of eight columns, zeros behind the last column
    const uint32_t row_pieces = a.chunk * 64u, pieces = m * row_pieces;
    auto piece = [&](uint32_t ch, uint32_t p) {
        const uint32_t row = p / row_pieces, col = p - row * row_pieces + ch * row_pieces;
        u4_t v = {0, 0, 0, 0};
        if (p < pieces && col < a.blocks * 4u) v = *(const u4_t*)(xg + ((uint64_t)row * a.blocks * 32u + col * 8u));
        return v;
    };
    auto place = [&](uint32_t ch, uint32_t p, u4_t v) {
        const uint32_t row = p / row_pieces;
        if (p < pieces) *(u4_t*)(qw_gemv_lds + (ch & 1u) * buffer + row * pitch + (p - row * row_pieces) * 16u) = v;
    };

    qw_mx_gemv_load now, next;
    auto fetch = [&](uint32_t tile, uint32_t step, qw_mx_gemv_load& l) {
        const uint64_t base = (uint64_t)min(tile * 16u + i, a.n - 1u) * a.ld32;
        const uint32_t b = step * QW_MX_GEMV_STEP;
        if (b + QW_MX_GEMV_STEP <= a.blocks) qw_mx_gemv_fetch<false>(a.blocks, a.codes + base * 16u, a.scales + base, b, g, l);
        else qw_mx_gemv_fetch<true>(a.blocks, a.codes + base * 16u, a.scales + base, b, g, l);
    };
    const uint32_t hop = gridDim.x * a.row_tiles;
    uint32_t tile = blockIdx.x * a.row_tiles + rt, flip = 0;
    if (way < steps) fetch(tile, way, now);
    for (uint32_t p0 = 0; p0 < pieces; p0 += threads) place(0, p0 + tid, piece(0, p0 + tid));
    __syncthreads();
    for (uint32_t first = blockIdx.x * a.row_tiles; first < tiles; first += hop, tile += hop) {   // the same count for every wave
        f4_t acc[2] = {};
        for (uint32_t ch = 0; ch < a.chunks; ++ch) {
            u4_t ahead[QW_MX_GEMV_AHEAD];
            if (CHUNKED && ch + 1u < a.chunks) {
#pragma unroll
                for (uint32_t k = 0; k < QW_MX_GEMV_AHEAD; ++k) ahead[k] = piece(ch + 1u, k * threads + tid);
            }
            const uint32_t end = min((ch + 1u) * a.chunk, steps);
            for (uint32_t st = ch * a.chunk + way; st < end; st += a.ways) {
                // the next step's weights, this tile's or the next one's, are on their way while this one's are multiplied
                const bool last = st + a.ways >= steps;
                fetch(last ? tile + hop : tile, last ? way : st + a.ways, next);
                __builtin_amdgcn_sched_barrier(0);
                qw_mx_gemv_multiply<DT>(now, xlds + (ch & 1u) * buffer + (st - ch * a.chunk) * 1024u, g, acc);
                now = next;
            }
            if (CHUNKED && ch + 1u < a.chunks) {
#pragma unroll
                for (uint32_t k = 0; k < QW_MX_GEMV_AHEAD; ++k) place(ch + 1u, k * threads + tid, ahead[k]);
                __syncthreads();
            }
        }
        acc[0] += acc[1];
        part[flip * waves * 64u + wave * 64u + lane] = acc[0];
        __syncthreads();
        if (way == 0u) {
            for (uint32_t w = 1; w < a.ways; ++w) acc[0] += part[flip * waves * 64u + (wave + w) * 64u + lane];
            const uint32_t col = tile * 16u + i;
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t t = 4u * g + r;
                if (col < a.n && t < m) {
                    if (a.y16) a.y16[(uint64_t)(row_first + t) * a.n + col] = (h1_t)acc[0][r];
                    if (a.y32) a.y32[(uint64_t)(row_first + t) * a.n + col] = acc[0][r];
                }
            }
        }
        flip ^= 1u;   // the next tile's sums go beside these: one barrier a tile
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
    const uint32_t blocks = w->k / 32u, tiles = qwhip_cdiv(w->n, 16u), steps = qwhip_cdiv(blocks, QW_MX_GEMV_STEP);
    // 16 waves a compute unit carry what its memory pipe needs in flight: in four workgroups where four copies of x and of the sums fit its
    // LDS, in two, in one (banks in the last-level cache, rows of 5120, 17408 outputs, one row: 12.1 / 12.5 / 13.5 us with 4 / 8 / 16 ways;
    // 17408 -> 5120: 14.6 / 14.1 / 15.2; eight rows of 5120: 39.4 / 16.3 / 16.3).  Past that x passes through LDS in chunks of a step a way, the next one carried in registers.
    const uint64_t row = (uint64_t)steps * 1024u + 16u, lds_bytes = 160u << 10;
    uint64_t lds = 0;
    uint32_t row_tiles = 1, ways = 4, chunk = steps, chunks = 1, group = m;
    for (; ways <= 16u; ways *= 2u) {
        lds = m * row + 2u * min(ways, steps) * 1024u;
        if (lds * (16u / ways) <= lds_bytes) break;
    }
    const bool chunked = ways > 16u;
    if (chunked) {
        // nine and more rows: four tiles a workgroup, unless two groups of rows, each with the weights and two tiles a workgroup, still run in
        // one round of the units (banks in the last-level cache; 9 rows of 8768: 17.9 -> 11.8 us on 20 to 64 fours of tiles, 17.9 .. 20.2 ->
        // 20.8 .. 32.7 on 72 to 160; 16 rows of 17408: 29.7 -> 18.3, then 34.1 .. 37.5 -> 33.7 .. 58.0)
        if (m > 8u && qwhip_cdiv(tiles, 4u) <= 64u) group = (m + 1u) / 2u;
        row_tiles = group > 8u ? 4u : 2u, ways = 16u / row_tiles;
        chunk = ways, chunks = qwhip_cdiv(steps, chunk);
        lds = 2u * group * (chunk * 1024u + 16u) + 16u * 1024u;   // at most 144 KB
    }
    const uint32_t resident = chunked ? tiles : 256u * 16u / ways;   // a workgroup keeps x and walks over tiles
    ways = min(ways, steps);
    const qw_mx_gemv_args a = {(const uint8_t*)w->codes, (const uint8_t*)w->scales, (const uint16_t*)x, (h1_t*)y16, y32, w->n, blocks, qw_mxfp4_ld(w) / 32u, m,
                               row_tiles, ways, chunk, chunks, group};
    const dim3 grid(min(qwhip_cdiv(tiles, row_tiles), resident), qwhip_cdiv(m, group)), block(64u * row_tiles * ways);
    void (*const kernel)(qw_mx_gemv_args) = x_dtype == QWHIP_F16 ? (chunked ? qw_mx_gemv_kernel<QWHIP_F16, true> : qw_mx_gemv_kernel<QWHIP_F16, false>)
                                                                  : (chunked ? qw_mx_gemv_kernel<QWHIP_BF16, true> : qw_mx_gemv_kernel<QWHIP_BF16, false>);
    if (lds > 65536u) QWHIP_TRY_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 << 10));
    hipLaunchKernelGGL(kernel, grid, block, (size_t)lds, s->stream, a);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
