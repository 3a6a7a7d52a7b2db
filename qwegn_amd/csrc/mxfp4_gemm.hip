// Product of two MXFP4 operands, Y[m, n] = X[m, k] . W[n, k]^T, on the scaled fp4 matrix instruction.
#include <math.h>

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

__device__ __forceinline__ f4_t qw_mx_mfma(u4_t a, uint32_t sa, u4_t b, uint32_t sb, f4_t c) {
    const i8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

template <int DT>
__device__ __forceinline__ void qw_mx_store(void* y, uint64_t at, float v) {
    if constexpr (DT == QWHIP_F32) ((float*)y)[at] = v;
    else if constexpr (DT == QWHIP_F16) ((h1_t*)y)[at] = (h1_t)v;
    else ((__bf16*)y)[at] = (__bf16)v;
}

// ------------------------------------------------------------------------------------------------
// Few tiles: a workgroup owns 32 x 32 of Y and deals the columns to its waves in steps of 16 blocks (512 columns), operands straight from
// memory; the waves' sums meet in LDS in the order of the waves.
// ------------------------------------------------------------------------------------------------
struct qw_mx_rows_load {   // a fragment's blocks g, 4 + g, 8 + g, 12 + g of a step and the step's scales of its row
    u4_t q[4], sc;
};
__device__ __forceinline__ void qw_mx_rows_fetch(const uint8_t* codes, const uint8_t* scales, uint32_t b, uint32_t blocks, uint32_t g, qw_mx_rows_load& l) {
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) l.q[u] = *(const u4_t*)(codes + (uint64_t)min(b + 4u * u + g, blocks - 1u) * 16u);
    if (b + 16u <= blocks) {
        __builtin_memcpy(&l.sc, scales + b, 16);
    } else {   // behind the last block zeros: of both operands, so that what stands there adds 2^-254 times a finite code
        l.sc = u4_t{0, 0, 0, 0};
        for (uint32_t k = 0; k < 16u && b + k < blocks; ++k) {
            const uint32_t v = (uint32_t)scales[b + k] << (8u * (k & 3u));
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) l.sc[u] |= (k >> 2) == u ? v : 0u;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(1024) void qw_mx_gemm_rows_kernel(qw_mx_operand w, qw_mx_operand x, uint32_t blocks, void* __restrict__ y, uint32_t ldy) {
    __shared__ f4_t part[16][4][64];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = blockDim.x >> 6, i = lane & 15u, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * 32u, m0 = blockIdx.y * 32u;
    const uint8_t *codes[4], *scales[4];
#pragma unroll
    for (uint32_t f = 0; f < 4; ++f) {
        const qw_mx_operand& o = f < 2u ? w : x;
        const uint64_t row = (uint64_t)min((f < 2u ? n0 : m0) + 16u * (f & 1u) + i, o.rows - 1u) * o.ld32;
        codes[f] = o.codes + row * 16u, scales[f] = o.scales + row;
    }
    f4_t acc[2][2] = {};
    for (uint32_t b = wave * 16u; b < blocks; b += waves * 16u) {
        qw_mx_rows_load l[4];
#pragma unroll
        for (uint32_t f = 0; f < 4; ++f) qw_mx_rows_fetch(codes[f], scales[f], b, blocks, g, l[f]);
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int c = 0; c < 2; ++c) acc[a][c] = qw_mx_mfma(l[a].q[u], l[a].sc[u] >> (8u * g), l[2 + c].q[u], l[2 + c].sc[u] >> (8u * g), acc[a][c]);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) part[wave][f][lane] = acc[f >> 1][f & 1];
    __syncthreads();
    const uint32_t take = min(waves, 4u);   // the first waves sum the fragments
    if (wave < take)
        for (uint32_t f = wave; f < 4u; f += take) {
            f4_t v = part[0][f][lane];
            for (uint32_t p = 1; p < waves; ++p) v += part[p][f][lane];
            const uint32_t n = n0 + 16u * (f >> 1) + 4u * g, m = m0 + 16u * (f & 1u) + i;
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
                if (n + r < w.rows && m < x.rows) qw_mx_store<DT>(y, (uint64_t)m * ldy + n + r, v[r]);
        }
}

// ------------------------------------------------------------------------------------------------
// The tiled kernel.  A workgroup of WM x WN waves owns a tile of X's rows by W's rows, a wave 16 MF x 16 NF of it, all sums in registers.
// Both operands pass through LDS in stages of 256 columns: a row's 128 bytes as eight pieces of 16 (one block each), piece c of row r at
// place c ^ ((r >> 1) & 7), so that the 16 rows that a fragment read touches lie on all banks.  Scales come in steps of two stages, 16
// bytes of a row: the scales of four fragments' rows in one block column form one word (the matrix instruction picks the byte), transposed
// inside lane quads on their way into LDS.
// 4096 x 17408 x 5120 on 256 x 256 tiles: 190 .. 194 us by card = 3.8 PFLOP/s, the matrix unit busy 48 % of the cycles at the 1.77 GHz that it
// holds under this load (17.3 cycles an instruction, 7.9 PFLOP/s, where nothing else runs), LDS 27 %: a stage's fragments and scales are 204 KB,
// 1170 cycles by the counter, against 2048 of matrix instructions on each of the four SIMDs.  Without the stores 179, without the loads into
// LDS 153.
// ------------------------------------------------------------------------------------------------
template <int N, int I = 0, class F>
__device__ __forceinline__ void qw_static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        qw_static_for<N, I + 1>(f);
    }
}

// c += a . b under bytes OA and OB of the scale words.  Written out so that the sums stay in one set of accumulation registers: a tile's 256
// of them and what else is alive fill the file, and left to itself the compiler moved sums about (250 moves beside 128 of these in the loop).
// Operands come from LDS reads, for which the compiler waits, or from vector instructions, which need the two wait states in front (they
// pass while the unit is busy with the instruction before); sums are written by nothing but these and read behind QW_MX_DRAIN.
template <int OA, int OB>
__device__ __forceinline__ void qw_mx_mfma_at(u4_t a, uint32_t sa, u4_t b, uint32_t sb, f4_t& c) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                 : "+a"(c)
                 : "v"(a), "v"(b), "v"(sa), "v"(sb), "n"(OA & 1), "n"(OB & 1), "n"(OA >> 1), "n"(OB >> 1));
}
// All of a wave's loads and LDS accesses done, then the workgroup's; by builtins, so that the compiler knows that nothing is left to wait for.
#define QW_MX_BARRIER()                                          \
    do {                                                         \
        asm volatile("" ::: "memory");                           \
        __builtin_amdgcn_s_waitcnt(0x0070); /* vmcnt, lgkmcnt */ \
        __builtin_amdgcn_s_barrier();                            \
        asm volatile("" ::: "memory");                           \
    } while (0)
#define QW_MX_DRAIN() asm volatile("s_nop 15\n\ts_nop 15" ::: "memory")   // more wait states than a matrix instruction's result takes

struct qw_mx_tile_args {
    qw_mx_operand w, x;
    void* y;
    uint32_t blocks, ldy, tiles_m, tiles_n;
    uint32_t range;   // stages of a K range (even), blockIdx.y its index: ranges write fp32 planes of m * ldy elements
};

template <int MF, int NF, int WM, int WN>
struct qw_mx_tile {
    static constexpr uint32_t WAVES = WM * WN, THREADS = 64u * WAVES, BM = 16u * MF * WM, BN = 16u * NF * WN, ROWS = BM + BN;
    static constexpr uint32_t GX = (MF + 3) / 4, GW = (NF + 3) / 4, GROUPS = WM * GX + WN * GW;   // groups of four fragments, a wave's own
    static constexpr uint32_t CODES = ROWS * 128u;                    // a stage's codes; two of them, then two steps' scales
    static constexpr uint32_t SCALES = GROUPS * 1024u;
    static constexpr uint32_t STEP = THREADS / 8u;                    // a lane loads 16-byte pieces of rows STEP apart
    static constexpr uint32_t XPIECES = BM / STEP, PIECES = ROWS / STEP;
    static constexpr uint32_t SROWS = (GROUPS + WAVES - 1u) / WAVES;  // rows whose scales of a step a thread carries
    static_assert(BM % STEP == 0 && BN % STEP == 0, "whole pieces");
    static constexpr uint32_t LDS = 2u * (CODES + SCALES);
};

template <int MF, int NF, int WM, int WN, int DT>
__global__ __launch_bounds__(64 * WM * WN, WM * WN / 4) void qw_mx_gemm_tile_kernel(const qw_mx_tile_args a) {
    using T = qw_mx_tile<MF, NF, WM, WN>;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), i = lane & 15u, g = lane >> 4;
    const uint32_t wm = wave % WM, wn = wave / WM;

    // workgroups are dealt to the eight XCDs in turn: an XCD takes a contiguous run of labels, and labels walk bands four tiles tall
    const uint32_t total = a.tiles_m * a.tiles_n, per_xcd = (total + 7u) / 8u, label = (blockIdx.x & 7u) * per_xcd + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per_xcd || label >= total) return;
    const uint32_t band = label / (4u * a.tiles_n), in_band = label - band * 4u * a.tiles_n, tall = min(4u, a.tiles_m - 4u * band);
    // the last tile of a side ends with the operand: the rows that it shares with its neighbour get the same bits from both
    const uint32_t n0 = min((in_band / tall) * T::BN, a.w.rows - T::BN), m0 = min((4u * band + in_band % tall) * T::BM, a.x.rows - T::BM);

    // what a lane loads of a stage: piece c of rows tid / 8 + STEP j, X's rows, then W's
    const uint32_t row0 = tid >> 3, c = (tid & 7u) ^ ((row0 >> 1) & 7u);
    const uint32_t xpitch = a.x.ld32 * 16u, wpitch = a.w.ld32 * 16u, xrow = row0 * xpitch, wrow = row0 * wpitch;
    const uint8_t* const xc = a.x.codes + (uint64_t)m0 * xpitch;
    const uint8_t* const wc = a.w.codes + (uint64_t)n0 * wpitch;
    // the scales that it carries: of row i of fragment f of a group, lanes 4 i + f; a step's 16 bytes
    const uint8_t* sbase[T::SROWS];
    uint32_t srow[T::SROWS], sgroup[T::SROWS];
#pragma unroll
    for (uint32_t t = 0; t < T::SROWS; ++t) {
        const uint32_t grp = min(T::WAVES * t + wave, T::GROUPS - 1u);
        const bool of_x = grp < WM * T::GX;
        const uint32_t gg = of_x ? grp : grp - WM * T::GX, per = of_x ? T::GX : T::GW, span = of_x ? 16u * MF : 16u * NF;
        const uint32_t at = min((gg / per) * span + (gg % per) * 64u + 16u * (lane & 3u) + (lane >> 2), (of_x ? T::BM : T::BN) - 1u);
        sgroup[t] = grp;
        sbase[t] = of_x ? a.x.scales + (uint64_t)m0 * a.x.ld32 : a.w.scales + (uint64_t)n0 * a.w.ld32;
        srow[t] = at * (of_x ? a.x.ld32 : a.w.ld32);
    }

    u4_t sstaged[T::SROWS];
    const uint32_t begin = blockIdx.y * a.range, stages = min(begin + a.range, (a.blocks + 7u) / 8u);   // its stages: begin .. stages - 1
    // 1 KB of a stage from memory into LDS, eight rows of a wave: lane l's 16 bytes land at place l & 7 of row l >> 3
    auto fetch_codes = [&](uint32_t st, uint32_t into, auto j) {
        const uint32_t off = min(st * 8u + c, a.blocks - 1u) * 16u;   // behind the last block: any block, under scales of zero
        constexpr uint32_t J = decltype(j)::value;
        const uint8_t* const from = J < T::XPIECES ? xc + (uint64_t)(T::STEP * J) * xpitch + (xrow + off) : wc + (uint64_t)(T::STEP * (J - T::XPIECES)) * wpitch + (wrow + off);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                         (__attribute__((address_space(3))) void*)(lds + (into & 1u) * T::CODES + (T::STEP * J + 8u * wave) * 128u), 16, 0, 0);
    };
    auto fetch_scales = [&](uint32_t step) {
        const uint32_t b = step * 16u;
        if (b + 16u <= a.blocks) {
#pragma unroll
            for (uint32_t t = 0; t < T::SROWS; ++t) __builtin_memcpy(&sstaged[t], sbase[t] + (srow[t] + b), 16);
        } else {   // behind the last block zeros: of both operands, so that what stands there adds 2^-254 times a finite code
#pragma unroll
            for (uint32_t t = 0; t < T::SROWS; ++t)
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) {
                    uint32_t v = 0;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        if (b + 4u * q + k < a.blocks) v |= (uint32_t)sbase[t][srow[t] + b + 4u * q + k] << (8u * k);
                    sstaged[t][q] = v;
                }
        }
    };
    // word q of lane 4 i + f has the scales of half stage q of row (f, i), a byte for each block column: after the transpose inside the quad
    // it has the scales of block column f, a byte for each fragment
    const uint32_t pick1 = (lane & 1u) ? 0x03070105u : 0x06020400u, pick2 = (lane & 2u) ? 0x03020706u : 0x05040100u;
    auto park_scales = [&](uint32_t step) {
#pragma unroll
        for (uint32_t t = 0; t < T::SROWS; ++t) {
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {   // to [group][half stage][row][block column]
                const uint32_t v = sstaged[t][q], p = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
                const uint32_t u = __builtin_amdgcn_perm(p, v, pick1), r = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xF, 0xF, true);
                *(uint32_t*)(lds + 2u * T::CODES + (step & 1u) * T::SCALES + sgroup[t] * 1024u + q * 256u + lane * 4u) = __builtin_amdgcn_perm(r, u, pick2);
            }
        }
    };
    // a wave's fragments and scales of half a stage: W's fragments are each read again when their matrix instructions are out, the rest twice
    u4_t x[2][MF], w[NF];
    uint32_t sx[2][T::GX], sw[2][T::GW];
    const uint32_t key = (i >> 1) & 7u;   // (row >> 1) & 7 of every fragment's row i: rows of fragments are 16 apart
    const uint32_t xat = (wm * 16u * MF + i) * 128u, wat = (T::BM + wn * 16u * NF + i) * 128u;
    const uint32_t place[2] = {((g ^ key) << 4), (((4u + g) ^ key) << 4)};
    auto read_x = [&](uint32_t st, auto h, auto j) {
        x[decltype(h)::value][decltype(j)::value] = *(const u4_t*)(lds + (st & 1u) * T::CODES + xat + place[decltype(h)::value] + 2048u * decltype(j)::value);
    };
    auto read_w = [&](uint32_t st, auto h, auto j) {
        w[decltype(j)::value] = *(const u4_t*)(lds + (st & 1u) * T::CODES + wat + place[decltype(h)::value] + 2048u * decltype(j)::value);
    };
    const uint32_t sat = 2u * T::CODES + (4u * i + g) * 4u;
    auto read_scales = [&](uint32_t st, auto h) {
        constexpr int H = decltype(h)::value;
        const uint32_t at = sat + ((st >> 1) & 1u) * T::SCALES + (2u * (st & 1u) + H) * 256u;
#pragma unroll
        for (uint32_t q = 0; q < T::GX; ++q) sx[H][q] = *(const uint32_t*)(lds + at + (wm * T::GX + q) * 1024u);
#pragma unroll
        for (uint32_t q = 0; q < T::GW; ++q) sw[H][q] = *(const uint32_t*)(lds + at + (WM * T::GX + wn * T::GW + q) * 1024u);
    };
    f4_t acc[NF][MF];
#pragma unroll
    for (int n = 0; n < NF; ++n)
#pragma unroll
        for (int m = 0; m < MF; ++m) {
            acc[n][m] = f4_t{0.f, 0.f, 0.f, 0.f};
            asm volatile("" : "+a"(acc[n][m]));   // in place before the wait below
        }
    QW_MX_DRAIN();
    auto multiply = [&](auto h, auto n) {
        constexpr int N = decltype(n)::value, H = decltype(h)::value;
        qw_static_for<MF>([&](auto m) {
            constexpr int M = decltype(m)::value;
            qw_mx_mfma_at<N & 3, M & 3>(w[N], sw[H][N >> 2], x[H][M], sx[H][M >> 2], acc[N][M]);
        });
    };

    fetch_scales(begin >> 1);
    qw_static_for<T::PIECES>([&](auto j) { fetch_codes(begin, 0, j); });
    park_scales(begin >> 1);
    fetch_scales(min((begin >> 1) + 1u, (stages - 1u) >> 1));
    QW_MX_BARRIER();
    qw_static_for<T::PIECES>([&](auto j) { fetch_codes(min(begin + 1u, stages - 1u), 1, j); });
    constexpr std::integral_constant<int, 0> H0{};
    constexpr std::integral_constant<int, 1> H1{};
    read_scales(begin, H0);
    qw_static_for<MF>([&](auto j) { read_x(0, H0, j); });
    qw_static_for<NF>([&](auto j) { read_w(0, H0, j); });
    // A stage.  First half: its matrix instructions, the second half's fragments on their way in, the next stage into the other buffer.
    // Second half: the stage after the next one is asked for, the next one's first fragments are on their way in.  Behind the last stage
    // the last one again, into a buffer that nobody reads.
    constexpr int PER = (int)(T::PIECES + NF - 1) / NF, PERX = (MF + NF - 1) / NF;   // beside the MF matrix instructions of a fragment of W
    auto stage = [&](uint32_t st, auto parity) {
        constexpr int P = decltype(parity)::value;
        const uint32_t after = min(st + 2u, stages - 1u), step = st >> 1;
        qw_static_for<NF>([&](auto n) {
            constexpr int N = decltype(n)::value;
            multiply(H0, n);
            if constexpr (N == 0) read_scales(st, H1);
            qw_static_for<PERX>([&](auto k) {
                constexpr int J = N * PERX + decltype(k)::value;
                if constexpr (J < MF) read_x(st, H1, std::integral_constant<int, J>{});
            });
            read_w(st, H1, n);
            __builtin_amdgcn_sched_barrier(0);
        });
        QW_MX_BARRIER();
        qw_static_for<NF>([&](auto n) {
            constexpr int N = decltype(n)::value;
            multiply(H1, n);
            if constexpr (N == 0) read_scales(st + 1u, H0);
            qw_static_for<PERX>([&](auto k) {
                constexpr int J = N * PERX + decltype(k)::value;
                if constexpr (J < MF) read_x(st + 1u, H0, std::integral_constant<int, J>{});
            });
            read_w(st + 1u, H0, n);
            // scales: asked for a step ahead, into LDS here, where no load is under way (a store to LDS waits for the ones into it)
            if constexpr (P == 0 && N == 0) park_scales(step + 1u);
            if constexpr (P == 1 && N == 0) fetch_scales(min(step + 2u, (stages - 1u) >> 1));
            qw_static_for<PER>([&](auto k) {
                constexpr int J = N * PER + decltype(k)::value;
                if constexpr (J < (int)T::PIECES) fetch_codes(after, st, std::integral_constant<int, J>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    for (uint32_t st = begin; st < stages; st += 2u) {
        stage(st, std::integral_constant<int, 0>{});
        if (st + 1u < stages) stage(st + 1u, std::integral_constant<int, 1>{});
    }

    QW_MX_DRAIN();
#pragma unroll
    for (int n = 0; n < NF; ++n)
#pragma unroll
        for (int m = 0; m < MF; ++m) asm volatile("" : "+a"(acc[n][m]));   // not read before the wait above
    // Out through LDS, 16 rows of a wave at a time, so that a row leaves as whole lines: a lane has four columns of one row.
    using E = std::conditional_t<DT == QWHIP_F32, float, std::conditional_t<DT == QWHIP_F16, h1_t, __bf16>>;
    typedef E e4_t __attribute__((ext_vector_type(4)));
    constexpr uint32_t PITCH = 16u * NF * sizeof(E) + 16u, ROW16 = NF * sizeof(E);   // bytes of a row in LDS; its 16-byte pieces
    static_assert(T::WAVES * 16u * PITCH <= T::LDS, "the waves' rows fit the stages' place");
    QW_MX_BARRIER();
    uint8_t* const own = lds + wave * 16u * PITCH;
    const bool pieces = (((uint64_t)a.ldy | n0) * sizeof(E) & 15u) == 0u && ((uintptr_t)a.y & 15u) == 0u;
#pragma unroll
    for (uint32_t m = 0; m < MF; ++m) {
        E* const y = (E*)a.y + (uint64_t)blockIdx.y * a.x.rows * a.ldy + (uint64_t)(m0 + wm * 16u * MF + 16u * m) * a.ldy + (n0 + wn * 16u * NF);
#pragma unroll
        for (uint32_t n = 0; n < NF; ++n) {
            const f4_t v = acc[n][m];
            *(e4_t*)(own + i * PITCH + (16u * n + 4u * g) * sizeof(E)) = e4_t{(E)v[0], (E)v[1], (E)v[2], (E)v[3]};
        }
        if (pieces) {
#pragma unroll
            for (uint32_t k = 0; k < 16u * ROW16 / 64u; ++k) {
                const uint32_t id = 64u * k + lane, r = id / ROW16, p = id % ROW16;
                __builtin_nontemporal_store(*(const u4_t*)(own + r * PITCH + 16u * p), (u4_t*)((uint8_t*)(y + (uint64_t)r * a.ldy) + 16u * p));
            }
        } else {
#pragma unroll 1
            for (uint32_t id = lane; id < 256u * NF; id += 64u) {
                const uint32_t r = id / (16u * NF), p = id % (16u * NF);
                y[(uint64_t)r * a.ldy + p] = *(const E*)(own + r * PITCH + sizeof(E) * p);
            }
        }
    }
}

// Sum of a product's planes in their order, four columns of a row a thread.
template <int DT>
__global__ __launch_bounds__(256) void qw_mx_gemm_planes_kernel(const float* __restrict__ planes, uint32_t ranges, uint32_t m, uint32_t n, uint32_t pitch, void* __restrict__ y,
                                                                 uint32_t ldy) {
    const uint32_t quads = pitch / 4u;
    const uint64_t id = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (id >= (uint64_t)m * quads) return;
    const uint32_t row = (uint32_t)(id / quads), col = (uint32_t)(id - (uint64_t)row * quads) * 4u;
    const float* from = planes + (uint64_t)row * pitch + col;
    f4_t v = *(const f4_t*)from;
    for (uint32_t r = 1; r < ranges; ++r) v += *(const f4_t*)(from + (uint64_t)r * m * pitch);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (col + e < n) qw_mx_store<DT>(y, (uint64_t)row * ldy + col + e, v[e]);
}

template <int MF, int NF, int WM, int WN>
static void qw_mx_launch_tile(qwhip_stream_t s, qw_mx_tile_args a, uint32_t ranges, uint32_t y_dtype) {
    using T = qw_mx_tile<MF, NF, WM, WN>;
    a.tiles_m = qwhip_cdiv(a.x.rows, T::BM), a.tiles_n = qwhip_cdiv(a.w.rows, T::BN);
    const dim3 grid(8u * qwhip_cdiv(a.tiles_m * a.tiles_n, 8u), ranges), block(T::THREADS);
    if (y_dtype == QWHIP_F32) hipLaunchKernelGGL((qw_mx_gemm_tile_kernel<MF, NF, WM, WN, QWHIP_F32>), grid, block, 0, s->stream, a);
    else if (y_dtype == QWHIP_F16) hipLaunchKernelGGL((qw_mx_gemm_tile_kernel<MF, NF, WM, WN, QWHIP_F16>), grid, block, 0, s->stream, a);
    else hipLaunchKernelGGL((qw_mx_gemm_tile_kernel<MF, NF, WM, WN, QWHIP_BF16>), grid, block, 0, s->stream, a);
}

// The forms by what they cost, in microseconds, as measured: a tile on a compute unit `base + per_stage * stages`, where two fit a unit a
// pair of them `base2 + per_stage2 * stages`; the rows kernel 3.5 and for a step (512 columns) 2.5e-3 a workgroup, 0.4 at least.  K ranges
// add the sum's launch and its bytes at 3 TB/s, and run where that still pays: on few tiles of many columns.
struct qw_mx_form {
    uint32_t bm, bn, a_unit;
    float base, per_stage, base2, per_stage2;
};
static const qw_mx_form g_mx_forms[] = {
    {256, 256, 1, 5.0f, 1.65f, 0.0f, 0.0f},
    {256, 192, 1, 4.5f, 1.45f, 0.0f, 0.0f},
    {128, 128, 2, 5.0f, 0.8f, 6.0f, 1.1f},
    {64, 128, 2, 5.0f, 0.65f, 6.0f, 0.75f},
};
constexpr uint32_t QW_MX_FORMS = 4, QW_MX_ROWS_FORM = QW_MX_FORMS;
static void qw_mx_launch_form(qwhip_stream_t s, uint32_t form, const qw_mx_tile_args& a, uint32_t ranges, uint32_t y_dtype) {
    if (form == 0u) qw_mx_launch_tile<4, 8, 4, 2>(s, a, ranges, y_dtype);
    else if (form == 1u) qw_mx_launch_tile<4, 6, 4, 2>(s, a, ranges, y_dtype);
    else if (form == 2u) qw_mx_launch_tile<2, 4, 4, 2>(s, a, ranges, y_dtype);
    else qw_mx_launch_tile<1, 4, 4, 2>(s, a, ranges, y_dtype);
}

struct qw_mx_plan {
    uint32_t form, ranges, range;
};
static uint32_t qw_mx_pitch(uint32_t n) { return (n + 3u) & ~3u; }   // of a plane
static qw_mx_plan qw_mx_choose(uint32_t m, uint32_t n, uint32_t blocks, bool tiles_ok, uint64_t room) {
    const uint32_t stages = qwhip_cdiv(blocks, 8u), steps = qwhip_cdiv(blocks, 16u);
    qw_mx_plan best = {QW_MX_ROWS_FORM, 1u, 0u};
    float least = 3.5f + (float)steps * fmaxf(0.4f, 2.5e-3f * (float)qwhip_cdiv(n, 32u) * (float)qwhip_cdiv(m, 32u));
    for (uint32_t f = 0; f < QW_MX_FORMS && tiles_ok; ++f) {
        const qw_mx_form& t = g_mx_forms[f];
        if (m < t.bm || n < t.bn) continue;
        const uint64_t tiles = (uint64_t)qwhip_cdiv(m, t.bm) * qwhip_cdiv(n, t.bn), plane = (uint64_t)m * qw_mx_pitch(n) * 4u;
        if (tiles > (1u << 22)) continue;   // 2^31 threads
        for (uint32_t want = 1; want <= 16u; ++want) {
            const uint32_t range = (qwhip_cdiv(stages, want) + 1u) & ~1u, ranges = qwhip_cdiv(stages, range);   // whole steps of scales
            if (want > 1u && (ranges != want || ranges * plane > room || tiles * ranges > 512u)) continue;
            const uint64_t a_unit = (tiles * ranges + 255u) / 256u;
            const float one = t.base + t.per_stage * (float)range, two = t.base2 + t.per_stage2 * (float)range;
            float cost = t.a_unit == 1u ? (float)a_unit * one : (float)(a_unit / 2u) * two + (float)(a_unit % 2u) * one;
            if (ranges > 1u) cost += 1.5f + ((float)ranges + 0.5f) * (float)plane / 3e6f;
            if (cost < least) least = cost, best = {f, ranges, range};
        }
    }
    return best;
}

extern "C" uint32_t qwhip_mxfp4_gemm_form(uint32_t m, uint32_t n, uint32_t k, uint64_t workspace_bytes, uint32_t* ranges) {
    const bool some = m != 0 && n != 0 && k != 0 && k % 32u == 0;
    const qw_mx_plan plan = some ? qw_mx_choose(m, n, k / 32u, true, workspace_bytes) : qw_mx_plan{QW_MX_ROWS_FORM, 1u, 0u};
    if (ranges) *ranges = plan.ranges;
    return plan.form;
}

extern "C" uint64_t qwhip_mxfp4_gemm_workspace_bytes(uint32_t m, uint32_t n, uint32_t k) {
    if (m == 0 || n == 0 || k == 0 || k % 32u != 0) return 0;
    const qw_mx_plan plan = qw_mx_choose(m, n, k / 32u, true, ~(uint64_t)0);
    return plan.ranges > 1u ? (uint64_t)plan.ranges * m * qw_mx_pitch(n) * 4u : 0u;
}

extern "C" qwhip_status qwhip_mxfp4_gemm(qwhip_stream_t s, const qwhip_mxfp4_view* w, const qwhip_mxfp4_view* x, void* y, uint32_t y_dtype, uint32_t ldy,
                                         void* workspace, uint64_t workspace_bytes) {
    QWHIP_REQUIRE(s);
    qwhip_status st = qwhip_mxfp4_view_validate(w);
    if (st != QWHIP_OK) return st;
    QWHIP_REQUIRE(x);
    if (w->k != x->k) return qwhip_fail(QWHIP_E_BAD_SHAPE, "the operands have %u and %u columns", w->k, x->k);
    if (x->n == 0) return QWHIP_OK;   // no rows
    st = qwhip_mxfp4_view_validate(x);
    if (st != QWHIP_OK) return st;
    QWHIP_REQUIRE(y);
    if (y_dtype != QWHIP_F32 && y_dtype != QWHIP_F16 && y_dtype != QWHIP_BF16)
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMM output must be f32, f16 or bf16, got dtype %u", y_dtype);
    if (ldy == 0) ldy = w->n;
    if (ldy < w->n) return qwhip_fail(QWHIP_E_BAD_SHAPE, "output row pitch %u is under n=%u", ldy, w->n);
    if ((uintptr_t)y & (y_dtype == QWHIP_F32 ? 3u : 1u)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMM output is not aligned to its elements");
    if ((uintptr_t)workspace & 15u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "GEMM workspace must be 16-byte aligned");
    QW_ON_DEVICE_OF(s);
    const qw_mx_operand ow = {(const uint8_t*)w->codes, (const uint8_t*)w->scales, w->n, qw_mxfp4_ld(w) / 32u};
    const qw_mx_operand ox = {(const uint8_t*)x->codes, (const uint8_t*)x->scales, x->n, qw_mxfp4_ld(x) / 32u};
    const uint32_t blocks = w->k / 32u;
    const bool tiles_ok = ow.ld32 < (1u << 18) && ox.ld32 < (1u << 18);   // 32-bit offsets inside a tile
    const qw_mx_plan plan = qw_mx_choose(x->n, w->n, blocks, tiles_ok, workspace ? workspace_bytes : 0u);
    if (plan.ranges > 1u) {
        const uint32_t pitch = qw_mx_pitch(w->n);
        qw_mx_launch_form(s, plan.form, {ow, ox, workspace, blocks, pitch, 0, 0, plan.range}, plan.ranges, QWHIP_F32);
        const dim3 grid((unsigned)(((uint64_t)x->n * (pitch / 4u) + 255u) / 256u)), block(256);
#define QW_MX_PLANES(DT) \
    hipLaunchKernelGGL(qw_mx_gemm_planes_kernel<DT>, grid, block, 0, s->stream, (const float*)workspace, plan.ranges, x->n, w->n, pitch, y, ldy)
        if (y_dtype == QWHIP_F32) QW_MX_PLANES(QWHIP_F32);
        else if (y_dtype == QWHIP_F16) QW_MX_PLANES(QWHIP_F16);
        else QW_MX_PLANES(QWHIP_BF16);
#undef QW_MX_PLANES
    } else if (plan.form != QW_MX_ROWS_FORM) {
        qw_mx_launch_form(s, plan.form, {ow, ox, y, blocks, ldy, 0, 0, plan.range}, 1, y_dtype);
    } else {
        // slabs of rows that one launch's grid and threads hold: one in all but extreme calls
        constexpr uint32_t SLAB_N = 1u << 26, SLAB_M = 65535u * 32u;
        const dim3 block(64u * min(16u, qwhip_cdiv(blocks, 16u)));
        for (uint64_t n0 = 0; n0 < w->n; n0 += SLAB_N)
            for (uint64_t m0 = 0; m0 < x->n; m0 += SLAB_M) {
                const qw_mx_operand sw = {ow.codes + n0 * ow.ld32 * 16u, ow.scales + n0 * ow.ld32, (uint32_t)min((uint64_t)SLAB_N, w->n - n0), ow.ld32};
                const qw_mx_operand sx = {ox.codes + m0 * ox.ld32 * 16u, ox.scales + m0 * ox.ld32, (uint32_t)min((uint64_t)SLAB_M, x->n - m0), ox.ld32};
                void* const sy = (uint8_t*)y + (m0 * ldy + n0) * (y_dtype == QWHIP_F32 ? 4u : 2u);
                const dim3 grid(qwhip_cdiv(sw.rows, 32u), qwhip_cdiv(sx.rows, 32u));
                if (y_dtype == QWHIP_F32) hipLaunchKernelGGL(qw_mx_gemm_rows_kernel<QWHIP_F32>, grid, block, 0, s->stream, sw, sx, blocks, sy, ldy);
                else if (y_dtype == QWHIP_F16) hipLaunchKernelGGL(qw_mx_gemm_rows_kernel<QWHIP_F16>, grid, block, 0, s->stream, sw, sx, blocks, sy, ldy);
                else hipLaunchKernelGGL(qw_mx_gemm_rows_kernel<QWHIP_BF16>, grid, block, 0, s->stream, sw, sx, blocks, sy, ldy);
            }
    }
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
