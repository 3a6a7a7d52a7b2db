// Between the LM head and the token: penalties for repeated tokens, biases, a grammar's mask, and the token that wins.
#include "qw_mxfp4.h"

// ------------------------------------------------------------------------------------------------
// A workgroup takes a slice of one row's vocabulary.  What the row's history says about a token of the slice is counted in LDS: the
// workgroup reads the whole history (a few kB that stay in the L2) and counts the tokens that fall into its slice - the low half of a
// word how often in the answer, the top bit whether at all.  Integer additions commute: the counts do not depend on the order.  The
// biases of the slice go through a second word per token, the largest entry index + 1: of two entries for a token the later one holds.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t QW_LG_SLICE = 2048, QW_LG_THREADS = 256;

struct qw_logits_args {
    qwhip_logits_rules r;
    const void* logits;
    void* out;
    unsigned long long* keys;
    int32_t* tokens;
    uint32_t n, ld, ld_out, parts;
};

// The bits of a float made monotone; NaN is below everything but a hole (key 0).
__device__ __forceinline__ uint32_t qw_lg_sortable(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    return (u & 0x80000000u) ? ~u : (u ^ 0x80000000u);
}

template <int DT>
__global__ __launch_bounds__(QW_LG_THREADS) void qw_logits_kernel(const qw_logits_args a) {
    __shared__ uint32_t seen[QW_LG_SLICE], biased[QW_LG_SLICE];
    __shared__ unsigned long long best_w[QW_LG_THREADS / 64];
    const uint32_t tid = threadIdx.x, part = blockIdx.x, row = blockIdx.y, lo = part * QW_LG_SLICE, len = min(QW_LG_SLICE, a.n - lo);
    for (uint32_t i = tid; i < QW_LG_SLICE; i += QW_LG_THREADS) seen[i] = 0u, biased[i] = 0u;
    __syncthreads();
    if (a.r.history) {
        const int32_t total = max(0, min(a.r.total_len[row], (int32_t)a.r.ld_history));
        const int32_t prompt = a.r.prompt_len ? a.r.prompt_len[row] : 0;
        const int32_t* h = a.r.history + (uint64_t)row * a.r.ld_history;
        for (int32_t i = (int32_t)tid; i < total; i += (int32_t)QW_LG_THREADS) {
            const uint32_t t = (uint32_t)h[i] - lo;   // a negative token is past every slice
            if (t < len) {
                if (i >= prompt) atomicAdd(&seen[t], 1u);
                atomicOr(&seen[t], 0x80000000u);
            }
        }
    }
    if (a.r.bias_off) {
        const uint32_t from = (uint32_t)max(0, a.r.bias_off[row]), to = min((uint32_t)max(0, a.r.bias_off[row + 1]), a.r.bias_count);
        for (uint32_t e = from + tid; e < to; e += QW_LG_THREADS) {
            const uint32_t t = (uint32_t)a.r.bias_tok[e] - lo;
            if (t < len) atomicMax(&biased[t], e + 1u);
        }
    }
    __syncthreads();
    const float rep = a.r.repetition ? a.r.repetition[row] : 1.0f, pres = a.r.presence ? a.r.presence[row] : 0.0f, freq = a.r.frequency ? a.r.frequency[row] : 0.0f;
    const uint32_t* mask = nullptr;
    if (a.r.allowed) {
        const int32_t at = a.r.allowed_row ? a.r.allowed_row[row] : (int32_t)row;
        if (at >= 0 && (uint32_t)at < a.r.allowed_rows) mask = a.r.allowed + (uint64_t)at * a.r.ld_allowed;
    }
    unsigned long long best = 0ull;
    for (uint32_t i = tid; i < len; i += QW_LG_THREADS) {
        const uint32_t tok = lo + i;
        float l = qw_load_f32<DT>(a.logits, (uint64_t)row * a.ld + tok);
        const uint32_t sn = seen[i], count = sn & 0x7FFFFFFFu;
        if (sn) {
            l = l > 0.0f ? l / rep : l * rep;
            if (count) l = (l - freq * (float)count) - pres;
        }
        if (biased[i]) l = l + a.r.bias_val[biased[i] - 1u];
        if (mask && ((mask[tok >> 5] >> (tok & 31u)) & 1u) == 0u) l = -__builtin_inff();
        const unsigned long long key = ((unsigned long long)qw_lg_sortable(l) << 32) | (uint32_t)~tok;
        best = key > best ? key : best;
        if (a.out) {
            const uint64_t o = (uint64_t)row * a.ld_out + tok;
            if constexpr (DT == QWHIP_F32) ((float*)a.out)[o] = l;
            else if constexpr (DT == QWHIP_F16) ((h1_t*)a.out)[o] = (h1_t)l;
            else ((uint16_t*)a.out)[o] = qw_f32_to_bf16(l);
        }
    }
    if (!a.tokens) return;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor(best, off, 64);
        best = o > best ? o : best;
    }
    if ((tid & 63u) == 0u) best_w[tid >> 6] = best;
    __syncthreads();
    if (tid == 0u) {
        for (uint32_t w = 1; w < QW_LG_THREADS / 64; ++w) best = best_w[w] > best ? best_w[w] : best;
        a.keys[(uint64_t)row * a.parts + part] = best;
    }
}

// The row's token out of its slices' keys; -1 where nothing is above -inf (its key is 0x007FFFFF).
__global__ __launch_bounds__(64) void qw_logits_token_kernel(const unsigned long long* __restrict__ keys, uint32_t parts, int32_t* __restrict__ tokens) {
    unsigned long long best = 0ull;
    for (uint32_t i = threadIdx.x; i < parts; i += 64u) {
        const unsigned long long k = keys[(uint64_t)blockIdx.x * parts + i];
        best = k > best ? k : best;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor(best, off, 64);
        best = o > best ? o : best;
    }
    if (threadIdx.x == 0u) tokens[blockIdx.x] = (uint32_t)(best >> 32) <= 0x007FFFFFu ? -1 : (int32_t)~(uint32_t)best;
}

extern "C" uint64_t qwhip_logits_workspace_bytes(uint32_t rows, uint32_t n) { return (uint64_t)rows * qwhip_cdiv(n, QW_LG_SLICE) * 8u; }

extern "C" qwhip_status qwhip_logits_process(qwhip_stream_t s, const qwhip_logits_rules* rules, const void* logits, uint32_t dtype, uint32_t rows, uint32_t n,
                                             uint32_t ld, void* out, uint32_t ld_out, int32_t* tokens, void* workspace, uint64_t workspace_bytes) {
    QWHIP_REQUIRE(s);
    QWHIP_REQUIRE(rules);
    if (dtype != QWHIP_F32 && dtype != QWHIP_F16 && dtype != QWHIP_BF16) return qwhip_fail(QWHIP_E_BAD_SHAPE, "logits must be f32, f16 or bf16, got dtype %u", dtype);
    if (n == 0 || n >= (1u << 30)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "a row of %u logits", n);
    if (ld == 0) ld = n;
    if (ld_out == 0) ld_out = n;
    if (ld < n || ld_out < n) return qwhip_fail(QWHIP_E_BAD_SHAPE, "row pitches %u, %u under n=%u", ld, ld_out, n);
    if (rows > 65535u) return qwhip_fail(QWHIP_E_BAD_SHAPE, "%u rows do not fit one launch", rows);
    if (rows == 0) return QWHIP_OK;
    QWHIP_REQUIRE(logits);
    if (!out && !tokens) return qwhip_fail(QWHIP_E_NULL, "neither an output nor tokens are asked for");
    const uint32_t size = dtype == QWHIP_F32 ? 4u : 2u;
    if (((uintptr_t)logits | (uintptr_t)out) & (size - 1u)) return qwhip_fail(QWHIP_E_BAD_SHAPE, "logits are not aligned to their elements");
    if (out == logits && ld_out != ld) return qwhip_fail(QWHIP_E_BAD_SHAPE, "in place the row pitches are one (%u, %u)", ld, ld_out);
    if (rules->history && !rules->total_len) return qwhip_fail(QWHIP_E_NULL, "a history needs total_len");
    if (rules->history && rules->ld_history > 0x3FFFFFFFu) return qwhip_fail(QWHIP_E_BAD_SHAPE, "history rows of %u tokens", rules->ld_history);
    if (rules->bias_off && rules->bias_count && (!rules->bias_tok || !rules->bias_val)) return qwhip_fail(QWHIP_E_NULL, "biases need their tokens and values");
    if (rules->allowed && rules->allowed_rows && rules->ld_allowed < qwhip_cdiv(n, 32u))
        return qwhip_fail(QWHIP_E_BAD_SHAPE, "mask rows of %u words for %u tokens", rules->ld_allowed, n);
    if (tokens) {
        QWHIP_REQUIRE(workspace);
        if (workspace_bytes < qwhip_logits_workspace_bytes(rows, n) || ((uintptr_t)workspace & 7u))
            return qwhip_fail(QWHIP_E_BAD_SHAPE, "tokens need an 8-byte aligned workspace of %llu bytes, got %llu", (unsigned long long)qwhip_logits_workspace_bytes(rows, n),
                              (unsigned long long)workspace_bytes);
    }
    QW_ON_DEVICE_OF(s);
    const uint32_t parts = qwhip_cdiv(n, QW_LG_SLICE);
    const qw_logits_args a = {*rules, logits, out, (unsigned long long*)workspace, tokens, n, ld, ld_out, parts};
    const dim3 grid(parts, rows), block(QW_LG_THREADS);
    if (dtype == QWHIP_F32) hipLaunchKernelGGL(qw_logits_kernel<QWHIP_F32>, grid, block, 0, s->stream, a);
    else if (dtype == QWHIP_F16) hipLaunchKernelGGL(qw_logits_kernel<QWHIP_F16>, grid, block, 0, s->stream, a);
    else hipLaunchKernelGGL(qw_logits_kernel<QWHIP_BF16>, grid, block, 0, s->stream, a);
    if (tokens) hipLaunchKernelGGL(qw_logits_token_kernel, dim3(rows), dim3(64), 0, s->stream, (const unsigned long long*)workspace, parts, tokens);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
