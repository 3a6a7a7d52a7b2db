// Between the LM head and the token: penalties for repeated tokens, biases, a grammar's mask, and the token that wins.
#include "qw_mxfp4.h"

// ------------------------------------------------------------------------------------------------
// A workgroup of 1024 threads takes a slice of one row's vocabulary, E tokens a thread, whose logits are on their way while it looks
// through the row's history (a few kB that stay in the L2) and counts in LDS the tokens that fall into its slice: the low bits of a word how
// often in the answer, the top bit whether at all.  Integer additions commute: the counts do not depend on the order.  Where the row has
// biases the same words then hold the largest index + 1 of a token's entries: of two entries for a token the later one holds.
// Bound by the logits' bytes for a full batch: 256 rows of 151936 fp32, history 2048, 64 masks: 71 us = 4.4 TB/s (82 with cached stores); by
// the work on a token for 16-bit logits, half the bytes in 57 us (a 2-byte load and store a lane); by latency for one row (history 4096):
// 7.3 us with the token's launch.  More tokens a thread pay for a workgroup's chain of loads and the
// history's reading less often (the batch with 1 / 2 / 4 / 8 / 16: 259 / 186 / 124 / 77 / 73 us), fewer leave the row's slices on more
// compute units (one row: 7.3 / 7.6 / 8.1 / 8.8 / 11.5).
// ------------------------------------------------------------------------------------------------
constexpr uint32_t QW_LG_THREADS = 1024;

struct qw_logits_args {
    qwhip_logits_rules r;
    const void* logits;
    void* out;
    unsigned long long* keys;
    int32_t* tokens;
    uint32_t n, ld, ld_out, parts;
};

// A key's token; -1 where nothing is above -inf (whose key is 0x007FFFFF).
__device__ __forceinline__ int32_t qw_lg_token(unsigned long long key) { return (uint32_t)(key >> 32) <= 0x007FFFFFu ? -1 : (int32_t)~(uint32_t)key; }

template <int DT, int E>
__global__ __launch_bounds__(QW_LG_THREADS) void qw_logits_kernel(const qw_logits_args a) {
    constexpr uint32_t SLICE = QW_LG_THREADS * E;
    __shared__ uint32_t word[SLICE];
    __shared__ unsigned long long best_w[QW_LG_THREADS / 64];
    const uint32_t tid = threadIdx.x, part = blockIdx.x, row = blockIdx.y, lo = part * SLICE, len = min(SLICE, a.n - lo);
    float l[E];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) l[e] = qw_load_f32<DT>(a.logits, (uint64_t)row * a.ld + lo + min(tid + e * QW_LG_THREADS, len - 1u));
    const int32_t* const h = a.r.history + (uint64_t)row * a.r.ld_history;
    const int32_t h0 = a.r.history && a.r.ld_history ? h[min(tid, a.r.ld_history - 1u)] : 0;
    const int32_t total = a.r.history ? max(0, min(a.r.total_len[row], (int32_t)a.r.ld_history)) : 0;
    uint32_t from = 0, to = 0;
    if (a.r.bias_off) from = (uint32_t)max(0, a.r.bias_off[row]), to = min((uint32_t)max(0, a.r.bias_off[row + 1u]), a.r.bias_count);
    const uint32_t* mask = nullptr;
    if (a.r.allowed) {
        const int32_t at = a.r.allowed_row ? a.r.allowed_row[row] : (int32_t)row;
        if (at >= 0 && (uint32_t)at < a.r.allowed_rows) mask = a.r.allowed + (uint64_t)at * a.r.ld_allowed;
    }
    uint32_t allowed[E];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) allowed[e] = mask ? mask[(lo + min(tid + e * QW_LG_THREADS, len - 1u)) >> 5] : 0xFFFFFFFFu;
    if (total > 0) {
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) word[tid + e * QW_LG_THREADS] = 0u;
        __syncthreads();
        const int32_t prompt = a.r.prompt_len ? a.r.prompt_len[row] : 0;
        for (int32_t i = (int32_t)tid; i < total; i += (int32_t)QW_LG_THREADS) {
            const uint32_t t = (uint32_t)(i == (int32_t)tid ? h0 : h[i]) - lo;   // a negative token is past every slice
            if (t < len) {
                if (i >= prompt) atomicAdd(&word[t], 1u);
                atomicOr(&word[t], 0x80000000u);
            }
        }
        __syncthreads();
        const float rep = a.r.repetition ? a.r.repetition[row] : 1.0f, pres = a.r.presence ? a.r.presence[row] : 0.0f, freq = a.r.frequency ? a.r.frequency[row] : 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            const uint32_t seen = word[tid + e * QW_LG_THREADS], count = seen & 0x7FFFFFFFu;
            if (seen) {
                l[e] = l[e] > 0.0f ? l[e] / rep : l[e] * rep;
                if (count) l[e] = (l[e] - freq * (float)count) - pres;
            }
        }
    }
    if (from < to) {
        // a thread clears the words that it alone has read
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) word[tid + e * QW_LG_THREADS] = 0u;
        __syncthreads();
        for (uint32_t i = from + tid; i < to; i += QW_LG_THREADS) {
            const uint32_t t = (uint32_t)a.r.bias_tok[i] - lo;
            if (t < len) atomicMax(&word[t], i + 1u);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            const uint32_t entry = word[tid + e * QW_LG_THREADS];
            if (entry) l[e] = l[e] + a.r.bias_val[entry - 1u];
        }
    }
    uint32_t key = 0u, at = 0u;   // a thread's tokens rise: a later one wins by a larger key alone
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        const uint32_t i = tid + e * QW_LG_THREADS, tok = lo + i;
        if (i < len) {
            if (((allowed[e] >> (tok & 31u)) & 1u) == 0u) l[e] = -__builtin_inff();
            const uint32_t k = qw_sortable_f32(l[e]);
            if (k > key) key = k, at = tok;
            if (a.out) {
                const uint64_t o = (uint64_t)row * a.ld_out + tok;
                if constexpr (DT == QWHIP_F32) __builtin_nontemporal_store(l[e], (float*)a.out + o);
                else if constexpr (DT == QWHIP_F16) __builtin_nontemporal_store((h1_t)l[e], (h1_t*)a.out + o);
                else __builtin_nontemporal_store((__bf16)l[e], (__bf16*)a.out + o);
            }
        }
    }
    if (!a.tokens) return;
    unsigned long long best = ((unsigned long long)key << 32) | (uint32_t)~at;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor(best, off, 64);
        best = o > best ? o : best;
    }
    if ((tid & 63u) == 0u) best_w[tid >> 6] = best;
    __syncthreads();
    if (tid == 0u) {
        for (uint32_t w = 1; w < QW_LG_THREADS / 64; ++w) best = best_w[w] > best ? best_w[w] : best;
        if (a.parts == 1u) a.tokens[row] = qw_lg_token(best);
        else a.keys[(uint64_t)row * a.parts + part] = best;
    }
}

// The row's token out of its slices' keys.
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
    if (threadIdx.x == 0u) tokens[blockIdx.x] = qw_lg_token(best);
}

extern "C" uint64_t qwhip_logits_workspace_bytes(uint32_t rows, uint32_t n) { return (uint64_t)rows * qwhip_cdiv(n, QW_LG_THREADS) * 8u; }

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
    // the most tokens a thread that leave two workgroups a compute unit (both sides at the kernel)
    uint32_t each = 16;
    while (each > 1u && (uint64_t)rows * qwhip_cdiv(n, QW_LG_THREADS * each) < 512u) each /= 2u;
    const uint32_t parts = qwhip_cdiv(n, QW_LG_THREADS * each);
    const qw_logits_args a = {*rules, logits, out, (unsigned long long*)workspace, tokens, n, ld, ld_out, parts};
    const dim3 grid(parts, rows), block(QW_LG_THREADS);
#define QW_LG(DT)                                                                                            \
    do {                                                                                                     \
        if (each == 16u) hipLaunchKernelGGL((qw_logits_kernel<DT, 16>), grid, block, 0, s->stream, a);       \
        else if (each == 8u) hipLaunchKernelGGL((qw_logits_kernel<DT, 8>), grid, block, 0, s->stream, a);         \
        else if (each == 4u) hipLaunchKernelGGL((qw_logits_kernel<DT, 4>), grid, block, 0, s->stream, a);    \
        else if (each == 2u) hipLaunchKernelGGL((qw_logits_kernel<DT, 2>), grid, block, 0, s->stream, a);    \
        else hipLaunchKernelGGL((qw_logits_kernel<DT, 1>), grid, block, 0, s->stream, a);                    \
    } while (0)
    if (dtype == QWHIP_F32) QW_LG(QWHIP_F32);
    else if (dtype == QWHIP_F16) QW_LG(QWHIP_F16);
    else QW_LG(QWHIP_BF16);
#undef QW_LG
    if (tokens && parts > 1u)
        hipLaunchKernelGGL(qw_logits_token_kernel, dim3(rows), dim3(64), 0, s->stream, (const unsigned long long*)workspace, parts, tokens);
    QWHIP_TRY_HIP(hipGetLastError());
    return QWHIP_OK;
}
