// Logits of a decode step before the sampler: penalties for repeated tokens, a bias, a grammar's bit mask; and the tokens' history.
//
//   x = seen ? (x > 0 ? x / r : x r) : x;   x -= f count + p [count > 0];   x += bias;   x = -inf where the mask forbids the token
//
// One pass, bound by memory: 8 bytes per logit out of place.  What is seldom needed is only read where it is: a lane looks at its four tokens' bits of
// `seen` (1/32 of the logits' bytes) and reads counts only behind a set bit; in place and without a bias the logits themselves are only touched
// behind a set `seen` bit or a cleared `allowed` bit.  Penalised logits are computed in 64 bits and rounded once (they are few).
#include "common.h"

namespace {

struct LogitArgs {
    const float* in;
    float* out;
    long ld, ld_out, ld_bias;
    int vocab, words;
    const int *seen, *counts, *allowed, *allowed_row;
    int n_masks;
    float rep, freq, pres;
    const float *rep_dev, *freq_dev, *pres_dev, *bias;
    int in_place;
};

constexpr int LU = 4;              // float4 groups per thread

template <bool VEC>
__global__ __launch_bounds__(256) void process_logits_kernel(const LogitArgs A) {
    const int b = blockIdx.y;
    const float* in = A.in + (long)b * A.ld;
    float* out = A.out + (long)b * A.ld_out;
    const float* bias = A.bias ? A.bias + (long)b * A.ld_bias : nullptr;
    const uint8_t* seen = A.seen ? (const uint8_t*)(A.seen + (long)b * A.words) : nullptr;
    const int* counts = A.counts ? A.counts + (long)b * A.vocab : nullptr;
    const uint8_t* mask = nullptr;
    if (A.allowed) {
        const int m = A.allowed_row ? A.allowed_row[b] : A.n_masks == 1 ? 0 : b;
        if (m >= 0 && m < A.n_masks) mask = (const uint8_t*)(A.allowed + (long)m * A.words);
    }
    const float r = A.rep_dev ? A.rep_dev[b] : A.rep, f = A.freq_dev ? A.freq_dev[b] : A.freq, pr = A.pres_dev ? A.pres_dev[b] : A.pres;
    auto penal = [&](float x, int v) -> float {            // token v, seen: everything but the mask
        double d = x;
        d = d > 0.0 ? d / (double)r : d * (double)r;
        if (counts) {
            const int n = counts[v];
            d -= (double)f * n + (n > 0 ? (double)pr : 0.0);
        }
        if (bias) d += (double)bias[v];
        return (float)d;
    };
    const int base = blockIdx.x * (256 * 4 * LU) + threadIdx.x * 4;
    uint32_t s4[LU], a4[LU];
#pragma unroll
    for (int u = 0; u < LU; ++u) {
        const int v = base + u * 1024;
        s4[u] = 0; a4[u] = 15;
        if (v < A.vocab) {                                 // (bits of a byte past the vocabulary belong to the row's last word: readable)
            if (seen) s4[u] = (seen[v >> 3] >> (v & 4)) & 15u;
            if (mask) a4[u] = (mask[v >> 3] >> (v & 4)) & 15u;
        }
    }
    float4 x[LU], bb[LU];
    bool full[LU], need[LU];
#pragma unroll
    for (int u = 0; u < LU; ++u) {
        const int v = base + u * 1024;
        full[u] = VEC && v + 4 <= A.vocab;
        need[u] = v < A.vocab && (!A.in_place || bias || (s4[u] & a4[u]));
        bb[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (full[u] && need[u]) {
            x[u] = *(const float4*)(in + v);
            if (bias) bb[u] = *(const float4*)(bias + v);
        }
    }
#pragma unroll
    for (int u = 0; u < LU; ++u) {
        const int v = base + u * 1024;
        if (v >= A.vocab) continue;
        if (full[u]) {
            if (!need[u]) {                                // in place: nothing to compute, perhaps tokens to forbid
                if (a4[u] == 15u) continue;
                if (a4[u] == 0u) { *(float4*)(out + v) = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); continue; }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!((a4[u] >> e) & 1)) out[v + e] = -INFINITY;
                continue;
            }
            float y[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
            const float be[4] = {bb[u].x, bb[u].y, bb[u].z, bb[u].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = ((s4[u] >> e) & 1) ? penal(y[e], v + e) : bias ? y[e] + be[e] : y[e];
                if (!((a4[u] >> e) & 1)) y[e] = -INFINITY;
            }
            *(float4*)(out + v) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            for (int e = 0; e < 4 && v + e < A.vocab; ++e) {
                const bool sn = (s4[u] >> e) & 1, al = (a4[u] >> e) & 1;
                if (!al) out[v + e] = -INFINITY;
                else if (sn) out[v + e] = penal(in[v + e], v + e);
                else if (bias) out[v + e] = in[v + e] + bias[v + e];
                else if (!A.in_place) out[v + e] = in[v + e];
            }
        }
    }
}

// One thread per id.  A prompt repeats its placeholder token thousands of times: the bit is read before the atomic that would set it.
__global__ __launch_bounds__(256) void token_history_kernel(int* __restrict__ seen, int* __restrict__ counts, int vocab, int words,
                                                            const int64_t* __restrict__ ids, long ld, int n, const int* __restrict__ len) {
    const int b = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n || (len && i >= len[b])) return;
    const int64_t v = ids[(long)b * ld + i];
    if (v < 0 || v >= vocab) return;
    int* w = seen + (long)b * words + (v >> 5);
    const int bit = (int)(1u << (v & 31));
    if (!(__hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & bit)) atomicOr(w, bit);
    if (counts) atomicAdd(counts + (long)b * vocab + v, 1);
}

}  // namespace

extern "C" int spacer_token_history_add(int* seen, int* counts, int B, int vocab, const int64_t* ids, long ld, int n, const int* len, spacer_stream_t stream) {
    SP_REQUIRE(vocab > 0 && B >= 0 && n >= 0, SPACER_EINVAL, "token_history_add: B = %d, vocab = %d, n = %d", B, vocab, n);
    if (B == 0 || n == 0) return SPACER_OK;
    SP_REQUIRE(seen && ids, SPACER_EINVAL, "token_history_add: seen and ids required");
    SP_REQUIRE(B <= 65535, SPACER_EINVAL, "token_history_add: %d rows (at most 65535)", B);
    hipLaunchKernelGGL(token_history_kernel, dim3(cdiv(n, 256), B), dim3(256), 0, (hipStream_t)stream, seen, counts, vocab, (vocab + 31) / 32, ids, ld, n, len);
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}

extern "C" int spacer_process_logits(const float* logits, long ld, float* out, long ld_out, int B, int vocab, const int* seen, const int* counts,
                                     float repetition, const float* repetition_dev, float frequency, const float* frequency_dev, float presence,
                                     const float* presence_dev, const float* bias, long ld_bias, const int* allowed, int n_masks,
                                     const int* allowed_row, spacer_stream_t stream) {
    SP_REQUIRE(vocab > 0 && B >= 0, SPACER_EINVAL, "process_logits: B = %d, vocab = %d", B, vocab);
    if (B == 0) return SPACER_OK;
    SP_REQUIRE(logits && out, SPACER_EINVAL, "process_logits: logits and out required");
    SP_REQUIRE(B <= 65535, SPACER_EINVAL, "process_logits: %d rows (at most 65535)", B);
    SP_REQUIRE(repetition_dev || repetition > 0.f, SPACER_EINVAL, "process_logits: repetition penalty %g must be above 0", (double)repetition);
    SP_REQUIRE(seen || !counts, SPACER_EINVAL, "process_logits: counts without seen");
    SP_REQUIRE(counts || !(frequency_dev || presence_dev || frequency != 0.f || presence != 0.f), SPACER_EINVAL, "process_logits: frequency and presence penalties need counts");
    SP_REQUIRE(!allowed || (allowed_row ? n_masks > 0 : (n_masks == 1 || n_masks == B)), SPACER_EINVAL, "process_logits: %d masks for %d rows", n_masks, B);
    const bool in_place = logits == out && ld == ld_out;
    LogitArgs A = {logits, out, ld, ld_out, ld_bias, vocab, (vocab + 31) / 32, seen, counts, allowed, allowed_row, n_masks, repetition, frequency, presence,
                   repetition_dev, frequency_dev, presence_dev, bias, in_place ? 1 : 0};
    const bool vec = (((uintptr_t)logits | (uintptr_t)out | (uintptr_t)bias) & 15) == 0 && ((ld | ld_out | (bias ? ld_bias : 0)) & 3) == 0;
    const dim3 grid(cdiv(vocab, 256 * 4 * LU), B);
    if (vec) hipLaunchKernelGGL(process_logits_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, A);
    else hipLaunchKernelGGL(process_logits_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, A);
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}
