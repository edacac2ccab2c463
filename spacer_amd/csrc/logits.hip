// Logits of a decode step before the sampler: penalties for repeated tokens, a bias, a grammar's bit mask; and the tokens' history.
//
//   x = seen ? (x > 0 ? x / r : x r) : x;   x -= f count + p [count > 0];   x += bias;   x = -inf where the mask forbids the token
//
// One pass, bound by memory: 8 bytes per logit out of place.  What is seldom needed is only read where it is: a lane looks at its four tokens' bits of
// `seen` (1/32 of the logits' bytes) and reads counts only behind a set bit; in place and without a bias the logits themselves are only touched
// behind a set `seen` bit or a cleared `allowed` bit.  Penalised logits are computed in 64 bits and rounded once (they are few).
// Measured, vocabulary 152064, out of place: 64 rows with a bias per row 24.7 us (4.7 TB/s of logits and bias), 128 rows with one bias 37.5 us (4.2 TB/s of
// logits alone, beside the scattered counts), 8 rows 5.6 us.
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
};

constexpr int LU = 4;              // float4 groups per thread
constexpr int MAX_VOCAB = 1 << 30; // (columns and ids of a row are counted in 32 bits)

template <bool VEC, bool IN_PLACE>
__global__ __launch_bounds__(256) void process_logits_kernel(const LogitArgs A) {
    const int b = blockIdx.y;
    const float* in = A.in + (long)b * A.ld;
    float* out = A.out + (long)b * A.ld_out;
    const float* bias = A.bias ? A.bias + (long)b * A.ld_bias : nullptr;
    const uint8_t* seen = A.seen ? (const uint8_t*)(A.seen + (long)b * A.words) : nullptr;
    const int* counts = A.counts ? A.counts + (long)b * A.vocab : nullptr;
    const int base = blockIdx.x * (256 * 4 * LU) + threadIdx.x * 4;
    // out of place every logit is read: first of all, beside the bits
    float4 x[LU], bb[LU];
    uint32_t s4[LU], a4[LU];
    if (VEC && !IN_PLACE) {
#pragma unroll
        for (int u = 0; u < LU; ++u) {
            const int v = base + u * 1024;
            if (v + 4 <= A.vocab) x[u] = *(const float4*)(in + v);
        }
    }
    const uint8_t* mask = nullptr;
    if (A.allowed) {
        const int m = A.allowed_row ? A.allowed_row[b] : A.n_masks == 1 ? 0 : b;
        if (m >= 0 && m < A.n_masks) mask = (const uint8_t*)(A.allowed + (long)m * A.words);
    }
#pragma unroll
    for (int u = 0; u < LU; ++u) {
        const int v = base + u * 1024;
        s4[u] = 0; a4[u] = 15;
        bb[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (v < A.vocab) {                                 // (bits of a byte past the vocabulary belong to the row's last word: readable)
            if (seen) s4[u] = (seen[v >> 3] >> (v & 4)) & 15u;
            if (mask) a4[u] = (mask[v >> 3] >> (v & 4)) & 15u;
            if (VEC && bias && v + 4 <= A.vocab) bb[u] = *(const float4*)(bias + v);
        }
    }
    const double r = A.rep_dev ? A.rep_dev[b] : A.rep, inv_r = 1.0 / r;
    const double f = A.freq_dev ? A.freq_dev[b] : A.freq, pr = A.pres_dev ? A.pres_dev[b] : A.pres;
    auto penal = [&](float xf, int n, float be) -> float { // a seen token with n occurrences in the completion
        double d = xf;
        d *= d > 0.0 ? inv_r : r;
        if (counts) d -= f * n + (n > 0 ? pr : 0.0);
        return (float)(bias ? d + (double)be : d);
    };
    if (VEC && IN_PLACE) {
#pragma unroll
        for (int u = 0; u < LU; ++u) {
            const int v = base + u * 1024;
            if (v + 4 <= A.vocab && (bias || (s4[u] & a4[u]))) x[u] = *(const float4*)(in + v);
        }
    }
    int n4[LU][4];
    if (VEC && counts) {                                   // the counts behind all set bits, in flight together
#pragma unroll
        for (int u = 0; u < LU; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = base + u * 1024 + e;
                n4[u][e] = 0;
                if (((s4[u] & a4[u]) >> e) & 1 && base + u * 1024 + 4 <= A.vocab) n4[u][e] = counts[v];
            }
    }
#pragma unroll
    for (int u = 0; u < LU; ++u) {
        const int v = base + u * 1024;
        if (v >= A.vocab) continue;
        if (VEC && v + 4 <= A.vocab) {
            if (IN_PLACE && !bias && !(s4[u] & a4[u])) {   // nothing to compute, perhaps tokens to forbid
                if (a4[u] == 15u) continue;
                if (a4[u] == 0u) { *(float4*)(out + v) = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); continue; }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!((a4[u] >> e) & 1)) out[v + e] = -INFINITY;
                continue;
            }
            float y[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
            const float be[4] = {bb[u].x, bb[u].y, bb[u].z, bb[u].w};
            if (s4[u] & a4[u]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = penal(y[e], counts ? n4[u][e] : 0, be[e]);
                    y[e] = ((s4[u] >> e) & 1) ? z : bias ? y[e] + be[e] : y[e];
                }
            } else if (bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += be[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!((a4[u] >> e) & 1)) y[e] = -INFINITY;
            *(float4*)(out + v) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            for (int e = 0; e < 4 && v + e < A.vocab; ++e) {
                const bool sn = (s4[u] >> e) & 1, al = (a4[u] >> e) & 1;
                const float be = bias ? bias[v + e] : 0.f;
                if (!al) out[v + e] = -INFINITY;
                else if (sn) out[v + e] = penal(in[v + e], counts ? counts[v + e] : 0, be);
                else if (bias) out[v + e] = in[v + e] + be;
                else if (!IN_PLACE) out[v + e] = in[v + e];
            }
        }
    }
}

// Counts an id per active lane.  Prompts repeat a placeholder token for thousands of positions, and atomics on one address go one by one: lanes that hold
// the same id as the first one share an atomic, then those of the first one left, the others go alone.  (8 rows of 2051
// ids, 7/8 of them the same: 37 us without this, 4.4 with it.)
__device__ __forceinline__ void add_ids(int* counts, int* seen, int v) {
#pragma unroll
    for (int round = 0; round < 3; ++round) {
        const int lead = __builtin_amdgcn_readfirstlane(v);
        const uint64_t same = round < 2 ? __ballot(v == lead) : 0ull;
        if (round < 2 && v != lead) continue;
        if (round == 2 || __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0)) == 0) {
            if (seen) atomicOr(seen + (v >> 5), (int)(1u << (v & 31)));
            if (counts) atomicAdd(counts + v, round < 2 ? (int)__popcll(same) : 1);
        }
        return;
    }
}

// Few ids: one thread each, bits and counts by atomics in memory.
__global__ __launch_bounds__(256) void token_history_kernel(int* __restrict__ seen, int* __restrict__ counts, int vocab, int words,
                                                            const int64_t* __restrict__ ids, long ld, int n, const int* __restrict__ len) {
    const int b = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n || (len && i >= len[b])) return;
    const int64_t v = ids[(long)b * ld + i];
    if (v < 0 || v >= vocab) return;
    add_ids(counts ? counts + (long)b * vocab : nullptr, seen + (long)b * words, (int)v);
}

// Many ids: workgroup 0 of a row collects its bits in LDS and owns the row's words, so that they are merged without atomics; the others count 4096 ids each.
__global__ __launch_bounds__(1024) void token_history_row_kernel(int* __restrict__ seen, int* __restrict__ counts, int vocab, int words,
                                                                 const int64_t* __restrict__ ids, long ld, int n, const int* __restrict__ len) {
    extern __shared__ int bits[];
    const int b = blockIdx.y, part = (int)blockIdx.x - 1;
    const int m = len ? min(n, len[b]) : n;
    if (part < 0) {
        for (int i = threadIdx.x; i < words; i += 1024) bits[i] = 0;
        __syncthreads();
    }
    const int end = part < 0 ? m : min(m, (part + 1) * 4096);
    for (int i0 = max(part, 0) * 4096 + threadIdx.x; i0 < end; i0 += 4096) {
        int64_t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = i0 + u * 1024 < end ? ids[(long)b * ld + i0 + u * 1024] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (v[u] < 0 || v[u] >= vocab) continue;
            const int bit = (int)(1u << (v[u] & 31));
            if (part >= 0) add_ids(counts + (long)b * vocab, nullptr, (int)v[u]);
            else if (!(bits[v[u] >> 5] & bit)) atomicOr(bits + (v[u] >> 5), bit);
        }
    }
    if (part >= 0) return;
    __syncthreads();
    int* w = seen + (long)b * words;
    for (int i = threadIdx.x; i < words; i += 1024)
        if (bits[i]) w[i] |= bits[i];
}

}  // namespace

extern "C" int spacer_token_history_add(int* seen, int* counts, int B, int vocab, const int64_t* ids, long ld, int n, const int* len, spacer_stream_t stream) {
    SP_REQUIRE(vocab > 0 && vocab <= MAX_VOCAB && B >= 0 && n >= 0 && n <= MAX_VOCAB, SPACER_EINVAL, "token_history_add: B = %d, vocab = %d, n = %d (both at most %d)",
               B, vocab, n, MAX_VOCAB);
    if (B == 0 || n == 0) return SPACER_OK;
    SP_REQUIRE(seen && ids, SPACER_EINVAL, "token_history_add: seen and ids required");
    SP_REQUIRE(B <= 65535, SPACER_EINVAL, "token_history_add: %d rows (at most 65535)", B);
    const int words = (vocab + 31) / 32;
    // Both forms, few-id | many-id (us, a clear of the bits included, vocabulary 152064): 8 x 2051 ids 4.9 | 7.1, 64 x 1024 8.3 | 6.7, 128 x 1024 13.3 | 9.7,
    // 128 x 2051 23.0 | 14.7 (different ids, counted: scattered atomics at 28 per ns bound both); with 7/8 of a row the same 4.4 | 6.3, 4.5 | 6.2, 5.2 | 6.7, 7.2 | 7.4
    if ((long)B * n >= 100000 && words * 4 <= 64 * 1024)
        hipLaunchKernelGGL(token_history_row_kernel, dim3(1 + (counts ? cdiv(n, 4096) : 0), B), dim3(1024), words * 4, (hipStream_t)stream, seen, counts, vocab, words,
                           ids, ld, n, len);
    else hipLaunchKernelGGL(token_history_kernel, dim3(cdiv(n, 256), B), dim3(256), 0, (hipStream_t)stream, seen, counts, vocab, words, ids, ld, n, len);
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}

extern "C" int spacer_process_logits(const float* logits, long ld, float* out, long ld_out, int B, int vocab, const int* seen, const int* counts,
                                     float repetition, const float* repetition_dev, float frequency, const float* frequency_dev, float presence,
                                     const float* presence_dev, const float* bias, long ld_bias, const int* allowed, int n_masks,
                                     const int* allowed_row, spacer_stream_t stream) {
    SP_REQUIRE(vocab > 0 && vocab <= MAX_VOCAB && B >= 0, SPACER_EINVAL, "process_logits: B = %d, vocab = %d (at most %d)", B, vocab, MAX_VOCAB);
    if (B == 0) return SPACER_OK;
    SP_REQUIRE(logits && out, SPACER_EINVAL, "process_logits: logits and out required");
    SP_REQUIRE(B <= 65535, SPACER_EINVAL, "process_logits: %d rows (at most 65535)", B);
    SP_REQUIRE(B == 1 || (ld >= 0 && ld_out >= vocab), SPACER_EINVAL, "process_logits: rows of out (stride %ld) overlap", ld_out);
    const bool in_place = logits == out && (ld == ld_out || B == 1);
    if (!in_place && logits < out + (B - 1) * ld_out + vocab && out < logits + (B - 1) * ld + vocab) {      // side by side in rows of one stride, or refused
        const long off = ((out - logits) % (ld ? ld : 1) + ld) % (ld ? ld : 1);
        SP_REQUIRE(B > 1 && ld == ld_out && off >= vocab && off <= ld - vocab, SPACER_EINVAL, "process_logits: out overlaps the logits without being them");
    }
    SP_REQUIRE(repetition_dev || repetition > 0.f, SPACER_EINVAL, "process_logits: repetition penalty %g must be above 0", (double)repetition);
    SP_REQUIRE(seen || !counts, SPACER_EINVAL, "process_logits: counts without seen");
    SP_REQUIRE(counts || !(frequency_dev || presence_dev || frequency != 0.f || presence != 0.f), SPACER_EINVAL, "process_logits: frequency and presence penalties need counts");
    SP_REQUIRE(!allowed || (allowed_row ? n_masks > 0 : (n_masks == 1 || n_masks == B)), SPACER_EINVAL, "process_logits: %d masks for %d rows", n_masks, B);
    LogitArgs A = {logits, out, ld, ld_out, ld_bias, vocab, (vocab + 31) / 32, seen, counts, allowed, allowed_row, n_masks, repetition, frequency, presence,
                   repetition_dev, frequency_dev, presence_dev, bias};
    const bool vec = (((uintptr_t)logits | (uintptr_t)out | (uintptr_t)bias) & 15) == 0 && ((ld | ld_out | (bias ? ld_bias : 0)) & 3) == 0;
    const dim3 grid(cdiv(vocab, 256 * 4 * LU), B);
    hipStream_t s = (hipStream_t)stream;
    if (vec && in_place) hipLaunchKernelGGL((process_logits_kernel<true, true>), grid, dim3(256), 0, s, A);
    else if (vec) hipLaunchKernelGGL((process_logits_kernel<true, false>), grid, dim3(256), 0, s, A);
    else if (in_place) hipLaunchKernelGGL((process_logits_kernel<false, true>), grid, dim3(256), 0, s, A);
    else hipLaunchKernelGGL((process_logits_kernel<false, false>), grid, dim3(256), 0, s, A);
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}
