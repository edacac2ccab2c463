// Writers and reader of the rollout's key/value cache (bf16, e4m3 or int8 rows; layout and row arithmetic: kv_cache.h).
//
//   kv_write    one source row per (sequence, position) slot: a prompt batch's K / V columns of the packed q|k|v rows -> the cache
//   kv_append   the N newest tokens of every sequence -> positions len .. len + N - 1 of its own cache
//   kv_read     the cache's values as bf16 or fp32 rows [sequence, position, kv head, D]
//   decode_qkv_finish_cache   the decode step's form of kv_append: split-K sums + bias + rotary -> q, and K / V into the cache
//
// All four move each byte once and are bound by memory: D / 8 lanes hold a row (16-byte loads), K and V of a row are in flight together.  Measured, D = 128:
// 4 prompts of up to 16384 positions x 4 heads to e4m3 39.6 us (181 MB, 4.6 TB/s) and back to bf16 35.7 us (203 MB, 5.7 TB/s); 8 x 1391 x 4 to int8 10.0 us
// and back to fp32 13.5 us; a step's 64 tokens x 4 heads 3.8 us, which is a launch.
#include "kv_cache.h"

namespace {

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
__device__ __forceinline__ u16x2 max2(u16x2 a, u16x2 b) { return __builtin_elementwise_max(a, b); }
template <int CTRL>
__device__ __forceinline__ u16x2 max_dpp(u16x2 x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return max2(x, __builtin_bit_cast(u16x2, (uint32_t)__builtin_amdgcn_update_dpp((int)u, (int)u, CTRL, 0xf, 0xf, true)));
}
// (max |k|, max |v|) of a row's 8 or 16 lanes, as the bits of |bf16|: packed 16-bit maxima, lanes exchanged by DPP (pairs, quads, halves, rows)
template <int LPR>
__device__ __forceinline__ u16x2 row_amax(const uint4 k, const uint4 v) {
    auto abs2 = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7fff7fffu); };
    const u16x2 a = max2(max2(abs2(k.x), abs2(k.y)), max2(abs2(k.z), abs2(k.w))), b = max2(max2(abs2(v.x), abs2(v.y)), max2(abs2(v.z), abs2(v.w)));
    u16x2 m = max2((u16x2){a[0], b[0]}, (u16x2){a[1], b[1]});
    m = max_dpp<0xb1>(m);
    m = max_dpp<0x4e>(m);
    m = max_dpp<0x141>(m);
    if (LPR == 16) m = max_dpp<0x140>(m);
    return m;
}

template <int FMT>
__device__ __forceinline__ void store_row(char* dst, float* scale, const uint4 x, uint32_t amax, int lane_in_row) {
    if (FMT == KV_BF16) {
        *(uint4*)(dst + lane_in_row * 16) = x;
        return;
    }
    const RowScale r = row_scale<FMT>(amax);
    *(uint2*)(dst + lane_in_row * 8) = FMT == KV_INT8 ? codes8_int8(x, r, int8_row(r, amax))
        : make_uint2(code2<FMT>(x.x, r) | (code2<FMT>(x.y, r) << 16), code2<FMT>(x.z, r) | (code2<FMT>(x.w, r) << 16));
    if (lane_in_row == 0) *scale = r.scale;
}

// Rows of a pass: sequence (blockIdx.x / chunks, a scalar), then row = position * Hkv + head inside it (32 bits), so that the heads of a token,
// side by side in the source, fall to one wave.  A lane holds a piece of RU rows of K and V: all loads are in flight before the first use, without a
// branch between them (rows that are not stored read row 0).
// (1 row a lane 40 us for the 16384-position prompts, 4 rows or several steps per workgroup 58.)
constexpr int RU = 2;
template <int D> constexpr int rows_per_block() { return 4 * (512 / D) * RU; }

// APPEND == false: slot (sequence, position) takes source row rows[slot] (below 0, or >= n_src: the slot stays as it is)
// APPEND == true : source row sequence * N + i goes to position len[sequence] + i (outside the cache: dropped)
template <int FMT, int D, bool APPEND>
__global__ __launch_bounds__(256) void kv_store_kernel(const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, long ld, int n_src,
                                                       const int* __restrict__ rows, const int* __restrict__ len, int len_stride, int N,
                                                       KvView c, unsigned Hkv, unsigned chunks) {
    constexpr int LPR = D / 8, RPW = 64 / LPR;       // lanes per row, rows per wave
    const int lane = threadIdx.x & 63, lr = lane % LPR;
    const unsigned seq = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const unsigned total = (unsigned)(APPEND ? N : c.cap) * Hkv;
    const unsigned r0 = chunk * rows_per_block<D>() + (threadIdx.x >> 6) * (RPW * RU) + lane / LPR;
    int pos[RU], h[RU];
    long src[RU];
    if (APPEND) {
        const long first = (long)len[(long)seq * len_stride];
#pragma unroll
        for (int u = 0; u < RU; ++u) {
            const unsigned r = r0 + u * RPW, i = r / Hkv;
            const long p = first + i;
            h[u] = (int)(r - i * Hkv);
            pos[u] = (int)p;
            src[u] = r < total && p >= 0 && p < c.cap ? (long)seq * N + i : -1;
        }
    } else {
        int at[RU];
#pragma unroll
        for (int u = 0; u < RU; ++u) {
            const unsigned r = r0 + u * RPW, i = r / Hkv;
            h[u] = (int)(r - i * Hkv);
            pos[u] = (int)i;
            at[u] = rows[(long)seq * c.cap + min(i, (unsigned)c.cap - 1)];
        }
#pragma unroll
        for (int u = 0; u < RU; ++u) src[u] = r0 + u * RPW < total && at[u] < n_src ? at[u] : -1;
    }
    uint4 xk[RU], xv[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const long o = max(src[u], 0L) * ld + h[u] * D + lr * 8;
        xk[u] = *(const uint4*)(k + o);
        xv[u] = *(const uint4*)(v + o);
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const u16x2 top = FMT == KV_BF16 ? (u16x2){0, 0} : row_amax<LPR>(xk[u], xv[u]);
        if (src[u] < 0) continue;
        const long at = (seq * c.s_seq + h[u] * c.s_head + pos[u] * c.s_pos) * kv_size<FMT>();
        const long sat = seq * c.c_seq + h[u] * c.c_head + pos[u] * c.c_pos;
        store_row<FMT>(c.k + at, c.ks + sat, xk[u], top[0], lr);
        store_row<FMT>(c.v + at, c.vs + sat, xv[u], top[1], lr);
    }
}

template <int FMT>
__device__ __forceinline__ void values8(const char* p, float s, float (&f)[8]) {
    if (FMT == KV_BF16) {
        const uint4 x = *(const uint4*)p;
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = bf_lo(w[i]); f[2 * i + 1] = bf_hi(w[i]); }
        return;
    }
    const uint2 x = *(const uint2*)p;
    const uint32_t w[2] = {x.x, x.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (FMT == KV_E4M3) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
            f[4 * i] = a[0]; f[4 * i + 1] = a[1]; f[4 * i + 2] = b[0]; f[4 * i + 3] = b[1];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[4 * i + j] = (float)(int8_t)((w[i] >> (8 * j)) & 0xffu);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= s;
}

template <int FMT, int D, bool F32>
__global__ __launch_bounds__(256) void kv_read_kernel(KvView c, const int* __restrict__ len, void* __restrict__ ko, void* __restrict__ vo,
                                                      unsigned Hkv, unsigned chunks) {
    constexpr int LPR = D / 8, RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, lr = lane % LPR;
    const unsigned seq = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const unsigned total = (unsigned)c.cap * Hkv;
    const unsigned r0 = chunk * rows_per_block<D>() + (threadIdx.x >> 6) * (RPW * RU) + lane / LPR;
    const int n = len ? len[seq] : c.cap;
    float a[RU][8], b[RU][8], sk[RU], sv[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const unsigned r = min(r0 + u * RPW, total - 1), i = r / Hkv, h = r - i * Hkv;
        const long sat = seq * c.c_seq + h * c.c_head + i * c.c_pos;
        sk[u] = FMT == KV_BF16 ? 1.f : c.ks[sat];
        sv[u] = FMT == KV_BF16 ? 1.f : c.vs[sat];
        const long at = (seq * c.s_seq + h * c.s_head + i * c.s_pos + lr * 8) * kv_size<FMT>();
        values8<FMT>(c.k + at, sk[u], a[u]);
        values8<FMT>(c.v + at, sv[u], b[u]);
        if ((int)i >= n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) a[u][e] = b[u][e] = 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const unsigned r = r0 + u * RPW;
        if (r >= total) continue;
        const long o = ((long)seq * total + r) * D + lr * 8;
        if (F32) {
            float *kp = (float*)ko + o, *vp = (float*)vo + o;
            *(float4*)kp = make_float4(a[u][0], a[u][1], a[u][2], a[u][3]); *(float4*)(kp + 4) = make_float4(a[u][4], a[u][5], a[u][6], a[u][7]);
            *(float4*)vp = make_float4(b[u][0], b[u][1], b[u][2], b[u][3]); *(float4*)(vp + 4) = make_float4(b[u][4], b[u][5], b[u][6], b[u][7]);
        } else {
            *(uint4*)((bf16_t*)ko + o) = make_uint4(pack_bf2(a[u][0], a[u][1]), pack_bf2(a[u][2], a[u][3]), pack_bf2(a[u][4], a[u][5]), pack_bf2(a[u][6], a[u][7]));
            *(uint4*)((bf16_t*)vo + o) = make_uint4(pack_bf2(b[u][0], b[u][1]), pack_bf2(b[u][2], b[u][3]), pack_bf2(b[u][4], b[u][5]), pack_bf2(b[u][6], b[u][7]));
        }
    }
}

// One wave per (sequence, head) of the step's q|k|v sums; lane j < D / 2 holds the rotary pair (j, j + D / 2).  K and V are rounded to
// bf16 first and quantised from there, so that the cache holds what kv_append makes of the same bf16 rows.
template <int FMT>
__global__ __launch_bounds__(256) void decode_qkv_finish_cache_kernel(float* __restrict__ acc, const bf16_t* __restrict__ bias,
                                                                      const float* __restrict__ cs, const float* __restrict__ sn,
                                                                      bf16_t* __restrict__ q_out, KvView c, const int* __restrict__ tail_len,
                                                                      int len_stride, int B, int Hq, int Hkv, int D,
                                                                      const float* __restrict__ rowss, float* __restrict__ rowss_zero,
                                                                      int norm_cols, float eps) {
    const int lane = threadIdx.x & 63, half = D / 2, heads = Hq + 2 * Hkv;
    if (rowss_zero && blockIdx.x == 0 && threadIdx.x < B) rowss_zero[threadIdx.x] = 0.f;
    const int wid = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wid >= B * heads) return;
    const int b = wid / heads, hh = wid % heads;
    const int j = min(lane, half - 1);
    const bool on = lane < half;
    float* a = acc + (long)wid * D;
    // every load before the first use: absent operands read a valid dummy address, whose bits (those of a float: they may spell an infinity or NaN, which a
    // product with 0 would keep) are cleared
    const bf16_t* bias_p = bias ? bias + (long)hh * D : (const bf16_t*)cs;
    const float bias_on = bias ? 1.f : 0.f;
    const int pos = tail_len[(long)b * len_stride];
    const float rsum = rowss ? rowss[b] : 0.f;
    const float a1 = a[j], a2 = a[j + half];
    const bf16_t bias_bits = bias ? 0xffffu : 0u, b1 = bias_p[bias ? j : 0] & bias_bits, b2 = bias_p[bias ? j + half : 0] & bias_bits;
    const float c1 = cs[(long)b * D + j], s1 = sn[(long)b * D + j], c2 = cs[(long)b * D + j + half], s2 = sn[(long)b * D + j + half];
    const float rs = rowss ? rsqrtf(rsum / (float)norm_cols + eps) : 1.f;
    float x1 = a1 * rs + bias_on * bf2f(b1), x2 = a2 * rs + bias_on * bf2f(b2);
    if (on) { a[j] = 0.f; a[j + half] = 0.f; }
    if (hh < Hq + Hkv) {
        const float r1 = x1 * c1 - x2 * s1, r2 = x2 * c2 + x1 * s2;
        x1 = r1; x2 = r2;
    }
    const uint32_t w = pack_bf2(x1, x2);
    if (hh < Hq) {
        bf16_t* dst = q_out + ((long)b * Hq + hh) * D;
        if (on) { dst[j] = (bf16_t)(w & 0xffffu); dst[j + half] = (bf16_t)(w >> 16); }
        return;
    }
    if (pos < 0 || pos >= c.cap) return;
    const bool is_k = hh < Hq + Hkv;
    const int h = hh - Hq - (is_k ? 0 : Hkv);
    char* dst = (is_k ? c.k : c.v) + (b * c.s_seq + h * c.s_head + pos * c.s_pos) * kv_size<FMT>();
    if (FMT == KV_BF16) {
        if (on) { ((bf16_t*)dst)[j] = (bf16_t)(w & 0xffffu); ((bf16_t*)dst)[j + half] = (bf16_t)(w >> 16); }
        return;
    }
    uint32_t m = amax2(w);                           // (lanes past half repeat the last pair: the maximum is the same)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    const RowScale r = row_scale<FMT>(m);
    const uint32_t q = code2<FMT>(w, r);
    if (on) { dst[j] = (char)(q & 0xffu); dst[j + half] = (char)(q >> 8); }
    if (lane == 0) (is_k ? c.ks : c.vs)[b * c.c_seq + h * c.c_head + pos * c.c_pos] = r.scale;
}

}  // namespace

// ---- host: one check of a cache for every entry that takes one
int spacer_check_kv_cache(const spacer_kv_cache* c, const char* who) {
    SP_REQUIRE(c, SPACER_EINVAL, "%s: no cache", who);
    SP_REQUIRE(c->struct_bytes == (int)sizeof(spacer_kv_cache), SPACER_EINVAL, "%s: spacer_kv_cache: struct_bytes = %d but this library's has %d bytes",
               who, c->struct_bytes, (int)sizeof(spacer_kv_cache));
    SP_REQUIRE(c->format == KV_BF16 || c->format == KV_E4M3 || c->format == KV_INT8, SPACER_EINVAL, "%s: cache format %d unknown", who, c->format);
    SP_REQUIRE(c->head_dim == 64 || c->head_dim == 128, SPACER_EINVAL, "%s: head_dim %d unsupported (64, 128)", who, c->head_dim);
    SP_REQUIRE(c->n_seq > 0 && c->capacity > 0 && c->kv_heads > 0, SPACER_EINVAL, "%s: empty cache (%d sequences, %d positions, %d heads)", who,
               c->n_seq, c->capacity, c->kv_heads);
    SP_REQUIRE(c->capacity <= 1 << 30, SPACER_EINVAL, "%s: %d positions (at most 2^30)", who, c->capacity);
    SP_REQUIRE(c->k && c->v, SPACER_EINVAL, "%s: cache without k or v", who);
    const long size = c->format == KV_BF16 ? 2 : 1;
    SP_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0 && ((c->stride_seq | c->stride_head | c->stride_pos) * size) % 16 == 0, SPACER_EINVAL,
               "%s: cache rows must start at multiples of 16 bytes", who);
    SP_REQUIRE(c->stride_pos >= 0 && c->stride_pos * size < (1L << 26) && c->scale_stride_pos >= 0 && c->scale_stride_pos < (1L << 26), SPACER_EINVAL,
               "%s: positions of a cache must be less than 64 MiB (scales: 2^26 floats) apart", who);
    SP_REQUIRE(c->format == KV_BF16 || (c->k_scale && c->v_scale), SPACER_EINVAL, "%s: 8-bit cache without scales", who);
    return SPACER_OK;
}

// A cache that is written: no two rows (or scales) at one address, as the sequences of an expanded view would be
static bool apart(const spacer_kv_cache* c, long s0, long s1, long s2, long extent) {
    long s[3] = {s0, s1, s2}, n[3] = {c->n_seq, c->kv_heads, c->capacity};
    for (int i = 0; i < 3; ++i) {                         // dimensions by stride, each at least as wide as all below it
        int at = -1;
        for (int j = 0; j < 3; ++j)
            if (n[j] > 1 && (at < 0 || s[j] < s[at])) at = j;
        if (at < 0) break;
        if (s[at] < extent) return false;
        extent += s[at] * (n[at] - 1);
        n[at] = 1;
    }
    return true;
}
static int check_target(const spacer_kv_cache* c, const char* who) {
    if (int rc = spacer_check_kv_cache(c, who)) return rc;
    SP_REQUIRE(c->k != c->v && apart(c, c->stride_seq, c->stride_head, c->stride_pos, c->head_dim), SPACER_EINVAL, "%s: rows of the cache share memory", who);
    SP_REQUIRE(c->format == KV_BF16 || (c->k_scale != c->v_scale && apart(c, c->scale_stride_seq, c->scale_stride_head, c->scale_stride_pos, 1)),
               SPACER_EINVAL, "%s: scales of the cache share memory", who);
    return SPACER_OK;
}

// Does a row of k meet a row of v?  With every dimension at least as wide as all below it (`apart`), v's first number lies at delta from k's and a row pair at
// delta - sum_j d_j s_j, |d_j| < n_j: a dimension's d_j is the quotient of what the wider ones left, or one more.
static bool meet(long delta, const long* s, const long* n, int dims, long extent) {
    if (dims == 0) return delta > -extent && delta < extent;
    long q = delta / s[0];
    if (delta % s[0] < 0) --q;
    for (long d = q; d <= q + 1; ++d)
        if (d > -n[0] && d < n[0] && meet(delta - d * s[0], s + 1, n + 1, dims - 1, extent)) return true;
    return false;
}
static bool pair_apart(const spacer_kv_cache* c, const void* k, const void* v, long s0, long s1, long s2, long extent, long size) {
    long all[3] = {s0, s1, s2}, count[3] = {c->n_seq, c->kv_heads, c->capacity}, s[3], n[3];
    int dims = 0;
    for (;;) {                                            // dimensions by falling stride, in bytes
        int at = -1;
        for (int j = 0; j < 3; ++j)
            if (count[j] > 1 && (at < 0 || all[j] > all[at])) at = j;
        if (at < 0) break;
        s[dims] = all[at] * size; n[dims++] = count[at];
        count[at] = 1;
    }
    return !meet((long)((uintptr_t)v - (uintptr_t)k), s, n, dims, extent * size);
}
// ... of a cache that check_target has passed, where something is written
static int check_pair(const spacer_kv_cache* c, const char* who) {
    SP_REQUIRE(pair_apart(c, c->k, c->v, c->stride_seq, c->stride_head, c->stride_pos, c->head_dim, c->format == KV_BF16 ? 2 : 1), SPACER_EINVAL,
               "%s: rows of k and v share memory", who);
    SP_REQUIRE(c->format == KV_BF16 || pair_apart(c, c->k_scale, c->v_scale, c->scale_stride_seq, c->scale_stride_head, c->scale_stride_pos, 1, 4), SPACER_EINVAL,
               "%s: scales of k and v share memory", who);
    return SPACER_OK;
}

KvView spacer_kv_view(const spacer_kv_cache* c) {
    return KvView{(char*)c->k, (char*)c->v, c->k_scale, c->v_scale, c->stride_seq, c->stride_head, c->stride_pos, c->scale_stride_seq,
                  c->scale_stride_head, c->scale_stride_pos, c->n_seq, c->capacity};
}

// Workgroups of a sequence's `rows` rows, `per` each, or 0 where the launch would not fit
static unsigned row_chunks(long n_seq, long rows, int per) {
    const long chunks = (rows + per - 1) / per;
    return rows < 0x7fffffffL - 4096 && n_seq * chunks <= 0x7fffffffL ? (unsigned)chunks : 0u;
}
static int check_source(const void* k, const void* v, long ld, const char* who) {
    SP_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ld % 8 == 0, SPACER_EINVAL, "%s: source rows must start at multiples of 16 bytes", who);
    return SPACER_OK;
}

extern "C" int spacer_kv_write(const spacer_kv_cache* c, const void* k, const void* v, long ld, int n_src, const int* rows, spacer_stream_t stream) {
    if (int rc = check_target(c, "kv_write")) return rc;
    SP_REQUIRE(n_src >= 0 && rows, SPACER_EINVAL, "kv_write: rows required, n_src >= 0");
    if (n_src == 0) return SPACER_OK;
    if (int rc = check_pair(c, "kv_write")) return rc;
    if (int rc = check_source(k, v, ld, "kv_write")) return rc;
    const long per_seq = (long)c->capacity * c->kv_heads;
    const unsigned chunks = row_chunks(c->n_seq, per_seq, 4 * (512 / c->head_dim) * RU);
    SP_REQUIRE(chunks, SPACER_EINVAL, "kv_write: cache too large");
#define CALL(F, D)                                                                                                                                   \
    hipLaunchKernelGGL((kv_store_kernel<F, D, false>), dim3(c->n_seq * chunks), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)k, (const bf16_t*)v, \
                       ld, n_src, rows, (const int*)nullptr, 0, 1, spacer_kv_view(c), c->kv_heads, chunks)
    KV_DISPATCH(c, CALL);
#undef CALL
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}

extern "C" int spacer_kv_append(const spacer_kv_cache* c, const void* k, const void* v, long ld, int N, const int* len, int len_per_seq,
                                spacer_stream_t stream) {
    if (int rc = check_target(c, "kv_append")) return rc;
    SP_REQUIRE(N >= 0 && len, SPACER_EINVAL, "kv_append: lengths required, N >= 0");
    if (N == 0) return SPACER_OK;
    if (int rc = check_pair(c, "kv_append")) return rc;
    if (int rc = check_source(k, v, ld, "kv_append")) return rc;
    const long per_seq = (long)N * c->kv_heads;
    const unsigned chunks = row_chunks(c->n_seq, per_seq, 4 * (512 / c->head_dim) * RU);
    SP_REQUIRE(chunks && (long)c->n_seq * N <= 0x7fffffffL, SPACER_EINVAL, "kv_append: %d sequences x %d tokens are too many", c->n_seq, N);
#define CALL(F, D)                                                                                                                                  \
    hipLaunchKernelGGL((kv_store_kernel<F, D, true>), dim3(c->n_seq * chunks), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)k, (const bf16_t*)v, \
                       ld, c->n_seq * N, (const int*)nullptr, len, len_per_seq ? 1 : 0, N, spacer_kv_view(c), c->kv_heads, chunks)
    KV_DISPATCH(c, CALL);
#undef CALL
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}

extern "C" int spacer_kv_read(const spacer_kv_cache* c, const int* len, void* k_out, void* v_out, int out_f32, spacer_stream_t stream) {
    if (int rc = spacer_check_kv_cache(c, "kv_read")) return rc;
    SP_REQUIRE(k_out && v_out && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, SPACER_EINVAL, "kv_read: outputs must be 16-byte aligned");
    const unsigned chunks = row_chunks(c->n_seq, (long)c->capacity * c->kv_heads, 4 * (512 / c->head_dim) * RU);
    SP_REQUIRE(chunks, SPACER_EINVAL, "kv_read: cache too large");
#define CALL(F, D)                                                                                                                                   \
    do {                                                                                                                                             \
        if (out_f32)                                                                                                                                 \
            hipLaunchKernelGGL((kv_read_kernel<F, D, true>), dim3(c->n_seq * chunks), dim3(256), 0, (hipStream_t)stream, spacer_kv_view(c), len, k_out, \
                               v_out, c->kv_heads, chunks);                                                                                           \
        else                                                                                                                                         \
            hipLaunchKernelGGL((kv_read_kernel<F, D, false>), dim3(c->n_seq * chunks), dim3(256), 0, (hipStream_t)stream, spacer_kv_view(c), len, k_out, \
                               v_out, c->kv_heads, chunks);                                                                                           \
    } while (0)
    KV_DISPATCH(c, CALL);
#undef CALL
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}

extern "C" int spacer_decode_qkv_finish_cache(float* acc32, const void* bias, const float* cos_t, const float* sin_t, void* q_out,
                                              const spacer_kv_cache* c, const int* tail_len, int len_per_seq, const float* rowss, float* rowss_zero,
                                              int norm_cols, float eps, int Hq, spacer_stream_t stream) {
    if (int rc = check_target(c, "decode_qkv_finish_cache")) return rc;
    if (int rc = check_pair(c, "decode_qkv_finish_cache")) return rc;
    const int B = c->n_seq, heads = Hq + 2 * c->kv_heads;
    SP_REQUIRE(acc32 && cos_t && sin_t && q_out && tail_len, SPACER_EINVAL, "decode_qkv_finish_cache: missing operand");
    SP_REQUIRE(Hq > 0, SPACER_EINVAL, "decode_qkv_finish_cache: Hq = %d", Hq);
    SP_REQUIRE(!rowss || norm_cols > 0, SPACER_EINVAL, "decode_qkv_finish_cache: norm_cols = %d", norm_cols);
    // (one workgroup clears rowss_zero while the others still read rowss)
    SP_REQUIRE(!rowss || !rowss_zero || rowss + B <= rowss_zero || rowss_zero + B <= rowss, SPACER_EINVAL, "decode_qkv_finish_cache: rowss_zero overlaps rowss");
    SP_REQUIRE(!rowss_zero || B <= 256, SPACER_EINVAL, "decode_qkv_finish_cache: at most 256 rows with rowss_zero, got %d", B);
    const dim3 grid(cdiv((long)B * heads, 4)), block(256);
#define CALL(F)                                                                                                                                     \
    hipLaunchKernelGGL((decode_qkv_finish_cache_kernel<F>), grid, block, 0, (hipStream_t)stream, acc32, (const bf16_t*)bias, cos_t, sin_t, (bf16_t*)q_out, \
                       spacer_kv_view(c), tail_len, len_per_seq ? 1 : 0, B, Hq, c->kv_heads, c->head_dim, rowss, rowss_zero, norm_cols, eps)
    if (c->format == KV_BF16) CALL(KV_BF16);
    else if (c->format == KV_E4M3) CALL(KV_E4M3);
    else CALL(KV_INT8);
#undef CALL
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}
