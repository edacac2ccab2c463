// Device view of a key/value cache (spacer_kv_cache) and the row arithmetic that its writers share.
//
// A cache row is one token's D numbers x of one kv head.  8-bit rows carry one fp32 scale s and stand for code * s:
//   e4m3  s = the smallest power of two >= 2^-126 with amax / s <= 448.  A power of two because a floating-point code keeps its
//         relative precision whatever the scale, x / s is then exact (the code is the only rounding) and so is the code as bf16
//   int8  s = amax / 127 rounded to fp32; code = the integer nearest to x / s, ties to even.  A fixed-point code needs the whole range
// A row with a NaN or an infinity gets s = NaN and codes 0: it stands for NaN everywhere, as loud as the bf16 row would be.
#pragma once
#include "common.h"

constexpr int KV_BF16 = SPACER_KV_BF16, KV_E4M3 = SPACER_KV_E4M3, KV_INT8 = SPACER_KV_INT8;

struct KvView {
    char *k, *v;
    float *ks, *vs;
    long s_seq, s_head, s_pos;      // elements between sequences, heads, positions of k and of v
    long c_seq, c_head, c_pos;      // floats between them in the scales
    int n_seq, cap;
};

int spacer_check_kv_cache(const spacer_kv_cache* c, const char* who);
KvView spacer_kv_view(const spacer_kv_cache* c);

#define KV_DISPATCH(c, CALL)                                                         \
    do {                                                                             \
        if ((c)->head_dim == 128) {                                                  \
            if ((c)->format == KV_BF16) CALL(KV_BF16, 128);                          \
            else if ((c)->format == KV_E4M3) CALL(KV_E4M3, 128);                     \
            else CALL(KV_INT8, 128);                                                 \
        } else {                                                                     \
            if ((c)->format == KV_BF16) CALL(KV_BF16, 64);                           \
            else if ((c)->format == KV_E4M3) CALL(KV_E4M3, 64);                      \
            else CALL(KV_INT8, 64);                                                  \
        }                                                                            \
    } while (0)

namespace {

template <int FMT> constexpr int kv_size() { return FMT == KV_BF16 ? 2 : 1; }

struct RowScale {
    float scale;       // what is stored
    float s, pre;      // divisor, and an exact power of two both sides are multiplied by first (1, except for tiny int8 rows)
    float inv;
    bool finite;
};

// a / 127 rounded to nearest: the product with the rounded 1 / 127 and one step with its exact remainder (equal to the division for every finite bf16 a
// of 2^-96 and more; below, the division itself)
__device__ __forceinline__ float div127(float a) {
    if (a < 1.2621774e-29f) return a / 127.f;
    const float c = 1.f / 127.f, y = a * c;
    return fmaf(fmaf(-127.f, y, a), c, y);
}

// amax as the bits of |bf16|: NaN > infinity > every finite value, so one integer maximum finds both
template <int FMT>
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    r.finite = amax_bits < 0x7f80u;
    r.pre = 1.f;
    if (FMT == KV_E4M3) {
        // amax = m 2^e, 1 <= m < 2; 448 = 1.75 * 2^8: s = 2^(e-8), one more when m > 1.75 (96 = 0.75 * 128)
        const int b = max(1, (int)(amax_bits >> 7) - 8 + ((amax_bits & 0x7fu) > 96u ? 1 : 0));
        r.s = r.finite ? __uint_as_float((uint32_t)b << 23) : __uint_as_float(0x7fc00000u);
        r.scale = r.s;
        r.inv = __uint_as_float((uint32_t)(254 - b) << 23);
    } else {
        const float amax = __uint_as_float(amax_bits << 16);
        r.scale = r.finite ? div127(amax) : __uint_as_float(0x7fc00000u);
        if (amax < 1.2621774e-29f) r.pre = 18446744073709551616.f;      // 2^-96, 2^64: keeps 1 / s finite
        r.s = r.scale * r.pre;
        r.inv = (r.finite && r.s > 0.f) ? 1.f / r.s : 0.f;
    }
    return r;
}

// the integer nearest to x / s: the product with 1 / s can only be one off where the quotient is next to a half, and x - s q is exact
// there (a multiple of s's last place, below s), so its comparison with s / 2 decides as the exact quotient would
__device__ __forceinline__ float quotient_rne(float x, const RowScale& r) {
    const float xs = x * r.pre;
    float q = rintf(xs * r.inv);
    const float e = fmaf(-r.s, q, xs), half = 0.5f * r.s, ae = fabsf(e);
    if (ae > half || (ae == half && ((int)q & 1))) q += copysignf(1.f, e);
    return fminf(fmaxf(q, -127.f), 127.f);
}

// two bf16 (packed) -> two codes in the low 16 bits
template <int FMT>
__device__ __forceinline__ uint32_t code2(uint32_t w, const RowScale& r) {
    if (!r.finite) return 0u;
    const float a = bf_lo(w), b = bf_hi(w);
    if (FMT == KV_E4M3) return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * r.inv, b * r.inv, 0, false) & 0xffffu;
    if (r.inv == 0.f) return 0u;
    return ((uint32_t)(int)quotient_rne(a, r) & 0xffu) | (((uint32_t)(int)quotient_rne(b, r) & 0xffu) << 8);
}

// What the eight-code form below needs of an int8 row.  1 / s comes from the hardware reciprocal (1 ulp) and is moved by at most 4 ulp so that max|x| / 2, which
// every other wave holds and whose quotient 63.5 (1 + error of s) lies next to a half, falls on the side of 63.5 that the exact quotient lies on (a
// tie's even neighbour is 64, outside).  Other numbers next to a half go the exact way.
struct Int8Row {
    float inv;
    uint32_t half;       // max|x| / 2 as bf16 bits
    bool exact;          // tiny, zero or non-finite row
};
__device__ __forceinline__ Int8Row int8_row(const RowScale& r, uint32_t amax_bits) {
    Int8Row q;
    const float amax = __uint_as_float(amax_bits << 16), inv = __builtin_amdgcn_rcpf(r.scale);
    const bool outside = fmaf(-127.f, r.scale, amax) >= 0.f, is = fmaf(amax, inv, -127.f) >= 0.f;
    q.inv = __uint_as_float(__float_as_uint(inv) + (outside == is ? 0 : outside ? 4 : -4));
    q.half = amax_bits - (1u << 7);
    q.exact = amax_bits < (31u << 7) || !r.finite;                                  // (31 << 7: 2^-96)
    return q;
}
// Eight int8 codes: u = x (1 / s) + 1.5 2^23 rounds the product to an integer in u's low bits.  1 / s is off by less than 5 2^-23 of itself, so the product
// by less than 7.6e-5: the integer is the right one where the product is further than 1e-4 from a half.  A wave that holds another number there (one in
// ten) or an exact row takes the comparison of quotient_rne for all.
__device__ __forceinline__ uint2 codes8_int8(const uint4 x, const RowScale& r, const Int8Row& q) {
    const float magic = 12582912.f;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    float u[8], far = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = (i & 1) ? bf_hi(w[i >> 1]) : bf_lo(w[i >> 1]);
        u[i] = fmaf(f, q.inv, magic);
        const float off = fmaf(f, q.inv, magic - u[i]);
        far = fmaxf(far, fabsf(f) == __uint_as_float(q.half << 16) ? 0.f : fabsf(off));
    }
    if (__any(q.exact || !(far < 0.4999f)))
        return make_uint2(code2<KV_INT8>(x.x, r) | (code2<KV_INT8>(x.y, r) << 16), code2<KV_INT8>(x.z, r) | (code2<KV_INT8>(x.w, r) << 16));
    uint32_t o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(u[4 * i + 1]), __float_as_uint(u[4 * i]), 0x0c0c0400u);
        const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(u[4 * i + 3]), __float_as_uint(u[4 * i + 2]), 0x04000c0cu);
        o[i] = ab | cd;
    }
    return make_uint2(o[0], o[1]);
}

__device__ __forceinline__ uint32_t amax2(uint32_t w) { return max(w & 0x7fffu, (w >> 16) & 0x7fffu); }

}  // namespace
