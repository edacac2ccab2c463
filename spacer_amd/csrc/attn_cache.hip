// Decode attention over bf16 / e4m3 / int8 key-value caches (kv_cache.h): one new token per sequence or a tree of drafted tokens.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i),   k_j = s^k_j K_j,  v_j = s^v_j V_j  (codes K, V; row scales s)
//
// Columns and rows.  A column is one query (node i of sequence b, head h); the columns of a kv head that read the same keys are the N side of
// 16x16x32 bf16 matrix products: the prompt's keys meet every (rollout, node, head) column of the prompt at once, a sequence's own keys its
// (node, head) columns.  The codes become bf16 in registers (e4m3 and int8 numbers are exact in bf16); s^k multiplies the fp32 scores and s^v
// the fp32 weights before they are rounded to bf16 for the second product, so no scale costs an operation per element.  l sums the weights as rounded, so
// that a rounding common to numerator and denominator drops out (relative error against 64 bits of 2 x 12 heads over 220 positions, int8: 2.9e-3 with the
// unrounded sum, now 2.1e-3; the output's own rounding alone gives 1.9e-3).
//   S^T[key, col] = K . Q^T     A = K rows straight from memory, B = Q fragments
//   O^T[d, col]  += V^T . P^T   A = V through a wave-private LDS image and the transposing LDS read, B = the weights just computed: the C layout of S^T
//                               (lane = column, registers = keys) is the B layout of the second product under a permutation of the keys that the
//                               image's row order repeats, so no lane exchange lies between the two
// Work split.  Workgroup = (prompt or sequence, kv head, column block of 16 NC, range of keys); its 4 waves take 32-key tiles in turn and never meet
// inside the loop: the next tile's K, V and scales are requested while the current one is worked on, so 8 waves per CU keep 64 KB in flight (8 bits).
// The waves' (O, m, l) are joined through LDS, the ranges' through fp32 records and a second small launch.  Short contexts take one launch of 8 waves
// per workgroup that walk the prompt's and the sequence's keys and write the output themselves (plan_attn).
// Measured (kernels alone): 2 x 12 heads over 220 int8 positions 6.2 us; 8 x 8 rollouts x 28 heads over 1391 + 300 e4m3 positions 14 us, over 16384 + 700 of
// int8 42 + 5 (join); 8 trees of 13 over 2311 + 211 bf16 positions 16 + 4; 32 trees of 32 over 5498 + 333 e4m3 positions of D = 64 52 + 5.  Many columns per
// key are bound by the softmax's and the conversions' VALU work (about 160 operations and 16 exponentials beside 18 products a tile of 32 x 32, D = 64), few by
// the latency of a tile's rows.
#include <math.h>

#include "kv_cache.h"

namespace {

constexpr int TK = 32;            // keys per wave and step
constexpr float LOG2E = 1.4426950408889634f;
constexpr float TINY = 8.0779357e-28f;      // 2^-90

// n / d for 0 <= n < 2^31 by a multiplication (d is the same for a whole launch): m = floor(2^(31 + s) / d) + 1 with 2^s >= d is exact there
struct FastDiv {
    unsigned m, s, d;
    __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : (int)(__umulhi((unsigned)n, m) >> (s - 1)); }
};

struct AttnCacheArgs {
    const bf16_t* q;
    long q_ld;
    KvView prompt, tail;
    const int *prompt_len, *tail_len, *row0;
    const int64_t* tree;
    int len_stride, tree_stride;
    int n_prompts, rows, B, N, Hq, Hkv;
    int sa, sb, cba, cbb;         // key ranges and column blocks of the prompt and of the sequence role
    int na;                       // workgroups of the prompt role (a multiple of 8)
    FastDiv per_row, rep;         // by N * Hq / Hkv and by Hq / Hkv
    float scale;
    float* rec_o;                 // [sa + sb][B * N * Hq][D]
    float2* rec_ml;               // [sa + sb][B * N * Hq]: maximum (log2 domain) and sum
    bf16_t* o;
};

// eight codes as bf16, exact; e4m3 codes times their row's scale, a power of two
template <int FMT>
__device__ __forceinline__ bf16x8 codes_to_bf16(uint2 w, float s) {
    uint32_t o[4];
    if (FMT == KV_E4M3) {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, false));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, true));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, false));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, true));
    } else {
        const uint32_t a[2] = {w.x, w.y};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                o[2 * i + j] = pack_bf2((float)(int8_t)((a[i] >> (16 * j)) & 0xffu), (float)(int8_t)((a[i] >> (16 * j + 8)) & 0xffu));
    }
    return __builtin_bit_cast(bf16x8, make_uint4(o[0], o[1], o[2], o[3]));
}

// An e4m3 scale that is neither a power of two of 2^-126 or more nor 0: the conversion above takes its exponent alone, and the sum of the rounded weights
// its reciprocal as a bf16 number, so that it would be one number here and another to kv_read
__device__ __forceinline__ bool no_power_of_two(float s) { return (__float_as_uint(s) & 0x807fffffu) != 0u; }

// maximum over the four 16-lane groups (lanes of the same column)
__device__ __forceinline__ float group_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t w = __float_as_uint(y);
    const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int FMT, int D, int NC>
struct Tile {
    static constexpr int ES = kv_size<FMT>();
    static constexpr int RB = D * ES;                   // bytes of a row
    static constexpr int CPR = RB / 16;                 // 16-byte chunks of a row
    static constexpr int KL = RB / 64;                  // K loads per lane and 16-key fragment
    static constexpr int VL = TK * CPR / 64;            // V loads per lane
    static constexpr int STEPS = D / 32;
    static constexpr int IMG = TK * RB;                 // bytes of a V image
    // rows that share the 64 LDS banks' 256 bytes take the same chunk order, the next ones another: fragment reads of 16 rows hit all banks once
    static __device__ __forceinline__ int swz(int row) { return (row / (RB >= 256 ? 1 : 256 / RB)) & (CPR - 1); }
};

// Column blocks of a workgroup: 1 or 2.  (4 leave one lane 128 registers of O: e4m3 rollouts 8 x 8 over 1391 + 300 positions 18.0 instead of 13.8 us, bf16
// 33 instead of 21; at D = 64 the two are level.)
constexpr int SCALES = TK * (4 + 4 + 2 + 2);      // a wave's row scales: K's (int8), V's, and 1 / V's as two bf16 numbers
constexpr int lds_bytes(int es, int D, int nc, int nw) {
    const int work = nw * (TK * D * es + SCALES), join = nc * 16 * nw * ((D + 4) * 4 + 8);      // 4 waves: at most 69 KB, two workgroups per CU; 8: 139 KB
    return work > join ? work : join;
}

// Keys [0, total) of one (sequence, kv head), this workgroup's share of them, and the first key that the nodes' masks speak of (total: none)
struct KeySegment {
    const char *k, *v;
    const float *ks, *vs;
    int row_b, c_pos;                 // bytes between positions, floats between their scales
    int total, base, t0, t1;          // t0, t1: in 32-key tiles
};

// The state of one workgroup's 16 NC columns and what it does with a segment of keys.  ColInfo: (c, row, head, node) -> the query of column c, or false.
template <int FMT, int D, int NC, int NW, class ColInfo>
struct Columns {
    using T = Tile<FMT, D, NC>;
    static constexpr int DF = D / 16;

    const AttnCacheArgs& A;
    const ColInfo& info;
    const int c0, lane, wave, l15, g;
    char* vimg;
    float* sc;
    bf16x8 qreg[NC][T::STEPS];
    f32x4 oacc[NC][DF];
    float m_run[NC], l_run[NC];
    uint4 kr[2][T::KL], vr[T::VL];
    float scr, kscr[2];               // row scales: of K (lanes .. 31) and of V (lanes 32 ..); e4m3: kscr, K's again for the rows that a lane converts

    __device__ __forceinline__ Columns(const AttnCacheArgs& args, const ColInfo& ci, char* smem, int first, int tid = threadIdx.x)
        : A(args), info(ci), c0(first), lane(tid & 63), wave(__builtin_amdgcn_readfirstlane(tid >> 6)), l15(tid & 15),
          g((tid & 63) >> 4), scr(0.f), kscr{1.f, 1.f} {
        vimg = smem + wave * T::IMG;
        sc = (float*)(smem + NW * T::IMG + wave * SCALES);
#pragma unroll
        for (int cb = 0; cb < NC; ++cb) {
            m_run[cb] = -INFINITY; l_run[cb] = 0.f;
#pragma unroll
            for (int d = 0; d < DF; ++d) oacc[cb][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }

    // fragment (cb, step): for column l15 the 8 numbers that the step's slots of lane group g stand for
    __device__ __forceinline__ bf16x8 q_frag(int cb, int step) const {
        int row, head, node;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (info(c0 + cb * 16 + l15, row, head, node)) {
            const int d = T::ES == 2 ? step * 32 + g * 8 : (step >> 1) * 64 + g * 16 + (step & 1) * 8;
            x = *(const uint4*)(A.q + ((long)row * A.N + node) * A.q_ld + (long)head * D + d);
        }
        return __builtin_bit_cast(bf16x8, x);
    }
    __device__ __forceinline__ void load_queries() {
#pragma unroll
        for (int cb = 0; cb < NC; ++cb)
#pragma unroll
            for (int s = 0; s < T::STEPS; ++s) qreg[cb][s] = q_frag(cb, s);
    }

    // Requests for tile t: 64-bit arithmetic stays in scalars, a lane adds 32 bits (32 rows span less than 2^31 bytes: checked on the host).
    // Keys behind the last repeat it, so every address lies inside the cache.
    __device__ __forceinline__ void fetch_k(const KeySegment& s, int t) {
        const int k0 = t * TK, last = s.total - 1 - k0;
        const char* kb = s.k + (long)k0 * s.row_b;
#pragma unroll
        for (int kf = 0; kf < 2; ++kf) {
            const int row = last >= TK - 1 ? kf * 16 + l15 : min(kf * 16 + l15, last);
            const uint32_t off = (uint32_t)(row * s.row_b + g * 16);
#pragma unroll
            for (int h = 0; h < T::KL; ++h) kr[kf][h] = *(const uint4*)(kb + off + h * 64);
            if (FMT == KV_E4M3) kscr[kf] = s.ks[(long)k0 * s.c_pos + row * s.c_pos];
        }
    }
    __device__ __forceinline__ void fetch_v(const KeySegment& s, int t) {
        const int k0 = t * TK, last = s.total - 1 - k0;
        const char* vb = s.v + (long)k0 * s.row_b;
        if (FMT != KV_BF16) {
            const float* sb = (lane >= TK ? s.vs : s.ks) + (long)k0 * s.c_pos;
            scr = sb[min(lane & (TK - 1), last) * s.c_pos];
        }
#pragma unroll
        for (int i = 0; i < T::VL; ++i) {
            const int row = lane / T::CPR + i * (64 / T::CPR);
            vr[i] = *(const uint4*)(vb + (uint32_t)((last >= TK - 1 ? row : min(row, last)) * s.row_b + (lane % T::CPR) * 16));
        }
    }
    __device__ __forceinline__ void fetch(const KeySegment& s, int t) { fetch_k(s, t); fetch_v(s, t); }

    // tiles first, first + NW, ... < s.t1 of a segment; the tile `first` has been requested by fetch()
    __device__ __forceinline__ void run(const KeySegment& s, int first) {
        int t = first;
        const int plain = min(s.t1, s.base / TK);         // from here on some key of a tile is a node or lies behind the last key
        for (; t < plain; t += NW) tile<false>(s, t);
        for (; t < s.t1; t += NW) tile<true>(s, t);
    }

    template <bool EDGE>
    __device__ __forceinline__ void tile(const KeySegment& s, int t) {
        const int k0 = t * TK;
        // ---- S^T = K . Q^T
        f32x4 st[NC][2];
#pragma unroll
        for (int cb = 0; cb < NC; ++cb) st[cb][0] = st[cb][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int step = 0; step < T::STEPS; ++step) {
            bf16x8 kf8[2];
#pragma unroll
            for (int kf = 0; kf < 2; ++kf) {
                if (FMT == KV_BF16) kf8[kf] = __builtin_bit_cast(bf16x8, kr[kf][FMT == KV_BF16 ? step : 0]);
                else {
                    const uint4 x = kr[kf][FMT == KV_BF16 ? 0 : step >> 1];
                    kf8[kf] = codes_to_bf16<FMT>((step & 1) ? make_uint2(x.z, x.w) : make_uint2(x.x, x.y), kscr[kf]);
                }
            }
#pragma unroll
            for (int cb = 0; cb < NC; ++cb) {
                st[cb][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf8[0], qreg[cb][step], st[cb][0], 0, 0, 0);
                st[cb][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf8[1], qreg[cb][step], st[cb][1], 0, 0, 0);
            }
        }
        if (t + NW < s.t1) fetch_k(s, t + NW);              // K's registers are free: the next tile's rows are under way during the rest, V's as soon as
                                                          // they lie in LDS
        // ---- V and the scales into the wave's image; (the previous tile's LDS reads stay in front of these writes: LDS is in order)
        asm volatile("" ::: "memory");
        uint16_t* inv_v = (uint16_t*)(sc + 2 * TK);       // [2][TK]
        bool tiny = false;                                // a V row below 2^-90 (a row of zeros): its weights are counted before they meet the scale
        if (FMT != KV_BF16) {
            sc[lane] = FMT == KV_INT8 && lane < TK ? scr * (A.scale * LOG2E) : scr;
            // (rare) a key whose K or V scale is no power of two counts as NaN, by its V scale, which hidden keys drop
            if (FMT == KV_E4M3 && __any(no_power_of_two(scr)) && no_power_of_two(scr)) sc[TK + (lane & (TK - 1))] = __uint_as_float(0x7fc00000u);
            if (lane >= TK) {
                const float inv = scr >= TINY && scr < INFINITY ? __builtin_amdgcn_rcpf(scr) : 0.f;
                const uint32_t hi = pack_bf2(inv, 0.f) & 0xffffu;
                inv_v[lane - TK] = (uint16_t)hi;
                if (FMT == KV_INT8) inv_v[lane] = (uint16_t)pack_bf2(inv - __uint_as_float(hi << 16), 0.f);
            }
            tiny = __any(lane >= TK && scr < TINY);
        }
        bool odd_v = false;                               // a NaN or an infinity in a bf16 V row that some columns must not see
#pragma unroll
        for (int i = 0; i < T::VL; ++i) {
            const int row = lane / T::CPR + i * (64 / T::CPR);
            uint4 x = vr[i];
            if (FMT == KV_E4M3 && EDGE) {                 // a row with a NaN code (the writers make none) counts as NaN: by its scale, which hidden rows drop
                auto nan4 = [](uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
                if (nan4(x.x) | nan4(x.y) | nan4(x.z) | nan4(x.w)) {
                    x = make_uint4(0, 0, 0, 0);
                    sc[TK + row] = __uint_as_float(0x7fc00000u);
                }
            }
            *(uint4*)(vimg + row * T::RB + (((lane % T::CPR) ^ T::swz(row)) * 16)) = x;
            if (FMT == KV_BF16 && EDGE) {
                const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) odd_v |= amax2(w[e]) >= 0x7f80u;
            }
        }
        if (t + NW < s.t1) fetch_v(s, t + NW);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // image and scales complete before any lane reads them
        __builtin_amdgcn_wave_barrier();
        f32x4 ksv[2], vsv[2];
        if (FMT != KV_BF16) {
#pragma unroll
            for (int kf = 0; kf < 2; ++kf) {
                if (FMT == KV_INT8) ksv[kf] = *(const f32x4*)(sc + kf * 16 + g * 4);
                vsv[kf] = *(const f32x4*)(sc + TK + kf * 16 + g * 4);
            }
        }
        // ---- online softmax in the log2 domain; the running maximum follows only in steps of more than 2^8 (weights stay below 2^8, far
        //      inside fp32 and bf16), so that O is rescaled a few times per range and not once per tile.  x = the score up to the factor kmul > 0,
        //      which for int8 is in the row scales; elsewhere it is applied by the exponential's fma
        const float kmul = FMT == KV_INT8 ? 1.f : A.scale * LOG2E;
        bf16x8 pf[NC];
        uint64_t see[NC];
        auto visible = [&](int cb, int key) -> bool { return key < s.base || (key < s.total && ((see[cb] >> (key - s.base)) & 1)); };
#pragma unroll
        for (int cb = 0; cb < NC; ++cb) {
            bool vis[2][4];
            if (EDGE) {                                   // nodes that the column's node sees
                int row, head, node;
                see[cb] = 0;
                if (s.base < s.total && info(c0 + cb * 16 + l15, row, head, node))
                    see[cb] = A.tree ? (uint64_t)A.tree[(long)row * A.tree_stride + node] : (node >= 63 ? ~0ull : (2ull << node) - 1);
#pragma unroll
                for (int kf = 0; kf < 2; ++kf)
#pragma unroll
                    for (int r = 0; r < 4; ++r) vis[kf][r] = visible(cb, k0 + kf * 16 + g * 4 + r);
            }
            float p[2][4], mx = -INFINITY;
#pragma unroll
            for (int kf = 0; kf < 2; ++kf)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = FMT == KV_INT8 ? st[cb][kf][r] * ksv[kf][r] : st[cb][kf][r];
                    if (EDGE && !vis[kf][r]) x = -INFINITY;
                    p[kf][r] = x;
                    mx = fmaxf(mx, x);
                }
            mx = group_max(mx) * kmul;
            if (__any(mx > m_run[cb] + 8.f)) {
                const float m_new = mx > m_run[cb] + 8.f ? mx : m_run[cb];
                const float alpha = m_run[cb] == m_new ? 1.f : __builtin_amdgcn_exp2f(m_run[cb] - m_new);
                m_run[cb] = m_new;
                l_run[cb] *= alpha;
#pragma unroll
                for (int d = 0; d < DF; ++d) oacc[cb][d] *= alpha;
            }
            const float m = m_run[cb] == -INFINITY ? 0.f : m_run[cb];     // nothing seen yet, or only scores of -infinity: every weight is 0
#pragma unroll
            for (int kf = 0; kf < 2; ++kf)
#pragma unroll
                for (int r = 0; r < 4; ++r) p[kf][r] = __builtin_amdgcn_exp2f(FMT == KV_INT8 ? p[kf][r] - m : fmaf(p[kf][r], kmul, -m));
            if (FMT != KV_BF16) {
                if (tiny) {
                    float sum = 0.f;
#pragma unroll
                    for (int kf = 0; kf < 2; ++kf)
#pragma unroll
                        for (int r = 0; r < 4; ++r) sum += vsv[kf][r] < TINY ? p[kf][r] : 0.f;
                    sum += __shfl_xor(sum, 16, 64);
                    l_run[cb] += sum + __shfl_xor(sum, 32, 64);
                }
#pragma unroll
                for (int kf = 0; kf < 2; ++kf)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        p[kf][r] *= vsv[kf][r];
                        if (EDGE && !vis[kf][r]) p[kf][r] = 0.f;    // (the scale of a hidden row may be NaN)
                    }
            }
            const uint4 pk = make_uint4(pack_bf2(p[0][0], p[0][1]), pack_bf2(p[0][2], p[0][3]), pack_bf2(p[1][0], p[1][1]), pack_bf2(p[1][2], p[1][3]));
            pf[cb] = __builtin_bit_cast(bf16x8, pk);
            // the sum counts the weights as the second product sees them, rounded: a row's rounding then scales numerator and denominator alike, and
            // a key that outweighs the others comes out exactly
            if (FMT == KV_BF16) {
                l_run[cb] += ((bf_lo(pk.x) + bf_hi(pk.x)) + (bf_lo(pk.y) + bf_hi(pk.y))) + ((bf_lo(pk.z) + bf_hi(pk.z)) + (bf_lo(pk.w) + bf_hi(pk.w)));
            } else {                                      // ... without the scale they carry: one more product, with 1 / s^v (e4m3: exact; int8: to 2^-17)
                f32x4 sum = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int part = 0; part < (FMT == KV_INT8 ? 2 : 1); ++part) {
                    const uint2 a = *(const uint2*)(inv_v + part * TK + 4 * g), b = *(const uint2*)(inv_v + part * TK + 16 + 4 * g);
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y)), pf[cb], sum, 0, 0, 0);
                }
                l_run[cb] += sum[0];
            }
        }
        // ---- O^T += V^T . P^T; slot j of lane group g is key (j >> 2) * 16 + 4 g + (j & 3)
        if (FMT == KV_BF16 && EDGE && __any(odd_v)) {     // rare: a product with a hidden NaN or infinity would be NaN; add visible keys one by one
#pragma unroll 1
            for (int key = 0; key < TK; ++key)
#pragma unroll
                for (int cb = 0; cb < NC; ++cb) {
                    // the key's weight sits in the lanes of group (key & 15) >> 2, pair (key >> 4, (key & 3) >> 1) of the packed operand
                    const uint4 pk = __builtin_bit_cast(uint4, pf[cb]);
                    const uint32_t mine = key < 16 ? ((key & 2) ? pk.y : pk.x) : ((key & 2) ? pk.w : pk.z);
                    const uint32_t pair = (uint32_t)__shfl((int)mine, ((key & 15) >> 2) * 16 + l15, 64);
                    const float w = (key & 1) ? bf_hi(pair) : bf_lo(pair);
                    const bool on = visible(cb, k0 + key);
#pragma unroll
                    for (int df = 0; df < DF; ++df)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int d = df * 16 + g * 4 + r;
                            const float x = bf2f(*(const bf16_t*)(vimg + key * T::RB + (((d >> 3) ^ T::swz(key)) * 16) + (d & 7) * 2));
                            if (on) oacc[cb][df][r] += w * x;
                        }
                }
            return;
        }
#pragma unroll
        for (int df = 0; df < DF; ++df) {
            bf16x8 vf;
            if (FMT == KV_BF16) {
                const int chunk = df * 2 + ((l15 & 3) >> 1), sub = (l15 & 1) * 8, r0 = 4 * g + (l15 >> 2), r1 = r0 + 16;
                typedef __attribute__((ext_vector_type(4))) short s16x4;
                typedef __attribute__((ext_vector_type(8))) short s16x8;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vimg + r0 * T::RB + ((chunk ^ T::swz(r0)) * 16) + sub));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vimg + r1 * T::RB + ((chunk ^ T::swz(r1)) * 16) + sub));
                const s16x8 both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                vf = __builtin_bit_cast(bf16x8, both);
            } else {
                // (lane i of a 16-lane group supplies 8 bytes of row i >> 1, columns 8 (i & 1) ..; it receives column i of the 8 rows)
                typedef __attribute__((ext_vector_type(2))) int i32x2;
                const int r = l15 >> 1, row = (r >> 2) * 16 + 4 * g + (r & 3);
                const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(vimg + row * T::RB + ((df ^ T::swz(row)) * 16) + (l15 & 1) * 8));
                vf = codes_to_bf16<FMT>(make_uint2((uint32_t)x[0], (uint32_t)x[1]), 1.f);
            }
#pragma unroll
            for (int cb = 0; cb < NC; ++cb) oacc[cb][df] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[cb], oacc[cb][df], 0, 0, 0);
        }
    }

    // joins the waves ([wave][column][D + 4 floats], [wave][column] (m, l) in LDS) and writes the record `slot` of every column, or with slot < 0 its output
    __device__ __forceinline__ void finish(char* smem, int slot) {
        constexpr int JC = NC * 16, TPC = 64 * NW / JC < D / 4 ? 64 * NW / JC : D / 4, PER = D / TPC;      // columns, threads per column, floats per thread
        const int tid = threadIdx.x;
        float* jo = (float*)smem;
        float2* jm = (float2*)(smem + NW * JC * (D + 4) * 4);
        const int jc = tid / TPC, jd = (tid % TPC) * 4;       // (a thread's float4 lie TPC * 4 floats apart: neighbouring threads, neighbouring banks)
        const long ncol_all = (long)A.B * A.N * A.Hq;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < NC; ++r) {
            float l = l_run[r];
            if (FMT == KV_BF16) {                         // (8-bit: every lane of a column holds its sum)
                l += __shfl_xor(l, 16, 64);
                l += __shfl_xor(l, 32, 64);
            }
#pragma unroll
            for (int df = 0; df < DF; ++df)
                *(f32x4*)(jo + (wave * JC + r * 16 + l15) * (D + 4) + df * 16 + g * 4) = oacc[r][df];
            if (g == 0) jm[wave * JC + r * 16 + l15] = make_float2(m_run[r], l);
        }
        __syncthreads();
        int row, head, node;
        if (jc >= JC || !info(c0 + jc, row, head, node)) return;
        float M = -INFINITY, L = 0.f, f[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, jm[w * JC + jc].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 ml = jm[w * JC + jc];
            f[w] = ml.x == -INFINITY ? 0.f : ml.x == M ? 1.f : __builtin_amdgcn_exp2f(ml.x - M);
            L += ml.y * f[w];
        }
        const long col = ((long)row * A.N + node) * A.Hq + head;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int i = 0; i < PER / 4; ++i) {
            const int d = jd + i * TPC * 4;
            f32x4 O = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) O += *(const f32x4*)(jo + (w * JC + jc) * (D + 4) + d) * f[w];
            if (slot < 0) *(uint2*)(A.o + col * D + d) = make_uint2(pack_bf2(O[0] * inv, O[1] * inv), pack_bf2(O[2] * inv, O[3] * inv));
            else *(f32x4*)(A.rec_o + ((long)slot * ncol_all + col) * D + d) = O;
        }
        if (slot >= 0 && tid % TPC == 0) A.rec_ml[(long)slot * ncol_all + col] = make_float2(M, L);
    }
    // no keys: the columns' records say so by their maximum and their sum, and hold no O
    __device__ __forceinline__ void finish_empty(int slot) const {
        int row, head, node;
        if (threadIdx.x < NC * 16 && info(c0 + threadIdx.x, row, head, node))
            A.rec_ml[(long)slot * A.B * A.N * A.Hq + ((long)row * A.N + node) * A.Hq + head] = make_float2(-INFINITY, 0.f);
    }
};

template <int FMT>
__device__ __forceinline__ KeySegment segment_of(const KvView& c, int seq, int hk, int total, int base, int splits, int sp) {
    KeySegment s;
    const long kv = ((long)seq * c.s_seq + (long)hk * c.s_head) * kv_size<FMT>(), ks = (long)seq * c.c_seq + (long)hk * c.c_head;
    s.k = c.k + kv; s.v = c.v + kv; s.ks = c.ks + ks; s.vs = c.vs + ks;
    s.row_b = (int)(c.s_pos * kv_size<FMT>()); s.c_pos = (int)c.c_pos;
    s.total = total; s.base = base;
    const int nt = (total + TK - 1) / TK, per = (nt + splits - 1) / splits;
    s.t0 = sp * per; s.t1 = min(nt, s.t0 + per);
    return s;
}

// rows [r0, r1) of the batch that prompt pr serves
__device__ __forceinline__ void rows_of(const AttnCacheArgs& A, int pr, int& r0, int& r1) {
    r0 = A.row0 ? min(max(A.row0[pr], 0), A.B) : min(pr * A.rows, A.B);
    r1 = A.row0 ? min(max(A.row0[pr + 1], r0), A.B) : min((pr + 1) * A.rows, A.B);
}

// AGAIN: row0 may give a prompt more sequences than the launch was cut for (A.rows); a workgroup then goes on to the columns behind the launch's.  A form of
// its own, for row0 with rows below the batch, because the loop costs registers: 80 rollouts of 12 prompts (8 or 4 each) over 1391 and 16384 positions take
// 26.9 and 122 us with it and 23.0 and 112 without in bf16, 8-bit caches are level (e4m3 27.2 and 55.3, int8 31.5 and 70.8).
template <int FMT, int D, int NCA, int NCB, bool AGAIN>
__global__ __launch_bounds__(256, 2) void attn_cache_kernel(const AttnCacheArgs A) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int rep = A.rep.d;
    const bool role_a = (int)blockIdx.x < A.na;
    // column blocks of one (keys, range) go to one XCD (workgroups are dealt to the 8 XCDs in turn), next to each other: its L2 serves all but the first
    const int idx = role_a ? blockIdx.x : blockIdx.x - A.na, cbs = role_a ? A.cba : A.cbb;
    const int cb = (idx >> 3) % cbs, job = ((idx >> 3) / cbs) * 8 + (idx & 7);
    if (role_a) {
        const int sp = job % A.sa, hk = (job / A.sa) % A.Hkv, pr = job / (A.sa * A.Hkv);
        if (pr >= A.n_prompts) return;
        int r0, r1;
        rows_of(A, pr, r0, r1);
        const int per_row = A.N * rep, ncol = (r1 - r0) * per_row;
        int c0 = cb * 16 * NCA, tid = threadIdx.x;
        if (c0 >= ncol) return;
        const int total = min(max(A.prompt_len[pr], 0), A.prompt.cap);
        const KeySegment s = segment_of<FMT>(A.prompt, pr, hk, total, total, A.sa, sp);
        auto info = [&](int c, int& row, int& head, int& node) -> bool {
            const int r = A.per_row(c), x = c - r * per_row;
            row = r0 + r; node = A.rep(x); head = hk * rep + x - node * rep;
            return c < ncol;
        };
        do {
            if (AGAIN) asm volatile("" : "+v"(tid));      // (addresses from the lane's number are worked out anew, not kept from round to round)
            Columns<FMT, D, NCA, 4, decltype(info)> W(A, info, smem, c0, tid);
            if (s.t0 >= s.t1) W.finish_empty(sp);
            else {
                const int first = s.t0 + W.wave;
                if (first < s.t1) W.fetch(s, first);
                W.load_queries();
                W.run(s, first);
                W.finish(smem, sp);
            }
            c0 += A.cba * 16 * NCA;
            if (AGAIN) __syncthreads();                   // the join's reads of LDS stay in front of the next columns' writes
        } while (AGAIN && c0 < ncol);
    } else {
        const int sp = job % A.sb, hk = (job / A.sb) % A.Hkv, b = job / (A.sb * A.Hkv);
        if (b >= A.B) return;
        const int ncol = A.N * rep, c0 = cb * 16 * NCB;
        if (c0 >= ncol) return;
        const int base = min(max(A.tail_len[(long)b * A.len_stride], 0), A.tail.cap), total = min(base + A.N, A.tail.cap);
        const KeySegment s = segment_of<FMT>(A.tail, b, hk, total, base, A.sb, sp);
        auto info = [&](int c, int& row, int& head, int& node) -> bool {
            row = b; node = A.rep(c); head = hk * rep + c - node * rep;
            return c < ncol;
        };
        Columns<FMT, D, NCB, 4, decltype(info)> W(A, info, smem, c0);
        if (s.t0 >= s.t1) return W.finish_empty(A.sa + sp);
        const int first = s.t0 + W.wave;
        if (first < s.t1) W.fetch(s, first);
        W.load_queries();
        W.run(s, first);
        W.finish(smem, A.sa + sp);
    }
}

// The prompt that serves row b (-1: none), found by all lanes of a wave at once
__device__ __forceinline__ int prompt_of_row(const AttnCacheArgs& A, int b) {
    if (!A.row0) return min(b / A.rows, A.n_prompts - 1);
    for (int p0 = 0; p0 < A.n_prompts; p0 += 64) {
        const int p = p0 + (threadIdx.x & 63);
        const bool hit = p < A.n_prompts && b >= A.row0[p] && b < A.row0[p + 1];
        const uint64_t m = __ballot(hit);
        if (m) return p0 + __ffsll((unsigned long long)m) - 1;
    }
    return -1;
}

// Short contexts: one workgroup takes the prompt's and the sequence's keys of its columns and writes their output itself.
template <int FMT, int D, int NC>
__global__ __launch_bounds__(512, 2) void attn_cache_solo_kernel(const AttnCacheArgs A) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int rep = A.rep.d, cb = blockIdx.x % A.cbb, hk = (blockIdx.x / A.cbb) % A.Hkv, b = blockIdx.x / (A.cbb * A.Hkv);
    const int ncol = A.N * rep;
    auto info = [&](int c, int& row, int& head, int& node) -> bool {
        row = b; node = A.rep(c); head = hk * rep + c - node * rep;
        return c < ncol;
    };
    Columns<FMT, D, NC, 8, decltype(info)> W(A, info, smem, cb * 16 * NC);
    W.load_queries();
    int nt = 0;
    if (A.n_prompts) {
        const int pr = __builtin_amdgcn_readfirstlane(prompt_of_row(A, b));
        if (pr >= 0) {
            const int total = min(max(A.prompt_len[pr], 0), A.prompt.cap);
            const KeySegment s = segment_of<FMT>(A.prompt, pr, hk, total, total, 1, 0);
            if (W.wave < s.t1) W.fetch(s, W.wave);
            W.run(s, W.wave);
            nt = s.t1;
        }
    }
    if (A.tail.k) {
        const int base = min(max(A.tail_len[(long)b * A.len_stride], 0), A.tail.cap), total = min(base + A.N, A.tail.cap);
        const KeySegment s = segment_of<FMT>(A.tail, b, hk, total, base, 1, 0);
        const int first = (W.wave - nt) & 7;              // the waves go on in turn
        if (first < s.t1) W.fetch(s, first);
        W.run(s, first);
    }
    W.finish(smem, -1);
}

// o = the softmax-weighted join of a column's records; D / 4 lanes per column.  A sequence that no prompt owns has no prompt records.
template <int D>
__global__ __launch_bounds__(256) void attn_cache_join_kernel(const AttnCacheArgs A) {
    constexpr int LPC = D / 4;
    const long ncol = (long)A.B * A.N * A.Hq;
    const long col = (long)blockIdx.x * (256 / LPC) + threadIdx.x / LPC;
    if (col >= ncol) return;
    const int d = (threadIdx.x % LPC) * 4, b = (int)(col / ((long)A.N * A.Hq));
    int first = 0;
    if (A.sa) {
        const int lo = A.row0 ? A.row0[0] : 0, hi = A.row0 ? A.row0[A.n_prompts] : A.n_prompts * A.rows;
        if (b < lo || b >= hi) first = A.sa;
    }
    const int ns = A.sa + A.sb;
    float M = -INFINITY, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = first; s0 < ns; s0 += 8) {              // eight records per memory round trip
        float2 ml[8];
        float4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long at = min(s0 + i, ns - 1) * ncol + col;
            ml[i] = A.rec_ml[at];
            x[i] = *(const float4*)(A.rec_o + at * D + d);
        }
        float m = M;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, ml[i].x);
        const float f0 = M == m ? 1.f : __builtin_amdgcn_exp2f(M - m);
        M = m;
        L *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] *= f0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // an empty range has no O and says so by its sum; NaN scores alone leave the maximum at -infinity too, but a sum of NaN, which stays
            if (s0 + i >= ns || (ml[i].x == -INFINITY && ml[i].y == 0.f)) continue;
            const float f = ml[i].x == M ? 1.f : __builtin_amdgcn_exp2f(ml[i].x - M);
            L += ml[i].y * f;
            O[0] += x[i].x * f; O[1] += x[i].y * f; O[2] += x[i].z * f; O[3] += x[i].w * f;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *(uint2*)(A.o + col * D + d) = make_uint2(pack_bf2(O[0] * inv, O[1] * inv), pack_bf2(O[2] * inv, O[3] * inv));
}

struct AttnPlan {
    int solo, nca, ncb, cba, cbb, sa, sb;
    long cols;
};

// How a launch is cut, from the shapes alone (the capacities stand for the lengths, which only the device knows; half of the tail's, which fills up while a
// rollout runs).
// Short contexts go in one launch, whose 8 waves per workgroup walk all keys of its columns and which fills the card once 256 of them (one per CU) are
// there.  Its bound counts 128-byte key rows per workgroup; both sides measured, one launch | two, e4m3, D = 128 unless said otherwise:
//   up to 64 workgroups    7.8 |  8.5 us at 700 positions,   9.4 |  8.5 at 1000 (1 x 2 and 1 x 8 rollouts; bf16 crosses at 400)
//   up to 192             10.0 | 11.5 us at 1013,           13.3 | 12.9 at 1513 (1 x 4 trees of 15)
//   up to 384             14.2 | 16.1 us at 1903 (8 x 8 rollouts), 21.3 | 23.4 at 3064 (trees of 64), D = 64 16.5 | 17.6 at 3005
//   more                  13.4 | 14.1 us at 400, but 10 to 20 % slower from 700 on at 512: a second round of workgroups
// 16 columns per workgroup while these are no more than the CUs (narrow 256: 14.2 us, with 32 columns 16.8; narrow 384, D = 64: 13.6 | 11.9).
// Others: of the widths (16 or 32 columns) and numbers of key ranges (sa, sb) the one whose estimate (us) is least: 512 workgroups run at once (two per CU), one
// costs a constant and its 32-key tiles per wave, a record of a column its bytes.  The constants were fitted to 2964 launches of 96 settings (1 to 16
// prompts of equal and of falling lengths, 4 to 4096 columns, 1300 to 30000 positions, all formats): the choice is 3.6 % behind the best of them in the mean,
// 15 % at worst.
// (8 waves per workgroup here too: level with 4 for single long prompts, 2 to 20 % behind elsewhere, so this form has 4.)
AttnPlan plan_attn(const spacer_kv_cache* prompt, const spacer_kv_cache* tail, int rows, int B, int N, int Hq) {
    const spacer_kv_cache* c = prompt ? prompt : tail;
    const long rep = Hq / c->kv_heads, cb = N * rep, ca = prompt ? rows * cb : 0, most = ca > cb ? ca : cb;
    const long positions = (long)(prompt ? prompt->capacity : 0) + (tail ? tail->capacity : 0), narrow = (long)B * c->kv_heads * cdiv(cb, 16);
    AttnPlan p = {};
    p.cols = (long)B * N * Hq;
    const long key_rows = positions * c->head_dim * (c->format == KV_BF16 ? 2 : 1) / 128;
    p.solo = key_rows <= (narrow <= 64 ? 900 : narrow <= 192 ? 1400 : narrow <= 384 ? 3000 : 600);
    if (p.solo) {
        p.ncb = cb <= 16 || narrow <= 256 ? 1 : 2;
        p.cbb = cdiv(cb, 16 * p.ncb);
        return p;
    }
    static const int ranges[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
    const double once = 6.7, tile = c->head_dim == 64 ? 0.8 : 1, ta = prompt ? prompt->capacity / (4.0 * TK) : 0, tb = tail ? tail->capacity / (8.0 * TK) : 0;      // tiles per wave
    double best = 1e300;
    for (int nc = 1; nc <= (most > 16 ? 2 : 1); ++nc) {
        const int ncb = cb <= 16 ? 1 : nc, cba = prompt ? cdiv(ca, 16 * nc) : 0, cbb = tail ? cdiv(cb, 16 * ncb) : 0;
        const double ja = (prompt ? (double)prompt->n_seq : 0) * c->kv_heads * cba, jb = (double)B * c->kv_heads * cbb;
        for (int ia = 0; ia < 10; ++ia) {
            const int sa = prompt ? ranges[ia] : 0;
            if (ia > 0 && (!prompt || ta < sa)) break;
            for (int sb = tail ? 1 : 0; sb <= (tail ? 4 : 0); sb = sb ? 2 * sb : 1) {
                if (sb > 1 && tb < sb) break;
                const double a = sa ? ceil(ta / sa) * (0.17 + 0.42 * nc) * tile : 0, b = sb ? ceil(tb / sb) * (0.17 + 0.42 * ncb) * tile : 0;
                const double work = (ja * sa * (once + a) + jb * sb * (once + b)) / 512, longest = a > b ? a : b;
                double t = work > longest ? work : longest;
                if (ja * sa + jb * sb > 512) t += 0.19 * (once + (sa && sb ? (a < b ? a : b) : a + b));
                t += 0.59e-4 * p.cols * (sa + sb) + 0.55 * cdiv(sa + sb, 8);
                if (t < best) { best = t; p.nca = nc; p.ncb = ncb; p.cba = cba; p.cbb = cbb; p.sa = sa; p.sb = sb; }
            }
        }
    }
    return p;
}

}  // namespace

static FastDiv fast_div(unsigned d) {
    FastDiv f = {0, 0, d};
    while ((1u << f.s) < d) ++f.s;
    f.m = (unsigned)((1ull << (31 + f.s)) / d) + 1;
    return f;
}

static int check_attn(const spacer_kv_cache* prompt, const spacer_kv_cache* tail, int rows, int B, int N, int Hq) {
    SP_REQUIRE(prompt || tail, SPACER_EINVAL, "attn_cache: no cache");
    if (prompt)
        if (int rc = spacer_check_kv_cache(prompt, "attn_cache")) return rc;
    if (tail)
        if (int rc = spacer_check_kv_cache(tail, "attn_cache")) return rc;
    SP_REQUIRE(!prompt || !tail || (prompt->format == tail->format && prompt->kv_heads == tail->kv_heads && prompt->head_dim == tail->head_dim),
               SPACER_EINVAL, "attn_cache: prompt and tail caches differ in format, kv_heads or head_dim");
    const spacer_kv_cache* c = prompt ? prompt : tail;
    SP_REQUIRE(B >= 0 && N >= 1 && N <= 64, SPACER_EINVAL, "attn_cache: %d sequences, %d nodes (1 .. 64)", B, N);
    SP_REQUIRE(Hq > 0 && Hq % c->kv_heads == 0, SPACER_EINVAL, "attn_cache: %d query heads over %d kv heads", Hq, c->kv_heads);
    SP_REQUIRE(!prompt || rows > 0, SPACER_EINVAL, "attn_cache: rows = %d per prompt", rows);
    SP_REQUIRE(!tail || tail->n_seq == B, SPACER_EINVAL, "attn_cache: tail cache of %d sequences, %d queries", tail ? tail->n_seq : 0, B);
    SP_REQUIRE((long)B * N * Hq <= 0x3fffffffL && (long)rows * N * Hq <= 0x3fffffffL, SPACER_EINVAL, "attn_cache: too many queries");
    return SPACER_OK;
}

extern "C" long spacer_attn_cache_workspace_bytes(const spacer_kv_cache* prompt, const spacer_kv_cache* tail, int rows, int B, int N, int Hq) {
    if (check_attn(prompt, tail, rows, B, N, Hq)) return -1;
    const AttnPlan p = plan_attn(prompt, tail, rows, B, N, Hq);
    const int D = prompt ? prompt->head_dim : tail->head_dim;
    return (p.sa + p.sb) * p.cols * (D + 2) * 4L;
}

extern "C" int spacer_attn_cache(const void* q, long q_ld, const spacer_kv_cache* prompt, const int* prompt_len, const int* row0, int rows,
                                 const spacer_kv_cache* tail, const int* tail_len, int len_per_seq, const int64_t* tree, int tree_per_seq, void* o,
                                 int B, int N, int Hq, float scale, void* workspace, long workspace_bytes, spacer_stream_t stream) {
    if (int rc = check_attn(prompt, tail, rows, B, N, Hq)) return rc;
    if (B == 0) return SPACER_OK;
    const spacer_kv_cache* c = prompt ? prompt : tail;
    const int D = c->head_dim, Hkv = c->kv_heads;
    SP_REQUIRE(q && o && (((uintptr_t)q | (uintptr_t)o) & 15) == 0 && q_ld % 8 == 0, SPACER_EINVAL, "attn_cache: q and o rows must start at multiples of 16 bytes");
    SP_REQUIRE(scale > 0.f && scale < INFINITY, SPACER_EINVAL, "attn_cache: scale %g must be a positive number", (double)scale);
    SP_REQUIRE(!prompt || prompt_len, SPACER_EINVAL, "attn_cache: prompt_len required");
    SP_REQUIRE(!prompt || row0 || (long)prompt->n_seq * rows == B, SPACER_EINVAL, "attn_cache: %d prompts x %d rows, %d sequences", prompt ? prompt->n_seq : 0, rows, B);
    SP_REQUIRE(!tail || tail_len, SPACER_EINVAL, "attn_cache: tail_len required");
    const AttnPlan p = plan_attn(prompt, tail, rows, B, N, Hq);
    const long need = (p.sa + p.sb) * p.cols * (D + 2) * 4L;
    SP_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), SPACER_ENOMEM, "attn_cache: workspace of %ld bytes, %ld needed",
               workspace ? workspace_bytes : 0L, need);
    AttnCacheArgs A = {};
    A.q = (const bf16_t*)q; A.q_ld = q_ld;
    if (prompt) { A.prompt = spacer_kv_view(prompt); A.n_prompts = prompt->n_seq; }
    if (tail) A.tail = spacer_kv_view(tail);
    A.prompt_len = prompt_len; A.tail_len = tail_len; A.row0 = row0; A.tree = tree;
    A.len_stride = len_per_seq ? 1 : 0; A.tree_stride = tree_per_seq ? N : 0;
    A.rows = rows; A.B = B; A.N = N; A.Hq = Hq; A.Hkv = Hkv;
    A.sa = p.sa; A.sb = p.sb; A.cba = p.cba; A.cbb = p.cbb;
    A.scale = scale;
    A.rep = fast_div(Hq / Hkv);
    A.per_row = fast_div(N * (Hq / Hkv));
    A.rec_o = (float*)workspace;
    A.rec_ml = (float2*)(A.rec_o + (p.sa + p.sb) * p.cols * D);
    A.o = (bf16_t*)o;
    hipStream_t s = (hipStream_t)stream;
    if (p.solo) {
        const long n = (long)B * Hkv * p.cbb;
        SP_REQUIRE(n <= 0x7fffffffL, SPACER_EINVAL, "attn_cache: too many workgroups");
#define LAUNCH(F, DD, NC)                                                                                                                           \
    do {                                                                                                                                            \
        constexpr int lds = lds_bytes(kv_size<F>(), DD, NC, 8);                                                                                         \
        static const hipError_t once = hipFuncSetAttribute((const void*)attn_cache_solo_kernel<F, DD, NC>, hipFuncAttributeMaxDynamicSharedMemorySize, lds); \
        (void)once;                                                                                                                                 \
        hipLaunchKernelGGL((attn_cache_solo_kernel<F, DD, NC>), dim3((unsigned)n), dim3(512), lds, s, A);                                            \
    } while (0)
#define CALL(F, DD)                                                                                                                                 \
    do {                                                                                                                                            \
        if (p.ncb == 1) LAUNCH(F, DD, 1);                                                                                                           \
        else LAUNCH(F, DD, 2);                                                                                                                      \
    } while (0)
        KV_DISPATCH(c, CALL);
#undef CALL
#undef LAUNCH
        SP_CHECK_LAUNCH();
        return SPACER_OK;
    }
    const long ja = prompt ? (long)prompt->n_seq * Hkv * p.sa : 0, jb = tail ? (long)B * Hkv * p.sb : 0;
    const long na = (ja + 7) / 8 * 8 * p.cba, nb = (jb + 7) / 8 * 8 * p.cbb;
    SP_REQUIRE(na + nb <= 0x7fffffffL, SPACER_EINVAL, "attn_cache: too many workgroups");
    A.na = (int)na;
    const bool again = row0 && rows < B;
#define LAUNCH_AS(F, DD, NA, NB, AGAIN)                                                                                                             \
    do {                                                                                                                                            \
        constexpr int lds = lds_bytes(kv_size<F>(), DD, NA > NB ? NA : NB, 4);                                                                          \
        static const hipError_t once = hipFuncSetAttribute((const void*)attn_cache_kernel<F, DD, NA, NB, AGAIN>, hipFuncAttributeMaxDynamicSharedMemorySize, lds); \
        (void)once;                                                                                                                                 \
        hipLaunchKernelGGL((attn_cache_kernel<F, DD, NA, NB, AGAIN>), dim3((unsigned)(na + nb)), dim3(256), lds, s, A);                              \
    } while (0)
#define LAUNCH(F, DD, NA, NB)                                                                                                                       \
    do {                                                                                                                                            \
        if (again) LAUNCH_AS(F, DD, NA, NB, true);                                                                                                  \
        else LAUNCH_AS(F, DD, NA, NB, false);                                                                                                       \
    } while (0)
#define CALL(F, DD)                                                                                                                                 \
    do {                                                                                                                                            \
        if (p.nca == 1) LAUNCH(F, DD, 1, 1);                                                                                                        \
        else if (p.ncb == 1) LAUNCH(F, DD, 2, 1);                                                                                                   \
        else LAUNCH(F, DD, 2, 2);                                                                                                                   \
    } while (0)
    KV_DISPATCH(c, CALL);
#undef CALL
#undef LAUNCH
#undef LAUNCH_AS
    if (D == 128) hipLaunchKernelGGL(attn_cache_join_kernel<128>, dim3(cdiv(p.cols, 8)), dim3(256), 0, s, A);
    else hipLaunchKernelGGL(attn_cache_join_kernel<64>, dim3(cdiv(p.cols, 16)), dim3(256), 0, s, A);
    SP_CHECK_LAUNCH();
    return SPACER_OK;
}
