// Shared device helpers of the 8-bit paged cache (tq_kv8_*.hip): the tile, its codes and their values.
//
// A tile holds block_size tokens of one (physical block, KV head): block_size * 128 codes and one fp32
// scale, a power of two.  Every conversion between the two is then exact but for the one rounding to the
// code: x / scale, code * scale and a change of scale are changes of exponent (the rounding shows only where an
// e4m3 code becomes subnormal, and for int8), results do not depend on how a division rounds, and
// appending rows one at a time requantises a block at most once per doubling of its largest value.
#pragma once

#include "tq_common.h"

constexpr int kKv8ScaleBytes = 16;  // fp32 scale and padding behind a tile's codes

typedef _Float16 kv8_half2 __attribute__((ext_vector_type(2)));

template <int ENC>
struct Kv8Code;

template <>
struct Kv8Code<TQ_E4M3> {
    // smallest e with top <= 448 * 2^e: 448 = 1.75 * 2^8, so one is carried where top's mantissa is over 0.75
    static __device__ __forceinline__ int exponent(uint32_t top_bits) { return (int)((top_bits + 0x1fffffu) >> 23) - 127 - 8; }
    // four codes of values times inv, the first in the low byte; ODD: some may not be finite
    template <bool ODD>
    static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d, float inv) {
        a = clamp<ODD>(a * inv);
        b = clamp<ODD>(b * inv);
        c = clamp<ODD>(c * inv);
        d = clamp<ODD>(d * inv);
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
    // (only infinities are outside; NaN stays)
    template <bool ODD>
    static __device__ __forceinline__ float clamp(float x) {
        const float y = __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
        return ODD && x == x ? y : x;
    }
    static __device__ __forceinline__ float value(uint32_t w, int i) {
        return i == 0   ? __builtin_amdgcn_cvt_f32_fp8((int)w, 0)
               : i == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 1)
               : i == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 2)
                        : __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
    // fp16 of codes 2h and 2h + 1 of w, times s (a power of two)
    static __device__ __forceinline__ kv8_half2 half2(uint32_t w, int h, float s) {
        return h == 0 ? __builtin_bit_cast(kv8_half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false))
                      : __builtin_bit_cast(kv8_half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true));
    }
};

template <>
struct Kv8Code<TQ_INT8> {
    // 127 = 1.984375 * 2^6
    static __device__ __forceinline__ int exponent(uint32_t top_bits) { return (int)((top_bits + 0x1ffffu) >> 23) - 127 - 6; }
    // x * inv + 1.5 * 2^23 holds the nearest whole number (ties to even) in its low bits
    template <bool ODD>
    static __device__ __forceinline__ uint32_t code(float x, float inv) {
        if (ODD) x = __builtin_amdgcn_fmed3f(x == x ? x * inv : 0.f, -127.f, 127.f);
        return __float_as_uint(__builtin_fmaf(x, ODD ? 1.f : inv, 12582912.f));
    }
    template <bool ODD>
    static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d, float inv) {
        const uint32_t lo = __builtin_amdgcn_perm(code<ODD>(b, inv), code<ODD>(a, inv), 0x0c0c0400u);
        return __builtin_amdgcn_perm(code<ODD>(d, inv), code<ODD>(c, inv), 0x04000c0cu) | lo;
    }
    static __device__ __forceinline__ float value(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }
    // The byte b = code + 128 under the exponent byte 0x64 is the fp16 number 1024 + b; s * (that) - 1152 s is
    // exact in one fused step (1152 s is a 4-bit multiple of a power of two).
    static __device__ __forceinline__ kv8_half2 half2(uint32_t w, int h, float s) {
        const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, h == 0 ? 0x04010400u : 0x04030402u);
        const _Float16 hs = (_Float16)s, hb = (_Float16)(-1152.f * s);
        return __builtin_elementwise_fma(__builtin_bit_cast(kv8_half2, x), kv8_half2{hs, hs}, kv8_half2{hb, hb});
    }
};

// 2^e as fp32, -126 <= e <= 127
__device__ __forceinline__ float kv8_exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// ---- attention over the tiles: what the decode and prefill kernels share ----
constexpr float kKv8NegInf = -__builtin_huge_valf();
constexpr float kKv8None = -3.4e38f;  // exponent base of a row that has seen no token
constexpr float kKv8Far = 4194304.f;  // 2^22: scores from here on have no room for a base beside the largest one
constexpr int kKv8MaxLen = 0x7fff0000;  // tokens of a sequence
constexpr float kKv8Log2e = 1.4426950408889634f;

struct Kv8Attn {
    tq_kv8_attn_args a;
    tq_udiv tpb_div;  // 16-token tiles per block
    tq_udiv group_div;
    int tpb, group, cap;  // cap: tokens a block table can hold
    int workers;          // at most
    float* ws_acc;        // [slot][row][128]: a piece's output, divided by its sum
    float* ws_ml;         // [slot][row][2]: exponent base (log2), sum
    int* ends;            // decode: [segment][2], the waves with its first and its last step
    // a window with sinks, and accumulated weights (tq_kv8_window_args)
    int window, sinks;    // (no window: one of 2^31 - 1 tokens)
    float* mass;
    int64_t mass_stride_block, mass_stride_head;
    float* scores;        // decode: [segment][most_steps][2 tiles][group][16], log2 units
    float* ws_me;         // decode: [slot][row][2]: exponent base (log2) and unrounded sum of every piece
    int most_steps;
};

// first token of the window of a query that sees `seen` tokens without one (below 0: a row before its sequence's start)
__device__ __forceinline__ int kv8_window_from(int seen, int window) { return seen > window ? seen - window : 0; }

// The steps of 32 tokens that hold what the positions first .. last see (first's window begins at lo, last sees the
// tokens below hi): steps 0 .. ns - 1 of the sinks, then b0 .. ; n in all.
struct Kv8Span {
    int lo, ns, b0, n;
    // the sequence's step that is number j here
    __device__ __forceinline__ int step(int j) const { return j < ns ? j : j + b0 - ns; }
};
__device__ __forceinline__ Kv8Span kv8_span(int lo, int hi, int sinks) {
    Kv8Span r;
    r.lo = lo;
    r.ns = (int)(((uint32_t)(sinks < lo ? sinks : lo) + 31) >> 5);
    r.b0 = lo >> 5 > r.ns ? lo >> 5 : r.ns;
    r.n = hi > 0 ? r.ns + (int)(((uint32_t)hi + 31) >> 5) - r.b0 : 0;
    return r;
}

// The factor +-2^k that brings a query row with the largest |x| m to [1, 4), and 2^-k.  Rows that are all zero or
// not finite keep k = 0.
__device__ __forceinline__ float kv8_query_factor(float m, bool negate, float& back) {
    const uint32_t b = __float_as_uint(m) >> 23;
    int k = 127 - (int)b;
    if (b == 0 || b == 255) k = 0;
    k = k > 126 ? 126 : k < -126 ? -126 : k;
    back = kv8_exp2i(-k);
    return negate ? -kv8_exp2i(k) : kv8_exp2i(k);
}
// x * f as fp16; with FINE, lo gets what the rounding left
template <bool FINE>
__device__ __forceinline__ void kv8_query_half(const float (&x)[32], float f, tq_half8 (&hi)[4], tq_half8 (&lo)[4]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float y = x[i] * f;
        hi[i >> 3][i & 7] = (_Float16)y;
        if (FINE) lo[i >> 3][i & 7] = (_Float16)(y - (float)hi[i >> 3][i & 7]);
    }
}

// 16 elements from element off on and 16 from off + second on (16-byte aligned)
__device__ __forceinline__ void kv8_load32(const void* base, int64_t off, int second, int dt, float (&x)[32]) {
    if (dt == TQ_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 v = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off + (i < 4 ? 0 : second - 16))[i];
            x[4 * i] = v.x;
            x[4 * i + 1] = v.y;
            x[4 * i + 2] = v.z;
            x[4 * i + 3] = v.w;
        }
    } else {
        tq_u32x4 raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            raw[i] = reinterpret_cast<const tq_u32x4*>(static_cast<const uint16_t*>(base) + off + (i < 2 ? 0 : second - 16))[i];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t b = (raw[i >> 3][(i >> 1) & 3] >> (16 * (i & 1))) & 0xffffu;
            x[i] = dt == TQ_BF16 ? tq_bf16_to_f32(b) : tq_f16_to_f32(b);
        }
    }
}

typedef __bf16 kv8_bf162 __attribute__((ext_vector_type(2)));

// N (a multiple of 4) consecutive elements to element off (8-byte aligned for 16-bit types, N = 4)
template <int N>
__device__ __forceinline__ void kv8_store(void* base, int64_t off, int dt, const float* o) {
    if (dt == TQ_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(base) + off);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) d[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        return;
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
        w[i] = dt == TQ_BF16 ? __builtin_bit_cast(uint32_t, kv8_bf162{(__bf16)o[2 * i], (__bf16)o[2 * i + 1]})
                             : __builtin_bit_cast(uint32_t, kv8_half2{(_Float16)o[2 * i], (_Float16)o[2 * i + 1]});
    uint16_t* d = static_cast<uint16_t*>(base) + off;
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i)
            reinterpret_cast<tq_u32x4*>(d)[i] = tq_u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    } else {
        *reinterpret_cast<tq_u32x2*>(d) = tq_u32x2{w[0], w[1]};
    }
}

// fp16 pairs of p; with FINE, lo gets the remainders
template <bool FINE>
__device__ __forceinline__ void kv8_prob8(const float (&p)[8], tq_half8& hi, tq_half8& lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = (_Float16)p[i];
        if (FINE) lo[i] = (_Float16)(p[i] - (float)hi[i]);
    }
}

// Their sum in fp32: of the numbers that the product with V sees, so that the rounding of a probability that
// dominates its row cancels.
template <bool FINE>
__device__ __forceinline__ float kv8_sum8(const float (&p)[8], const tq_half8& hi) {
    if (FINE) return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    const kv8_half2 one = {(_Float16)1.f, (_Float16)1.f};
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = __builtin_amdgcn_fdot2(kv8_half2{hi[2 * k], hi[2 * k + 1]}, one, sum, false);
    return sum;
}

// A tile's V scale relative to the largest (a power of two); below the smallest fp16 number it counts as zero
__device__ __forceinline__ float kv8_relative(float s, float inv) {
    const float r = s * inv;
    return r < 5.9604645e-8f ? 0.f : r;
}

// The same from the difference of their exponents
__device__ __forceinline__ float kv8_step(int d) { return d < -24 ? 0.f : kv8_exp2i(d); }
// A scale from its fp32 exponent field (0: zero)
__device__ __forceinline__ float kv8_scale(int e) { return __uint_as_float((uint32_t)e << 23); }

// Eight fp16 of two code words, four values each, times sa and sb
template <int ENC>
__device__ __forceinline__ tq_half8 kv8_half8(uint32_t a, uint32_t b, float sa, float sb) {
    const kv8_half2 x0 = Kv8Code<ENC>::half2(a, 0, sa), x1 = Kv8Code<ENC>::half2(a, 1, sa);
    const kv8_half2 x2 = Kv8Code<ENC>::half2(b, 0, sb), x3 = Kv8Code<ENC>::half2(b, 1, sb);
    return tq_half8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

// N more pieces of a cut segment into the running mean a with exponent base M (none yet: -inf) and sum l; a piece has base
// mp (-inf: no piece), sum lp and mean v; Mn is the largest of all bases
template <int N>
__device__ __forceinline__ void kv8_join(float& M, float& l, float4& a, float Mn, const float (&mp)[N], const float (&lp)[N],
                                         const float4 (&v)[N]) {
    float w[N];
    l *= M == kKv8NegInf ? 0.f : __builtin_amdgcn_exp2f(M - Mn);
    float sum = l;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        w[k] = mp[k] == kKv8NegInf ? 0.f : __builtin_amdgcn_exp2f(mp[k] - Mn) * lp[k];
        sum += w[k];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float keep = l * inv;
    a.x *= keep;
    a.y *= keep;
    a.z *= keep;
    a.w *= keep;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float f = w[k] * inv;
        a.x = __builtin_fmaf(f, v[k].x, a.x);
        a.y = __builtin_fmaf(f, v[k].y, a.y);
        a.z = __builtin_fmaf(f, v[k].z, a.z);
        a.w = __builtin_fmaf(f, v[k].w, a.w);
    }
    M = Mn;
    l = sum;
}

// The word's bytes of the first n of its four tokens
__device__ __forceinline__ uint32_t kv8_keep(int n) { return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }

// 0x80 in the bytes that are an e4m3 NaN
__device__ __forceinline__ uint32_t kv8_nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// host: checks that decode and prefill share, and the derived fields
int tq_kv8_attn_setup(const tq_kv8_attn_args* a, Kv8Attn* p);
// host: the same with a window and accumulated weights
int tq_kv8_window_setup(const tq_kv8_window_args* a, Kv8Attn* p);
// host: compute units of the current device (0: unknown)
int tq_kv8_cus();
