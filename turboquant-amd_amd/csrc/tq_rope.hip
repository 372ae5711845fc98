// Rotary positions on query and key rows.
//
// Pair i of a row turns by angle 2 pi * position * turns[i]: (x, y) -> m (x cos - y sin, y cos + x sin).  The
// turns are a product in 64 bits of which the whole part is dropped, so an angle far out is as good as one near
// 0; sine and cosine are then fp32 functions of at most half a turn.  A wave takes a token: lane i
// works out pair i's cosine and sine, LDS deals them, and 8 lanes share a row, each with 16 elements that hold
// whole pairs: chunks of 8 at 8j and rotary_dim / 2 + 8j, or 16 consecutive ones when interleaved.  In
// both, lane j's pairs are 8j .. 8j + 7, so its factors stay in registers for all heads.  Lanes beyond
// rotary_dim / 16 copy.  Rows that this does not fit (rotary_dim not a multiple of 16, unaligned rows) take one
// pair or element per lane.
//
// Bound: memory, each row read and written once: 16384 tokens of 48 + 8 heads in bf16, 470 MB, take 99 us, 4.75 TB/s
// where a large copy moves 4.9 (with loads or stores past the caches it is slower).  64 tokens: 3.6 us of
// latency, behind the caller's own 10.
#include "tq_common.h"

namespace {

constexpr int kWaves = 4;

struct Rope {
    tq_rope_args a;
    int split;    // waves that share a token's rows
    int in_place; // elements behind rotary_dim need no copy
};

__device__ __forceinline__ double position(const Rope& p, int64_t t) {
    return p.a.position_dtype == TQ_I64 ? (double)static_cast<const int64_t*>(p.a.positions)[t]
                                        : (double)static_cast<const int32_t*>(p.a.positions)[t];
}
// magnitude * (cos, sin) of pair i at position pos
__device__ __forceinline__ float2 factors(const Rope& p, double pos, int i) {
    // (the fused step rounds once, after the whole part is gone, so far positions lose nothing)
    const double t = p.a.turns[i];
    const float r = (float)__builtin_fma(pos, t, -__builtin_rint(pos * t));  // [-1/2, 1/2]
    float s, c;
    sincospif(2.0f * r, &s, &c);
    return make_float2(c * p.a.magnitude, s * p.a.magnitude);
}
__device__ __forceinline__ void rotate(float& x, float& y, float2 f) {
    const float a = __builtin_fmaf(x, f.x, -(y * f.y)), b = __builtin_fmaf(y, f.x, x * f.y);
    x = a;
    y = b;
}

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t off, float* x) {
    if (DT == TQ_F32) {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
        const float4 a = s[0], b = s[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const tq_u32x4 w = *reinterpret_cast<const tq_u32x4*>(static_cast<const uint16_t*>(base) + off);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t b = (w[k >> 1] >> (16 * (k & 1))) & 0xffffu;
            x[k] = DT == TQ_BF16 ? tq_bf16_to_f32(b) : tq_f16_to_f32(b);
        }
    }
}
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t off, const float* x) {
    if (DT == TQ_F32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(base) + off);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        tq_u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = DT == TQ_BF16 ? (tq_f32_to_bf16_bits(x[2 * k]) | tq_f32_to_bf16_bits(x[2 * k + 1]) << 16)
                                 : tq_pack_half2(x[2 * k], x[2 * k + 1]);
        *reinterpret_cast<tq_u32x4*>(static_cast<uint16_t*>(base) + off) = w;
    }
}

// row r of the token: q's heads, then k's
__device__ __forceinline__ void row_at(const Rope& p, int64_t t, int r, const void*& in, void*& out, int64_t& io, int64_t& oo) {
    const bool isq = r < p.a.q_heads;
    const int h = isq ? r : r - p.a.q_heads;
    in = isq ? p.a.q : p.a.k;
    out = isq ? p.a.q_out : p.a.k_out;
    io = isq ? t * p.a.q_stride_token + h * p.a.q_stride_head : t * p.a.k_stride_token + h * p.a.k_stride_head;
    oo = isq ? t * p.a.q_out_stride_token + h * p.a.q_out_stride_head : t * p.a.k_out_stride_token + h * p.a.k_out_stride_head;
}

template <int DT, bool INTERLEAVED>
__global__ __launch_bounds__(64 * kWaves) void rope_kernel(Rope p) {
    __shared__ float2 s_f[kWaves][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * kWaves + wave;
    const int64_t t = unit / p.split;
    const int part = (int)(unit - t * p.split);
    if (t >= p.a.num_tokens) return;
    if (lane < p.a.rotary_dim / 2) s_f[wave][lane] = factors(p, position(p, t), lane);
    __builtin_amdgcn_wave_barrier();  // (LDS of this wave alone: its accesses stay in order)
    const int j = lane & 7, sub = lane >> 3;
    const bool turns = 16 * j < p.a.rotary_dim;
    float2 f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = turns ? s_f[wave][8 * j + i] : make_float2(1.f, 0.f);
    const int half = p.a.rotary_dim >> 1;
    const int a0 = INTERLEAVED || !turns ? 16 * j : 8 * j;
    const int a1 = INTERLEAVED || !turns ? 16 * j + 8 : half + 8 * j;
    const int rows = p.a.q_heads + p.a.k_heads;
    for (int r = 8 * part + sub; r < rows; r += 8 * p.split) {
        const void* in;
        void* out;
        int64_t io, oo;
        row_at(p, t, r, in, out, io, oo);
        if (!turns && p.in_place) continue;
        float x[16];
        load8<DT>(in, io + a0, x);
        load8<DT>(in, io + a1, x + 8);
        if (turns) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (INTERLEAVED)
                    rotate(x[2 * i], x[2 * i + 1], f[i]);
                else
                    rotate(x[i], x[8 + i], f[i]);
            }
        }
        store8<DT>(out, oo + a0, x);
        store8<DT>(out, oo + a1, x + 8);
    }
}

// any even rotary_dim, any alignment: lane i takes pair i, then an element behind them
__global__ __launch_bounds__(64 * kWaves) void rope_any_kernel(Rope p) {
    const int lane = threadIdx.x & 63;
    const int wave = threadIdx.x >> 6;
    const int64_t unit = (int64_t)blockIdx.x * kWaves + wave;
    const int64_t t = unit / p.split;
    const int part = (int)(unit - t * p.split);
    if (t >= p.a.num_tokens) return;
    const int half = p.a.rotary_dim >> 1;
    const bool turns = lane < half;
    const float2 f = turns ? factors(p, position(p, t), lane) : make_float2(1.f, 0.f);
    const int a = p.a.interleaved ? 2 * lane : lane, b = p.a.interleaved ? 2 * lane + 1 : half + lane;
    const int rows = p.a.q_heads + p.a.k_heads;
    for (int r = part; r < rows; r += p.split) {
        const void* in;
        void* out;
        int64_t io, oo;
        row_at(p, t, r, in, out, io, oo);
        if (turns) {
            float x = tq_load1(in, io + a, p.a.dtype), y = tq_load1(in, io + b, p.a.dtype);
            rotate(x, y, f);
            tq_store1(out, oo + a, p.a.dtype, x);
            tq_store1(out, oo + b, p.a.dtype, y);
        }
        if (!p.in_place)
            for (int i = p.a.rotary_dim + lane; i < TQ_HEAD_DIM; i += 64)
                tq_store1(out, oo + i, p.a.dtype, tq_load1(in, io + i, p.a.dtype));
    }
}

}  // namespace

extern "C" int tq_rope(const tq_rope_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    if (a->head_dim != TQ_HEAD_DIM) return TQ_ERR_HEAD_DIM;
    if (a->dtype != TQ_F32 && a->dtype != TQ_F16 && a->dtype != TQ_BF16) return TQ_ERR_DTYPE;
    if (a->position_dtype != TQ_I32 && a->position_dtype != TQ_I64) return TQ_ERR_DTYPE;
    if (a->num_tokens < 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads > (1 << 20) || a->k_heads > (1 << 20) ||
        a->rotary_dim < 2 || a->rotary_dim > TQ_HEAD_DIM || a->rotary_dim % 2)
        return TQ_ERR_INVALID_ARGUMENT;
    if (a->num_tokens == 0 || a->q_heads + a->k_heads == 0) return TQ_OK;
    if (!a->positions || !a->turns || (a->q_heads && (!a->q || !a->q_out)) || (a->k_heads && (!a->k || !a->k_out)))
        return TQ_ERR_INVALID_ARGUMENT;
    const uintptr_t size = a->dtype == TQ_F32 ? 4 : 2;
    uintptr_t ptrs = 0;
    int64_t el = 0;
    bool same = true;
    if (a->q_heads) {
        ptrs |= (uintptr_t)a->q | (uintptr_t)a->q_out;
        el |= a->q_stride_token | a->q_stride_head | a->q_out_stride_token | a->q_out_stride_head;
        same = same && a->q == a->q_out;
        if (a->q == a->q_out && (a->q_stride_token != a->q_out_stride_token || a->q_stride_head != a->q_out_stride_head))
            return TQ_ERR_INVALID_ARGUMENT;
    }
    if (a->k_heads) {
        ptrs |= (uintptr_t)a->k | (uintptr_t)a->k_out;
        el |= a->k_stride_token | a->k_stride_head | a->k_out_stride_token | a->k_out_stride_head;
        same = same && a->k == a->k_out;
        if (a->k == a->k_out && (a->k_stride_token != a->k_out_stride_token || a->k_stride_head != a->k_out_stride_head))
            return TQ_ERR_INVALID_ARGUMENT;
    }
    if (ptrs % size || (uintptr_t)a->turns % 8 || (uintptr_t)a->positions % (a->position_dtype == TQ_I64 ? 8 : 4))
        return TQ_ERR_ALIGNMENT;
    Rope p = {};
    p.a = *a;
    p.in_place = same;
    const bool wide = a->rotary_dim % 16 == 0 && ptrs % 16 == 0 && el % 8 == 0;
    // Few tokens: a token's rows over several waves, one pass of 8 rows each, up to about two waves per SIMD
    const int rows = a->q_heads + a->k_heads;
    const int passes = wide ? (rows + 7) / 8 : rows;
    int64_t split = 2048 / a->num_tokens;
    split = split < 1 ? 1 : split < passes ? split : passes;
    p.split = (int)split;
    const int64_t units = a->num_tokens * split;
    const int64_t grid = (units + kWaves - 1) / kWaves;
    if (grid > 0xffffff) return TQ_ERR_INVALID_ARGUMENT;  // (a launch's threads stay below 2^32)
    const void* kern = (const void*)rope_any_kernel;
    if (wide) {
#define TQ_ROPE(D) \
    if (a->dtype == D) kern = a->interleaved ? (const void*)rope_kernel<D, true> : (const void*)rope_kernel<D, false>;
        TQ_ROPE(TQ_F32) TQ_ROPE(TQ_F16) TQ_ROPE(TQ_BF16)
#undef TQ_ROPE
    }
    void* args[] = {&p};
    hipError_t e = hipLaunchKernel(kern, dim3((unsigned)grid), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
