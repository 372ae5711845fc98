// Prefill / extend attention over the 8-bit paged caches: several query tokens per sequence (tiles: tq_kv8.h).
//
// A row is one (new token, query head of the GQA group) pair, token-major; a workgroup takes 128 rows of a
// (sequence, KV head), each of its 4 waves 32 of them, and walks the keys in steps of 32 (two 16-token tiles).
// MFMA layout, lane l, n = l % 32, h = l / 32:
//   S^T [32 tokens x 32 rows] = K . Q^T      8 x mfma_f32_32x32x16_f16; slice c covers dims 64h + 8c + (0..7), so the
//                                            lane's operand is 64 bytes of token n
//   O^T [dim 4m + d][row] += V^T . P^T       4 x mfma_f32_32x32x16_f16 per tile, k = 8h + i being tokens 4h + i and 8 + 4h + i:
//                                            what S^T leaves in the lane, and two words of the values layout
#include "tq_kv8.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;

template <int ENC, bool FINE>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_prefill_kernel(Kv8Attn p, int row_blocks) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hkv = p.a.num_kv_heads;
    // longest row blocks first
    const int per = p.a.num_seqs * hkv;
    const int rb = row_blocks - 1 - (int)(blockIdx.x / (uint32_t)per);
    const int s = (int)(blockIdx.x % (uint32_t)per) / hkv, kh = (int)(blockIdx.x % (uint32_t)per) % hkv;
    const int q0 = p.a.cu_seqlens_q[s];
    int nq = p.a.cu_seqlens_q[s + 1] - q0;
    const int64_t first = (int64_t)rb * kRows + wave * kWaveRows;
    const int computed = nq < p.a.max_q_len ? nq : p.a.max_q_len;
    if (first >= (int64_t)computed * p.group) return;
    int L = p.a.seq_lens[s];
    L = L < p.cap ? L : p.cap;
    L = L > 0 ? L : 0;
    const bool causal = p.a.flags & TQ_PREFILL_CAUSAL;

    // this lane's row
    const uint32_t row = (uint32_t)first + n;
    const int i = (int)tq_udiv_apply(row, p.group_div);
    const int head = kh * p.group + (int)(row - (uint32_t)i * (uint32_t)p.group);
    const bool real = i < computed;
    int seen = causal ? L - nq + i + 1 : L;  // tokens that the row sees
    seen = real && seen > 0 ? (seen < L ? seen : L) : 0;
    // of the wave's rows: most and least
    int last = (int)tq_udiv_apply((uint32_t)first + kWaveRows - 1, p.group_div);
    last = last < computed ? last : computed - 1;
    int most = causal ? L - nq + last + 1 : L;
    most = most > 0 ? most : 0;
    const int least = causal ? L - nq + (int)tq_udiv_apply((uint32_t)first, p.group_div) + 1 : L;

    tq_half8 qh[8], ql[8];
    float c1;
    {
        float x[32];
        tq_half8 hi[4], lo[4];
        // both halves are scaled by the row's factor: the larger of the two maxima decides
        const int64_t off = (int64_t)(q0 + (real ? i : 0)) * p.a.q_stride_token + (int64_t)(real ? head : 0) * p.a.q_stride_head + 64 * h;
        float y[32], m = 0.f;
        kv8_load32(p.a.q, off, p.a.q_dtype, x);
        kv8_load32(p.a.q, off + 32, p.a.q_dtype, y);
#pragma unroll
        for (int k = 0; k < 32; ++k) m = fmaxf(m, fmaxf(__builtin_fabsf(x[k]), __builtin_fabsf(y[k])));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        float back;
        const float f = kv8_query_factor(m, p.a.sm_scale < 0.f, back);
        kv8_query_half<FINE>(x, f, hi, lo);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            qh[k] = hi[k];
            ql[k] = lo[k];
        }
        kv8_query_half<FINE>(y, f, hi, lo);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            qh[4 + k] = hi[k];
            ql[4 + k] = lo[k];
        }
        c1 = __builtin_fabsf(p.a.sm_scale) * kKv8Log2e * back;
    }

    const uint8_t* kb = static_cast<const uint8_t*>(p.a.k_cache) + kh * p.a.k_stride_head;
    const uint8_t* vb = static_cast<const uint8_t*>(p.a.v_cache) + kh * p.a.v_stride_head;
    const int32_t* bt = p.a.block_tables + s * p.a.block_table_stride;
    const int last_tile = L > 0 ? (L - 1) >> 4 : 0;
    const uint32_t scale_at = (uint32_t)p.a.block_size * TQ_HEAD_DIM;

    float M = kKv8None, lsum = 0.f, vref = 0.f;
    f32x16 acc[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[d][v] = 0.f;

    const int steps = (most + 31) >> 5;
    for (int j = 0; j < steps; ++j) {
        int64_t kt[2], vt[2];
        float ks[2], vs[2];
        int nv[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int ti = 2 * j + t, tc = ti < last_tile ? ti : last_tile;
            const int b = (int)tq_udiv_apply((uint32_t)tc, p.tpb_div);
            int blk = __builtin_amdgcn_readfirstlane(bt[b]);
            nv[t] = L - 16 * ti;
            if ((uint32_t)blk >= (uint64_t)p.a.num_blocks) {
                blk = 0;
                nv[t] = 0;
            }
            const int64_t in = (int64_t)(tc - p.tpb * b) * (16 * TQ_HEAD_DIM);
            ks[t] = *reinterpret_cast<const float*>(kb + blk * p.a.k_stride_block + scale_at);
            vs[t] = *reinterpret_cast<const float*>(vb + blk * p.a.v_stride_block + scale_at);
            kt[t] = blk * p.a.k_stride_block + in;
            vt[t] = blk * p.a.v_stride_block + in;
        }
        // ---- scores ----
        tq_u32x4 kw[4], vw[2][2];
        {
            const tq_u32x4* src = reinterpret_cast<const tq_u32x4*>(kb + (n < 16 ? kt[0] : kt[1]) + 128 * (n & 15) + 64 * h);
#pragma unroll
            for (int c = 0; c < 4; ++c) kw[c] = src[c];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    vw[t][k] = *reinterpret_cast<const tq_u32x4*>(vb + vt[t] + 512 * (h + 2 * k) + 16 * n);
        }
        f32x16 sc;
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const tq_half8 a = kv8_half8<ENC>(kw[c >> 1][2 * (c & 1)], kw[c >> 1][2 * (c & 1) + 1], 1.f, 1.f);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], sc, 0, 0, 0);
            if (FINE) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[c], sc, 0, 0, 0);
        }
        float sv[16];
        const float f[2] = {c1 * ks[0], c1 * ks[1]};
#pragma unroll
        for (int v = 0; v < 16; ++v) sv[v] = sc[v] * f[v >> 3];
        if (32 * j + 32 > least || nv[0] < 16 || nv[1] < 16) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int t = v >> 3, in = 8 * ((v >> 2) & 1) + 4 * h + (v & 3);
                if (in >= nv[t] || 32 * j + 16 * t + in >= seen) sv[v] = kKv8NegInf;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (nv[t] <= 0) vs[t] = 0.f;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t keep = kv8_keep(nv[t] - 8 * k - 4 * h);
#pragma unroll
                    for (int d = 0; d < 4; ++d) vw[t][k][d] &= keep;
                }
            }
        }
        // ---- online softmax ----
        float mx = sv[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) mx = fmaxf(mx, sv[v]);
        if (__builtin_amdgcn_ballot_w64(mx > M)) {
            const float Mn = fmaxf(M, fmaxf(mx, __shfl_xor(mx, 32, 64)));
            const float alpha = __builtin_amdgcn_exp2f(M - Mn);
            lsum *= alpha;
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= alpha;
            M = Mn;
        }
        const float vmax = fmaxf(vs[0], vs[1]);
        if (vmax > vref) {  // wave-uniform
            const float r = vref / vmax;
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= r;
            vref = vmax;
        }
        const float rv = vref > 0.f ? 1.f / vref : 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float pr[8];
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                pr[v] = __builtin_amdgcn_exp2f(sv[8 * t + v] - M);
                lsum += pr[v];
            }
            tq_half8 ph, pl;
            kv8_prob8<FINE>(pr, ph, pl);
            const float vf = kv8_relative(vs[t], rv);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const tq_half8 a = kv8_half8<ENC>(vw[t][0][d], vw[t][1][d], vf, vf);
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph, acc[d], 0, 0, 0);
                if (FINE) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl, acc[d], 0, 0, 0);
            }
        }
    }

    // ---- acc[d][4q + r] is dim 32q + 16h + 4r + d of row n ----
    const float l = lsum + __shfl_xor(lsum, 32, 64);
    if (!real) return;
    const float inv = l == 0.f ? 0.f : vref / l;
    const int64_t out = (int64_t)(q0 + i) * p.a.out_stride_token + (int64_t)head * p.a.out_stride_head + 16 * h;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float o[16];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < 4; ++d) o[4 * r + d] = acc[d][4 * q + r] * inv;
        kv8_store<16>(p.a.out, out + 32 * q, p.a.out_dtype, o);
    }
}

}  // namespace

extern "C" int64_t tq_kv8_prefill_workspace_bytes(int num_seqs, int max_q_len, int num_q_heads, int num_kv_heads) {
    return 0;
}

extern "C" int tq_kv8_prefill(const tq_kv8_attn_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    Kv8Attn p = {};
    const int rc = tq_kv8_attn_setup(a, &p);
    if (rc != TQ_OK) return rc;
    if (a->max_q_len < 0 || (a->flags & ~TQ_PREFILL_CAUSAL)) return TQ_ERR_INVALID_ARGUMENT;
    if (a->num_seqs == 0 || a->max_q_len == 0) return TQ_OK;
    if (!a->q || !a->out || !a->k_cache || !a->v_cache || !a->block_tables || !a->seq_lens || !a->cu_seqlens_q)
        return TQ_ERR_INVALID_ARGUMENT;
    const int64_t rows = (int64_t)a->max_q_len * p.group;
    if (rows > 0x7fffff00) return TQ_ERR_INVALID_ARGUMENT;
    int blocks = (int)((rows + kRows - 1) / kRows);
    const int64_t grid = (int64_t)blocks * a->num_seqs * a->num_kv_heads;
    if (grid > 0x7fffffff) return TQ_ERR_INVALID_ARGUMENT;
    const bool fine = a->q_dtype == TQ_F32 || a->out_dtype == TQ_F32;
    const void* kern = a->encoding == TQ_E4M3 ? (fine ? (const void*)kv8_prefill_kernel<TQ_E4M3, true> : (const void*)kv8_prefill_kernel<TQ_E4M3, false>)
                                              : (fine ? (const void*)kv8_prefill_kernel<TQ_INT8, true> : (const void*)kv8_prefill_kernel<TQ_INT8, false>);
    void* args[] = {&p, &blocks};
    hipError_t e = hipLaunchKernel(kern, dim3((unsigned)grid), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
