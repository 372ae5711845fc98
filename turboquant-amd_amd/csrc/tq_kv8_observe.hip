// Accumulated attention weights of prompts over the 8-bit paged caches, from their last queries (tiles: tq_kv8.h).
//
//   mass[t] = (t new ? 0 : mass[t]) + sum over rows r of 2^(s[r][t] - M[r]) / l[r],  s = sm log2(e) q_r . k_t
//
// A row is one (query, head of the GQA group) pair; 128 rows are a block.  Two kernels, both with S^T [32 tokens x 32
// rows] = K . Q^T on mfma_f32_32x32x16_f16 (lane l, n = l % 32, h = l / 32; operands as in tq_kv8_prefill.hip) and the
// block's query operands in LDS, where a workgroup's four waves share them:
//   kv8_observe_stats_kernel  M and l of a row block over a chunk of the steps that its rows see
//   kv8_observe_sum_kernel    a wave keeps the keys of 64 tokens in registers and goes over all row blocks; the sums over
//                             rows stay in registers until the end, so that no two waves add to a number and the
//                             order of the sums is fixed
// Products are done twice: keeping the scores would move 4 bytes a (row, token) twice, where a token's keys
// are 128 bytes for all rows.
#include "tq_kv8.h"

namespace {

constexpr int kWaves = 4;
constexpr int kRows = 128;      // of a row block: 32 a wave to load
constexpr int kTokens = 64;     // of a wave of the sums
constexpr int kSpread = 1024;   // workgroups of the statistics, at least, where the keys allow

struct Observe {
    Kv8Attn at;
    int max_q, last, blocks, chunks, chunk_steps;  // blocks: of a segment, at most
    float2* part;                                  // [segment][block][chunk][128]: M, l
};

struct Rows {  // a sequence's observed rows
    int q0, nq, L, count, first;  // rows; number of the first observed new token
};
__device__ __forceinline__ Rows rows_of(const Observe& p, int s) {
    Rows r;
    r.q0 = __builtin_amdgcn_readfirstlane(p.at.a.cu_seqlens_q[s]);
    const int nq = __builtin_amdgcn_readfirstlane(p.at.a.cu_seqlens_q[s + 1]) - r.q0;
    const int L = __builtin_amdgcn_readfirstlane(p.at.a.seq_lens[s]);
    r.nq = nq > 0 ? nq : 0;
    r.L = L < 0 ? 0 : L < p.at.cap ? L : p.at.cap;
    int n = r.nq < p.last ? r.nq : p.last;
    n = n < p.max_q ? n : p.max_q;
    r.first = r.nq - n;
    r.count = n * p.at.group;
    return r;
}
// position of row `row`'s query (below 0 where the sequence is shorter than its new tokens)
__device__ __forceinline__ int position(const Observe& p, const Rows& r, int row) {
    return r.L - r.nq + r.first + (int)tq_udiv_apply((uint32_t)row, p.at.group_div);
}
__device__ __forceinline__ int last_row(const Rows& r, int rb) {
    const int x = rb * kRows + kRows - 1;
    return x < r.count - 1 ? x : r.count - 1;
}
// the steps that a row block sees
__device__ __forceinline__ Kv8Span span_of(const Observe& p, const Rows& r, int rb) {
    const int lo = kv8_window_from(position(p, r, rb * kRows) + 1, p.at.window), hi = position(p, r, last_row(r, rb)) + 1;
    return kv8_span(lo, hi, p.at.sinks);
}

// A row block's operands in LDS: row tile rt, slice k of lane l at q[(rt * 8 + k) * 64 + l]
template <bool FINE>
struct Block {
    tq_half8 hi[4 * 8 * 64];
    tq_half8 lo[FINE ? 4 * 8 * 64 : 1];
    float c1[kRows], M[kRows], inv[kRows];
    int seen[kRows];
};
// Wave w loads rows 32 w ..; a row that `use` denies becomes zeros
template <bool FINE, typename Use>
__device__ __forceinline__ void load_rows(const Observe& p, const Rows& r, int kh, int rb, Block<FINE>& b, Use use) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5, rt = threadIdx.x >> 6;
    const tq_kv8_attn_args& a = p.at.a;
    const int row = rb * kRows + 32 * rt + n;
    const bool real = row < r.count;
    const int i = real ? (int)tq_udiv_apply((uint32_t)row, p.at.group_div) : 0;
    const int head = kh * p.at.group + (real ? row - i * p.at.group : 0);
    const int64_t off = (int64_t)(r.q0 + r.first + i) * a.q_stride_token + (int64_t)head * a.q_stride_head + 16 * h;
    float x[32], y[32], m = 0.f;
    kv8_load32(a.q, off, 32, a.q_dtype, x);
    kv8_load32(a.q, off + 64, 32, a.q_dtype, y);
#pragma unroll
    for (int k = 0; k < 32; ++k) m = fmaxf(m, fmaxf(__builtin_fabsf(x[k]), __builtin_fabsf(y[k])));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    float back;
    float f = kv8_query_factor(m, a.sm_scale < 0.f, back);
    if (!real || !use(32 * rt + n)) {
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] = y[k] = 0.f;
    }
    tq_half8 hi[2][4], lo[2][4];
    kv8_query_half<FINE>(x, f, hi[0], lo[0]);
    kv8_query_half<FINE>(y, f, hi[1], lo[1]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        b.hi[(rt * 8 + k) * 64 + lane] = hi[k >> 2][k & 3];
        if (FINE) b.lo[(rt * 8 + k) * 64 + lane] = lo[k >> 2][k & 3];
    }
    if (h == 0) {
        const int pos = position(p, r, row);
        b.c1[32 * rt + n] = __builtin_fabsf(a.sm_scale) * kKv8Log2e * back;
        b.seen[32 * rt + n] = real && pos >= 0 ? pos + 1 : 0;
    }
}

// The 32 tokens of step js: keys as fp16 operands, scales and rows in use of both tiles
struct Keys {
    tq_half8 k[8];
    float ks[2];
    int nv[2];
};
template <int ENC, bool CLEAN>
__device__ __forceinline__ void load_keys(const Observe& p, int s, int kh, int L, int js, Keys& out) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const tq_kv8_attn_args& a = p.at.a;
    const uint8_t* kb = static_cast<const uint8_t*>(a.k_cache) + kh * a.k_stride_head;
    const uint8_t* tile[2];
    const int last_tile = L > 0 ? (L - 1) >> 4 : 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int ti = 2 * js + t, tc = ti < last_tile ? ti : last_tile;
        const int b = (int)tq_udiv_apply((uint32_t)tc, p.at.tpb_div);
        int blk = __builtin_amdgcn_readfirstlane(a.block_tables[s * a.block_table_stride + b]);
        int nv = L - 16 * ti;
        nv = nv < 16 ? (nv > 0 ? nv : 0) : 16;
        if ((uint32_t)blk >= (uint64_t)a.num_blocks) {
            blk = 0;
            nv = 0;
        }
        tile[t] = kb + blk * a.k_stride_block + (int64_t)(tc - p.at.tpb * b) * (16 * TQ_HEAD_DIM);
        out.ks[t] = *reinterpret_cast<const float*>(kb + blk * a.k_stride_block + (int64_t)a.block_size * TQ_HEAD_DIM);
        out.nv[t] = nv;
    }
    const tq_u32x4* src = reinterpret_cast<const tq_u32x4*>((n < 16 ? tile[0] : tile[1]) + 128 * (n & 15) + 16 * h);
    tq_u32x4 w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = src[2 * c];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        uint32_t u = w[c >> 1][2 * (c & 1)], v = w[c >> 1][2 * (c & 1) + 1];
        if (CLEAN && ENC == TQ_E4M3) {
            // (NaN codes become 0: the rows that see one count for nothing)
            const uint32_t x = kv8_nan_bytes(u), y = kv8_nan_bytes(v);
            u &= ~((x << 1) - (x >> 7));
            v &= ~((y << 1) - (y >> 7));
        }
        out.k[c] = kv8_half8<ENC>(u, v, 1.f, 1.f);
    }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Scores in log2 units of a step's 32 tokens and row tile rt: lane n's row, token 16 t + 8 (v / 4) + 4h + v % 4 in
// sv[8 t + v]; -inf where the row does not see the token.
template <bool FINE>
__device__ __forceinline__ void scores(const Observe& p, const Block<FINE>& b, const Keys& k, int rt, int js, bool edge, float (&sv)[16]) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    f32x16 sc;
#pragma unroll
    for (int v = 0; v < 16; ++v) sc[v] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.k[c], b.hi[(rt * 8 + c) * 64 + lane], sc, 0, 0, 0);
        if (FINE) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.k[c], b.lo[(rt * 8 + c) * 64 + lane], sc, 0, 0, 0);
    }
    const float c1 = b.c1[32 * rt + n], f[2] = {c1 * k.ks[0], c1 * k.ks[1]};
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        sv[v] = sc[v] * f[v >> 3];
        asm("" : "+v"(sv[v]));  // (rounded here in both kernels: far scores then differ from M as they should)
    }
    if (edge) {
        const int seen = b.seen[32 * rt + n], lo = kv8_window_from(seen, p.at.window);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int at = 32 * js + 16 * t + 4 * h;
            const int upto = seen - at < k.nv[t] - 4 * h ? seen - at : k.nv[t] - 4 * h;
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                const int x = 8 * (v >> 2) + (v & 3);
                if (x >= upto || (x >= p.at.sinks - at && x < lo - at)) sv[8 * t + v] = kKv8NegInf;
            }
        }
    }
}
// some row of block rb may not see all tokens of step js
__device__ __forceinline__ bool at_edge(const Observe& p, const Rows& r, int rb, int js, const Keys& k) {
    const int least = position(p, r, rb * kRows) + 1, lo = kv8_window_from(position(p, r, last_row(r, rb)) + 1, p.at.window);
    return 32 * js + 32 > least || (32 * js < lo && 32 * js + 32 > p.at.sinks) || k.nv[0] + k.nv[1] != 32;
}

// (M, l) and (m, x) joined
__device__ __forceinline__ void join(float& M, float& l, float m, float x) {
    const float Mn = fmaxf(M, m);
    l = l * __builtin_amdgcn_exp2f(M - Mn) + x * __builtin_amdgcn_exp2f(m - Mn);
    M = Mn;
}

template <int ENC, bool FINE>
__global__ __launch_bounds__(64 * kWaves) void kv8_observe_stats_kernel(Observe p) {
    __shared__ Block<FINE> b;
    __shared__ float2 s_part[kWaves][kRows];
    const int lane = threadIdx.x & 63, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t x = blockIdx.x;
    const int chunk = (int)(x % (uint32_t)p.chunks);
    x /= (uint32_t)p.chunks;
    const int rb = (int)(x % (uint32_t)p.blocks);
    const uint32_t seg = x / (uint32_t)p.blocks;
    const int s = (int)(seg / (uint32_t)p.at.a.num_kv_heads), kh = (int)seg - s * p.at.a.num_kv_heads;
    const Rows r = rows_of(p, s);
    if (rb * kRows >= r.count) return;
    const Kv8Span span = span_of(p, r, rb);
    const int j0 = chunk * p.chunk_steps, j1 = j0 + p.chunk_steps < span.n ? j0 + p.chunk_steps : span.n;
    float M[4], l[4];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
        M[rt] = kKv8None;
        l[rt] = 0.f;
    }
    if (j0 < j1) {
        load_rows<FINE>(p, r, kh, rb, b, [](int) { return true; });
        __syncthreads();
        for (int j = j0 + wave; j < j1; j += kWaves) {
            const int js = span.step(j);
            Keys k;
            load_keys<ENC, false>(p, s, kh, r.L, js, k);
            const bool edge = at_edge(p, r, rb, js, k);
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                float sv[16];
                scores<FINE>(p, b, k, rt, js, edge, sv);
                float m = M[rt];
#pragma unroll
                for (int v = 0; v < 16; ++v) m = fmaxf(m, sv[v]);
                float sum = 0.f;
#pragma unroll
                for (int v = 0; v < 16; ++v) sum += __builtin_amdgcn_exp2f(sv[v] - m);
                l[rt] = l[rt] * __builtin_amdgcn_exp2f(M[rt] - m) + sum;
                M[rt] = m;
            }
        }
    }
#pragma unroll
    for (int rt = 0; rt < 4; ++rt) {
        join(M[rt], l[rt], __shfl_xor(M[rt], 32, 64), __shfl_xor(l[rt], 32, 64));
        if (lane < 32) s_part[wave][32 * rt + n] = make_float2(M[rt], l[rt]);
    }
    __syncthreads();
    if (threadIdx.x < kRows) {
        float2 m = s_part[0][threadIdx.x];
        for (int w = 1; w < kWaves; ++w) join(m.x, m.y, s_part[w][threadIdx.x].x, s_part[w][threadIdx.x].y);
        p.part[(((int64_t)seg * p.blocks + rb) * p.chunks + chunk) * kRows + threadIdx.x] = m;
    }
}

template <int ENC, bool FINE>
__global__ __launch_bounds__(64 * kWaves) void kv8_observe_sum_kernel(Observe p, int token_blocks) {
    __shared__ Block<FINE> b;
    __shared__ float s_sum[kWaves][kTokens];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t seg = blockIdx.x / (uint32_t)token_blocks;
    const int s = (int)(seg / (uint32_t)p.at.a.num_kv_heads), kh = (int)seg - s * p.at.a.num_kv_heads;
    const Rows r = rows_of(p, s);
    const int t_wg = (int)(blockIdx.x - seg * (uint32_t)token_blocks) * (kWaves * kTokens);
    if (r.nq == 0 || t_wg >= r.L) return;
    const int t0 = t_wg + wave * kTokens;
    Keys k[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) load_keys<ENC, true>(p, s, kh, r.L, (t0 >> 5) + i, k[i]);
    float acc[2][16];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][v] = 0.f;
    const int nrb = (r.count + kRows - 1) / kRows;
    for (int rb = 0; rb < nrb; ++rb) {
        // (rows that see none of the workgroup's tokens; the same for all its waves)
        const Kv8Span span = span_of(p, r, rb);
        const int hi = position(p, r, last_row(r, rb)) + 1;
        if (t_wg >= hi || (t_wg + kWaves * kTokens <= span.lo && t_wg >= p.at.sinks)) continue;
        __syncthreads();
        // ---- the rows' statistics, then their operands ----
        if (threadIdx.x < kRows) {
            float M = kKv8None, l = 0.f;
            const float2* part = p.part + ((int64_t)seg * p.blocks + rb) * p.chunks * kRows + threadIdx.x;
            const int used = (span.n + p.chunk_steps - 1) / p.chunk_steps;
            for (int c = 0; c < used; ++c) join(M, l, part[(int64_t)c * kRows].x, part[(int64_t)c * kRows].y);
            const bool good = rb * kRows + (int)threadIdx.x < r.count && l > 0.f && l < __builtin_huge_valf();
            b.M[threadIdx.x] = good ? M : 0.f;
            b.inv[threadIdx.x] = good ? 1.f / l : 0.f;
        }
        __syncthreads();
        load_rows<FINE>(p, r, kh, rb, b, [&](int row) { return b.inv[row] > 0.f; });
        __syncthreads();
        if (t0 >= hi) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int js = (t0 >> 5) + i;
            const bool edge = at_edge(p, r, rb, js, k[i]);
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                float sv[16];
                scores<FINE>(p, b, k[i], rt, js, edge, sv);
                const float M = b.M[32 * rt + n], inv = b.inv[32 * rt + n];
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][v] = __builtin_fmaf(__builtin_amdgcn_exp2f(sv[v] - M), inv, acc[i][v]);
            }
        }
    }
    // ---- sums over the rows: the 32 lanes of a half ----
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            float x = acc[i][v];
            for (int m = 1; m < 32; m <<= 1) x += __shfl_xor(x, m, 64);
            if (n == v) s_sum[wave][32 * i + 16 * (v >> 3) + 8 * ((v & 7) >> 2) + 4 * h + (v & 3)] = x;
        }
    __syncthreads();
    const int t = t0 + lane;
    if (t >= r.L) return;
    const int tb = (int)tq_udiv_apply((uint32_t)(t >> 4), p.at.tpb_div);
    const int blk = p.at.a.block_tables[s * p.at.a.block_table_stride + tb];
    if ((uint32_t)blk >= (uint64_t)p.at.a.num_blocks) return;
    float* dst = p.at.mass + blk * p.at.mass_stride_block + kh * p.at.mass_stride_head + (t - tb * p.at.a.block_size);
    *dst = (t >= r.L - r.nq ? 0.f : *dst) + s_sum[wave][lane];
}

// row blocks of a segment, and chunks of the statistics, at most
void counts(int64_t segs, int64_t max_q, int64_t last, int64_t group, int64_t& blocks, int64_t& chunks) {
    blocks = ((max_q < last ? max_q : last) * group + kRows - 1) / kRows;
    chunks = blocks * segs >= kSpread ? 1 : (kSpread + blocks * segs - 1) / (blocks * segs);
}

}  // namespace

extern "C" int64_t tq_kv8_observe_workspace_bytes(int num_seqs, int max_q_len, int last, int num_q_heads, int num_kv_heads) {
    if (num_seqs <= 0 || max_q_len <= 0 || last <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return 0;
    int64_t blocks, chunks;
    const int64_t segs = (int64_t)num_seqs * num_kv_heads;
    counts(segs, max_q_len, last, num_q_heads / num_kv_heads, blocks, chunks);
    return segs * blocks * chunks * kRows * 8;
}

extern "C" int tq_kv8_observe(const tq_kv8_window_args* w, tq_stream_t stream) {
    if (!w) return TQ_ERR_INVALID_ARGUMENT;
    const tq_kv8_attn_args* a = &w->attn;
    Observe p = {};
    const int rc = tq_kv8_window_setup(w, &p.at);
    if (rc != TQ_OK) return rc;
    if (a->max_q_len < 0 || a->max_seq_len < 0 || w->last <= 0 || a->flags != TQ_PREFILL_CAUSAL) return TQ_ERR_INVALID_ARGUMENT;
    p.at.cap = p.at.cap < a->max_seq_len ? p.at.cap : a->max_seq_len;
    if (a->num_seqs == 0 || a->max_q_len == 0 || p.at.cap == 0) return TQ_OK;
    if (!a->q || !a->k_cache || !w->mass || !a->block_tables || !a->seq_lens || !a->cu_seqlens_q) return TQ_ERR_INVALID_ARGUMENT;
    p.max_q = a->max_q_len;
    p.last = w->last;
    const int64_t segs = (int64_t)a->num_seqs * a->num_kv_heads;
    int64_t blocks, chunks;
    counts(segs, p.max_q, p.last, p.at.group, blocks, chunks);
    const int64_t need = tq_kv8_observe_workspace_bytes(a->num_seqs, a->max_q_len, w->last, a->num_q_heads, a->num_kv_heads);
    if (!a->workspace || (uintptr_t)a->workspace % 256 || a->workspace_bytes < need) return TQ_ERR_WORKSPACE;
    // the steps that a row block sees, at most (its rows lie over 128 / group tokens)
    int64_t steps = ((int64_t)p.at.cap + 31) / 32;
    if (w->window) {
        const int64_t m = ((int64_t)w->window + kRows / p.at.group + 1 + 31) / 32 + 1 + ((int64_t)w->sinks + 31) / 32;
        steps = m < steps ? m : steps;
    }
    // (a wave takes two steps at least)
    const int64_t most = (steps + 2 * kWaves - 1) / (2 * kWaves);
    chunks = chunks < most ? chunks : most;
    const int64_t token_blocks = ((int64_t)p.at.cap + kWaves * kTokens - 1) / (kWaves * kTokens);
    // (a launch's threads stay below 2^32, row numbers below 2^31)
    if (segs > 0xffffff || blocks > 0xffffff || segs * blocks > 0xffffff || segs * blocks * chunks > 0xffffff || segs * token_blocks > 0xffffff)
        return TQ_ERR_INVALID_ARGUMENT;
    p.blocks = (int)blocks;
    p.chunk_steps = (int)((steps + chunks - 1) / chunks);
    p.chunks = (int)((steps + p.chunk_steps - 1) / p.chunk_steps);
    p.part = static_cast<float2*>(a->workspace);
    const bool fine = a->q_dtype == TQ_F32;
    const void *stats = nullptr, *sum = nullptr;
#define TQ_OBSERVE(E, F)                                          \
    if (a->encoding == E && fine == F) {                          \
        stats = (const void*)kv8_observe_stats_kernel<E, F>;      \
        sum = (const void*)kv8_observe_sum_kernel<E, F>;          \
    }
    TQ_OBSERVE(TQ_E4M3, false) TQ_OBSERVE(TQ_E4M3, true) TQ_OBSERVE(TQ_INT8, false) TQ_OBSERVE(TQ_INT8, true)
#undef TQ_OBSERVE
    int tb = (int)token_blocks;
    void* args[] = {&p, &tb};
    hipError_t e = hipLaunchKernel(stats, dim3((unsigned)(segs * blocks * p.chunks)), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess) e = hipLaunchKernel(sum, dim3((unsigned)(segs * token_blocks)), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
