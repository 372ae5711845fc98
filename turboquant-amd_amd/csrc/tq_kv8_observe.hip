// Accumulated attention weights of prompts over the 8-bit paged caches, from their last queries (tiles: tq_kv8.h).
//
//   mass[t] = (t new ? 0 : mass[t]) + sum over rows r of 2^(s[r][t] - M[r]) / l[r],  s = sm log2(e) q_r . k_t
//
// A row is one (query, head of the GQA group) pair; 256 rows (128 with FINE) are a block, whose query operands stay in LDS
// while a workgroup's four waves go over steps of 32 tokens.  S^T [32 tokens x 32 rows] = K . Q^T on
// mfma_f32_32x32x16_f16 (lane l, n = l % 32, h = l / 32; operands as in tq_kv8_prefill.hip):
//   kv8_observe_stats_kernel  M and l of a row block over a chunk of the steps that its rows see
//   kv8_observe_sum_kernel    a range of tokens and a group of row blocks: each wave adds its steps' weights over the rows, the
//                             sums lie in LDS, one wave to a token, so that their order is fixed; one group of row blocks
//                             goes to mass at once, several to the workspace and
//   kv8_observe_add_kernel    adds those up
// Products are done twice: keeping the scores would move 4 bytes a (row, token) twice, where a token's keys
// are 128 bytes for all rows.
//
// Bound: few rows by the start (lengths, block table, keys or rows, statistics: a chain of some 12 us in either kernel), many by a
// SIMD's two waves: by counters (the second call below) 990 cycles for 32 x 32 scores in the statistics and 1200 in the sums, of which the
// products take 256 and other vector instructions, the exponentials above all, 550 and 660; the two hardly overlap.  Four prompts of
// 8192 tokens, last 32 queries of 48 / 8 heads: 28 + 32 us (13 GFLOP); 384 to 512 queries of 32 / 8 heads after 1000 to 8000 tokens of two
// sequences: 53 + 70 + 5.  f32 queries: twice the products, 94 and 165 us a call instead of 55 and 113.  Tried: a row tile at a time with four
// waves per SIMD (8 waves a workgroup): 62 -> 67 us and 120 as before; rows of 128 with 64 tokens' keys in registers: 155 and 183.
#include "tq_kv8.h"

namespace {

constexpr int kWaves = 4;
constexpr int kSpread = 512;    // workgroups of a kernel that the device holds at once: more where the work allows
constexpr int kMaxTokens = 512; // of a workgroup of the sums
constexpr int kGroups = 16;     // of row blocks, at most

struct Observe {
    Kv8Attn at;
    int max_q, last, rows, blocks;  // rows of a block; blocks of a segment, at most
    int chunks, chunk_steps;        // of the statistics
    int most_chunks;                // that the workspace has room for: no fewer with more steps
    int tokens, ranges, groups;     // of the sums: tokens of a workgroup, ranges of a segment, groups of row blocks
    float2* part;                   // [segment][block][chunk][rows]: M, l
    float* sums;                    // [segment][group][range][tokens]
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
__device__ __forceinline__ int last_row(const Observe& p, const Rows& r, int rb) {
    const int x = rb * p.rows + p.rows - 1;
    return x < r.count - 1 ? x : r.count - 1;
}
// the steps that a row block sees
__device__ __forceinline__ Kv8Span span_of(const Observe& p, const Rows& r, int rb) {
    const int lo = kv8_window_from(position(p, r, rb * p.rows) + 1, p.at.window), hi = position(p, r, last_row(p, r, rb)) + 1;
    return kv8_span(lo, hi, p.at.sinks);
}

// A row block's operands in LDS: row tile rt, slice k of lane l at hi[(rt * 8 + k) * 64 + l]
template <bool FINE>
struct Block {
    static constexpr int kTiles = FINE ? 4 : 8, kRows = 32 * kTiles;
    tq_half8 hi[kTiles * 8 * 64];
    tq_half8 lo[FINE ? kTiles * 8 * 64 : 1];
    float c1[kRows], M[kRows], inv[kRows];
    int seen[kRows];
};
// Row tile rt by a wave
template <bool FINE>
__device__ __forceinline__ void load_rows(const Observe& p, const Rows& r, int kh, int rb, int rt, Block<FINE>& b) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const tq_kv8_attn_args& a = p.at.a;
    const int row = rb * p.rows + 32 * rt + n;
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
    if (!real) {
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
        // (rows that do not exist: scores of 0 * 0, whatever the row whose place they took)
        b.c1[32 * rt + n] = real ? __builtin_fabsf(a.sm_scale) * kKv8Log2e * back : 0.f;
        b.seen[32 * rt + n] = real && pos >= 0 ? pos + 1 : 0;
    }
}

// 64 tiles of 16 tokens, one per lane: where their keys are, scale, rows in use.  span: 32 steps from number j on
struct Tiles {
    uint32_t lo, hi;
    float ks;
    int nv;
};
__device__ __forceinline__ Tiles tiles_from(const Observe& p, int s, int kh, int L, const Kv8Span& span, int j) {
    const int lane = threadIdx.x & 63;
    const tq_kv8_attn_args& a = p.at.a;
    const uint8_t* kb = static_cast<const uint8_t*>(a.k_cache) + kh * a.k_stride_head;
    const int last_tile = L > 0 ? (L - 1) >> 4 : 0;
    const int ti = 2 * span.step(j + (lane >> 1)) + (lane & 1), tc = ti < last_tile ? ti : last_tile;
    const int b = (int)tq_udiv_apply((uint32_t)tc, p.at.tpb_div);
    int blk = a.block_tables[s * a.block_table_stride + b];
    int nv = L - 16 * ti;
    nv = nv < 16 ? (nv > 0 ? nv : 0) : 16;
    if ((uint32_t)blk >= (uint64_t)a.num_blocks) {
        blk = 0;
        nv = 0;
    }
    const uint8_t* block = kb + blk * a.k_stride_block;
    const uint64_t at = (uint64_t)block + (uint64_t)(tc - p.at.tpb * b) * (16 * TQ_HEAD_DIM);
    return {(uint32_t)at, (uint32_t)(at >> 32), *reinterpret_cast<const float*>(block + (int64_t)a.block_size * TQ_HEAD_DIM), nv};
}
// Codes of the step whose tiles are those of lanes i and i + 1: 16 bytes of token n's dims 32c + 16h .. in w[c]
struct Codes {
    tq_u32x4 w[4];
};
__device__ __forceinline__ Codes load_codes(const Tiles& t, int i) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    auto address = [&](int k) -> uint64_t {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)t.lo, k) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)t.hi, k) << 32;
    };
    const uint64_t a0 = address(i), a1 = address(i + 1);
    // (named as global memory: a load that may be from LDS is waited for with the operands')
    using GlobalWords = const __attribute__((address_space(1))) tq_u32x4*;
    const GlobalWords src = (GlobalWords)((n < 16 ? a0 : a1) + 128 * (n & 15) + 16 * h);
    Codes out;
#pragma unroll
    for (int c = 0; c < 4; ++c) out.w[c] = src[2 * c];
    return out;
}
// scales and rows in use of a step's tiles
struct Step {
    float ks[2];
    int nv[2];
};
__device__ __forceinline__ Step step_of(const Tiles& t, int i) {
    Step x;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        x.ks[k] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(t.ks), i + k));
        x.nv[k] = __builtin_amdgcn_readlane(t.nv, i + k);
    }
    return x;
}
template <int ENC>
__device__ __forceinline__ void convert(const Codes& x, tq_half8 (&k)[8]) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        k[c] = kv8_half8<ENC>(x.w[c >> 1][2 * (c & 1)], x.w[c >> 1][2 * (c & 1) + 1], 1.f, 1.f);
    }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Scores in log2 units of a step's 32 tokens and row tiles rt and rt + 1 (two chains of products): lane n's row, token
// 16 t + 8 (v / 4) + 4h + v % 4 in sv[.][8 t + v]; -inf where the row does not see the token.
template <bool FINE>
__device__ __forceinline__ void scores(const Observe& p, const Block<FINE>& b, const tq_half8 (&k)[8], const Step& x, int rt, int js, bool edge,
                                       float (&sv)[2][16]) {
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    f32x16 sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[i][v] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[c], b.hi[((rt + i) * 8 + c) * 64 + lane], sc[i], 0, 0, 0);
            if (FINE) sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[c], b.lo[((rt + i) * 8 + c) * 64 + lane], sc[i], 0, 0, 0);
        }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float c1 = b.c1[32 * (rt + i) + n], f[2] = {c1 * x.ks[0], c1 * x.ks[1]};
#pragma unroll
        for (int v = 0; v < 16; ++v) {
#pragma clang fp contract(off)
            sv[i][v] = sc[i][v] * f[v >> 3];  // (rounded here in both kernels: far scores then differ from M as they should)
        }
    }
    if (edge) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int seen = b.seen[32 * (rt + i) + n], lo = kv8_window_from(seen, p.at.window);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int at = 32 * js + 16 * t + 4 * h;
                const int upto = seen - at < x.nv[t] - 4 * h ? seen - at : x.nv[t] - 4 * h;
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    const int y = 8 * (v >> 2) + (v & 3);
                    if (y >= upto || (y >= p.at.sinks - at && y < lo - at)) sv[i][8 * t + v] = kKv8NegInf;
                }
            }
        }
    }
}
// some row of block rb may not see all tokens of step js
__device__ __forceinline__ bool at_edge(const Observe& p, const Rows& r, int rb, int js, const Step& x) {
    const int least = position(p, r, rb * p.rows) + 1, lo = kv8_window_from(position(p, r, last_row(p, r, rb)) + 1, p.at.window);
    return 32 * js + 32 > least || (32 * js < lo && 32 * js + 32 > p.at.sinks) || x.nv[0] + x.nv[1] != 32;
}

// (M, l) and (m, x) joined
__device__ __forceinline__ void join(float& M, float& l, float m, float x) {
    const float Mn = fmaxf(M, m);
    l = l * __builtin_amdgcn_exp2f(M - Mn) + x * __builtin_amdgcn_exp2f(m - Mn);
    M = Mn;
}

template <int ENC, bool FINE>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_observe_stats_kernel(Observe p) {
    constexpr int kTiles = Block<FINE>::kTiles, kRows = Block<FINE>::kRows;
    __shared__ Block<FINE> b;
    __shared__ float2 s_part[kWaves][kRows];
    const int lane = threadIdx.x & 63, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t of_chunks = blockIdx.x / (uint32_t)p.chunks;
    const int chunk = (int)(blockIdx.x - of_chunks * (uint32_t)p.chunks);
    const uint32_t seg = of_chunks / (uint32_t)p.blocks;
    const int rb = (int)(of_chunks - seg * (uint32_t)p.blocks);
    const int s = (int)(seg / (uint32_t)p.at.a.num_kv_heads), kh = (int)seg - s * p.at.a.num_kv_heads;
    const Rows r = rows_of(p, s);
    if (rb * kRows >= r.count) return;
    const Kv8Span span = span_of(p, r, rb);
    const int j0 = chunk * p.chunk_steps, j1 = j0 + p.chunk_steps < span.n ? j0 + p.chunk_steps : span.n;
    if (j0 >= j1) return;  // (the sums read the chunks that have steps)
    // row tiles, in pairs: rows that do not exist are zeros
    const int tiles = 2 * ((last_row(p, r, rb) - rb * kRows) / 64 + 1);
    float M[kTiles], l[kTiles];
#pragma unroll
    for (int rt = 0; rt < kTiles; ++rt) {
        M[rt] = kKv8None;
        l[rt] = 0.f;
    }
    Tiles after = tiles_from(p, s, kh, r.L, span, j0);
    for (int rt = wave; rt < tiles; rt += kWaves) load_rows<FINE>(p, r, kh, rb, rt, b);
    __syncthreads();
    for (int jg = j0; jg < j1; jg += 32) {
    const Tiles now = after;
    const int je = jg + 32 < j1 ? jg + 32 : j1;
    if (je < j1) after = tiles_from(p, s, kh, r.L, span, je);
    Codes next = load_codes(now, 2 * wave);
    for (int j = jg + wave; j < je; j += kWaves) {
        const int js = span.step(j), i = 2 * (j - jg);
        tq_half8 k[8];
        convert<ENC>(next, k);
        next = load_codes(now, i + 2 * kWaves < 62 ? i + 2 * kWaves : 62);  // (behind the last: a valid address)
        const Step x = step_of(now, i);
        const bool edge = at_edge(p, r, rb, js, x);
#pragma unroll
        for (int rt = 0; rt < kTiles; rt += 2) {
            if (rt >= tiles) break;
            float sv[2][16];
            scores<FINE>(p, b, k, x, rt, js, edge, sv);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float m = M[rt + i];
#pragma unroll
                for (int v = 0; v < 16; ++v) m = fmaxf(m, sv[i][v]);
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int v = 0; v < 16; ++v) sum[v & 3] += __builtin_amdgcn_exp2f(sv[i][v] - m);
                l[rt + i] = l[rt + i] * __builtin_amdgcn_exp2f(M[rt + i] - m) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                M[rt + i] = m;
            }
        }
    }
    }
#pragma unroll
    for (int rt = 0; rt < kTiles; ++rt) {
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

// mass of token t of a segment, if its table entry is good
__device__ __forceinline__ void put(const Observe& p, const Rows& r, int s, int kh, int t, float sum) {
    const int tb = (int)tq_udiv_apply((uint32_t)(t >> 4), p.at.tpb_div);
    const int blk = p.at.a.block_tables[s * p.at.a.block_table_stride + tb];
    if ((uint32_t)blk >= (uint64_t)p.at.a.num_blocks) return;
    float* dst = p.at.mass + blk * p.at.mass_stride_block + kh * p.at.mass_stride_head + (t - tb * p.at.a.block_size);
    *dst = (t >= r.L - r.nq ? 0.f : *dst) + sum;
}

template <int ENC, bool FINE>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_observe_sum_kernel(Observe p) {
    constexpr int kTiles = Block<FINE>::kTiles, kRows = Block<FINE>::kRows;
    __shared__ Block<FINE> b;
    __shared__ float s_sum[kMaxTokens];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t of_ranges = blockIdx.x / (uint32_t)p.ranges;
    const int range = (int)(blockIdx.x - of_ranges * (uint32_t)p.ranges);
    const uint32_t seg = of_ranges / (uint32_t)p.groups;
    const int group = (int)(of_ranges - seg * (uint32_t)p.groups);
    const int s = (int)(seg / (uint32_t)p.at.a.num_kv_heads), kh = (int)seg - s * p.at.a.num_kv_heads;
    const Rows r = rows_of(p, s);
    const int t0 = range * p.tokens, t1 = t0 + p.tokens < r.L ? t0 + p.tokens : r.L;
    if (r.nq == 0 || t0 >= t1) return;
    for (int i = threadIdx.x; i < p.tokens; i += 64 * kWaves) s_sum[i] = 0.f;
    const int nrb = (r.count + kRows - 1) / kRows;
    const Tiles now = tiles_from(p, s, kh, r.L, Kv8Span{0, 1 << 30, 0, 0}, t0 >> 5);
    // (the last row blocks, which see most tokens, dealt over the groups)
    for (int rb = group; rb < nrb; rb += p.groups) {
        // rows that see none of the range's tokens: the same for all waves
        const Kv8Span span = span_of(p, r, rb);
        const int hi = position(p, r, last_row(p, r, rb)) + 1;
        if (t0 >= hi || (t0 + p.tokens <= span.lo && t0 >= p.at.sinks)) continue;
        const int tiles = 2 * ((last_row(p, r, rb) - rb * kRows) / 64 + 1);
        const int behind = t1 < hi ? t1 : hi;
        int t = t0 + 32 * wave;
        Codes next = load_codes(now, 2 * wave);
        __syncthreads();
        for (int rt = wave; rt < tiles; rt += kWaves) load_rows<FINE>(p, r, kh, rb, rt, b);
        // ---- the rows' statistics ----
        bool bad = false;
        if (threadIdx.x < kRows) {
            float M = kKv8None, l = 0.f;
            const float2* part = p.part + ((int64_t)seg * p.blocks + rb) * p.chunks * kRows + threadIdx.x;
            const int used = (span.n + p.chunk_steps - 1) / p.chunk_steps;
            for (int c = 0; c < used; c += 16) {
                float2 y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = c + i < used ? part[(int64_t)(c + i) * kRows] : make_float2(kKv8None, 0.f);
#pragma unroll
                for (int i = 0; i < 16; ++i) join(M, l, y[i].x, y[i].y);
            }
            const bool real = rb * kRows + (int)threadIdx.x < r.count;
            bad = real && !(l < __builtin_huge_valf());
            const bool good = real && !bad && l > 0.f;
            b.M[threadIdx.x] = good ? M : 0.f;
            b.inv[threadIdx.x] = good ? 1.f / l : 0.f;
        }
        if (__syncthreads_or(bad)) {
            // rows whose weights are not numbers: operands and factors of zeros, which add nothing (a factor that passes fp32's range
            // with a block's scale would make NaN of a lane's sum, and other rows' weights are in it)
            if (threadIdx.x < kRows && !(b.inv[threadIdx.x] > 0.f)) b.c1[threadIdx.x] = 0.f;
            for (int i = threadIdx.x; i < kTiles * 8 * 64; i += 64 * kWaves) {
                const int row = 32 * (i >> 9) + (i & 31);
                if (rb * kRows + row < r.count && !(b.inv[row] > 0.f)) {
                    b.hi[i] = tq_half8{0, 0, 0, 0, 0, 0, 0, 0};
                    if (FINE) b.lo[FINE ? i : 0] = b.hi[i];
                }
            }
            __syncthreads();
        }
        for (; t < behind; t += 32 * kWaves) {
            tq_half8 k[8];
            convert<ENC>(next, k);
            const int lane0 = (t - t0) >> 4;
            next = load_codes(now, lane0 + 2 * kWaves < 62 ? lane0 + 2 * kWaves : 62);
            const Step x = step_of(now, lane0);
            const bool edge = at_edge(p, r, rb, t >> 5, x);
            float acc[16];
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[v] = 0.f;
            for (int rt = 0; rt < tiles; rt += 2) {
                float sv[2][16];
                scores<FINE>(p, b, k, x, rt, t >> 5, edge, sv);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float M = b.M[32 * (rt + i) + n], inv = b.inv[32 * (rt + i) + n];
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[v] = __builtin_fmaf(__builtin_amdgcn_exp2f(sv[i][v] - M), inv, acc[v]);
                }
            }
            // (NaN in a key: all rows that see its token count for nothing)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[v] = fmaxf(acc[v], 0.f);
            // ---- over the half's 32 lanes: each stage halves the lane's values; lane n ends with value n / 2 ----
#pragma unroll
            for (int m = 16; m >= 2; m >>= 1) {
                const bool up = n & m;
#pragma unroll
                for (int v = 0; v < m / 2; ++v) {
                    const float send = up ? acc[v] : acc[v + m / 2], keep = up ? acc[v + m / 2] : acc[v];
                    acc[v] = keep + __shfl_xor(send, m, 64);
                }
            }
            const float sum = acc[0] + __shfl_xor(acc[0], 1, 64);
            const int v = n >> 1;
            if (!(n & 1)) s_sum[t - t0 + 16 * (v >> 3) + 8 * ((v & 7) >> 2) + 4 * h + (v & 3)] += sum;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < t1 - t0; i += 64 * kWaves) {
        if (p.groups == 1) put(p, r, s, kh, t0 + i, s_sum[i]);
        else p.sums[(((int64_t)seg * p.groups + group) * p.ranges + range) * p.tokens + i] = s_sum[i];
    }
}

__global__ __launch_bounds__(256) void kv8_observe_add_kernel(Observe p) {
    const int per = (p.ranges * p.tokens + 255) / 256;
    const uint32_t seg = blockIdx.x / (uint32_t)per;
    const int t = (int)(blockIdx.x - seg * (uint32_t)per) * 256 + (int)threadIdx.x;
    const int s = (int)(seg / (uint32_t)p.at.a.num_kv_heads), kh = (int)seg - s * p.at.a.num_kv_heads;
    const Rows r = rows_of(p, s);
    if (r.nq == 0 || t >= r.L) return;
    float sum = 0.f;
    for (int g = 0; g < p.groups; ++g) sum += p.sums[((int64_t)seg * p.groups + g) * p.ranges * p.tokens + t];
    put(p, r, s, kh, t, sum);
}

// How a call is cut: workgroups of the statistics go by (row block, chunk of its steps), of the sums by (group of row blocks,
// range of tokens).
void cut(Observe& p, int64_t segs, int64_t max_q, int64_t last, int64_t group, bool fine, int64_t len, int64_t steps) {
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    p.rows = fine ? Block<true>::kRows : Block<false>::kRows;
    const int64_t blocks = up((max_q < last ? max_q : last) * group, p.rows);
    p.blocks = (int)(blocks < INT32_MAX ? blocks : INT32_MAX);
    // (a wave takes two steps at least)
    int64_t chunks = up(kSpread, segs * blocks), most = up(steps, 2 * kWaves);
    chunks = chunks < most ? chunks : most;
    p.most_chunks = (int)chunks;
    p.chunk_steps = (int)up(steps, chunks);
    p.chunks = (int)up(steps, p.chunk_steps);
    p.tokens = kMaxTokens;
    while (p.tokens > 32 * kWaves && segs * blocks * up(len, p.tokens) < kSpread) p.tokens /= 2;
    p.ranges = (int)up(len, p.tokens);
    int64_t groups = up(2 * kSpread, segs * p.ranges);
    groups = groups < blocks ? groups : blocks;
    p.groups = (int)(groups < kGroups ? groups : kGroups);
}
int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }
int64_t part_bytes(const Observe& p, int64_t segs) { return align256(segs * p.blocks * p.most_chunks * p.rows * 8); }

}  // namespace

// (steps without a window: with one there are no more chunks)
extern "C" int64_t tq_kv8_observe_workspace_bytes(int num_seqs, int max_q_len, int last, int num_q_heads, int num_kv_heads, int q_dtype,
                                                  int max_seq_len) {
    if (num_seqs <= 0 || max_q_len <= 0 || last <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || max_seq_len <= 0)
        return 0;
    Observe p = {};
    const int64_t segs = (int64_t)num_seqs * num_kv_heads;
    cut(p, segs, max_q_len, last, num_q_heads / num_kv_heads, q_dtype == TQ_F32, max_seq_len, ((int64_t)max_seq_len + 31) / 32);
    return part_bytes(p, segs) + (p.groups > 1 ? segs * p.groups * p.ranges * p.tokens * 4 : 0);
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
    const bool fine = a->q_dtype == TQ_F32;
    const int64_t need = tq_kv8_observe_workspace_bytes(a->num_seqs, a->max_q_len, w->last, a->num_q_heads, a->num_kv_heads, a->q_dtype, p.at.cap);
    if (!a->workspace || (uintptr_t)a->workspace % 256 || a->workspace_bytes < need) return TQ_ERR_WORKSPACE;
    // the steps that a row block sees, at most (its rows lie over rows / group tokens)
    int64_t steps = ((int64_t)p.at.cap + 31) / 32;
    if (w->window) {
        const int64_t m = ((int64_t)w->window + 256 / p.at.group + 1 + 31) / 32 + 1 + ((int64_t)w->sinks + 31) / 32;
        steps = m < steps ? m : steps;
    }
    cut(p, segs, p.max_q, p.last, p.at.group, fine, p.at.cap, steps);
    // (a launch's threads stay below 2^32, row numbers below 2^31)
    if (segs > 0xffffff || p.blocks > 0x7fffff || segs * p.blocks > 0xffffff || segs * p.blocks * p.chunks > 0xffffff ||
        segs * p.ranges * p.groups > 0xffffff || segs * (((int64_t)p.ranges * p.tokens + 255) / 256) > 0xffffff)
        return TQ_ERR_INVALID_ARGUMENT;
    p.part = static_cast<float2*>(a->workspace);
    p.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + part_bytes(p, segs));
    const void *stats = nullptr, *sum = nullptr;
#define TQ_OBSERVE(E, F)                                          \
    if (a->encoding == E && fine == F) {                          \
        stats = (const void*)kv8_observe_stats_kernel<E, F>;      \
        sum = (const void*)kv8_observe_sum_kernel<E, F>;          \
    }
    TQ_OBSERVE(TQ_E4M3, false) TQ_OBSERVE(TQ_E4M3, true) TQ_OBSERVE(TQ_INT8, false) TQ_OBSERVE(TQ_INT8, true)
#undef TQ_OBSERVE
    void* args[] = {&p};
    hipError_t e = hipLaunchKernel(stats, dim3((unsigned)(segs * p.blocks * p.chunks)), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess) e = hipLaunchKernel(sum, dim3((unsigned)(segs * p.groups * p.ranges)), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess && p.groups > 1)
        e = hipLaunchKernel((const void*)kv8_observe_add_kernel, dim3((unsigned)(segs * ((p.ranges * p.tokens + 255) / 256))), dim3(256), args, 0,
                            stream);
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
