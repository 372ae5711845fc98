// Decode attention over the 8-bit paged caches: one query token per sequence (tiles: tq_kv8.h).
//
// Work is the stream of 32-token steps of the (sequence, KV head) segments, sequences in order and a
// sequence's KV heads after each other.  Of P steps in all, wave w of R takes steps [floor(w P / R),
// floor((w + 1) P / R)): found on the device from seq_lens, so no length is needed on the host.  A
// segment inside one wave is written directly; the pieces of a cut one go to workspace slot w + (segment
// number), which never repeats since along the waves the segments never decrease, and
// kv8_decode_merge_kernel joins them: the waves with a segment's first and last step leave their numbers.  Each wave works alone: no LDS, no barriers.
//
// MFMA layout, lane l, n = l % 16, g = l / 16, tiles A and B of 16 tokens per step:
//   S^T [16 tokens x 16 heads] = K . Q^T   4 x mfma_f32_16x16x32_f16 per tile; slice cc covers dims 32g + 8cc + (0..7),
//                                          so the lane's operand is 32 bytes of token n
//   O^T [dim 8m + a][head] += V^T . P^T    8 x mfma_f32_16x16x32_f16 per step, k = 8g + i being tokens 4g..4g+3 of A, then
//                                          of B: what S^T leaves in the lane, and a word of the values layout each
// One pass with the running maximum and sum of the softmax.  The tile's K scale goes into the score's
// factor; V's scale, relative to the largest met so far, into the conversion to fp16, which is exact down to
// 2^-15 of that, where codes pass below fp16's numbers, and gives zeros from 2^-24 on (the accumulators are rescaled
// when a larger scale is met).
//
// Bound: HBM reads, 256 bytes per token and KV head: 64 x 32768 tokens of 8 heads in 762 us, 5.6 TB/s, where a large
// copy moves 4.9.  With a window the same per visible token: 64 sequences of 300 to 32768 tokens, window 4096, 384 MB in 82 us.
// With accumulated weights each step's scores are kept for kv8_decode_mass_kernel, 4 bytes a head and token: at 64 x 32768 tokens
// 402 MB more are written (409 by counters) and the kernel takes 1078 us instead of 762; the same stores into a buffer that stays in
// L2 cost 25 us, so it is the writes among the reads that memory takes badly (nontemporal stores and stores behind the next
// loads changed nothing, scores that lie by head instead of by token 1 %).  Reading the keys again instead would move 128 bytes a token for all heads,
// at six heads a KV head as long.  Small calls: launches, start-up (the search for the wave's part, block table, scales) and
// the merge, about 15 us.
#include "tq_kv8.h"

#include <atomic>

namespace {

constexpr int kWaves = 4;
// 16-token tiles of a step (4: one sequence of 4099 tokens 15.9 -> 14.9 us, 32 x 1K..8K 70.9 -> 75.2)
constexpr int kTiles = 2;
// Resident waves (12: 64 x 32768 tokens 759 -> 776 us, 32 x 1K..8K 70.9 -> 76.0; 6: 852 and 75)
constexpr int kWavesPerCu = 8;
constexpr int kMaxWorkers = 256 * kWavesPerCu;
constexpr int kMinSteps = 2;     // steps a wave takes at least (1 x 4099 tokens: 1 18.2 us, 2 16.9, 4 16.9, 8 18.9)
// A row's exponent base lies kUp below its largest score so far: as fp16 numbers the probabilities then keep 11 bits down
// to 2^-28 of the largest, and count as zero only below 2^-39 of it (with the base at the largest: 2^-14 and 2^-25; a long tail
// of small ones was lost).
constexpr float kUp = 14.f;

__device__ __forceinline__ int length_of(const Kv8Attn& p, int s) {
    int L = p.a.seq_lens[s];
    L = L < p.cap ? L : p.cap;
    return L > 0 ? L : 0;
}
// the steps of a sequence of L tokens that the window and the sinks touch
__device__ __forceinline__ Kv8Span span_of(const Kv8Attn& p, int L) { return kv8_span(kv8_window_from(L, p.window), L, p.sinks); }
template <bool WINDOW>
__device__ __forceinline__ int steps_of(const Kv8Attn& p, int s) {
    static_assert(kTiles == 2, "kv8_span counts steps of 32 tokens");
    if (WINDOW) return span_of(p, length_of(p, s)).n;
    return (int)(((uint32_t)length_of(p, s) + 16 * kTiles - 1) / (16 * kTiles));
}
// Steps (one KV head) of the 64 sequences from s0 on: this lane's, and the sum up to it (below 2^32: 64 times 2^26)
template <bool WINDOW>
__device__ __forceinline__ uint32_t scan_steps(const Kv8Attn& p, int s0, uint32_t& mine) {
    const int lane = threadIdx.x & 63;
    mine = s0 + lane < p.a.num_seqs ? (uint32_t)steps_of<WINDOW>(p, s0 + lane) : 0u;
    uint32_t in = mine;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t x = (uint32_t)__shfl_up((int)in, d, 64);
        if (lane >= d) in += x;
    }
    return in;
}
// floor(w P / R) = w floor(P / R) + floor(w (P mod R) / R), R waves in use
struct Share {
    int64_t each;
    uint32_t rest, R;
    __device__ __forceinline__ int64_t at(uint32_t w) const { return w * each + w * rest / R; }  // (w, R below 2^12)
};
__device__ __forceinline__ Share share_of(const Kv8Attn& p, int64_t P) {
    const int64_t m = P / kMinSteps;
    Share h;
    h.R = m < 1 ? 1u : m < p.workers ? (uint32_t)m : (uint32_t)p.workers;
    if (P >> 32) {
        h.each = P / h.R;
        h.rest = (uint32_t)(P - h.each * h.R);
    } else {
        h.each = (uint32_t)P / h.R;
        h.rest = (uint32_t)P - (uint32_t)h.each * h.R;
    }
    return h;
}

// WINDOW: each sequence's steps are those that its window and the sinks touch (all, where the window is 2^31 - 1); MASS: every
// step leaves its scores for the accumulated weights.
template <int ENC, bool FINE, bool WINDOW, bool MASS>
__global__ __launch_bounds__(64 * kWaves, kWavesPerCu / 4) void kv8_decode_kernel(Kv8Attn p) {
    using Code = Kv8Code<ENC>;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = (int64_t)blockIdx.x * kWaves + wave;
    const int hkv = p.a.num_kv_heads;
    uint32_t mine;
    uint32_t in = scan_steps<WINDOW>(p, 0, mine);
    int64_t P = (uint32_t)__builtin_amdgcn_readlane((int)in, 63);
    if (p.a.num_seqs > 64) {
        uint32_t u;
        for (int s0 = 64; s0 < p.a.num_seqs; s0 += 64) P += (uint32_t)__builtin_amdgcn_readlane((int)scan_steps<WINDOW>(p, s0, u), 63);
    }
    P *= hkv;
    const Share share = share_of(p, P);
    if (P == 0 || w >= share.R) return;
    int64_t pos = share.at((uint32_t)w);
    const int64_t end = share.at((uint32_t)w + 1);

    // ---- the sequence that holds step pos ----
    int s = 0;
    int64_t seq0 = 0;  // its first step
    for (int s0 = 0;;) {
        const uint64_t over = __builtin_amdgcn_ballot_w64((int64_t)in * hkv + seq0 > pos);
        if (over) {
            const int l = __builtin_ctzll(over);
            s = s0 + l;
            seq0 += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)(in - mine), l) * hkv;
            break;
        }
        seq0 += (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)in, 63) * hkv;
        s0 += 64;  // (pos is below the last one's end)
        in = scan_steps<WINDOW>(p, s0, mine);
    }
    s = __builtin_amdgcn_readfirstlane(s);
    int np = steps_of<WINDOW>(p, s);
    int kh = (int)((pos - seq0) / np);
    int64_t seg0 = seq0 + (int64_t)kh * np;

    while (pos < end) {
        int L = p.a.seq_lens[s];
        L = __builtin_amdgcn_readfirstlane(L < p.cap ? L : p.cap);
        const int j0 = __builtin_amdgcn_readfirstlane((int)(pos - seg0));
        const int j1 = __builtin_amdgcn_readfirstlane((int)(end - seg0 < np ? end - seg0 : np));
        const uint8_t* kb = static_cast<const uint8_t*>(p.a.k_cache) + kh * p.a.k_stride_head;
        const uint8_t* vb = static_cast<const uint8_t*>(p.a.v_cache) + kh * p.a.v_stride_head;
        const int32_t* bt = p.a.block_tables + s * p.a.block_table_stride;
        const int last_tile = (L - 1) >> 4;
        const uint32_t scale_at = (uint32_t)p.a.block_size * TQ_HEAD_DIM;
        const Kv8Span span = WINDOW ? span_of(p, L) : Kv8Span{0, 0, 0, 0};
        // the sequence's tile that is number ti here (behind the last: one past the sequence's end)
        auto tile_of = [&](int ti) -> int { return !WINDOW || ti < 2 * span.ns ? ti : ti + 2 * (span.b0 - span.ns); };

        // ---- 64 tiles' blocks and scales at a time, one per lane ----
        // block (tiles past the last and bad entries: a valid block and zero tokens), rows in use, scales
        struct Tiles {
            int blk, nv;
            float ks, vs;
        };
        auto tiles_from = [&](int t0) -> Tiles {
            Tiles t;
            const int ti = tile_of(t0 + lane);
            const int tc = ti < last_tile ? ti : last_tile;
            t.blk = bt[tq_udiv_apply((uint32_t)tc, p.tpb_div)];
            const int nv = L - 16 * ti;
            t.nv = nv < 16 ? (nv > 0 ? nv : 0) : 16;
            if ((uint32_t)t.blk >= (uint64_t)p.a.num_blocks) {
                t.blk = 0;
                t.nv = 0;
            }
            if (WINDOW) {
                // rows [from, upto) of it lie between the sinks and the window; all of them: no rows
                int from = p.sinks - 16 * ti, upto = span.lo - 16 * ti;
                from = from < 0 ? 0 : from < 16 ? from : 16;
                upto = upto < from ? from : upto < 16 ? upto : 16;
                t.nv = upto - from == 16 ? 0 : t.nv | from << 8 | upto << 16;
            }
            t.ks = *reinterpret_cast<const float*>(kb + t.blk * p.a.k_stride_block + scale_at);
            t.vs = *reinterpret_cast<const float*>(vb + t.blk * p.a.v_stride_block + scale_at);
            return t;
        };
        Tiles nxt = tiles_from(kTiles * j0);

        // ---- the query: heads kh * group + n ----
        tq_half8 qh[4], ql[4];
        float c1;
        {
            float x[32];
            const int64_t off = s * p.a.q_stride_token + (int64_t)(kh * p.group + (n < p.group ? n : 0)) * p.a.q_stride_head + 16 * g;
            kv8_load32(p.a.q, off, 64, p.a.q_dtype, x);
            float m = 0.f, back;
#pragma unroll
            for (int i = 0; i < 32; ++i) m = fmaxf(m, __builtin_fabsf(x[i]));
            const float f = kv8_query_factor(tq_max_over_groups(m), p.a.sm_scale < 0.f, back);
            kv8_query_half<FINE>(x, f, qh, ql);
            c1 = __builtin_fabsf(p.a.sm_scale) * kKv8Log2e * back;
        }

        uint32_t kw[kTiles][8], vw[kTiles][8];
        auto load = [&](const uint8_t* tile, uint32_t at, int second, uint32_t (&x)[8]) {
            const tq_u32x4* src = reinterpret_cast<const tq_u32x4*>(tile + at);
            // (each byte is read once: kept out of the caches' way, 64 x 32768 tokens 792 -> 759 us)
            const tq_u32x4 a = __builtin_nontemporal_load(src), b = __builtin_nontemporal_load(src + second);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i];
                x[4 + i] = b[i];
            }
        };
        // the tile's codes: block and row within it
        auto tile_at = [&](int number, int blk, int64_t stride) -> int64_t {
            const int ti = tile_of(number);
            const int tc = ti < last_tile ? ti : last_tile;
            return blk * stride + (int64_t)(tc - p.tpb * (int)tq_udiv_apply((uint32_t)tc, p.tpb_div)) * (16 * TQ_HEAD_DIM);
        };
        // (each load's lanes next to each other: a token's 64 bytes of keys, 256 bytes of values)
        const uint32_t k_off = 128 * n + 16 * g, v_off = 512 * g + 16 * n;
        struct Blocks {
            int b[kTiles];
        };
        auto load_keys = [&](const Blocks& b, int ti) {
#pragma unroll
            for (int h = 0; h < kTiles; ++h) load(kb + tile_at(ti + h, b.b[h], p.a.k_stride_block), k_off, 4, kw[h]);
        };
        auto load_values = [&](const Blocks& b, int ti) {
#pragma unroll
            for (int h = 0; h < kTiles; ++h) load(vb + tile_at(ti + h, b.b[h], p.a.v_stride_block), v_off, 16, vw[h]);
        };
        // (the loads of step j + 1 go out during step j without a condition, the last step repeats its own: where the
        // compiler cannot count what is under way, it waits for all of it)
        {
            Blocks b;
#pragma unroll
            for (int h = 0; h < kTiles; ++h) b.b[h] = __builtin_amdgcn_readlane(nxt.blk, h);
            load_keys(b, kTiles * j0);
            load_values(b, kTiles * j0);
        }

        float M = kKv8None, base = kKv8None, lsum = 0.f, vref = 0.f;  // M: largest score so far
        float lfull = 0.f;  // MASS: the sum of the probabilities before their rounding
        tq_floatx4 acc[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) acc[a] = tq_floatx4{0.f, 0.f, 0.f, 0.f};

        for (int jg = j0; jg < j1; jg += 64 / kTiles) {
        const int t0 = kTiles * jg, je = jg + 64 / kTiles < j1 ? jg + 64 / kTiles : j1;
        const Tiles cur = nxt;
        if (t0 + 64 < kTiles * j1) nxt = tiles_from(t0 + 64);
        for (int j = jg; j < je; ++j) {
            const int i = kTiles * j - t0;  // lane of the step's first tile in cur
            const bool more = j + 1 < j1;
            // the next step's tiles
            const int jn = more ? j + 1 : j, fi = (more ? i + kTiles : i) & 63;
            const bool over = more && i == 64 - kTiles;
            Blocks next;
            float ks[kTiles], vs[kTiles];
            int nv[kTiles], from[kTiles], upto[kTiles], all = 0;
#pragma unroll
            for (int h = 0; h < kTiles; ++h) {
                next.b[h] = over ? __builtin_amdgcn_readlane(nxt.blk, h) : __builtin_amdgcn_readlane(cur.blk, fi + h);
                ks[h] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(cur.ks), i + h));
                vs[h] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(cur.vs), i + h));
                nv[h] = __builtin_amdgcn_readlane(cur.nv, i + h);
                from[h] = upto[h] = 0;
                if (WINDOW) {
                    from[h] = (nv[h] >> 8) & 255;
                    upto[h] = nv[h] >> 16;
                    nv[h] &= 255;
                }
                all += nv[h] + from[h] - upto[h];
            }
            // ---- scores in log2 units: tokens 4g + r of each tile, head n ----
            float sv[4 * kTiles];
#pragma unroll
            for (int h = 0; h < kTiles; ++h) {
                tq_floatx4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) {
                    const tq_half8 a = kv8_half8<ENC>(kw[h][2 * cc], kw[h][2 * cc + 1], 1.f, 1.f);
                    sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[cc], sc, 0, 0, 0);
                    if (FINE) sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[cc], sc, 0, 0, 0);
                }
                const float f = c1 * ks[h];
#pragma unroll
                for (int r = 0; r < 4; ++r) sv[4 * h + r] = sc[r] * f;
            }
            load_keys(next, kTiles * jn);
            if (all != 16 * kTiles) {
#pragma unroll
                for (int r = 0; r < 4 * kTiles; ++r) {
                    const int t = 4 * g + (r & 3);
                    if (t >= nv[r >> 2] || (WINDOW && t >= from[r >> 2] && t < upto[r >> 2])) sv[r] = kKv8NegInf;
                }
#pragma unroll
                for (int h = 0; h < kTiles; ++h) {
                    uint32_t keep = kv8_keep(nv[h] - 4 * g);
                    if (WINDOW) keep &= ~kv8_keep(upto[h] - 4 * g) | kv8_keep(from[h] - 4 * g);
#pragma unroll
                    for (int a = 0; a < 8; ++a) vw[h][a] &= keep;
                    if (nv[h] == 0) vs[h] = 0.f;
                }
            }
            // ---- online softmax ----
            float mx = sv[0], vmax = vs[0];
#pragma unroll
            for (int r = 1; r < 4 * kTiles; ++r) mx = fmaxf(mx, sv[r]);
#pragma unroll
            for (int h = 1; h < kTiles; ++h) vmax = fmaxf(vmax, vs[h]);
            if (__builtin_amdgcn_ballot_w64(mx > M)) {
                const float Mn = fmaxf(M, tq_max_over_groups(mx));
                const float bn = __builtin_fabsf(Mn) < kKv8Far ? Mn - kUp : Mn;
                const float alpha = __builtin_amdgcn_exp2f(base - bn);
                lsum *= alpha;
                lfull *= alpha;
#pragma unroll
                for (int a = 0; a < 8; ++a) acc[a] *= alpha;
                M = Mn;
                base = bn;
            }
            if (vmax > vref) {  // wave-uniform
                const float f = vref / vmax;
#pragma unroll
                for (int a = 0; a < 8; ++a) acc[a] *= f;
                vref = vmax;
            }
            const float rv = vref > 0.f ? 1.f / vref : 0.f;
#pragma unroll
            for (int h = 0; h < kTiles; h += 2) {
                float pr[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) pr[r] = __builtin_amdgcn_exp2f(sv[4 * h + r] - base);
                tq_half8 ph, pl;
                kv8_prob8<FINE>(pr, ph, pl);
                lsum += kv8_sum8<FINE>(pr, ph);
                if (MASS) lfull += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
                const float va = kv8_relative(vs[h], rv), vb2 = kv8_relative(vs[h + 1], rv);
#pragma unroll
                for (int a = 0; a < 8; ++a) {
                    const tq_half8 v = kv8_half8<ENC>(vw[h][a], vw[h + 1][a], va, vb2);
                    acc[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, acc[a], 0, 0, 0);
                    if (FINE) acc[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, acc[a], 0, 0, 0);
                }
            }
            load_values(next, kTiles * jn);
            if (MASS) {
                // (behind the next step's loads, which would otherwise wait for them, and without a condition: lanes without a
                // head are out of the buffer's range)
                const uint32_t bytes = 128u * (uint32_t)p.group;
                const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
                    p.scores + (((int64_t)s * hkv + kh) * p.most_steps + j) * (32 * p.group), (short)0, (int)bytes, 0x00020000);
#pragma unroll
                for (int h = 0; h < kTiles; ++h) {
                    const uint32_t at = n < p.group ? (uint32_t)h * (bytes >> 1) + 64u * n + 16u * g : 0x40000000u;
                    __builtin_amdgcn_raw_buffer_store_b128(
                        tq_u32x4{__float_as_uint(sv[4 * h]), __float_as_uint(sv[4 * h + 1]), __float_as_uint(sv[4 * h + 2]), __float_as_uint(sv[4 * h + 3])},
                        rsrc, (int)at, 0, 0);
                }
            }
        }
        }

        // ---- acc[a][r] is dim 64 (a / 4) + 16g + 4r + a % 4 of head n ----
        const float l = tq_sum_over_groups(lsum);
        const bool complete = j0 == 0 && j1 == np;
        if (lane == 0) {
            int* ends = p.ends + 2 * ((int64_t)s * hkv + kh);
            if (j0 == 0) ends[0] = (int)w;
            if (j1 == np) ends[1] = (int)w;
        }
        if (MASS) {
            const float l1 = tq_sum_over_groups(lfull);
            if (g == 0 && n < p.group) {
                const int64_t row = (w + (int64_t)s * hkv + kh) * p.group + n;
                p.ws_me[2 * row] = base;
                p.ws_me[2 * row + 1] = l1;
            }
        }
        if (n < p.group) {
            float o[2][16];
            // (a piece is divided by its own sum: plain sums of large values pass fp32's range)
            const float f = l == 0.f ? 0.f : vref / l;
#pragma unroll
            for (int a = 0; a < 8; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[a >> 2][4 * r + (a & 3)] = acc[a][r] * f;
            const int64_t row = (w + (int64_t)s * hkv + kh) * p.group + n;
            const int64_t at = complete ? s * p.a.out_stride_token + (int64_t)(kh * p.group + n) * p.a.out_stride_head : row * TQ_HEAD_DIM;
#pragma unroll
            for (int k = 0; k < 2; ++k)
                kv8_store<16>(complete ? p.a.out : (void*)p.ws_acc, at + 64 * k + 16 * g, complete ? p.a.out_dtype : TQ_F32, o[k]);
            if (!complete) {
                if (g == 0) {
                    p.ws_ml[2 * row] = base;
                    p.ws_ml[2 * row + 1] = l;
                }
            }
        }
        // ---- next segment ----
        pos = seg0 + j1;
        if (j1 == np) {
            seg0 += np;
            if (++kh == hkv) {
                kh = 0;
                do {
                    if (++s >= p.a.num_seqs) return;
                    np = steps_of<WINDOW>(p, s);
                } while (np == 0);
            }
        }
    }
}

// Adds the weights of a segment's tokens, summed over its query heads, to what they had; the sequence's last token starts
// from 0.  Workgroup (segment, 32 steps): first each head's base and sum over the segment's pieces, then four tokens a
// thread.  A weight that is not a number counts as 0.  Bound: memory, 4 bytes of score a head and 8 of weight a token: 64 x 32768
// tokens of 48 / 8 heads, 537 MB, 113 us, 4.8 TB/s.
__global__ __launch_bounds__(256) void kv8_decode_mass_kernel(Kv8Attn p, int chunks) {
    __shared__ float2 s_stat[16];
    const uint32_t seg = blockIdx.x / (uint32_t)chunks, chunk = blockIdx.x - seg * (uint32_t)chunks;
    const int hkv = p.a.num_kv_heads, s = (int)(seg / (uint32_t)hkv), kh = (int)seg - s * hkv;
    const int L = length_of(p, s);
    const Kv8Span span = span_of(p, L);
    if ((int)chunk * 32 >= span.n) return;
    const int w0 = p.ends[2 * seg], w1 = p.ends[2 * seg + 1];
    const int lane = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < p.group; r += 4) {
        float M = kKv8None, l = 0.f;
        for (int w = w0 + lane; w <= w1; w += 64) {
            const int64_t row = ((int64_t)w + seg) * p.group + r;
            const float b = p.ws_me[2 * row], x = p.ws_me[2 * row + 1];
            const float Mn = fmaxf(M, b);
            l = l * __builtin_amdgcn_exp2f(M - Mn) + x * __builtin_amdgcn_exp2f(b - Mn);
            M = Mn;
        }
        for (int m = 1; m < 64; m <<= 1) {
            const float b = __shfl_xor(M, m, 64), x = __shfl_xor(l, m, 64);
            const float Mn = fmaxf(M, b);
            l = l * __builtin_amdgcn_exp2f(M - Mn) + x * __builtin_amdgcn_exp2f(b - Mn);
            M = Mn;
        }
        if (lane == 0) s_stat[r] = make_float2(M, l == 0.f ? 0.f : 1.f / l);
    }
    __syncthreads();
    const int j = 32 * (int)chunk + (int)(threadIdx.x >> 3);
    if (j >= span.n) return;
    const int in = 4 * (int)(threadIdx.x & 7);  // first token within the step
    const int t = 32 * span.step(j) + in;
    if (t >= L) return;
    const float* src = p.scores + (((int64_t)seg) * p.most_steps + j) * (32 * p.group) + (in >> 4) * (16 * p.group) + (in & 15);
    float add[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < p.group; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(src + 16 * r);
        const float2 st = s_stat[r];
        const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = __builtin_amdgcn_exp2f(y[k] - st.x) * st.y;
            add[k] += f == f ? f : 0.f;
        }
    }
    const int b = (int)tq_udiv_apply((uint32_t)(t >> 4), p.tpb_div);
    const int blk = p.a.block_tables[s * p.a.block_table_stride + b];
    if ((uint32_t)blk >= (uint64_t)p.a.num_blocks) return;
    float* dst = p.mass + blk * p.mass_stride_block + kh * p.mass_stride_head + (t - b * p.a.block_size);
    if (t + 4 <= L && (t >= span.lo || t + 4 <= p.sinks)) {
        float4 m = *reinterpret_cast<const float4*>(dst);
        if (t + 4 == L) m.w = 0.f;
        *reinterpret_cast<float4*>(dst) = make_float4(m.x + add[0], m.y + add[1], m.z + add[2], m.w + add[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (t + k < L && (t + k >= span.lo || t + k < p.sinks)) dst[k] = (t + k == L - 1 ? 0.f : dst[k]) + add[k];
    }
}

// Workgroup (s, head): out = sum_i w_i out_i / sum_i w_i, w_i = 2^(M_i - M) l_i, over the pieces of the head's segment, as a
// running mean, which stays within the values' range; nothing to do where one wave held it all, zeros where the
// sequence is empty.  The workgroup's 8 half-waves share the pieces, a lane has 4 dims.  (With a workgroup per KV
// head, one sequence of 4099 tokens: merge 13.6 -> 6.6 us.)
template <bool WINDOW>
__global__ __launch_bounds__(256) void kv8_decode_merge_kernel(Kv8Attn p) {
    __shared__ float4 s_acc[8][32];
    __shared__ float2 s_ml[8];
    const int hkv = p.a.num_kv_heads;
    const int s = (int)(blockIdx.x / (uint32_t)p.a.num_q_heads), head = (int)(blockIdx.x % (uint32_t)p.a.num_q_heads);
    const int kh = head / p.group, r = head - kh * p.group;
    const int* ends = p.ends + 2 * ((int64_t)s * hkv + kh);
    int w0 = ends[0], w1 = ends[1];
    if (steps_of<WINDOW>(p, s) == 0) {  // (no wave had it)
        w0 = 0;
        w1 = -1;
    }
    if (w0 == w1) return;
    const int half = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const int64_t seg = (int64_t)s * hkv + kh;
    float M = kKv8NegInf, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int wb = w0 + half; wb <= w1; wb += 4 * 8) {
        float mp[4], lp[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int wk = wb + k * 8;
            mp[k] = kKv8NegInf;
            lp[k] = 0.f;
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (wk <= w1) {
                const int64_t row = (wk + seg) * p.group + r;
                mp[k] = p.ws_ml[2 * row];
                lp[k] = p.ws_ml[2 * row + 1];
                v[k] = *reinterpret_cast<const float4*>(p.ws_acc + row * TQ_HEAD_DIM + 4 * l32);
            }
        }
        const float Mn = fmaxf(M, fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])));
        kv8_join<4>(M, l, a, Mn, mp, lp, v);
    }
    s_acc[half][l32] = a;
    if (l32 == 0) s_ml[half] = make_float2(M, l);
    __syncthreads();
    if (half) return;
    float Mn = kKv8NegInf;
#pragma unroll
    for (int k = 0; k < 8; ++k) Mn = fmaxf(Mn, s_ml[k].x);
    float mp[8], lp[8];
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        mp[k] = s_ml[k].x;
        lp[k] = s_ml[k].y;
        v[k] = s_acc[k][l32];
    }
    M = kKv8NegInf;
    l = 0.f;
    a = make_float4(0.f, 0.f, 0.f, 0.f);
    kv8_join<8>(M, l, a, Mn, mp, lp, v);
    const float o[4] = {a.x, a.y, a.z, a.w};
    kv8_store<4>(p.a.out, s * p.a.out_stride_token + (int64_t)head * p.a.out_stride_head + 4 * l32, p.a.out_dtype, o);
}

std::atomic<int> g_cus[64];

}  // namespace

int tq_kv8_cus() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 0;
    int cus = dev < 64 ? g_cus[dev].load(std::memory_order_relaxed) : 0;
    if (cus > 0) return cus;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 0;
    if (dev < 64) g_cus[dev].store(cus, std::memory_order_relaxed);
    return cus;
}

int tq_kv8_attn_setup(const tq_kv8_attn_args* a, Kv8Attn* p) {
    if (a->head_dim != TQ_HEAD_DIM) return TQ_ERR_HEAD_DIM;
    if (a->block_size <= 0 || a->block_size % 16 || a->block_size > 65536) return TQ_ERR_BLOCK_SIZE;
    for (const int dt : {a->q_dtype, a->out_dtype})
        if (dt != TQ_F32 && dt != TQ_F16 && dt != TQ_BF16) return TQ_ERR_DTYPE;
    if (a->encoding != TQ_E4M3 && a->encoding != TQ_INT8) return TQ_ERR_DTYPE;
    if (a->num_seqs < 0 || a->num_kv_heads <= 0 || a->num_q_heads <= 0 || a->num_blocks <= 0 || a->max_blocks_per_seq < 0 ||
        a->block_table_stride < a->max_blocks_per_seq || a->num_blocks > INT32_MAX)
        return TQ_ERR_INVALID_ARGUMENT;
    if (a->num_q_heads % a->num_kv_heads) return TQ_ERR_GQA;
    if (!(__builtin_fabsf(a->sm_scale) < __builtin_huge_valf())) return TQ_ERR_INVALID_ARGUMENT;
    const uintptr_t ptrs = (uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache;
    const int64_t el = a->q_stride_token | a->q_stride_head | a->out_stride_token | a->out_stride_head;
    const int64_t by = a->k_stride_block | a->k_stride_head | a->v_stride_block | a->v_stride_head;
    if (ptrs % 16 || el % 8 || by % 16) return TQ_ERR_ALIGNMENT;
    p->a = *a;
    p->tpb = a->block_size / 16;
    p->tpb_div = tq_make_udiv((uint32_t)p->tpb);
    p->group = a->num_q_heads / a->num_kv_heads;
    p->group_div = tq_make_udiv((uint32_t)p->group);
    // (positions stay below 2^31, those of the 64 tiles requested ahead included)
    const int64_t cap = (int64_t)a->max_blocks_per_seq * a->block_size;
    p->cap = (int)(cap < kKv8MaxLen ? cap : kKv8MaxLen);
    return TQ_OK;
}

int tq_kv8_window_setup(const tq_kv8_window_args* w, Kv8Attn* p) {
    const int rc = tq_kv8_attn_setup(&w->attn, p);
    if (rc != TQ_OK) return rc;
    if (w->window < 0 || w->sinks < 0 || (w->sinks && !w->window) || w->reserved) return TQ_ERR_INVALID_ARGUMENT;
    if (w->mass && ((uintptr_t)w->mass % 16 || (w->mass_stride_block | w->mass_stride_head) % 4)) return TQ_ERR_ALIGNMENT;
    p->window = w->window ? w->window : INT32_MAX;
    p->sinks = w->sinks;
    p->mass = w->mass;
    p->mass_stride_block = w->mass_stride_block;
    p->mass_stride_head = w->mass_stride_head;
    return TQ_OK;
}

extern "C" int64_t tq_kv8_decode_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads) {
    if (num_seqs < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return 0;
    const int64_t slots = kMaxWorkers + (int64_t)num_seqs * num_kv_heads;
    return slots * (num_q_heads / num_kv_heads) * (TQ_HEAD_DIM + 2) * 4 + (int64_t)num_seqs * num_kv_heads * 8;
}

namespace {

int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }
// steps of a sequence of up to len tokens (a window's tokens reach into one step more than they fill)
int64_t most_steps(int64_t len, int64_t window, int64_t sinks) {
    const int64_t all = (len + 31) / 32;
    if (!window) return all;
    const int64_t m = (window + 31) / 32 + 1 + (sinks + 31) / 32;
    return m < all ? m : all;
}

int launch_decode(Kv8Attn& p, bool window, int64_t need, tq_stream_t stream) {
    const tq_kv8_attn_args* a = &p.a;
    if (p.group > 16) return TQ_ERR_GQA;
    if (a->num_seqs == 0) return TQ_OK;
    // (a launch's threads stay below 2^32)
    if (a->max_seq_len < 0 || (int64_t)a->num_seqs * a->num_q_heads > 0xffffff) return TQ_ERR_INVALID_ARGUMENT;
    if (!a->q || !a->out || !a->k_cache || !a->v_cache || (!a->block_tables && a->max_blocks_per_seq) || !a->seq_lens) return TQ_ERR_INVALID_ARGUMENT;
    if (!a->workspace || (uintptr_t)a->workspace % 256 || a->workspace_bytes < need) return TQ_ERR_WORKSPACE;
    p.cap = p.cap < a->max_seq_len ? p.cap : a->max_seq_len;
    const int64_t slots = kMaxWorkers + (int64_t)a->num_seqs * a->num_kv_heads;
    p.ws_acc = static_cast<float*>(a->workspace);
    p.ws_ml = p.ws_acc + slots * p.group * TQ_HEAD_DIM;
    p.ends = reinterpret_cast<int*>(p.ws_ml + slots * p.group * 2);
    // tokens of a sequence that are read
    const int64_t most = window ? most_steps(p.cap, p.window == INT32_MAX ? 0 : p.window, p.sinks) : (p.cap + 16 * kTiles - 1) / (16 * kTiles);
    p.most_steps = (int)most;
    const int64_t chunks = (most + 31) / 32;
    if (p.mass) {
        uint8_t* at = static_cast<uint8_t*>(a->workspace) + align256(tq_kv8_decode_workspace_bytes(a->num_seqs, a->num_q_heads, a->num_kv_heads));
        p.ws_me = reinterpret_cast<float*>(at);
        p.scores = reinterpret_cast<float*>(at + align256(slots * p.group * 8));
        if ((int64_t)a->num_seqs * a->num_kv_heads * chunks > 0xffffff) return TQ_ERR_INVALID_ARGUMENT;
    }
    const int cus = tq_kv8_cus();
    if (cus <= 0) return (int)hipErrorNoDevice;
    // no more waves than the lengths can ask for
    const int64_t ask = (int64_t)a->num_seqs * a->num_kv_heads * most / kMinSteps;
    int64_t workers = (int64_t)cus * kWavesPerCu;
    workers = workers < kMaxWorkers ? workers : kMaxWorkers;
    workers = workers < ask ? workers : ask;
    p.workers = (int)(workers < 1 ? 1 : workers);
    const bool fine = a->q_dtype == TQ_F32 || a->out_dtype == TQ_F32;
    const void* kern = nullptr;
#define TQ_DECODE(E, F)                                                                      \
    if (a->encoding == E && fine == F)                                                       \
        kern = p.mass ? (const void*)kv8_decode_kernel<E, F, true, true>                     \
                      : window ? (const void*)kv8_decode_kernel<E, F, true, false> : (const void*)kv8_decode_kernel<E, F, false, false>;
    TQ_DECODE(TQ_E4M3, false) TQ_DECODE(TQ_E4M3, true) TQ_DECODE(TQ_INT8, false) TQ_DECODE(TQ_INT8, true)
#undef TQ_DECODE
    void* args[] = {&p};
    hipError_t e = hipLaunchKernel(kern, dim3((unsigned)((p.workers + kWaves - 1) / kWaves)), dim3(64 * kWaves), args, 0, stream);
    if (e == hipSuccess)
        e = hipLaunchKernel(window ? (const void*)kv8_decode_merge_kernel<true> : (const void*)kv8_decode_merge_kernel<false>,
                            dim3((unsigned)(a->num_seqs * a->num_q_heads)), dim3(256), args, 0, stream);
    if (e == hipSuccess && p.mass && chunks) {
        int n = (int)chunks;
        void* margs[] = {&p, &n};
        e = hipLaunchKernel((const void*)kv8_decode_mass_kernel, dim3((unsigned)(a->num_seqs * a->num_kv_heads * chunks)), dim3(256), margs, 0, stream);
    }
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}

}  // namespace

extern "C" int64_t tq_kv8_decode_window_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads, int max_seq_len, int window,
                                                        int sinks, int mass) {
    const int64_t plain = tq_kv8_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads);
    if (plain <= 0 || !mass || max_seq_len < 0 || window < 0 || sinks < 0) return plain;
    const int64_t slots = kMaxWorkers + (int64_t)num_seqs * num_kv_heads;
    return align256(plain) + align256(slots * (num_q_heads / num_kv_heads) * 8) +
           (int64_t)num_seqs * num_q_heads * most_steps(max_seq_len, window, sinks) * 32 * 4;
}

extern "C" int tq_kv8_decode(const tq_kv8_attn_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    Kv8Attn p = {};
    const int rc = tq_kv8_attn_setup(a, &p);
    return rc != TQ_OK ? rc : launch_decode(p, false, tq_kv8_decode_workspace_bytes(a->num_seqs, a->num_q_heads, a->num_kv_heads), stream);
}

extern "C" int tq_kv8_decode_window(const tq_kv8_window_args* w, tq_stream_t stream) {
    if (!w) return TQ_ERR_INVALID_ARGUMENT;
    const tq_kv8_attn_args* a = &w->attn;
    Kv8Attn p = {};
    const int rc = tq_kv8_window_setup(w, &p);
    if (rc != TQ_OK) return rc;
    if (!w->window && !w->mass)
        return launch_decode(p, false, tq_kv8_decode_workspace_bytes(a->num_seqs, a->num_q_heads, a->num_kv_heads), stream);
    const int len = p.cap < a->max_seq_len ? p.cap : a->max_seq_len;
    return launch_decode(p, true, tq_kv8_decode_window_workspace_bytes(a->num_seqs, a->num_q_heads, a->num_kv_heads, len, w->window,
                                                                       w->sinks, w->mass != nullptr), stream);
}
