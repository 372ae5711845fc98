// Prefill / extend attention over the 8-bit paged caches: several query tokens per sequence (tiles: tq_kv8.h).
//
// A row is one (new token, query head of the GQA group) pair, token-major; a segment is a block of 64 rows
// (32 with FINE) of a (sequence, KV head) with the keys that its rows see, walked in steps of 32 (two 16-token
// tiles).  A wave works on its own, without barriers.  MFMA layout, lane l, n = l % 32, h = l / 32:
//   S^T [32 tokens x 32 rows] = K . Q^T      8 x mfma_f32_32x32x16_f16; slices 2c and 2c + 1 cover dims 32c + 16h + (0..15):
//                                            16 bytes of token n, the lane halves' next to each other
//   O^T [dim 4m + d][row] += V^T . P^T       4 x mfma_f32_32x32x16_f16 per tile, k = 8h + i being tokens 4h + i and 8 + 4h + i:
//                                            what S^T leaves in the lane, and two words of the values layout
// A code converted to fp16 feeds both of the wave's 32-row tiles.  The query operands of 64 rows stay in LDS:
// that leaves two waves per SIMD their 256 registers, so that one's products hide the other's softmax.
//
// Work: the segments form one stream (sequences in order, a sequence's KV heads after each other, row blocks
// ascending) in which row block rb counts a + b rb tokens, what its last row sees rounded up to that form and a
// set-up share, so that positions are found in closed form from cu_seqlens_q and seq_lens.  Of P tokens
// in all, worker (wave) w of R takes positions [floor(w P / R), floor((w + 1) P / R)), and of a segment the
// steps that begin there.  A segment inside one worker is written directly; the pieces of a cut one (at most the
// first and the last of a worker, slots 2w and 2w + 1) go to the workspace and kv8_prefill_merge_kernel joins
// them.  (A workgroup's four waves on one segment, joined in LDS, leave a quarter of the pieces: 300 new after 2000
// tokens 58 -> 49 us, but 8 prompts of 900 to 1300 tokens 161 -> 290 and the six long extends 145 -> 147.)
//
// Bound: a SIMD's waves, whose products and vector instructions hardly overlap.  4 x 4096 tokens of 48 / 8 heads, 0.82
// TFLOP, take 867 us, 0.95 PFLOP/s, where a large fp16 matrix product reaches 1.22.  A step has 32 products and, over a
// whole launch, 245 other vector instructions (64 conversions, 64 of the exponentials and their scaling, 16 packings, 16
// sums; the rest moves operands and addresses): matrix unit 46 % busy, vector unit 57 %, 6 % of it the products'
// issue, 97 % together.  What keeps the two waves from overlapping more is open.  int8 takes 930 us (its conversions are
// more instructions), f32 1549 (twice the products; int8 1664).  Without the loads of K and V a step takes 9 % less,
// without the LDS reads 4.5 %, without the exponentials 5 %.  Tried and slower: 32 rows a wave (1180 us, two or three waves per SIMD), products ordered
// among the exponentials by hand (1130, spills), the same with one wave per SIMD (1540), a barrier per step so that a
// workgroup's waves share L1 (+ 3 %), a SIMD's two waves in turn by barriers (1115); raised priority around the
// products gives 0.7 % here and costs 4 x 2048 tokens 7 %.  Calls of few tokens: 20 us of start-up (search, query
// rows, first loads) and merge.
#include "tq_kv8.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;          // of a workgroup
constexpr int kWavesPerCu = 8;     // resident
constexpr int kMaxWorkers = 256 * kWavesPerCu;
constexpr int kMinTokens = 128;    // stream tokens a worker takes at least (32 or more: see the merge)
// A segment's set-up (query loads, first steps, output) in tokens (160, 320, 480, 640: 8 prompts of 900 to 1300 tokens 158, 158,
// 158, 162 us; 37 to 512 new after 1000 to 16000 of six sequences 134, 130, 129, 133)
constexpr int kSegTokens = 480;
// The cut pieces' set-up and their merge in tokens (1500: 8 to 40 new after 100 to 700 of 32 sequences 50.5 -> 53.6 us)
constexpr int kMergeTokens = 384;
// A row's exponent base lies `down` below the largest score of the step that set it, and moves only when a lane's
// 16 probabilities of a step sum to more than move_sum: no maximum is worked out otherwise, and fp16's normal range
// reaches from 2^15 above the base to 2^-14 below it.  In 16 bits the largest probability is thus 2^4 or more, and one
// below 2^-18 of it loses bits; FINE, whose two numbers resolve 2^-25, has it at 2^10 or more.  (The lower base moves
// more often: 4 x 4096 tokens in f32 1533 -> 1547 us; in bf16 it would take 883 -> 901.)
template <bool FINE>
struct Base {
    static constexpr float down = FINE ? 10.f : 4.f;
    static constexpr float move_sum = FINE ? 32768.f : 16384.f;
};
constexpr int kFirst = 2;          // query operands that stay in registers (1 .. 4: 4 x 4096 tokens 910, 906, 920, 921 us)

struct Cut {  // a segment that several workers share
    int q0, nq, kh, rb, slot0, w0, w1;  // w0 -1: none; worker 0's rb: the workers in use
};
struct Prefill {
    Kv8Attn at;
    int max_q, causal, rows, row_bits, step, grow;  // rows of a segment, their log2; tokens between row blocks; of the first
    Cut* cuts;
    int* tickets;  // one per XCD, zeroed; NULL where the call is too small to be dealt by tickets
};

// ---- the stream of segments ----
struct Seq {
    int q0, nq, L, nrb;
    int step;
    int64_t a, U;  // tokens of row block rb: a + step rb; of all row blocks
};
// A value that is the same in all lanes, in scalar registers (loads and shuffles leave it in vector registers)
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)(uint32_t)uniform((int)x) | (int64_t)uniform((int)(x >> 32)) << 32;
}
// (whole: every segment counts the same, so that a worker's share is one of them; SAME: s is the same in all lanes)
template <bool SAME>
__device__ __forceinline__ Seq seq_of(const Prefill& p, int s, bool whole) {
    Seq q;
    q.q0 = p.at.a.cu_seqlens_q[s];
    int nq = p.at.a.cu_seqlens_q[s + 1] - q.q0, L = p.at.a.seq_lens[s];
    if (SAME) {
        q.q0 = uniform(q.q0);
        nq = uniform(nq);
        L = uniform(L);
    }
    q.nq = nq > 0 ? nq : 0;
    const int computed = q.nq < p.max_q ? q.nq : p.max_q;  // (positions count all new tokens)
    q.L = L < 0 ? 0 : L < p.at.cap ? L : p.at.cap;
    q.nrb = (int)(((uint32_t)computed * (uint32_t)p.at.group + (uint32_t)p.rows - 1) >> p.row_bits);  // (host: below 2^31)
    const int past = q.L > q.nq ? q.L - q.nq : 0;
    q.a = whole ? kMinTokens : (p.causal ? past + p.grow : q.L) + kSegTokens;
    q.step = whole || !p.causal ? 0 : p.step;
    q.U = q.nrb * q.a + (int64_t)q.step * q.nrb * (q.nrb - 1) / 2;
    return q;
}
// tokens that the last row of row block rb sees
__device__ __forceinline__ int visible(const Prefill& p, const Seq& q, int rb) {
    if (!p.causal) return q.L;
    int i = (int)tq_udiv_apply((uint32_t)(rb * p.rows + p.rows - 1), p.at.group_div);
    i = i < q.nq - 1 ? i : q.nq - 1;
    const int v = q.L - q.nq + i + 1;
    return v > 0 ? v : 0;
}
__device__ __forceinline__ int64_t before(const Seq& q, int64_t rb) { return rb * q.a + (int64_t)q.step * rb * (rb - 1) / 2; }
// Tokens of the whole stream, and how it is dealt to the workers:
//   whole     the segments, at kMinTokens each, if they are no more than the workers and the longest takes no longer
//             than a cut one's worker and the merge;
//   tickets   whole segments, the next one to whoever is free, if there is one per worker and the ones that come last
//             are short against a worker's share (4 x 2048 tokens 235 -> 210 us, 4 x 4096 1055 -> 908; with half that
//             demand 64 prompts of 64 to 200 tokens 86 -> 131);
//   shares    otherwise.
enum { kShares, kWhole, kTickets };
__device__ __forceinline__ int64_t stream_total(const Prefill& p, int& dealt, int& most_rb) {
    const int lane = threadIdx.x & 63;
    int64_t P = 0, segs = 0;
    int longest = 0, last = 0, nrb = 0;
    for (int s = lane; s < p.at.a.num_seqs; s += 64) {
        const Seq q = seq_of<false>(p, s, false);
        P += q.U * p.at.a.num_kv_heads;
        segs += (int64_t)q.nrb * p.at.a.num_kv_heads;
        longest = q.nrb && q.L > longest ? q.L : longest;
        last = q.nrb && q.a > last ? (int)q.a : last;
        nrb = nrb > q.nrb ? nrb : q.nrb;
    }
    for (int m = 32; m >= 1; m >>= 1) {
        P += __shfl_xor(P, m, 64);
        segs += __shfl_xor(segs, m, 64);
        int o = __shfl_xor(longest, m, 64);
        longest = longest > o ? longest : o;
        o = __shfl_xor(last, m, 64);
        last = last > o ? last : o;
        o = __shfl_xor(nrb, m, 64);
        nrb = nrb > o ? nrb : o;
    }
    P = uniform(P);
    segs = uniform(segs);
    longest = uniform(longest);
    last = uniform(last);
    nrb = uniform(nrb);
    most_rb = nrb;
    dealt = kShares;
    if (segs <= p.at.workers && (int64_t)(longest - kMergeTokens) * p.at.workers <= P) dealt = kWhole;
    // (the tickets' numbers run over every sequence's row blocks as if all had the most; those that do not exist cost a
    // ticket)
    else if (p.tickets && (int64_t)nrb * p.at.a.num_seqs * p.at.a.num_kv_heads <= 2 * segs && segs >= p.at.workers &&
             (int64_t)longest * p.at.workers <= P && 4 * (int64_t)last * p.at.workers <= P)
        dealt = kTickets;
    return dealt == kWhole ? segs * kMinTokens : P;
}
// The workers' ranges: floor(w P / R) = w floor(P / R) + floor(w (P mod R) / R)
struct Share {
    int64_t each;
    uint32_t rest, R;
    __device__ __forceinline__ int64_t at(int64_t w) const { return w * each + (uint32_t)w * rest / R; }
};
__device__ __forceinline__ Share share_of(const Prefill& p, int64_t P, bool whole) {
    // (a SIMD's second wave pays from twice the tokens on: 300 new after 2000 tokens 57.0 -> 53.6 us; with that for all
    // waves 23 new after 700 take 28.6 instead of 24.8)
    constexpr int64_t half = kMaxWorkers / 2;
    int64_t m = P / kMinTokens;
    if (!whole && m > half) m = m >> 1 > half ? m >> 1 : half;
    Share h;
    h.R = m < 1 ? 1u : (uint32_t)(m < p.at.workers ? m : (int64_t)p.at.workers);
    h.each = P / h.R;
    h.rest = (uint32_t)(P - h.each * h.R);
    return h;
}
struct Place {
    int s, kh, rb;
    int64_t seg;  // stream position of the segment's start
};
// The segment that holds stream position pos (below the stream's total).
__device__ __forceinline__ Place find(const Prefill& p, int64_t pos, bool whole, Seq& q) {
    const int lane = threadIdx.x & 63;
    const int hkv = p.at.a.num_kv_heads;
    int64_t P = 0;
    Place at = {0, 0, 0, 0};
    for (int s0 = 0; s0 < p.at.a.num_seqs; s0 += 64) {
        const int64_t u = s0 + lane < p.at.a.num_seqs ? seq_of<false>(p, s0 + lane, whole).U * hkv : 0;
        int64_t in = u;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t x = __shfl_up(in, d, 64);
            if (lane >= d) in += x;
        }
        in += P;
        const uint64_t over = __builtin_amdgcn_ballot_w64(in > pos);
        if (over) {
            const int l = __builtin_ctzll(over);
            at.s = s0 + l;
            at.seg = __shfl(in - u, l, 64);
            break;
        }
        P = __shfl(in, 63, 64);
    }
    at.s = uniform(at.s);
    at.seg = uniform(at.seg);
    q = seq_of<true>(p, at.s, whole);
    int64_t off = pos - at.seg;
    // (estimates in double, put right in whole numbers)
    int kh = (int)((double)off / (double)q.U);
    kh = kh < hkv ? kh : hkv - 1;
    while (kh > 0 && kh * q.U > off) --kh;
    while (kh + 1 < hkv && (kh + 1) * q.U <= off) ++kh;
    kh = uniform(kh);
    off -= kh * q.U;
    const double h = (double)q.a - 0.5 * q.step;
    int rb = q.step ? (int)((__builtin_sqrt(h * h + 2.0 * q.step * (double)off) - h) / q.step) : (int)((double)off / h);
    rb = rb < 0 ? 0 : (rb < q.nrb ? rb : q.nrb - 1);
    while (rb > 0 && before(q, rb) > off) --rb;
    while (rb + 1 < q.nrb && before(q, rb + 1) <= off) ++rb;
    at.kh = uniform(kh);
    at.rb = uniform(rb);
    at.seg += at.kh * q.U + before(q, at.rb);
    return at;
}

template <int ENC, bool FINE>
__global__ __launch_bounds__(64 * kWaves, 2) void kv8_prefill_kernel(Prefill p) {
    constexpr int kRT = FINE ? 1 : 2;     // 32-row tiles of a segment
    constexpr bool kQLds = !FINE;         // query operands in LDS
    constexpr int kRows = 32 * kRT;
    extern __shared__ __attribute__((aligned(16))) uint8_t s_lds[];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const tq_kv8_attn_args& a = p.at.a;
    const int hkv = a.num_kv_heads, group = p.at.group;

    // ---- this worker's part of the stream ----
    int dealt, most_rb;
    const int64_t P = stream_total(p, dealt, most_rb);
    if (P == 0 || dealt == kTickets) {
        if (blockIdx.x == 0 && threadIdx.x == 0) p.cuts[0].rb = 0;  // nothing to merge
        if (P == 0) return;
    }
    const bool whole = dealt == kWhole;
    const Share share = share_of(p, P, whole);
    // consecutive workers share an XCD (workgroups go to the 8 XCDs in turn), so that its L2 holds few
    // sequences' keys; fewer workers than waves spread over all workgroups
    const int nwg = (int)gridDim.x;
    const int wg = (nwg & 7) ? (int)blockIdx.x : (int)((blockIdx.x & 7) * (nwg >> 3) + (blockIdx.x >> 3));
    const int first = (int)(share.R * (uint32_t)wg / (uint32_t)nwg), behind = (int)(share.R * (uint32_t)(wg + 1) / (uint32_t)nwg);
    const int w = first + wave;
    if (dealt != kTickets && w >= behind) return;  // (a workgroup has waves for all: R <= kWaves nwg)
    const int64_t p0 = share.at(w), p1 = share.at(w + 1);
    Seq q;
    int s = 0, kh = 0, rb = 0;
    int64_t seg = 0;
    if (dealt != kTickets) {
        const Place place = find(p, p0, whole, q);
        s = place.s;
        kh = place.kh;
        rb = place.rb;
        seg = place.seg;
        // for the merge: the segment that this worker's range begins inside of, if the worker before holds its
        // start and steps are left here
        Cut cut = {0, 0, 0, (int)share.R, 0, -1, 0};
        if (w > 0 && !whole) {
            const int nsteps = (visible(p, q, rb) + 31) >> 5;
            const int64_t before_this = share.at(w - 1), last = seg + 32 * (int64_t)(nsteps - 1);
            if (p0 > seg && before_this <= seg && nsteps > 0 && last >= p0) {
                int w1 = w;
                while (share.at(w1 + 1) <= last) ++w1;
                cut = {q.q0, q.nq, kh, rb, 2 * (w - 1) + (seg > before_this ? 1 : 0), w - 1, w1};
            }
        }
        if (lane == 0) p.cuts[w] = cut;
    }
    // Tickets: a workgroup's waves take kWaves neighbouring row blocks of a (sequence, KV head) pair, whose keys they
    // then share in L1.  One counter per XCD for the pairs x, x + 8, .., so that a pair's keys are read by one XCD, the
    // pairs' last (longest) row blocks first; an XCD without work left goes on with the next one's.  The next ticket is
    // taken while the one at hand is worked on.
    __shared__ int s_nan[kWaves];  // a NaN among the values of the segment's edge steps
    if (lane == 0) s_nan[wave] = 0;
    // the exponent base of rows whose scores lie beyond kKv8Far: their M stays kKv8None, so that every step moves it
    __shared__ float s_base[kWaves][kRT][64];
    __shared__ int s_ticket[2][2];  // pair (-1: none left), row blocks from the last
    const int pairs = a.num_seqs * hkv;
    const int turns = (most_rb + kWaves - 1) / kWaves;
    int xcd = (int)(blockIdx.x & 7), tried = 0, turn = 0;
    auto take_ticket = [&](int slot) {  // thread 0
        int pair = -1, back = 0;
        while (tried < 8) {
            const int mine = (pairs - xcd + 7) >> 3;  // pairs of this counter
            const int64_t items = mine > 0 ? (int64_t)mine * turns : 0;
            const int t = items > 0 ? atomicAdd(p.tickets + xcd, 1) : 0;
            if (t < items) {
                back = t / mine;
                pair = xcd + 8 * (t - back * mine);
                break;
            }
            ++tried;
            xcd = (xcd + 1) & 7;
        }
        s_ticket[slot][0] = pair;
        s_ticket[slot][1] = back;
    };
    // the ticket at hand: false when none is left
    auto use_ticket = [&]() -> bool {
        __syncthreads();
        const int pair = uniform(s_ticket[turn][0]), back = uniform(s_ticket[turn][1]);
        if (pair < 0) return false;
        turn ^= 1;
        if (threadIdx.x == 0) take_ticket(turn);
        s = pair / hkv;
        kh = pair - s * hkv;
        q = seq_of<true>(p, s, false);
        rb = q.nrb - 1 - (kWaves * back + wave);
        return true;
    };
    if (dealt == kTickets) {
        if (threadIdx.x == 0) take_ticket(0);
        if (!use_ticket()) return;
    }

    uint32_t q_at = (uint32_t)(wave * (8 * kRT * 64) + lane);
    const uint32_t scale_at = (uint32_t)a.block_size * TQ_HEAD_DIM;
    const uint32_t k_off = 128 * (n & 15) + 16 * h, v_off = 512 * h + 16 * n;

    while (dealt == kTickets || seg < p1) {
        const int64_t u = q.a + (int64_t)q.step * rb;
        const int nsteps = rb >= 0 ? (visible(p, q, rb) + 31) >> 5 : 0;
        int j0 = 0, j1 = nsteps;
        bool mine = dealt == kTickets ? rb >= 0 : seg >= p0;
        if (dealt == kShares) {
            // the steps that begin in [p0, p1)
            const int64_t from = p0 > seg ? p0 - seg : 0, to = p1 - seg < u ? p1 - seg : u;
            j0 = (int)((from + 31) >> 5);
            const int64_t je = (to + 31) >> 5;
            j1 = (int)(je < nsteps ? je : nsteps);
            mine = j0 < j1 || (nsteps == 0 && seg >= p0);
        }
        j0 = uniform(j0);
        j1 = uniform(j1);
        if (mine) {
            const int computed = q.nq < p.max_q ? q.nq : p.max_q;
            auto row_of = [&](int rt, int& i, int& head) {
                const uint32_t row = (uint32_t)(rb * kRows + 32 * rt + n);
                i = (int)tq_udiv_apply(row, p.at.group_div);
                head = kh * group + (int)(row - (uint32_t)i * (uint32_t)group);
            };
            // tokens that every row sees
            const int least = p.causal ? q.L - q.nq + (int)tq_udiv_apply((uint32_t)(rb * kRows), p.at.group_div) + 1 : q.L;

            // ---- the query rows ----
            int seen[kRT];
            float c1[kRT];
            tq_half8 qh[kQLds ? 1 : kRT][kQLds ? 1 : 8], ql[FINE ? kRT : 1][8];
            tq_half8* q_out = reinterpret_cast<tq_half8*>(s_lds) + q_at;
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                int i, head;
                row_of(rt, i, head);
                const bool real = i < computed;
                const int sn = p.causal ? q.L - q.nq + i + 1 : q.L;  // tokens that the row sees
                seen[rt] = real && sn > 0 ? (sn < q.L ? sn : q.L) : 0;
                const int64_t off = (int64_t)(q.q0 + (real ? i : 0)) * a.q_stride_token + (int64_t)(real ? head : 0) * a.q_stride_head + 16 * h;
                float x[32], y[32], m = 0.f;
                kv8_load32(a.q, off, 32, a.q_dtype, x);
                kv8_load32(a.q, off + 64, 32, a.q_dtype, y);
#pragma unroll
                for (int k = 0; k < 32; ++k) m = fmaxf(m, fmaxf(__builtin_fabsf(x[k]), __builtin_fabsf(y[k])));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                float back;
                const float f = kv8_query_factor(m, a.sm_scale < 0.f, back);
                tq_half8 hi[2][4], lo[2][4];
                kv8_query_half<FINE>(x, f, hi[0], lo[0]);
                kv8_query_half<FINE>(y, f, hi[1], lo[1]);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (kQLds) q_out[(k * kRT + rt) * 64] = hi[k >> 2][k & 3];
                    else qh[kQLds ? 0 : rt][kQLds ? 0 : k] = hi[k >> 2][k & 3];
                    if (FINE) ql[FINE ? rt : 0][k] = lo[k >> 2][k & 3];
                }
                c1[rt] = __builtin_fabsf(a.sm_scale) * kKv8Log2e * back;
            }

            const uint8_t* kb = static_cast<const uint8_t*>(a.k_cache) + kh * a.k_stride_head;
            const uint8_t* vb = static_cast<const uint8_t*>(a.v_cache) + kh * a.v_stride_head;
            const int32_t* bt = a.block_tables + s * a.block_table_stride;
            const int last_tile = q.L > 0 ? (q.L - 1) >> 4 : 0;

            // ---- 64 tiles at a time, one per lane: where their codes are, rows in use, the scales' exponents ----
            // (work on a tile's address is done here once; a scalar instruction per step costs a wave as much as a vector one)
            struct Tiles {
                uint32_t klo, khi, vlo, vhi;
                int what;  // rows in use, K's exponent << 8, V's exponent << 16, both + 127
            };
            auto tiles_from = [&](int t0) -> Tiles {
                const int ti = t0 + lane;
                const int tc = ti < last_tile ? ti : last_tile;  // (behind the last: a valid address, no rows)
                const int b = (int)tq_udiv_apply((uint32_t)tc, p.at.tpb_div);
                int blk = bt[b];
                int nv = q.L - 16 * ti;
                nv = nv < 16 ? (nv > 0 ? nv : 0) : 16;
                if ((uint32_t)blk >= (uint64_t)a.num_blocks) {
                    blk = 0;
                    nv = 0;
                }
                const uint64_t kblk = (uint64_t)kb + blk * a.k_stride_block, vblk = (uint64_t)vb + blk * a.v_stride_block;
                const uint32_t ke = *reinterpret_cast<const uint32_t*>(kb + blk * a.k_stride_block + scale_at) >> 23;
                const uint32_t ve = *reinterpret_cast<const uint32_t*>(vb + blk * a.v_stride_block + scale_at) >> 23;
                const uint32_t in = (uint32_t)(tc - p.at.tpb * b) * (16 * TQ_HEAD_DIM);
                return {(uint32_t)(kblk + in), (uint32_t)((kblk + in) >> 32), (uint32_t)(vblk + in), (uint32_t)((vblk + in) >> 32),
                        (int)((uint32_t)nv | (ke & 255u) << 8 | (nv ? ve & 255u : 0u) << 16)};
            };
            auto address = [](uint32_t lo, uint32_t hi, int i) -> uint64_t {
                return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)lo, i) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, i) << 32;
            };
            // (named as global memory: the compiler takes a number for any kind, and a load that may be from LDS keeps the
            // query operands' waits waiting)
            using GlobalWords = const __attribute__((address_space(1))) tq_u32x4*;
            tq_u32x4 kw[4], vw[2][2];
            auto load_keys = [&](const Tiles& t, int i) {
                const uint64_t a0 = address(t.klo, t.khi, i), a1 = address(t.klo, t.khi, i + 1);
                const GlobalWords src = (GlobalWords)((n < 16 ? a0 : a1) + k_off);
#pragma unroll
                for (int c = 0; c < 4; ++c) kw[c] = src[2 * c];
            };
            auto load_values = [&](const Tiles& t, int i) {
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const GlobalWords src = (GlobalWords)(address(t.vlo, t.vhi, i + v) + v_off);
#pragma unroll
                    for (int k = 0; k < 2; ++k) vw[v][k] = src[64 * k];
                }
            };

            float M[kRT], lsum[kRT];
            bool far = false;  // s_base holds the rows' bases
            int vref = 0;  // exponent + 127 of the largest V scale so far (0: none)
            f32x16 acc[kRT][4];
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                M[rt] = kKv8None;
                lsum[rt] = 0.f;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[rt][d][v] = 0.f;
            }

            // The loads of step j + 1 go out during step j without a condition (behind the last step, those of the sequence's last
            // tile): where the compiler cannot count what is under way, it waits for all of it.  31 steps use a group of 64
            // tiles, whose last two are the first of the next.
            Tiles nxt = {0, 0, 0, 0, 0};
            tq_half8 b_first[kFirst];  // the first query operands, the same in every step
            if (j0 < j1) {
                nxt = tiles_from(2 * j0);
                load_keys(nxt, 0);
                load_values(nxt, 0);
                if (kQLds) {
#pragma unroll
                    for (int i = 0; i < kFirst; ++i) b_first[i] = reinterpret_cast<const tq_half8*>(s_lds)[q_at + i * 64];
                }
            }
            for (int jg = j0; jg < j1; jg += 31) {
                const int je = jg + 31 < j1 ? jg + 31 : j1;
                const Tiles cur = nxt;
                nxt = tiles_from(2 * jg + 62);
                for (int j = jg; j < je; ++j) {
                    const int i = 2 * (j - jg);
                    int ke[2], ve[2], nv[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int w = __builtin_amdgcn_readlane(cur.what, i + t);
                        nv[t] = w & 255;
                        ke[t] = (w >> 8) & 255;
                        ve[t] = (w >> 16) & 255;
                    }
                    // ---- scores ----
                    // (the operands' place is hidden from the compiler, which would keep all of them in registers)
                    if (kQLds) asm volatile("" : "+v"(q_at));
                    const tq_half8* q_in = reinterpret_cast<const tq_half8*>(s_lds) + q_at;
                    f32x16 sc[kRT];
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
                        for (int v = 0; v < 16; ++v) sc[rt][v] = 0.f;
                    if (kQLds) {
                        // operand i = slice i / 2, row tile i % 2
                        tq_half8 k;
#pragma unroll
                        for (int i = 0; i < 8 * kRT; ++i) {
                            const int c = i / kRT, rt = i % kRT;
                            if (rt == 0) k = kv8_half8<ENC>(kw[c >> 1][2 * (c & 1)], kw[c >> 1][2 * (c & 1) + 1], 1.f, 1.f);
                            sc[rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, i < kFirst ? b_first[i < kFirst ? i : 0] : q_in[i * 64], sc[rt], 0, 0, 0);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const tq_half8 k = kv8_half8<ENC>(kw[c >> 1][2 * (c & 1)], kw[c >> 1][2 * (c & 1) + 1], 1.f, 1.f);
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt) {
                                sc[rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[kQLds ? 0 : rt][kQLds ? 0 : c], sc[rt], 0, 0, 0);
                                if (FINE) sc[rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[FINE ? rt : 0][c], sc[rt], 0, 0, 0);
                            }
                        }
                    }
                    load_keys(cur, i + 2);
                    if (32 * j + 32 > least || nv[0] + nv[1] != 32) {
#pragma unroll
                        for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const int sn = seen[rt] - 32 * j - 16 * t, upto = (sn < nv[t] ? sn : nv[t]) - 4 * h;
#pragma unroll
                                for (int v = 0; v < 8; ++v)
                                    if (8 * (v >> 2) + (v & 3) >= upto) sc[rt][8 * t + v] = kKv8NegInf;
                            }
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint32_t keep = kv8_keep(nv[t] - 8 * k - 4 * h);
#pragma unroll
                                for (int d = 0; d < 4; ++d) vw[t][k][d] &= keep;
                            }
                        }
                        // (a NaN among the values must not reach the rows that do not see its token, as 0 * NaN: here its code
                        // becomes 0, and the rows that do see it get theirs after the stores)
                        if (ENC == TQ_E4M3 && 32 * j + 32 > least) {
                            uint32_t nans = 0;
#pragma unroll
                            for (int t = 0; t < 2; ++t)
#pragma unroll
                                for (int k = 0; k < 2; ++k)
#pragma unroll
                                    for (int d = 0; d < 4; ++d) nans |= kv8_nan_bytes(vw[t][k][d]);
                            if (__builtin_amdgcn_ballot_w64(nans != 0)) {
#pragma unroll
                                for (int t = 0; t < 2; ++t)
#pragma unroll
                                    for (int k = 0; k < 2; ++k)
#pragma unroll
                                        for (int d = 0; d < 4; ++d) {
                                            const uint32_t nan = kv8_nan_bytes(vw[t][k][d]);
                                            vw[t][k][d] &= ~((nan << 1) - (nan >> 7));
                                        }
                                s_nan[wave] = 1;
                            }
                        }
                    }
                    // ---- online softmax ----
                    tq_half8 ph[kRT][2], pl[FINE ? kRT : 1][2];
#pragma unroll
                    for (int rt = 0; rt < kRT; ++rt) {
                        // (over zero, so that a masked score stays -inf)
                        float f[2] = {fmaxf(c1[rt] * kv8_scale(ke[0]), 1e-37f), fmaxf(c1[rt] * kv8_scale(ke[1]), 1e-37f)};
                        auto probabilities = [&](float base) -> float {
                            float sum[2];
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                float pr[8];
#pragma unroll
                                for (int v = 0; v < 8; ++v) pr[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rt][8 * t + v], f[t], -base));
                                kv8_prob8<FINE>(pr, ph[rt][t], pl[FINE ? rt : 0][t]);
                                sum[t] = kv8_sum8<FINE>(pr, ph[rt][t]);
                            }
                            return sum[0] + sum[1];
                        };
                        float sum = probabilities(M[rt]);
                        if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum > Base<FINE>::move_sum) != 0, 0)) {
                            float mt[2];
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                mt[t] = fmaxf(fmaxf(fmaxf(sc[rt][8 * t], sc[rt][8 * t + 1]), fmaxf(sc[rt][8 * t + 2], sc[rt][8 * t + 3])),
                                              fmaxf(fmaxf(sc[rt][8 * t + 4], sc[rt][8 * t + 5]), fmaxf(sc[rt][8 * t + 6], sc[rt][8 * t + 7])));
                            const float mx = fmaxf(mt[0] * f[0], mt[1] * f[1]);
                            const float top = fmaxf(mx, __shfl_xor(mx, 32, 64));
                            float old = M[rt];
                            if (far && old == kKv8None) old = s_base[wave][rt][lane];
                            const float Mn = fmaxf(old, __builtin_fabsf(top) < kKv8Far ? top - Base<FINE>::down : top);
                            const float alpha = __builtin_amdgcn_exp2f(old - Mn);
                            lsum[rt] *= alpha;
#pragma unroll
                            for (int d = 0; d < 4; ++d) acc[rt][d] *= alpha;
                            M[rt] = Mn;
                            float base = Mn;
                            if (far || __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(Mn) < kKv8Far) && Mn != kKv8None)) {
                                if (!far) {
#pragma unroll
                                    for (int r = 0; r < kRT; ++r) s_base[wave][r][lane] = M[r];
                                    far = true;
                                }
                                // far scores are rounded as their base was: what fp32 drops of a product may be many units
                                s_base[wave][rt][lane] = Mn;
                                if (!(__builtin_fabsf(Mn) < kKv8Far)) {
#pragma unroll
                                    for (int v = 0; v < 16; ++v) {
                                        float x = sc[rt][v] * f[v >> 3];
                                        asm("" : "+v"(x));  // (kept from becoming a fused step)
                                        sc[rt][v] = x - Mn;
                                    }
                                    f[0] = f[1] = 1.f;
                                    base = 0.f;
                                    M[rt] = kKv8None;
                                }
                            }
                            sum = probabilities(base);
                        }
                        lsum[rt] += sum;
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        // (tile by tile: a row that sees the first alone keeps all bits of it)
                        if (ve[t] > vref) {  // wave-uniform
                            const float r = kv8_scale(127 + vref - ve[t] > 0 ? 127 + vref - ve[t] : 0);
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
                                for (int d = 0; d < 4; ++d) acc[rt][d] *= r;
                            vref = ve[t];
                        }
                        const float vf = kv8_step(ve[t] - vref);
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const tq_half8 v = kv8_half8<ENC>(vw[t][0][d], vw[t][1][d], vf, vf);
#pragma unroll
                            for (int rt = 0; rt < kRT; ++rt) {
                                acc[rt][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[rt][t], acc[rt][d], 0, 0, 0);
                                if (FINE) acc[rt][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[FINE ? rt : 0][t], acc[rt][d], 0, 0, 0);
                            }
                        }
                    }
                    load_values(cur, i + 2);
                }
            }

            // ---- the piece's rows: acc[rt][d][4k + r] is dim 32k + 16h + 4r + d of row n ----
            const bool complete = j0 == 0 && j1 == nsteps;
#pragma unroll
            for (int rt = 0; rt < kRT; ++rt) {
                const float l = lsum[rt] + __shfl_xor(lsum[rt], 32, 64);
                int i, head;
                row_of(rt, i, head);
                // (a piece is divided by its own sum: plain sums of large values pass fp32's range)
                const float f = l == 0.f ? 0.f : kv8_scale(vref) / l;
                if (i < computed) {
                    const int64_t row = (int64_t)(2 * w + (seg > p0 ? 1 : 0)) * kRows + 32 * rt + n;
                    const int64_t at = complete ? (int64_t)(q.q0 + i) * a.out_stride_token + (int64_t)head * a.out_stride_head : row * TQ_HEAD_DIM;
                    void* dst = complete ? a.out : (void*)p.at.ws_acc;
                    const int dt = complete ? a.out_dtype : TQ_F32;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float o[16];
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int d = 0; d < 4; ++d) o[4 * r + d] = acc[rt][d][4 * k + r] * f;
                        kv8_store<16>(dst, at + 32 * k + 16 * h, dt, o);
                    }
                    if (!complete && h == 0) {
                        p.at.ws_ml[2 * row] = far && M[rt] == kKv8None ? s_base[wave][rt][lane] : M[rt];
                        p.at.ws_ml[2 * row + 1] = l;
                    }
                }
            }
            if (ENC == TQ_E4M3 && uniform(s_nan[wave])) {
                s_nan[wave] = 0;
                __threadfence_block();
                const int from = least > 32 * j0 ? least & ~31 : 32 * j0, to = 32 * j1 < q.L ? 32 * j1 : q.L;
                for (int t = from; t < to; ++t) {
                    const int b = (int)tq_udiv_apply((uint32_t)(t >> 4), p.at.tpb_div), in = t - b * a.block_size;
                    const int blk = bt[b];
                    if ((uint32_t)blk >= (uint64_t)a.num_blocks) continue;
                    const uint8_t* codes = vb + blk * a.v_stride_block + 512 * (in >> 2) + (in & 3);
                    for (int d = lane; d < TQ_HEAD_DIM; d += 64) {
                        if ((codes[4 * d] & 0x7f) != 0x7f) continue;
                        for (int r = 0; r < kRows; ++r) {
                            const uint32_t x = (uint32_t)(rb * kRows + r);
                            const int i = (int)tq_udiv_apply(x, p.at.group_div);
                            if (i >= computed || t >= (p.causal ? q.L - q.nq + i + 1 : q.L)) continue;
                            const int head = kh * group + (int)(x - (uint32_t)i * (uint32_t)group);
                            if (complete) tq_store1(a.out, (int64_t)(q.q0 + i) * a.out_stride_token + (int64_t)head * a.out_stride_head + d, a.out_dtype, __builtin_nanf(""));
                            else p.at.ws_acc[((int64_t)(2 * w + (seg > p0 ? 1 : 0)) * kRows + r) * TQ_HEAD_DIM + d] = __builtin_nanf("");
                        }
                    }
                }
            }
        }
        // next segment
        if (dealt == kTickets) {
            if (!use_ticket()) return;
            continue;
        }
        seg += u;
        if (++rb == q.nrb) {
            rb = 0;
            if (++kh == hkv) {
                kh = 0;
                do {
                    ++s;
                    if (s >= a.num_seqs) return;
                    q = seq_of<true>(p, s, whole);
                } while (q.nrb == 0);
            }
        }
    }
}

// Joins the pieces of the segments that several workers share: workgroup (w - 1, y) takes the segment that worker
// w's record names; 32 lanes per row (4 dims each), 8 rows, 8 pieces requested together.  Every piece
// holds at least one step: a worker's range is at least kMinTokens long.
// out = sum_i w_i out_i / sum_i w_i, w_i = 2^(M_i - M) l_i, as a running mean, which stays within the values' range.
__global__ __launch_bounds__(256) void kv8_prefill_merge_kernel(Prefill p) {
    const int w = (int)blockIdx.x + 1;
    if (w >= p.cuts[0].rb) return;
    const Cut cut = p.cuts[w];
    if (cut.w0 < 0) return;
    const tq_kv8_attn_args& args = p.at.a;
    const int l32 = threadIdx.x & 31;
    const int r0 = 8 * (int)blockIdx.y + (int)(threadIdx.x >> 5);
    const uint32_t row = (uint32_t)(cut.rb * p.rows + r0);
    const int i = (int)tq_udiv_apply(row, p.at.group_div);
    if (i >= (cut.nq < p.max_q ? cut.nq : p.max_q)) return;
    float M = kKv8NegInf, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int wb = cut.w0; wb <= cut.w1; wb += 8) {
        float mp[8], lp[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int wk = wb + k;
            mp[k] = kKv8NegInf;
            lp[k] = 0.f;
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (wk <= cut.w1) {
                const int64_t x = (int64_t)(wk == cut.w0 ? cut.slot0 : 2 * wk) * p.rows + r0;
                mp[k] = p.at.ws_ml[2 * x];
                lp[k] = p.at.ws_ml[2 * x + 1];
                v[k] = *reinterpret_cast<const float4*>(p.at.ws_acc + x * TQ_HEAD_DIM + 4 * l32);
            }
        }
        float Mn = M;
#pragma unroll
        for (int k = 0; k < 8; ++k) Mn = fmaxf(Mn, mp[k]);
        kv8_join<8>(M, l, a, Mn, mp, lp, v);
    }
    const float o[4] = {a.x, a.y, a.z, a.w};
    const int head = cut.kh * p.at.group + (int)(row - (uint32_t)i * (uint32_t)p.at.group);
    kv8_store<4>(args.out, (int64_t)(cut.q0 + i) * args.out_stride_token + (int64_t)head * args.out_stride_head + 4 * l32, args.out_dtype, o);
}

// workers that a call can use at most (counted for row blocks of 32: FINE's, and twice the others')
int64_t most_workers(int64_t num_seqs, int64_t max_q_len, int64_t group, int64_t hkv, int64_t cap) {
    const int64_t blocks = (max_q_len * group + 31) / 32;
    const int64_t per = (cap + kSegTokens + 2 * kMinTokens) / kMinTokens;
    if (num_seqs > kMaxWorkers || blocks > kMaxWorkers || hkv > kMaxWorkers || per > kMaxWorkers) return kMaxWorkers;
    // (each factor fits 12 bits)
    const int64_t m = num_seqs * blocks * hkv * per;
    return m < kMaxWorkers ? (m < 1 ? 1 : m) : kMaxWorkers;
}

__global__ void kv8_tickets_kernel(int* tickets) { tickets[threadIdx.x] = 0; }

}  // namespace

extern "C" int64_t tq_kv8_prefill_workspace_bytes(int num_seqs, int max_q_len, int num_q_heads, int num_kv_heads,
                                                  int max_blocks_per_seq, int block_size) {
    if (num_seqs <= 0 || max_q_len <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || max_blocks_per_seq < 0 ||
        block_size <= 0)
        return 0;
    const int64_t w = most_workers(num_seqs, max_q_len, num_q_heads / num_kv_heads, num_kv_heads, (int64_t)max_blocks_per_seq * block_size);
    // pieces (two per worker, 64 rows), the tickets, the cuts
    return w * (2 * 64 * (TQ_HEAD_DIM + 2) * 4 + (int64_t)sizeof(Cut)) + 8 * 4;
}

extern "C" int tq_kv8_prefill(const tq_kv8_attn_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    Prefill p = {};
    const int rc = tq_kv8_attn_setup(a, &p.at);
    if (rc != TQ_OK) return rc;
    if (a->max_q_len < 0 || (a->flags & ~TQ_PREFILL_CAUSAL)) return TQ_ERR_INVALID_ARGUMENT;
    if (a->num_seqs == 0 || a->max_q_len == 0) return TQ_OK;
    if (!a->q || !a->out || !a->k_cache || !a->v_cache || (!a->block_tables && a->max_blocks_per_seq) || !a->seq_lens || !a->cu_seqlens_q)
        return TQ_ERR_INVALID_ARGUMENT;
    // (row numbers and a row block's tokens stay in 32 bits)
    if ((int64_t)a->max_q_len * p.at.group > 0x7fffff00) return TQ_ERR_INVALID_ARGUMENT;
    const int64_t need = tq_kv8_prefill_workspace_bytes(a->num_seqs, a->max_q_len, a->num_q_heads, a->num_kv_heads,
                                                        a->max_blocks_per_seq, a->block_size);
    if (!a->workspace || (uintptr_t)a->workspace % 256 || a->workspace_bytes < need) return TQ_ERR_WORKSPACE;
    const int cus = tq_kv8_cus();
    if (cus <= 0) return (int)hipErrorNoDevice;
    const bool fine = a->q_dtype == TQ_F32 || a->out_dtype == TQ_F32;
    const int64_t most = most_workers(a->num_seqs, a->max_q_len, p.at.group, a->num_kv_heads, (int64_t)a->max_blocks_per_seq * a->block_size);
    const int64_t resident = (int64_t)cus * kWavesPerCu;
    p.at.workers = (int)(most < resident ? most : resident);
    p.max_q = a->max_q_len;
    p.causal = (a->flags & TQ_PREFILL_CAUSAL) != 0;
    p.row_bits = fine ? 5 : 6;
    p.rows = 1 << p.row_bits;
    p.step = (p.rows + p.at.group - 1) / p.at.group;
    p.grow = (p.rows - 1) / p.at.group + 1;
    p.at.ws_acc = static_cast<float*>(a->workspace);
    p.at.ws_ml = p.at.ws_acc + most * 2 * 64 * TQ_HEAD_DIM;
    int* tickets = reinterpret_cast<int*>(p.at.ws_ml + most * 2 * 64 * 2);
    p.cuts = reinterpret_cast<Cut*>(tickets + 8);
    // (at most as many segments as this)
    const int64_t pairs = (int64_t)a->num_seqs * a->num_kv_heads;
    const int64_t blocks = ((int64_t)a->max_q_len * p.at.group + p.rows - 1) / p.rows;
    if (pairs <= 0x7fffff && blocks <= 0x7fffffff / pairs && pairs * blocks >= resident && p.at.workers == resident && resident % 8 == 0)
        p.tickets = tickets;
    const void* kern = a->encoding == TQ_E4M3 ? (fine ? (const void*)kv8_prefill_kernel<TQ_E4M3, true> : (const void*)kv8_prefill_kernel<TQ_E4M3, false>)
                                              : (fine ? (const void*)kv8_prefill_kernel<TQ_INT8, true> : (const void*)kv8_prefill_kernel<TQ_INT8, false>);
    const unsigned lds = fine ? 0 : kWaves * 8 * 2 * 64 * 16;  // 64 KB
    // one wave per workgroup while the workers are few: they spread over the compute units
    int64_t grid = (int64_t)cus * (kWavesPerCu / kWaves);
    grid = grid < p.at.workers ? grid : p.at.workers;
    void* args[] = {&p};
    hipError_t e = hipSuccess;
    if (p.tickets) {
        void* zero[] = {&tickets};
        e = hipLaunchKernel((const void*)kv8_tickets_kernel, dim3(1), dim3(8), zero, 0, stream);
    }
    if (e == hipSuccess) e = hipLaunchKernel(kern, dim3((unsigned)grid), dim3(64 * kWaves), args, lds, stream);
    if (e == hipSuccess && p.at.workers > 1)
        e = hipLaunchKernel((const void*)kv8_prefill_merge_kernel, dim3((unsigned)p.at.workers - 1, (unsigned)p.rows / 8), dim3(256), args, 0, stream);
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
