// Eviction from the 8-bit paged caches by accumulated weight (tiles: tq_kv8.h).
//
// A segment is a (sequence, KV head).  The plan, a workgroup per segment, finds which tokens stay: the m-th largest number between
// the first and the last ones by three passes over 11, 11 and 10 bits of the numbers' order (counts in LDS; up to
// 32768 tokens' numbers stay in registers), then the tokens above it and the first ones equal to it, in order by one
// scan.  The kept rows move in units of 16, a wave each: their bytes, V's taken out of words of four tokens and put together
// again, and where a block's largest scale is another's, rescaled.  Three ways:
//   kv8_evict_segment_kernel  plan and move by one workgroup, a barrier between a round's loads and its stores: many segments
//   kv8_evict_move_kernel     any workgroup moves any unit; units wait for those that what they overwrite goes to: few segments
//   gather and scatter        through the workspace: blocks of more than 64 rows, whose scales take a kernel of their own
//
// Bound: memory, 512 bytes of codes a kept token: 32 x 4352 tokens of 8 heads cut to 4096, 546 MB in 192 us, 2.8 TB/s where a
// copy moves 4.7.  One compute unit has some 20 GB/s of it, so the segment kernel needs most of them busy and 16 to 20 kB a round
// under way; the move kernel pays for its flags (208 us there, some 50 less where nothing has to wait) and, where single tokens stay,
// for V's words of four tokens: 16 sequences of 3001 to 32768 tokens cut to 8190 need 168 MB of codes read and as much written, and by
// counters 279 MB are read, in 29 + 149 us.  One prompt of 32768: 31 us for the plan, one workgroup for 32768 numbers, and 11.
// (Kernel times of a fresh cache's first cut.  Cut again, its scales have met and fewer rows are rounded: 185, 29 + 130, 31 + 11.)
#include "tq_kv8.h"

namespace {

constexpr int kInPlace = 64;                      // rows of a block, at most, that move without the workspace
constexpr int kMove = 4;                          // waves, and units, of a ticket
// Segments from which on a workgroup takes a whole one: with most of them cut that keeps most compute units busy and needs no flags (kernel
// times; 4352 tokens cut to 4096, 8 heads, all sequences: 176 segments 166 us against the plan's and the move kernel's 161, 192: 177
// against 179, 256: 192 against 236; 128 segments, 80 of them of up to 26172 tokens cut to 8190: 350 against 177).  The lengths are on the
// device, so those that stay as they are count too, and a call of many sequences of which few are cut pays for it: of 256 segments
// 8 cut 135 against 41, 64: 147 against 83, 128: 166 against 135, 160: 177 against 161, 192: 181 against 186; one sequence of
// 32768 cut to 8190 among 24: 331 against 59.
constexpr int kSegments = 192;
constexpr int kPad = 32;                          // words between tickets: a cache line each
constexpr int kUnit = 16;                         // rows that a wave moves
constexpr int kStage = 2 * kUnit * TQ_HEAD_DIM;   // their codes

struct Evict {
    tq_kv8_evict_args a;
    tq_udiv tpb_div;
    int tpb, cap, units, blocks;  // units and blocks of what is kept
    int2* list;                   // [segment][16 units]: block (-1: a bad entry) and row of the kept tokens
    int32_t* ranks;               // [segment][units + 1]: kept tokens before token 16 u
    int32_t* loaded;              // [segment][units]: 1 once the unit's rows and scales are in registers
    int32_t* cut;                 // [segment]: 1 where the plan cuts the sequence, for all kernels
    int32_t* ticket;              // [segment][kPad]: the next one (away from what is only read)
    int items;                    // workgroups of a segment
    uint16_t* shift;              // [segment][16 units]: exponents that K's (low byte) and V's codes fall by; 63: zeros
    float2* scales;               // [segment][blocks]: K's and V's
    uint8_t* stage;               // [segment][units][kStage]
    float* stage_mass;            // [segment][16 units]
};

__device__ __forceinline__ int length_of(const Evict& p, int s) {
    const int L = p.a.seq_lens[s];
    return L < p.cap ? (L > 0 ? L : 0) : p.cap;
}
// order of the numbers as whole numbers: -0 as 0, NaN below all
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x == x)) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// block of tile t (16 tokens) of sequence s; -1: a bad entry
__device__ __forceinline__ int block_of(const Evict& p, int s, int tile, int& row) {
    const int b = (int)tq_udiv_apply((uint32_t)tile, p.tpb_div);
    row = 16 * (tile - b * p.tpb);
    const int blk = p.a.block_tables[s * p.a.block_table_stride + b];
    return (uint32_t)blk < (uint64_t)p.a.num_blocks ? blk : -1;
}

constexpr int kPlan = 1024;
constexpr int kQuads = 8;  // of tokens that a thread of the plan keeps in registers: 32768 tokens in all

// inclusive sum over the workgroup's threads in order; total: of all of them (two barriers)
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t* s_tot, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = (uint32_t)__shfl_up((int)x, d, 64);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) s_tot[wave] = x;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (int w = 0; w < kPlan / 64; ++w) {
        const uint32_t y = s_tot[w];
        before += w < wave ? y : 0u;
        total += y;
    }
    return x + before;
}

struct PlanLds {
    uint32_t hist[2048], tot[kPlan / 64], pick[2];
};
// (hist, at the end)
struct PlanSums {
    uint32_t kept[kQuads * (kPlan / 64)], equal[kQuads * (kPlan / 64)];
};

// The kept tokens of segment (s, kh), L > longer_than tokens long, to p.list.  REGS: L <= 4 kQuads kPlan, so that the numbers
// are read once.
template <bool REGS>
__device__ void plan(const Evict& p, uint32_t seg, int s, int kh, int L, PlanLds& lds) {
    const int tid = threadIdx.x;
    const int c0 = p.a.sinks, c1 = L - p.a.recent;  // candidates
    const float* mass = p.a.mass + kh * p.a.mass_stride_head;
    // keys of tokens t .. t + 3 (t a multiple of 4)
    auto load = [&](int t, uint32_t (&k)[4], int2& at) {
        int row;
        const int blk = block_of(p, s, t >> 4, row);
        at = make_int2(blk, row + (t & 15));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (blk >= 0) x = *reinterpret_cast<const float4*>(mass + blk * p.a.mass_stride_block + row + (t & 15));
        k[0] = blk < 0 ? 0u : key_of(x.x);
        k[1] = blk < 0 ? 0u : key_of(x.y);
        k[2] = blk < 0 ? 0u : key_of(x.z);
        k[3] = blk < 0 ? 0u : key_of(x.w);
    };
    uint32_t key[REGS ? kQuads : 1][4];
    int2 at[REGS ? kQuads : 1];
    if (REGS) {
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int t = 4 * (q * kPlan + tid);
            load(t < L ? t : 0, key[REGS ? q : 0], at[REGS ? q : 0]);
        }
    }
    // ---- the least key that stays, and how many of the tokens with it ----
    uint32_t least = 0xffffffffu, need = (uint32_t)(p.a.keep - p.a.sinks - p.a.recent), mask = 0;
    if (need) {
        least = 0;
        for (int pass = 0; pass < 3; ++pass) {
            const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < 2048; i += kPlan) lds.hist[i] = 0;
            __syncthreads();
            auto count = [&](int t, const uint32_t (&k)[4]) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i >= c0 && t + i < c1 && (k[i] & mask) == least) atomicAdd(&lds.hist[(k[i] >> sh) & (bins - 1)], 1u);
            };
            if (REGS) {
#pragma unroll
                for (int q = 0; q < kQuads; ++q) count(4 * (q * kPlan + tid), key[REGS ? q : 0]);
            } else {
                for (int t = 4 * tid; t < c1; t += 4 * kPlan) {
                    uint32_t k[4];
                    int2 x;
                    load(t, k, x);
                    count(t, k);
                }
            }
            __syncthreads();
            // bins from the largest on, two a thread
            const int top = 2047 - 2 * tid;
            const uint32_t a = lds.hist[top], b = lds.hist[top - 1];
            uint32_t total;
            const uint32_t in = scan(a + b, lds.tot, total), before = in - a - b;
            if (before < need && need <= in) {
                const bool first = need <= before + a;
                lds.pick[0] = (uint32_t)(first ? top : top - 1);
                lds.pick[1] = need - before - (first ? 0u : a);
            }
            __syncthreads();
            least |= lds.pick[0] << sh;
            mask |= (uint32_t)(bins - 1) << sh;
            need = lds.pick[1];
        }
    }
    // ---- the kept tokens, in order ----
    int2* list = p.list + (int64_t)seg * (kUnit * p.units);
    int32_t* ranks = p.ranks + (int64_t)seg * (p.units + 1);
    // what a token is: 1 stays, 2 has the least key; the quad's counts, those of the latter in the upper half
    auto classify = [&](int t, const uint32_t (&k)[4], int (&what)[4]) -> uint32_t {
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = t + i;
            what[i] = x >= L ? 0 : x < c0 || x >= c1 || k[i] > least ? 1 : k[i] == least ? 2 : 0;
            n += what[i] == 1 ? 1u : what[i] == 2 ? 0x10000u : 0u;
        }
        return n;
    };
    // g, e: tokens before the quad that stay and that have the least key
    auto emit = [&](int t, int2 first, const int (&what)[4], uint32_t g, uint32_t e) {
        if (!(t & 15) && t >> 4 <= p.units) ranks[t >> 4] = (int32_t)(g + (e < need ? e : need));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (what[i] == 1 || (what[i] == 2 && e < need)) list[g + (e < need ? e : need)] = make_int2(first.x, first.y + i);
            g += what[i] == 1;
            e += what[i] == 2;
        }
    };
    if (REGS) {
        // one pass over all quads: each wave's sums, then those before each of them
        const int lane = tid & 63, wave = tid >> 6;
        PlanSums& sums = *reinterpret_cast<PlanSums*>(lds.hist);
        uint32_t in[kQuads];
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            int what[4];
            in[q] = classify(4 * (q * kPlan + tid), key[REGS ? q : 0], what);
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t y = (uint32_t)__shfl_up((int)in[q], d, 64);
                if (lane >= d) in[q] += y;
            }
        }
        __syncthreads();
        constexpr int kSums = kQuads * (kPlan / 64);
        if (lane == 63) {
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                sums.kept[q * (kPlan / 64) + wave] = in[q] & 0xffffu;
                sums.equal[q * (kPlan / 64) + wave] = in[q] >> 16;
            }
        }
        __syncthreads();
        static_assert(kSums == 128, "two a lane");
        if (wave < 2) {
            uint32_t* x = wave ? sums.equal : sums.kept;
            const uint32_t a = x[2 * lane], b = x[2 * lane + 1];
            uint32_t y = a + b;
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t z = (uint32_t)__shfl_up((int)y, d, 64);
                if (lane >= d) y += z;
            }
            x[2 * lane] = y - a - b;
            x[2 * lane + 1] = y - b;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
            const int t = 4 * (q * kPlan + tid);
            int what[4];
            const uint32_t before = in[q] - classify(t, key[REGS ? q : 0], what);
            emit(t, at[REGS ? q : 0], what, sums.kept[q * (kPlan / 64) + wave] + (before & 0xffffu),
                 sums.equal[q * (kPlan / 64) + wave] + (before >> 16));
        }
    } else {
        uint32_t kept = 0, equal = 0;  // before this round
        for (int r0 = 0; r0 < L; r0 += 4 * kPlan) {
            const int t = r0 + 4 * tid;
            uint32_t k[4] = {0u, 0u, 0u, 0u};
            int2 x = make_int2(-1, 0);
            if (t < L) load(t, k, x);
            int what[4];
            const uint32_t n = classify(t, k, what);
            uint32_t total;
            const uint32_t before = scan(n, lds.tot, total) - n;
            emit(t, x, what, kept + (before & 0xffffu), equal + (before >> 16));
            kept += total & 0xffffu;
            equal += total >> 16;
        }
    }
}
// Plans the workgroup's segment; false: the sequence stays as it is
__device__ __forceinline__ bool plan_segment(const Evict& p, PlanLds& lds, int& s, int& kh) {
    const uint32_t seg = blockIdx.x;
    s = (int)(seg / (uint32_t)p.a.num_kv_heads);
    kh = (int)seg - s * p.a.num_kv_heads;
    const int L = length_of(p, s);
    const bool cut = L > p.a.longer_than;
    if (kh == 0 && threadIdx.x == 0) p.a.change[s] = cut ? p.a.keep - p.a.seq_lens[s] : 0;
    if (p.cut && threadIdx.x == 0) p.cut[seg] = cut;
    if (!cut) return false;
    if (p.loaded) {
        if (threadIdx.x == 0) p.ticket[seg * kPad] = 0;
        for (int u = threadIdx.x; u < p.units; u += kPlan) p.loaded[(int64_t)seg * p.units + u] = 0;
        if (threadIdx.x == 0 && kUnit * p.units >= L) p.ranks[(int64_t)seg * (p.units + 1) + p.units] = p.a.keep;
    }
    if (L <= 4 * kQuads * kPlan) plan<true>(p, seg, s, kh, L, lds);
    else plan<false>(p, seg, s, kh, L, lds);
    return true;
}
__global__ __launch_bounds__(kPlan) void kv8_evict_plan_kernel(Evict p) {
    __shared__ PlanLds lds;
    int s, kh;
    plan_segment(p, lds, s, kh);
}

// a tile's scale as its exponent + 127; 0: zero
__device__ __forceinline__ int exponent_at(const uint8_t* tile, const Evict& p) {
    return (int)(*reinterpret_cast<const uint32_t*>(tile + (int64_t)p.a.block_size * TQ_HEAD_DIM) >> 23) & 255;
}

// A wave per kept block: the largest scale of the blocks its rows come from, and what each row's codes fall by.
__global__ __launch_bounds__(256) void kv8_evict_scales_kernel(Evict p) {
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t seg = unit / (uint32_t)p.blocks;
    const int b = (int)(unit - seg * (uint32_t)p.blocks);
    if (seg >= (uint32_t)p.a.num_seqs * (uint32_t)p.a.num_kv_heads) return;
    const int s = (int)(seg / (uint32_t)p.a.num_kv_heads), kh = (int)seg - s * p.a.num_kv_heads;
    if (!p.cut[seg]) return;
    const int d0 = b * p.a.block_size, d1 = d0 + p.a.block_size < p.a.keep ? d0 + p.a.block_size : p.a.keep;
    const uint8_t* kc = static_cast<const uint8_t*>(p.a.k_cache) + kh * p.a.k_stride_head;
    const uint8_t* vc = static_cast<const uint8_t*>(p.a.v_cache) + kh * p.a.v_stride_head;
    const int64_t at = (int64_t)seg * (kUnit * p.units);
    auto exponents = [&](int d, int& ek, int& ev) {
        const int blk = p.list[at + d].x;
        ek = blk < 0 ? 0 : exponent_at(kc + blk * p.a.k_stride_block, p);
        ev = blk < 0 ? 0 : exponent_at(vc + blk * p.a.v_stride_block, p);
    };
    int mk = 0, mv = 0;
    for (int d = d0 + lane; d < d1; d += 64) {
        int ek, ev;
        exponents(d, ek, ev);
        mk = mk > ek ? mk : ek;
        mv = mv > ev ? mv : ev;
    }
    for (int m = 1; m < 64; m <<= 1) {
        const int x = __shfl_xor(mk, m, 64), y = __shfl_xor(mv, m, 64);
        mk = mk > x ? mk : x;
        mv = mv > y ? mv : y;
    }
    if (lane == 0) p.scales[(int64_t)seg * p.blocks + b] = make_float2(kv8_scale(mk), kv8_scale(mv));
    for (int d = d0 + lane; d < d1; d += 64) {
        int ek, ev;
        exponents(d, ek, ev);
        const int sk = ek && mk - ek < 63 ? mk - ek : 63, sv = ev && mv - ev < 63 ? mv - ev : 63;
        p.shift[at + d] = (uint16_t)(sk | sv << 8);
    }
}

// Codes of a word times f[i] (powers of two, or 0), rounded to nearest even
template <int ENC>
__device__ __forceinline__ uint32_t rescale(uint32_t w, float f0, float f1, float f2, float f3) {
    using Code = Kv8Code<ENC>;
    return Code::template pack<true>(Code::value(w, 0) * f0, Code::value(w, 1) * f1, Code::value(w, 2) * f2, Code::value(w, 3) * f3, 1.f);
}
__device__ __forceinline__ float factor_of(int shift) { return shift < 63 ? kv8_exp2i(-shift) : 0.f; }

// Where row lane of a unit (lanes 0 .. 15) comes from: block (-1: none, zeros), row in it, what its codes fall by
struct Source {
    int blk, row, sh;
};
// 16 kept rows in a wave's registers: K's rows lane / 8 and 8 + lane / 8, bytes 16 (lane % 8) ..; V's words with dims 2 lane and
// 2 lane + 1 of row i's group of four; row lane's number
struct Raw {
    tq_u32x4 k[2];
    tq_u32x2 w[kUnit];
    float mass;
};
__device__ __forceinline__ void load_raw(const Evict& p, int kh, int blk, int row, Raw& x) {
    const int lane = threadIdx.x & 63;
    x.mass = 0.f;
    if (blk >= 0 && lane < kUnit) x.mass = p.a.mass[blk * p.a.mass_stride_block + kh * p.a.mass_stride_head + row];
    {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int b = __shfl(blk, 8 * i + (lane >> 3), 64), r = __shfl(row, 8 * i + (lane >> 3), 64);
            x.k[i] = tq_u32x4{0, 0, 0, 0};
            if (b >= 0)
                x.k[i] = *reinterpret_cast<const tq_u32x4*>(static_cast<const uint8_t*>(p.a.k_cache) + b * p.a.k_stride_block +
                                                            kh * p.a.k_stride_head + (int64_t)r * TQ_HEAD_DIM + 16 * (lane & 7));
        }
    }
    const uint8_t* vc = static_cast<const uint8_t*>(p.a.v_cache) + kh * p.a.v_stride_head;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        const int b = __builtin_amdgcn_readlane(blk, i), r = __builtin_amdgcn_readlane(row, i);
        x.w[i] = tq_u32x2{0, 0};
        if (b >= 0) x.w[i] = reinterpret_cast<const tq_u32x2*>(vc + b * p.a.v_stride_block + (int64_t)(r >> 2) * 512)[lane];
    }
}
// the rows as they are stored: V's words of the unit's four groups
struct Unit {
    tq_u32x4 k[2];
    tq_u32x2 v[4];
    float mass;
};
template <int ENC>
__device__ __forceinline__ Unit arrange(const Raw& raw, int row, int sh) {
    const int lane = threadIdx.x & 63;
    Unit x;
    x.mass = raw.mass;
    x.k[0] = raw.k[0];
    x.k[1] = raw.k[1];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        x.v[g] = tq_u32x2{0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int from = 8 * (__builtin_amdgcn_readlane(row, 4 * g + i) & 3);
            x.v[g][0] |= ((raw.w[4 * g + i][0] >> from) & 255u) << (8 * i);
            x.v[g][1] |= ((raw.w[4 * g + i][1] >> from) & 255u) << (8 * i);
        }
    }
    if (__builtin_amdgcn_ballot_w64(lane < kUnit && sh != 0)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float fk = factor_of(__shfl(sh, 8 * i + (lane >> 3), 64) & 255);
            if (fk != 1.f) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x.k[i][j] = rescale<ENC>(x.k[i][j], fk, fk, fk, fk);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = factor_of(__builtin_amdgcn_readlane(sh, 4 * g + i) >> 8);
            if (f[0] != 1.f || f[1] != 1.f || f[2] != 1.f || f[3] != 1.f) {
                x.v[g][0] = rescale<ENC>(x.v[g][0], f[0], f[1], f[2], f[3]);
                x.v[g][1] = rescale<ENC>(x.v[g][1], f[0], f[1], f[2], f[3]);
            }
        }
    }
    return x;
}

// sc: the block's scales, written with its last kept rows
__device__ __forceinline__ void store_unit(const Evict& p, int s, int kh, int u, const Unit& x, float2 sc) {
    const int lane = threadIdx.x & 63;
    int row;
    const int blk = block_of(p, s, u, row);
    if (blk < 0) return;
    const int rows = p.a.keep - kUnit * u < kUnit ? p.a.keep - kUnit * u : kUnit;
    uint8_t* kt = static_cast<uint8_t*>(p.a.k_cache) + blk * p.a.k_stride_block + kh * p.a.k_stride_head;
    uint8_t* vt = static_cast<uint8_t*>(p.a.v_cache) + blk * p.a.v_stride_block + kh * p.a.v_stride_head;
    if (lane < rows) p.a.mass[blk * p.a.mass_stride_block + kh * p.a.mass_stride_head + row + lane] = x.mass;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (8 * i + (lane >> 3) < rows)
            *reinterpret_cast<tq_u32x4*>(kt + (int64_t)(row + 8 * i) * TQ_HEAD_DIM + 16 * lane) = x.k[i];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint32_t mine = kv8_keep(rows - 4 * g);
        tq_u32x2* dst = reinterpret_cast<tq_u32x2*>(vt + (int64_t)(row + 4 * g) * TQ_HEAD_DIM) + lane;
        if (mine == 0xffffffffu) {
            *dst = x.v[g];
        } else if (mine) {  // rows behind the kept ones stay
            const tq_u32x2 old = *dst;
            *dst = tq_u32x2{(x.v[g][0] & mine) | (old[0] & ~mine), (x.v[g][1] & mine) | (old[1] & ~mine)};
        }
    }
    if ((row + kUnit == p.a.block_size || u == p.units - 1) && lane == 0) {
        *reinterpret_cast<float*>(kt + (int64_t)p.a.block_size * TQ_HEAD_DIM) = sc.x;
        *reinterpret_cast<float*>(vt + (int64_t)p.a.block_size * TQ_HEAD_DIM) = sc.y;
    }
}

// wave -> (segment, unit); false: nothing to do
__device__ __forceinline__ bool unit_of(const Evict& p, uint32_t& seg, int& s, int& kh, int& u) {
    const uint32_t x = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    seg = x / (uint32_t)p.units;
    u = (int)(x - seg * (uint32_t)p.units);
    s = (int)(seg / (uint32_t)p.a.num_kv_heads);
    kh = (int)seg - s * p.a.num_kv_heads;
    return s < p.a.num_seqs && p.cut[seg];
}

template <int ENC>
__global__ __launch_bounds__(256) void kv8_evict_gather_kernel(Evict p) {
    uint32_t seg;
    int s, kh, u;
    if (!unit_of(p, seg, s, kh, u)) return;
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)seg * (kUnit * p.units) + kUnit * u;
    Source src = {-1, 0, 0};
    if (lane < p.a.keep - kUnit * u && lane < kUnit) {
        src.blk = p.list[at + lane].x;
        src.row = p.list[at + lane].y;
        src.sh = p.shift[at + lane];
    }
    Raw raw;
    load_raw(p, kh, src.blk, src.row, raw);
    const Unit x = arrange<ENC>(raw, src.row, src.sh);
    const int64_t n = (int64_t)seg * p.units + u;
    tq_u32x4* dst = reinterpret_cast<tq_u32x4*>(p.stage + n * kStage);
    dst[lane] = x.k[0];
    dst[64 + lane] = x.k[1];
#pragma unroll
    for (int g = 0; g < 4; ++g) reinterpret_cast<tq_u32x2*>(dst + 128)[64 * g + lane] = x.v[g];
    if (lane < kUnit) p.stage_mass[n * kUnit + lane] = x.mass;
}

__global__ __launch_bounds__(256) void kv8_evict_scatter_kernel(Evict p) {
    uint32_t seg;
    int s, kh, u;
    if (!unit_of(p, seg, s, kh, u)) return;
    const int lane = threadIdx.x & 63;
    const int64_t n = (int64_t)seg * p.units + u;
    const tq_u32x4* src = reinterpret_cast<const tq_u32x4*>(p.stage + n * kStage);
    Unit x;
    x.k[0] = src[lane];
    x.k[1] = src[64 + lane];
#pragma unroll
    for (int g = 0; g < 4; ++g) x.v[g] = reinterpret_cast<const tq_u32x2*>(src + 128)[64 * g + lane];
    x.mass = lane < kUnit ? p.stage_mass[n * kUnit + lane] : 0.f;
    store_unit(p, s, kh, u, x, p.scales[(int64_t)seg * p.blocks + tq_udiv_apply((uint32_t)u, p.tpb_div)]);
}

// The rows of blocks of up to 64 rows, in place.  A wave loads its unit's rows and scales, says so in p.loaded, waits until the
// units that what it overwrites goes to have said so, and stores.  A kept row's new place is not behind its old
// one, so those are units of the same segment up to this one; a segment's workgroups take its units in order by ticket, so that
// all lower ones are with running waves, and what those wait for is lower still: every wait ends.  (A load's data is in registers before its
// word is written, and the flags need no other order: what is stored is not read again in this launch.)
template <int ENC>
__global__ __launch_bounds__(64 * kMove, 8) void kv8_evict_move_kernel(Evict p) {
    __shared__ int s_ticket;
    // (the 8 XCDs have a segment's workgroups in turn: with all of them on one, 32 x 4352 tokens cut to 4096 took a third longer, 284 us)
    const uint32_t seg = blockIdx.x / (uint32_t)p.items;
    const int s = (int)(seg / (uint32_t)p.a.num_kv_heads), kh = (int)seg - s * p.a.num_kv_heads;
    if (!p.cut[seg]) return;
    if (threadIdx.x == 0) s_ticket = __hip_atomic_fetch_add(p.ticket + seg * kPad, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int u = __builtin_amdgcn_readfirstlane(s_ticket) * kMove + wave;
    if (u >= p.units) return;
    const int2* list = p.list + (int64_t)seg * (kUnit * p.units);
    const int32_t* ranks = p.ranks + (int64_t)seg * (p.units + 1);
    int32_t* loaded = p.loaded + (int64_t)seg * p.units;
    const uint8_t* kc = static_cast<const uint8_t*>(p.a.k_cache) + kh * p.a.k_stride_head;
    const uint8_t* vc = static_cast<const uint8_t*>(p.a.v_cache) + kh * p.a.v_stride_head;
    {
        const int b = (int)tq_udiv_apply((uint32_t)u, p.tpb_div), first = kUnit * (u - b * p.tpb);
        // ---- lane l: row l of the unit's block, its own rows being first .. first + 15 ----
        const int d = kUnit * u - first + lane;
        int blk = -1, row = 0;
        if (lane < p.a.block_size && d < p.a.keep) {
            blk = list[d].x;
            row = list[d].y;
        }
        const int ek = blk < 0 ? 0 : exponent_at(kc + blk * p.a.k_stride_block, p);
        const int ev = blk < 0 ? 0 : exponent_at(vc + blk * p.a.v_stride_block, p);
        const int mine = first + (lane & 15);
        const int from = __shfl(row, mine, 64);
        Raw raw;
        load_raw(p, kh, __shfl(blk, mine, 64), from, raw);
        // the units that the old rows here go to; with the block's last unit, which writes its scales, all units of the
        // blocks that rows of the old block go to
        const bool last = first + kUnit == p.a.block_size || u == p.units - 1;
        int w0, w1;
        if (last) {
            // (rows of the last block that lie behind the kept units count too)
            const int r0 = ranks[b * p.tpb], r1 = (b + 1) * p.tpb <= p.units ? ranks[(b + 1) * p.tpb] : p.a.keep;
            w0 = r0 < r1 ? (int)tq_udiv_apply((uint32_t)(r0 >> 4), p.tpb_div) * p.tpb : u;
            w1 = r0 < r1 ? ((int)tq_udiv_apply((uint32_t)((r1 - 1) >> 4), p.tpb_div) + 1) * p.tpb : u;
        } else {
            const int r0 = ranks[u], r1 = ranks[u + 1];
            w0 = r0 < r1 ? r0 >> 4 : u;
            w1 = r0 < r1 ? ((r1 - 1) >> 4) + 1 : u;
        }
        w1 = w1 < u ? w1 : u;
        // ---- what the rows' codes fall by ----
        int mk = ek, mv = ev;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int x = __shfl_xor(mk, m, 64), y = __shfl_xor(mv, m, 64);
            mk = mk > x ? mk : x;
            mv = mv > y ? mv : y;
        }
        const int sk = ek && mk - ek < 63 ? mk - ek : 63, sv = ev && mv - ev < 63 ? mv - ev : 63;
        const Unit x = arrange<ENC>(raw, from, __shfl(sk | sv << 8, mine, 64));
        asm volatile("s_waitcnt vmcnt(0)" ::"v"(x.mass) : "memory");
        if (lane == 0) __hip_atomic_store(loaded + u, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int w = w0 + lane; w < w1; w += 64)
            while (!__hip_atomic_load(loaded + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) __builtin_amdgcn_s_sleep(1);
        asm volatile("" ::: "memory");
        store_unit(p, s, kh, u, x, make_float2(kv8_scale(mk), kv8_scale(mv)));
    }
}

// All of it for a segment in one workgroup, for blocks of up to 64 rows: the plan, then rounds of 16 units, one a wave.  A kept row's
// new place is not behind its old one, so the units of a round overwrite nothing that later rounds read; a barrier keeps
// a round's stores behind its own loads, of rows and of scales, and the next round's loads go out before them.
template <int ENC>
__global__ __launch_bounds__(kPlan) void kv8_evict_segment_kernel(Evict p) {
    __shared__ PlanLds lds;
    int s, kh;
    if (!plan_segment(p, lds, s, kh)) return;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int kRound = kPlan / 64;
    const int2* list = p.list + (int64_t)blockIdx.x * (kUnit * p.units);
    const uint8_t* kc = static_cast<const uint8_t*>(p.a.k_cache) + kh * p.a.k_stride_head;
    const uint8_t* vc = static_cast<const uint8_t*>(p.a.v_cache) + kh * p.a.v_stride_head;
    // Lane l stands for row l of the unit's block (the unit's own rows are lanes first .. first + 15): where it is, then its exponents
    auto first_of = [&](int u) -> int {
        int row;
        const int b = (int)tq_udiv_apply((uint32_t)u, p.tpb_div);
        row = 16 * (u - b * p.tpb);
        return row;
    };
    auto place = [&](int u) -> int2 {
        const int d = kUnit * u - first_of(u) + lane;
        return u < p.units && lane < p.a.block_size && d < p.a.keep ? list[d] : make_int2(-1, 0);
    };
    struct Round {
        Raw raw;
        int row, ek, ev;  // row: of the unit's row lane; exponents: of the block's row lane
    };
    auto load = [&](int u, int2 at, Round& r) {
        const int blk = at.x, row = at.y;
        r.ek = blk < 0 ? 0 : exponent_at(kc + blk * p.a.k_stride_block, p);
        r.ev = blk < 0 ? 0 : exponent_at(vc + blk * p.a.v_stride_block, p);
        const int from = (first_of(u) + (lane & 15)) & 63;
        const int b = __shfl(blk, from, 64);
        r.row = __shfl(row, from, 64);
        load_raw(p, kh, b, r.row, r.raw);
    };
    Round cur;
    load(wave, place(wave), cur);
    int2 next = place(wave + kRound);
    const int rounds = (p.units + kRound - 1) / kRound;
    for (int r = 0; r < rounds; ++r) {
        const int u = r * kRound + wave;
        // ---- what the rows' codes fall by ----
        int mk = cur.ek, mv = cur.ev;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int x = __shfl_xor(mk, m, 64), y = __shfl_xor(mv, m, 64);
            mk = mk > x ? mk : x;
            mv = mv > y ? mv : y;
        }
        const int sk = cur.ek && mk - cur.ek < 63 ? mk - cur.ek : 63, sv = cur.ev && mv - cur.ev < 63 ? mv - cur.ev : 63;
        const int sh = __shfl(sk | sv << 8, (first_of(u) + (lane & 15)) & 63, 64);
        const Unit x = arrange<ENC>(cur.raw, cur.row, sh);
        // (all of the round's rows and scales are in registers before any wave stores; the compiler has the same wait at the top of the
        // loop, but nothing else here asks for it)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        load(u + kRound, next, cur);
        next = place(u + 2 * kRound);
        if (u < p.units) store_unit(p, s, kh, u, x, make_float2(kv8_scale(mk), kv8_scale(mv)));
    }
}

int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

}  // namespace

extern "C" int64_t tq_kv8_evict_workspace_bytes(int num_seqs, int num_kv_heads, int keep, int block_size) {
    if (num_seqs <= 0 || num_kv_heads <= 0 || keep <= 0 || block_size <= 0 || block_size % 16) return 0;
    const int64_t segs = (int64_t)num_seqs * num_kv_heads, units = ((int64_t)keep + kUnit - 1) / kUnit;
    const int64_t blocks = ((int64_t)keep + block_size - 1) / block_size;
    const int64_t cut = align256(segs * 4);
    if (block_size <= kInPlace) return cut + align256(segs * kPad * 4) + align256(segs * units * kUnit * 8) + align256(segs * (units + 1) * 4) + align256(segs * units * 4);
    return cut + align256(segs * units * kUnit * 8) + align256(segs * (units + 1) * 4) + align256(segs * units * kUnit * 2) +
           align256(segs * blocks * 8) + align256(segs * units * kUnit * 4) + segs * units * kStage;
}

extern "C" int tq_kv8_evict(const tq_kv8_evict_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    if (a->head_dim != TQ_HEAD_DIM) return TQ_ERR_HEAD_DIM;
    if (a->block_size <= 0 || a->block_size % 16 || a->block_size > 65536) return TQ_ERR_BLOCK_SIZE;
    if (a->encoding != TQ_E4M3 && a->encoding != TQ_INT8) return TQ_ERR_DTYPE;
    if (a->num_seqs < 0 || a->num_kv_heads <= 0 || a->num_blocks <= 0 || a->num_blocks > INT32_MAX || a->max_blocks_per_seq < 0 ||
        a->block_table_stride < a->max_blocks_per_seq || a->max_seq_len < 0 || a->reserved)
        return TQ_ERR_INVALID_ARGUMENT;
    if (a->keep <= 0 || a->sinks < 0 || a->recent < 0 || (int64_t)a->sinks + a->recent > a->keep || a->longer_than < a->keep)
        return TQ_ERR_INVALID_ARGUMENT;
    const uintptr_t ptrs = (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)a->mass;
    const int64_t by = a->k_stride_block | a->k_stride_head | a->v_stride_block | a->v_stride_head;
    if (ptrs % 16 || by % 16 || (a->mass_stride_block | a->mass_stride_head) % 4) return TQ_ERR_ALIGNMENT;
    if (a->num_seqs == 0) return TQ_OK;
    if (!a->k_cache || !a->v_cache || !a->mass || (!a->block_tables && a->max_blocks_per_seq) || !a->seq_lens || !a->change)
        return TQ_ERR_INVALID_ARGUMENT;
    Evict p = {};
    p.a = *a;
    p.tpb = a->block_size / 16;
    p.tpb_div = tq_make_udiv((uint32_t)p.tpb);
    int64_t cap = (int64_t)a->max_blocks_per_seq * a->block_size;
    cap = cap < a->max_seq_len ? cap : a->max_seq_len;
    p.cap = (int)(cap < kKv8MaxLen ? cap : kKv8MaxLen);
    const int64_t segs = (int64_t)a->num_seqs * a->num_kv_heads;
    // (a launch's threads stay below 2^32)
    if (segs > 0x3fffff) return TQ_ERR_INVALID_ARGUMENT;
    const bool any = p.cap > a->longer_than;
    void* args[] = {&p};
    if (any) {
        if (!a->workspace || (uintptr_t)a->workspace % 256 ||
            a->workspace_bytes < tq_kv8_evict_workspace_bytes(a->num_seqs, a->num_kv_heads, a->keep, a->block_size))
            return TQ_ERR_WORKSPACE;
        p.units = (a->keep + kUnit - 1) / kUnit;
        p.blocks = (a->keep + a->block_size - 1) / a->block_size;
        if (segs * ((p.units + kMove - 1) / kMove) > 0xffffff || segs * p.units > 0x3fffff0) return TQ_ERR_INVALID_ARGUMENT;
        uint8_t* at = static_cast<uint8_t*>(a->workspace);
        const int64_t rows = segs * p.units * kUnit;
        p.cut = reinterpret_cast<int32_t*>(at);
        at += align256(segs * 4);
        p.list = reinterpret_cast<int2*>(at);
        at += align256(rows * 8);
        p.ranks = reinterpret_cast<int32_t*>(at);
        at += align256(segs * (p.units + 1) * 4);
        if (a->block_size <= kInPlace) {
            p.loaded = reinterpret_cast<int32_t*>(at);
            p.ticket = reinterpret_cast<int32_t*>(at + align256(segs * p.units * 4));
            p.items = (p.units + kMove - 1) / kMove;
        } else {
            p.shift = reinterpret_cast<uint16_t*>(at);
            at += align256(rows * 2);
            p.scales = reinterpret_cast<float2*>(at);
            at += align256(segs * p.blocks * 8);
            p.stage_mass = reinterpret_cast<float*>(at);
            p.stage = at + align256(rows * 4);
        }
    }
    const bool whole = any && a->block_size <= kInPlace && segs >= kSegments;
    const void* first = !whole ? (const void*)kv8_evict_plan_kernel
                       : a->encoding == TQ_E4M3 ? (const void*)kv8_evict_segment_kernel<TQ_E4M3> : (const void*)kv8_evict_segment_kernel<TQ_INT8>;
    hipError_t e = hipLaunchKernel(first, dim3((unsigned)segs), dim3(kPlan), args, 0, stream);
    if (whole) {
    } else if (any && p.loaded) {
        const void* move = a->encoding == TQ_E4M3 ? (const void*)kv8_evict_move_kernel<TQ_E4M3> : (const void*)kv8_evict_move_kernel<TQ_INT8>;
        if (e == hipSuccess) e = hipLaunchKernel(move, dim3((unsigned)(segs * p.items)), dim3(64 * kMove), args, 0, stream);
    } else if (any) {
        const unsigned units = (unsigned)((segs * p.units + 3) / 4), blocks = (unsigned)((segs * p.blocks + 3) / 4);
        if (e == hipSuccess) e = hipLaunchKernel((const void*)kv8_evict_scales_kernel, dim3(blocks), dim3(256), args, 0, stream);
        const void* gather = a->encoding == TQ_E4M3 ? (const void*)kv8_evict_gather_kernel<TQ_E4M3> : (const void*)kv8_evict_gather_kernel<TQ_INT8>;
        if (e == hipSuccess) e = hipLaunchKernel(gather, dim3(units), dim3(256), args, 0, stream);
        if (e == hipSuccess) e = hipLaunchKernel((const void*)kv8_evict_scatter_kernel, dim3(units), dim3(256), args, 0, stream);
    }
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
