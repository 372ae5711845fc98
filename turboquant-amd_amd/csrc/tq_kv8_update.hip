// Quantisation of K and V rows into the 8-bit paged caches (tiles: tq_kv8.h).
//
// A run is a maximal stretch of tokens with consecutive slots inside one block, skipped tokens between them (at most
// 63 at a time) passed over; one wave takes one run of one head, so a block's scale, its requantisation and its
// rows have one owner and need no atomics.  Pass 1 finds the largest finite |x| of the run, pass 2 writes the codes;
// where the run lies in one 16-row sub-tile the rows stay in registers between the two.  Lane (c, g), c = lane % 16,
// g = lane / 16, holds dims 8c..8c+7 of rows 4g..4g+3 of a sub-tile: a wave's load is four whole rows, the
// keys' store four whole rows, and the values' store (whose words are four rows of one dim) 2 KB in one
// piece.  A row group that the run covers in part keeps its other rows' bytes by read and merge.
//
// The largest value is found on the rows as they are loaded, two 16-bit numbers at a time; infinities and NaN, which do
// not count, send a wave the longer way.  K and V of a head are one wave's work, so that both rows are under way at once.
//
// Bound: memory; 16384 tokens x 8 heads read 64 MB of bf16 and write 32 MB of codes in 23.3 us, 4.3 TB/s, where a large
// copy moves 4.9 (28.4 with clamps and a maximum of single values in every wave).  64 single tokens: 5 us of latency.
#include "tq_kv8.h"

namespace {

struct Kv8Update {
    tq_kv8_update_args a;
    int window;     // tokens whose runs one workgroup takes
    int window_wg;  // workgroups per window (over heads and tensors)
};

constexpr int kWaves = 4;

__device__ __forceinline__ int64_t slot_at(const Kv8Update& p, int64_t t) {
    return p.a.slot_dtype == TQ_I64 ? static_cast<const int64_t*>(p.a.slot_mapping)[t]
                                    : (int64_t)static_cast<const int32_t*>(p.a.slot_mapping)[t];
}

// 8 elements as fp32
template <int DT>
struct Raw {
    tq_u32x4 w[DT == TQ_F32 ? 2 : 1];
    __device__ __forceinline__ float get(int i) const {
        if (DT == TQ_F32) return __uint_as_float(w[i >> 2][i & 3]);
        const uint32_t b = (w[0][i >> 1] >> (16 * (i & 1))) & 0xffffu;
        return DT == TQ_BF16 ? tq_bf16_to_f32(b) : tq_f16_to_f32(b);
    }
};
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const void* base, int64_t off) {
    Raw<DT> r;
    if (DT == TQ_F32) {
        const tq_u32x4* s = reinterpret_cast<const tq_u32x4*>(static_cast<const float*>(base) + off);
        r.w[0] = s[0];
        r.w[DT == TQ_F32 ? 1 : 0] = s[1];
    } else {
        r.w[0] = *reinterpret_cast<const tq_u32x4*>(static_cast<const uint16_t*>(base) + off);
    }
    return r;
}

// The next rows of a run from token `at` on: the tokens of up to 16 of them to s_tok, and the token behind the last.
__device__ __forceinline__ int64_t next_tokens(const Kv8Update& p, int64_t at, int rows, int64_t slots, int* s_tok, int64_t t0) {
    const int lane = threadIdx.x & 63;
    for (int got = 0; got < rows;) {
        const int64_t u = at + lane;
        const int64_t s = u < p.a.num_tokens ? slot_at(p, u) : -1;
        const bool valid = s >= 0 && s < slots;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(valid);
        const int rank = got + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
        if (valid && rank < rows) s_tok[rank] = (int)(u - t0);
        const uint64_t last = __builtin_amdgcn_ballot_w64(valid && rank == rows - 1);
        if (last) return at + __builtin_ctzll(last) + 1;
        if (!mask) break;  // (a run's rows are there: not reached)
        got += __builtin_popcountll(mask);
        at += 64;
    }
    return at;
}

// Largest |x| of 8 elements as fp32 bits, not finite ones too: 16-bit types two at a time
template <int DT>
__device__ __forceinline__ uint32_t largest(const Raw<DT>& r, uint32_t top) {
    if (DT == TQ_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = r.w[i >> 2][i & 3] & 0x7fffffffu;
            top = b > top ? b : top;
        }
        return top;
    }
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 t = __builtin_bit_cast(u16x2, top);
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, r.w[0][i] & 0x7fff7fffu));
    return __builtin_bit_cast(uint32_t, t);
}
// the wave's largest, as fp32 bits
template <int DT>
__device__ __forceinline__ uint32_t wave_largest(uint32_t top) {
    if (DT != TQ_F32) {
        const uint32_t lo = top & 0xffffu, hi = top >> 16;
        top = lo > hi ? lo : hi;
        top = DT == TQ_BF16 ? top << 16 : __float_as_uint(tq_f16_to_f32(top));
    }
    auto with = [&](uint32_t o) { top = o > top ? o : top; };
    with((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x128, 0xf, 0xf, true));  // rotations within 16 lanes
    with((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x124, 0xf, 0xf, true));
    with((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x122, 0xf, 0xf, true));
    with((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x121, 0xf, 0xf, true));
    auto a = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = a[0] > a[1] ? a[0] : a[1];
    auto b = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = b[0] > b[1] ? b[0] : b[1];
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)top);
}

// Sub-tile `sub` of a tile: the codes of the run's rows [row0, end) in it (raw: 4 rows of this lane), other rows kept,
// and requantised by `ratio` where the scale grew.
template <int ENC, int DT, bool VALUES, bool ODD>
__device__ __forceinline__ void write_sub(uint8_t* at, const Raw<DT> (&raw)[4], int r0, int row0, int end, bool in_run, bool grew,
                                          float inv, float ratio) {
    using Code = Kv8Code<ENC>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    auto moved = [&](uint32_t w) {
        return Code::template pack<ODD>(Code::value(w, 0), Code::value(w, 1), Code::value(w, 2), Code::value(w, 3), ratio);
    };
    if (VALUES) {
        uint32_t word[8];
        const bool all = r0 >= row0 && r0 + 4 <= end, some = r0 < end && r0 + 4 > row0;
        tq_u32x4* q = reinterpret_cast<tq_u32x4*>(at + 512 * g + 32 * c);
        if (in_run) {
#pragma unroll
            for (int i = 0; i < 8; ++i) word[i] = Code::template pack<ODD>(raw[0].get(i), raw[1].get(i), raw[2].get(i), raw[3].get(i), inv);
        }
        if (!all && (some || grew)) {
            const tq_u32x4 a = q[0], b = q[1];
            uint32_t mine = 0;  // the bytes of the run's rows
#pragma unroll
            for (int r = 0; r < 4; ++r) mine |= in_run && r0 + r >= row0 && r0 + r < end ? 0xffu << (8 * r) : 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t old = i < 4 ? a[i] : b[i - 4];
                if (grew) old = moved(old);
                word[i] = in_run ? (word[i] & mine) | (old & ~mine) : old;
            }
        }
        if (all || some || grew) {
            q[0] = tq_u32x4{word[0], word[1], word[2], word[3]};
            q[1] = tq_u32x4{word[4], word[5], word[6], word[7]};
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = r0 + r;
            tq_u32x2* q = reinterpret_cast<tq_u32x2*>(at + (4 * g + r) * TQ_HEAD_DIM + 8 * c);
            if (in_run && row >= row0 && row < end) {
                const Raw<DT>& w = raw[r];
                *q = tq_u32x2{Code::template pack<ODD>(w.get(0), w.get(1), w.get(2), w.get(3), inv),
                              Code::template pack<ODD>(w.get(4), w.get(5), w.get(6), w.get(7), inv)};
            } else if (grew) {
                const tq_u32x2 w = *q;
                *q = tq_u32x2{moved(w[0]), moved(w[1])};
            }
        }
    }
}

// One head of K and of V: the run's n rows from token t0 on, at row row0 of its block.  gaps: tokens are skipped inside
// the run.
template <int ENC, int DT>
__device__ __forceinline__ void write_run(const Kv8Update& p, int64_t t0, int n, bool gaps, int* s_tok, int64_t block, int row0, int head) {
    using Code = Kv8Code<ENC>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int end = row0 + n;
    const int sub0 = row0 >> 4, sub1 = (end + 15) >> 4;
    const void* x[2] = {p.a.k, p.a.v};
    const int64_t xst[2] = {p.a.k_stride_token, p.a.v_stride_token};
    const int64_t xbase[2] = {head * p.a.k_stride_head + 8 * c, head * p.a.v_stride_head + 8 * c};
    uint8_t* tile[2] = {static_cast<uint8_t*>(p.a.k_cache) + block * p.a.k_stride_block + head * p.a.k_cache_stride_head,
                        static_cast<uint8_t*>(p.a.v_cache) + block * p.a.v_stride_block + head * p.a.v_cache_stride_head};
    const uint32_t scale_at = (uint32_t)p.a.block_size * TQ_HEAD_DIM;
    float old_scale[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) old_scale[kv] = *reinterpret_cast<const float*>(tile[kv] + scale_at);

    Raw<DT> raw[2][4];
    int64_t at_token = t0;  // of the next sub-tile's first row
    // rows outside the run repeat the first of the sub-tile's
    auto load = [&](int sub, bool next, int kv) {
        const int from = 16 * sub > row0 ? 16 * sub : row0, to = 16 * sub + 16 < end ? 16 * sub + 16 : end;
        if (gaps && next) at_token = next_tokens(p, sub == sub0 ? t0 : at_token, to - from, p.a.num_blocks * p.a.block_size, s_tok, t0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * sub + 4 * g + r;
            const bool in = row >= from && row < to;
            const int64_t t = gaps ? t0 + s_tok[in ? row - from : 0] : t0 + (in ? row : from) - row0;
            raw[kv][r] = load_raw<DT>(x[kv], t * xst[kv] + xbase[kv]);
        }
    };
    uint32_t top[2] = {0, 0};
    for (int sub = sub0; sub < sub1; ++sub) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) load(sub, kv == 0, kv);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int r = 0; r < 4; ++r) top[kv] = largest<DT>(raw[kv][r], top[kv]);
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        uint32_t t = wave_largest<DT>(top[kv]);
        const bool odd = t >= 0x7f800000u;  // infinities or NaN among the rows: they do not count
        if (odd) {
            uint32_t f = 0;
            for (int sub = sub0; sub < sub1; ++sub) {
                if (sub1 - sub0 > 1) load(sub, true, kv);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t b = __float_as_uint(raw[kv][r].get(i)) & 0x7fffffffu;
                        f = b < 0x7f800000u && b > f ? b : f;
                    }
            }
            t = wave_largest<TQ_F32>(f);
        }
        int e = Code::exponent(t);
        e = t == 0 || e < -126 ? -126 : e;
        const bool fresh = row0 == 0 || !(old_scale[kv] > 0.f);
        const int e_old = (int)(__float_as_uint(old_scale[kv]) >> 23) - 127;
        const bool grew = !fresh && e > e_old;
        if (!fresh && !grew) e = e_old;
        e = __builtin_amdgcn_readfirstlane(e);
        const float inv = kv8_exp2i(-e);
        // the factor of the codes that stay
        const float ratio = grew ? (e_old - e >= -126 ? kv8_exp2i(e_old - e) : 0.f) : 1.f;
        if (lane == 0 && (fresh || grew)) *reinterpret_cast<float*>(tile[kv] + scale_at) = kv8_exp2i(e);

        const int s0 = grew ? 0 : sub0, s1 = grew ? p.a.block_size >> 4 : sub1;
        for (int sub = s0; sub < s1; ++sub) {
            const bool in_run = sub >= sub0 && sub < sub1;  // wave-uniform
            if (in_run && sub1 - sub0 > 1) load(sub, true, kv);
            const int r0 = 16 * sub + 4 * g;
            uint8_t* at = tile[kv] + 16 * sub * TQ_HEAD_DIM;
            // (codes that stay may be NaN)
            if (odd || grew) {
                if (kv == 0) write_sub<ENC, DT, false, true>(at, raw[kv], r0, row0, end, in_run, grew, inv, ratio);
                else write_sub<ENC, DT, true, true>(at, raw[kv], r0, row0, end, in_run, grew, inv, ratio);
            } else {
                if (kv == 0) write_sub<ENC, DT, false, false>(at, raw[kv], r0, row0, end, in_run, false, inv, ratio);
                else write_sub<ENC, DT, true, false>(at, raw[kv], r0, row0, end, in_run, false, inv, ratio);
            }
        }
    }
}

// Workgroup (window, part): the runs that begin in the window's tokens, times heads and tensors, dealt to
// the waves of the window's workgroups.
template <int ENC, int DT>
__global__ __launch_bounds__(64 * kWaves) void kv8_update_kernel(Kv8Update p) {
    __shared__ int s_tok_all[kWaves][16];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int* s_tok = s_tok_all[wave];
    const int64_t t0 = (int64_t)(blockIdx.x / (uint32_t)p.window_wg) * p.window;
    const int part = (int)(blockIdx.x % (uint32_t)p.window_wg) * kWaves + wave;
    const int64_t slots = p.a.num_blocks * p.a.block_size;
    // lane i: token t0 + i (window <= 64), and token t0 - 64 + i for what lies before
    const int64_t t = t0 + lane;
    const int64_t slot = t < p.a.num_tokens ? slot_at(p, t) : -1;
    const int64_t early = t >= 64 ? slot_at(p, t - 64) : -1;
    const bool valid = slot >= 0 && slot < slots;
    const uint64_t here = __builtin_amdgcn_ballot_w64(valid), there = __builtin_amdgcn_ballot_w64(early >= 0 && early < slots);
    // the slot of the last token before this one that has one, of the 64 before it
    int64_t before = -2;
    {
        const uint64_t below = here & ((1ull << lane) - 1), reach = there & ~((1ull << lane) - 1);
        const int from = below ? 63 - __builtin_clzll(below) : reach ? 63 - __builtin_clzll(reach) : 0;
        const int64_t a = __shfl(slot, from, 64), b = __shfl(early, from, 64);
        before = below ? a : reach ? b : before;
    }
    const bool starts = lane < p.window && valid && !(before + 1 == slot && slot % p.a.block_size != 0);
    uint64_t heads_of = __builtin_amdgcn_ballot_w64(starts);
    const int jobs = p.a.num_heads;
    int first = part;  // this wave's next job of the run at hand
    while (heads_of) {
        const int i = __builtin_ctzll(heads_of);
        heads_of &= heads_of - 1;
        if (first < jobs) {
            const int64_t s = ((int64_t)__builtin_amdgcn_readlane((int)(slot >> 32), i) << 32) |
                              (uint32_t)__builtin_amdgcn_readlane((int)slot, i);
            const int64_t block = s / p.a.block_size;
            const int row0 = (int)(s - block * p.a.block_size);
            // the run's length: the 64 tokens behind its last one at a time
            const int most = p.a.block_size - row0;
            int n = 1;
            bool gaps = false;
            // (first those that this wave has at hand)
            bool at_hand = true;
            for (int64_t a = t0 + i + 1; n < most;) {
                int64_t su = __shfl(slot, (lane + i + 1) & 63, 64);
                if (!at_hand) su = a + lane < p.a.num_tokens ? slot_at(p, a + lane) : -1;
                else if (lane + i + 1 > 63) su = -1;
                const bool vu = su >= 0 && su < slots;
                const uint64_t mask = __builtin_amdgcn_ballot_w64(vu);
                if (!mask) {
                    if (!at_hand) break;
                    at_hand = false;
                    continue;
                }
                const int rank = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
                const uint64_t off = __builtin_amdgcn_ballot_w64(vu && (n + rank >= most || su != s + n + rank));
                // the tokens that follow: those with a slot before the first that does not
                const uint64_t follow = off ? mask & ((off & -off) - 1) : mask;
                if (!follow) break;
                const int last = 63 - __builtin_clzll(follow);
                gaps = gaps || follow != (last == 63 ? ~0ull : (1ull << (last + 1)) - 1);
                n += __builtin_popcountll(follow);
                if (off) break;
                a += last + 1;
                at_hand = false;
            }
            for (; first < jobs; first += kWaves * p.window_wg) write_run<ENC, DT>(p, t0 + i, n, gaps, s_tok, block, row0, first);
        }
        first -= jobs;
    }
}

}  // namespace

extern "C" int64_t tq_kv8_tile_bytes(int block_size) {
    if (block_size <= 0 || block_size % 16) return TQ_ERR_BLOCK_SIZE;
    return (int64_t)block_size * TQ_HEAD_DIM + kKv8ScaleBytes;
}

extern "C" int tq_kv8_update(const tq_kv8_update_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    if (a->head_dim != TQ_HEAD_DIM) return TQ_ERR_HEAD_DIM;
    if (a->block_size <= 0 || a->block_size % 16 || a->block_size > 65536) return TQ_ERR_BLOCK_SIZE;
    if (a->x_dtype != TQ_F32 && a->x_dtype != TQ_F16 && a->x_dtype != TQ_BF16) return TQ_ERR_DTYPE;
    if (a->slot_dtype != TQ_I32 && a->slot_dtype != TQ_I64) return TQ_ERR_DTYPE;
    if (a->encoding != TQ_E4M3 && a->encoding != TQ_INT8) return TQ_ERR_DTYPE;
    if (a->num_tokens < 0 || a->num_heads < 0 || a->num_heads > 65536 || a->num_blocks < 0 || a->num_blocks > INT64_MAX / a->block_size)
        return TQ_ERR_INVALID_ARGUMENT;
    if (a->num_tokens == 0 || a->num_heads == 0 || a->num_blocks == 0) return TQ_OK;
    if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->slot_mapping) return TQ_ERR_INVALID_ARGUMENT;
    const uintptr_t ptrs = (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache;
    const int64_t el = a->k_stride_token | a->k_stride_head | a->v_stride_token | a->v_stride_head;
    const int64_t by = a->k_stride_block | a->k_cache_stride_head | a->v_stride_block | a->v_cache_stride_head;
    if (ptrs % 16 || el % 8 || by % 16) return TQ_ERR_ALIGNMENT;
    if ((uintptr_t)a->slot_mapping % (a->slot_dtype == TQ_I64 ? 8 : 4)) return TQ_ERR_ALIGNMENT;
    Kv8Update p = {};
    p.a = *a;
    // A window of a block's length holds about one run of a prompt; single tokens of many sequences are a run
    // each, and a window of one token gives each run's heads waves of their own.  The host knows the tokens alone, not
    // the runs: short calls are taken for single tokens, long ones for prompts.  At the rule's border, 1024 tokens of 8
    // heads, a window of one and one of a block take 12.7 and 41 us (blocks of 64: 12.7 and 152) for single tokens, 13.1 and
    // 6.0 (23.4 and 12.3) for a prompt; 8192 single tokens, a block's window each: 76 (182).
    const int per_run = (a->num_heads + kWaves - 1) / kWaves;
    p.window = a->block_size < 64 ? a->block_size : 64;
    if (a->num_tokens * per_run <= 2048) p.window = 1;
    p.window_wg = per_run;
    const int64_t grid = (a->num_tokens + p.window - 1) / p.window * p.window_wg;
    if (grid > 0xffffff) return TQ_ERR_INVALID_ARGUMENT;  // (a launch's threads stay below 2^32)
    const void* kern = nullptr;
#define TQ_K8U(E, D) \
    if (a->encoding == E && a->x_dtype == D) kern = (const void*)kv8_update_kernel<E, D>;
    TQ_K8U(TQ_E4M3, TQ_F32) TQ_K8U(TQ_E4M3, TQ_F16) TQ_K8U(TQ_E4M3, TQ_BF16)
    TQ_K8U(TQ_INT8, TQ_F32) TQ_K8U(TQ_INT8, TQ_F16) TQ_K8U(TQ_INT8, TQ_BF16)
#undef TQ_K8U
    void* args[] = {&p};
    hipError_t err = hipLaunchKernel(kern, dim3((unsigned)grid), dim3(64 * kWaves), args, 0, stream);
    if (err == hipSuccess) err = hipGetLastError();
    return err == hipSuccess ? TQ_OK : (int)err;
}
