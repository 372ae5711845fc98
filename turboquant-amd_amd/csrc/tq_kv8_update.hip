// Quantisation of K and V rows into the 8-bit paged caches (tiles: tq_kv8.h).
//
// A run is a maximal stretch of tokens with consecutive slots inside one block, skipped tokens between them (at most
// 63 at a time) passed over; one wave takes one run of one head of K or of V, so a block's scale, its
// requantisation and its rows have one owner and need no atomics.  Pass 1 finds the largest finite |x| of the run, pass 2 writes the codes; where
// the run lies in one 16-row sub-tile the rows stay in registers between the two.  Lane (c, g), c = lane % 16,
// g = lane / 16, holds dims 8c..8c+7 of rows 4g..4g+3 of a sub-tile: a wave's load is four whole rows, the
// keys' store four whole rows, and the values' store (whose words are four rows of one dim) 2 KB in one
// piece.  A row group that the run covers in part keeps its other rows' bytes by read and merge.
//
// Bound: memory; 16384 tokens x 8 heads read 64 MB of bf16 and write 32 MB of codes.
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

// gaps: tokens are skipped inside the run
template <int ENC, int DT, bool VALUES>
__device__ __forceinline__ void write_run(const Kv8Update& p, int64_t t0, int n, bool gaps, int* s_tok, int64_t block, int row0, int head) {
    using Code = Kv8Code<ENC>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const void* x = VALUES ? p.a.v : p.a.k;
    const int64_t xst = VALUES ? p.a.v_stride_token : p.a.k_stride_token;
    const int64_t xsh = VALUES ? p.a.v_stride_head : p.a.k_stride_head;
    uint8_t* tile = static_cast<uint8_t*>(VALUES ? p.a.v_cache : p.a.k_cache) +
                    block * (VALUES ? p.a.v_stride_block : p.a.k_stride_block) +
                    head * (VALUES ? p.a.v_cache_stride_head : p.a.k_cache_stride_head);
    float* scale_at = reinterpret_cast<float*>(tile + p.a.block_size * TQ_HEAD_DIM);
    const float old_scale = *scale_at;
    const int end = row0 + n;
    const int sub0 = row0 >> 4, sub1 = (end + 15) >> 4;
    const int64_t xbase = head * xsh + 8 * c;

    Raw<DT> raw[4];
    int64_t at_token = t0;  // of the next sub-tile's first row
    auto load = [&](int sub) {
        const int from = 16 * sub > row0 ? 16 * sub : row0, to = 16 * sub + 16 < end ? 16 * sub + 16 : end;
        if (gaps) {
            if (sub == sub0) at_token = t0;
            at_token = next_tokens(p, at_token, to - from, p.a.num_blocks * p.a.block_size, s_tok, t0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * sub + 4 * g + r;
            const bool in = row >= from && row < to;
            const int64_t t = gaps ? t0 + s_tok[in ? row - from : 0] : t0 + (in ? row - row0 : 0);
            raw[r] = load_raw<DT>(x, t * xst + xbase);
        }
    };
    uint32_t top = 0;
    for (int sub = sub0; sub < sub1; ++sub) {
        load(sub);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // (rows outside the run repeat its first)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = __float_as_uint(raw[r].get(i)) & 0x7fffffffu;
                top = b < 0x7f800000u && b > top ? b : top;
            }
        }
    }
    for (int m = 32; m >= 1; m >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, m, 64);
        top = o > top ? o : top;
    }
    int e = Code::exponent(top);
    e = top == 0 || e < -126 ? -126 : e;
    const bool fresh = row0 == 0 || !(old_scale > 0.f);
    const int e_old = (int)(__float_as_uint(old_scale) >> 23) - 127;
    const bool grew = !fresh && e > e_old;
    if (!fresh && !grew) e = e_old;
    e = __builtin_amdgcn_readfirstlane(e);
    const float inv = kv8_exp2i(-e);
    // the factor of the codes that stay
    const float ratio = grew ? (e_old - e >= -126 ? kv8_exp2i(e_old - e) : 0.f) : 1.f;
    if (lane == 0 && (fresh || grew)) *scale_at = kv8_exp2i(e);

    const int s0 = grew ? 0 : sub0, s1 = grew ? p.a.block_size >> 4 : sub1;
    for (int sub = s0; sub < s1; ++sub) {
        const bool in_run = sub >= sub0 && sub < sub1;  // wave-uniform
        if (in_run && sub1 - sub0 > 1) load(sub);
        const int r0 = 16 * sub + 4 * g;
        uint8_t* at = tile + 16 * sub * TQ_HEAD_DIM;
        if (VALUES) {
            uint32_t word[8];
            const bool all = r0 >= row0 && r0 + 4 <= end, some = r0 < end && r0 + 4 > row0;
            tq_u32x4* q = reinterpret_cast<tq_u32x4*>(at + 512 * g + 32 * c);
            if (!all && (some || grew)) {
                const tq_u32x4 a = q[0], b = q[1];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    word[i] = a[i];
                    word[4 + i] = b[i];
                }
                if (grew) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        word[i] = Code::pack(Code::value(word[i], 0) * ratio, Code::value(word[i], 1) * ratio,
                                             Code::value(word[i], 2) * ratio, Code::value(word[i], 3) * ratio);
                }
            }
            if (in_run) {
                uint32_t mine = 0;  // the bytes of the run's rows
#pragma unroll
                for (int r = 0; r < 4; ++r) mine |= r0 + r >= row0 && r0 + r < end ? 0xffu << (8 * r) : 0u;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t w = Code::pack(raw[0].get(i) * inv, raw[1].get(i) * inv, raw[2].get(i) * inv, raw[3].get(i) * inv);
                    word[i] = all ? w : (w & mine) | (word[i] & ~mine);
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
                if (row >= row0 && row < end) {
                    const Raw<DT>& w = raw[r];
                    *q = tq_u32x2{Code::pack(w.get(0) * inv, w.get(1) * inv, w.get(2) * inv, w.get(3) * inv),
                                  Code::pack(w.get(4) * inv, w.get(5) * inv, w.get(6) * inv, w.get(7) * inv)};
                } else if (grew) {
                    tq_u32x2 w = *q;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        w[i] = Code::pack(Code::value(w[i], 0) * ratio, Code::value(w[i], 1) * ratio,
                                          Code::value(w[i], 2) * ratio, Code::value(w[i], 3) * ratio);
                    *q = w;
                }
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
    const bool in = lane < p.window && t < p.a.num_tokens;
    const int64_t slot = in ? slot_at(p, t) : -1;
    const int64_t early = t >= 64 ? slot_at(p, t - 64) : -1;
    const bool valid = slot >= 0 && slot < slots;
    const uint64_t here = __builtin_amdgcn_ballot_w64(valid), there = __builtin_amdgcn_ballot_w64(early >= 0 && early < slots);
    if (!here) return;
    // the slot of the last token before this one that has one, of the 64 before it
    int64_t before = -2;
    {
        const uint64_t below = here & ((1ull << lane) - 1), reach = there & ~((1ull << lane) - 1);
        const int from = below ? 63 - __builtin_clzll(below) : reach ? 63 - __builtin_clzll(reach) : 0;
        const int64_t a = __shfl(slot, from, 64), b = __shfl(early, from, 64);
        before = below ? a : reach ? b : before;
    }
    const bool starts = valid && !(before + 1 == slot && slot % p.a.block_size != 0);
    uint64_t heads_of = __builtin_amdgcn_ballot_w64(starts);
    const int jobs = 2 * p.a.num_heads;
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
            for (int64_t a = t0 + i + 1; n < most;) {
                const int64_t u = a + lane;
                const int64_t su = u < p.a.num_tokens ? slot_at(p, u) : -1;
                const bool vu = su >= 0 && su < slots;
                const uint64_t mask = __builtin_amdgcn_ballot_w64(vu);
                if (!mask) break;
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
            }
            for (; first < jobs; first += kWaves * p.window_wg) {
                if (first < p.a.num_heads)
                    write_run<ENC, DT, false>(p, t0 + i, n, gaps, s_tok, block, row0, first);
                else
                    write_run<ENC, DT, true>(p, t0 + i, n, gaps, s_tok, block, row0, first - p.a.num_heads);
            }
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
    // each, and a window of one token gives each run's heads waves of their own.
    const int jobs = 2 * a->num_heads;
    const int per_run = (jobs + kWaves - 1) / kWaves;
    p.window = a->block_size < 64 ? a->block_size : 64;
    if (a->num_tokens * per_run <= 4096) p.window = 1;
    p.window_wg = per_run;
    const int64_t grid = (a->num_tokens + p.window - 1) / p.window * p.window_wg;
    if (grid > 0x7fffffff) return TQ_ERR_INVALID_ARGUMENT;
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
