// Step planning: block tables, slots, positions and lengths of one engine step from the requests' lengths.
//
// plan_scan_kernel (one workgroup): per request the blocks it takes and gives up, prefix sums over the requests in
// order, which requests the ring can serve, the new lengths and the ring's new state.  plan_fill_kernel (many
// workgroups) writes table entries, the ring's end and the tokens' positions and slots from the
// records that the scan left in the workspace.  A new block's id is read from the ring where it is needed,
// not from the table, so that nothing in the fill waits for anything else in it.  Small steps run the
// fill inside the scan's workgroup: one launch.
//
// The ring needs no order between taking and giving: entries are taken from its occupied part and put behind it.
//
// Bound: launch and memory latency: 64 requests with a token each take 5.7 us in one launch; 500 requests with 36000
// tokens, 0.5 MB, take 4.3 + 5.6 us in two.
#include "tq_common.h"

namespace {

constexpr int kThreads = 512;
constexpr int kFillThreads = 256;

struct Record {       // of one request
    int past, have;   // tokens before; blocks before
    int take, give;   // blocks taken, given up (at most one is not 0)
    int first, put;   // ring index of the first one taken, of the first one given up
    int start;        // first token
    int given;        // whether new tokens get slots
};

struct Plan {
    tq_plan_args a;
    Record* rec;
    tq_udiv block_div;
};

// inclusive prefix sum over the workgroup's threads; total: the last one's
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* s_wave, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int i = 0; i < kThreads / 64; ++i) {
        if (i < wave) before += s_wave[i];
        total += s_wave[i];
    }
    __syncthreads();
    return x + before;
}

// place of the j-th entry from `from` on
__device__ __forceinline__ int ring_at(const Plan& p, int from, int j) {
    return (int)(((uint32_t)from + (uint32_t)j) % (uint32_t)p.a.num_blocks);
}

// Table entries of request s that change hands
__device__ __forceinline__ void fill_blocks(const Plan& p, int s, const Record& r, int from, int step) {
    int32_t* row = p.a.tables + s * p.a.table_stride;
    for (int j = from; j < r.take; j += step) row[r.have + j] = p.a.ring[ring_at(p, r.first, j)];
    for (int j = from; j < r.give; j += step)
        p.a.ring[ring_at(p, r.put, j)] = row[r.have - r.give + j];
}
// Token t of request s
__device__ __forceinline__ void fill_token(const Plan& p, int64_t t, int s, const Record& r) {
    const int pos = r.past + (int)(t - r.start);
    int64_t slot = -1;
    if (r.given) {
        const int b = (int)tq_udiv_apply((uint32_t)pos, p.block_div);
        const int j = b - r.have;
        const int blk = j >= 0 ? p.a.ring[ring_at(p, r.first, j)]
                               : p.a.tables[s * p.a.table_stride + b];
        slot = (int64_t)blk * p.a.block_size + (pos - b * p.a.block_size);
    }
    p.a.positions[t] = pos;
    p.a.slot_mapping[t] = slot;
}
// The request that token t belongs to: the last with start <= t (empty ones before it share its start)
template <class Start>
__device__ __forceinline__ int find_request(int n, int64_t t, Start start) {
    int lo = 0, hi = n;  // start(lo) <= t < start(hi)
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (start(m) <= t) lo = m;
        else hi = m;
    }
    return lo;
}

__global__ __launch_bounds__(kThreads) void plan_scan_kernel(Plan p, int fill) {
    __shared__ int64_t s_wave[kThreads / 64];
    __shared__ Record s_rec[kThreads];
    const tq_plan_args& a = p.a;
    const int tid = threadIdx.x;
    const uint32_t N = (uint32_t)a.num_blocks;
    const uint32_t head = (uint32_t)a.pool_in[0] % N;
    int count = a.pool_in[1];
    count = count < 0 ? 0 : count < a.num_blocks ? count : a.num_blocks;
    int64_t need0 = 0, give0 = 0, start0 = 0, taken = 0;
    for (int s0 = 0; s0 < a.num_seqs; s0 += kThreads) {
        const int s = s0 + tid;
        const bool in = s < a.num_seqs;
        int past = in ? a.past[s] : 0;
        past = past > 0 ? past : 0;
        const int add = in ? a.new_tokens[s] : 0;
        const uint32_t total = add >= 0 || past > -(int64_t)add ? (uint32_t)past + (uint32_t)add : 0u;
        const uint32_t bs = (uint32_t)a.block_size;
        const int have = (int)(((uint32_t)past + bs - 1) / bs);
        const int want = (int)(total / bs + (total % bs != 0));
        const bool fits = want <= a.max_blocks;
        const int need = fits && want > have ? want - have : 0;
        int64_t sum;
        const int64_t upto = need0 + block_scan(need, s_wave, sum);
        need0 += sum;
        const bool given = fits && (need == 0 || upto <= count);
        // (the requests that are served hold a prefix of the needs: upto only grows)
        int64_t got = 0;
        block_scan(given ? need : 0, s_wave, got);
        taken += got;
        // entries given up: those that the table has
        const int held = have < a.max_blocks ? have : a.max_blocks;
        const int give = held > want ? held - want : 0;
        const int64_t put = give0 + block_scan(give, s_wave, sum) - give;
        give0 += sum;
        const int n = add > 0 ? add : 0;
        // (a place no token has stands for all that 32 bits do not hold)
        int64_t start = start0 + block_scan(n, s_wave, sum) - n;
        start = start < 0x7fffffff ? start : 0x7fffffff;
        start0 += sum;
        if (in) {
            Record r;
            r.past = past;
            r.have = held;
            r.take = given ? need : 0;
            r.give = give;
            r.first = given ? (int)((head + (uint32_t)(upto - need)) % N) : 0;
            r.put = (int)((head + (uint32_t)count + (uint32_t)(put % N)) % N);
            r.start = (int)start;
            r.given = given;
            if (fill)
                s_rec[s] = r;  // (num_seqs <= kThreads)
            else
                p.rec[s] = r;
            a.seq_lens[s] = given ? (int)total : past;
            a.query_start_loc[s] = (int)start;
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.query_start_loc[a.num_seqs] = (int)(start0 < 0x7fffffff ? start0 : 0x7fffffff);
        const int64_t left = count - taken + give0;
        a.pool_out[0] = (int)((head + (uint32_t)taken) % N);
        a.pool_out[1] = (int)(left < a.num_blocks ? left : a.num_blocks);
    }
    if (!fill) return;
    const int lane = tid & 63, wave = tid >> 6;
    for (int s = wave; s < a.num_seqs; s += kThreads / 64) fill_blocks(p, s, s_rec[s], lane, 64);
    for (int64_t t = tid; t < a.num_tokens; t += kThreads) {
        if (t < start0) {
            const int s = find_request(a.num_seqs, t, [&](int i) -> int64_t { return s_rec[i].start; });
            fill_token(p, t, s, s_rec[s]);
        } else {
            a.positions[t] = 0;
            a.slot_mapping[t] = -1;
        }
    }
}

__global__ __launch_bounds__(kFillThreads) void plan_fill_kernel(Plan p) {
    const tq_plan_args& a = p.a;
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * (kFillThreads / 64);
    for (int64_t s = (int64_t)blockIdx.x * (kFillThreads / 64) + (threadIdx.x >> 6); s < a.num_seqs; s += waves)
        fill_blocks(p, (int)s, p.rec[s], lane, 64);
    const int64_t end = a.query_start_loc[a.num_seqs];
    for (int64_t t = (int64_t)blockIdx.x * kFillThreads + threadIdx.x; t < a.num_tokens; t += (int64_t)gridDim.x * kFillThreads) {
        if (t < end) {
            const int s = find_request(a.num_seqs, t, [&](int i) -> int64_t { return a.query_start_loc[i]; });
            fill_token(p, t, s, p.rec[s]);
        } else {
            a.positions[t] = 0;
            a.slot_mapping[t] = -1;
        }
    }
}

}  // namespace

extern "C" int64_t tq_plan_step_workspace_bytes(int num_seqs) {
    return num_seqs < 0 || num_seqs > (1 << 20) ? 0 : (int64_t)num_seqs * (int64_t)sizeof(Record);
}

extern "C" int tq_plan_step(const tq_plan_args* a, tq_stream_t stream) {
    if (!a) return TQ_ERR_INVALID_ARGUMENT;
    if (a->block_size <= 0 || a->block_size % 16) return TQ_ERR_BLOCK_SIZE;
    if (a->num_seqs < 0 || a->num_seqs > (1 << 20) || a->num_tokens < 0 || a->num_tokens > 0x7fffffff || a->num_blocks <= 0 ||
        a->num_blocks > (1 << 30) || a->max_blocks < 0 || (int64_t)a->max_blocks * a->block_size > 0x7fffffff ||
        a->table_stride < a->max_blocks)
        return TQ_ERR_INVALID_ARGUMENT;
    if (!a->ring || !a->pool_in || !a->pool_out || !a->query_start_loc ||
        (a->num_seqs && (!a->past || !a->new_tokens || !a->tables || !a->seq_lens)) ||
        (a->num_tokens && (!a->positions || !a->slot_mapping)))
        return TQ_ERR_INVALID_ARGUMENT;
    const int64_t need = tq_plan_step_workspace_bytes(a->num_seqs);
    if (need && (!a->workspace || (uintptr_t)a->workspace % 16 || a->workspace_bytes < need)) return TQ_ERR_WORKSPACE;
    Plan p = {};
    p.a = *a;
    p.rec = static_cast<Record*>(a->workspace);
    p.block_div = tq_make_udiv((uint32_t)a->block_size);
    // A second launch costs 2.5 us from the host, a round of the one workgroup's threads 0.9 (64 requests, 64 / 1024 / 2000 /
    // 4000 tokens, one launch 13 us from Python and 6.1 / 8.3 / 9.8 / 12.8 in a graph, two 15.5 and 6.7 / 8.6 / 8.6 / 8.5).
    int fill = a->num_seqs <= kThreads && a->num_tokens <= 4 * kThreads;
    void* args[] = {&p, &fill};
    hipError_t e = hipLaunchKernel((const void*)plan_scan_kernel, dim3(1), dim3(kThreads), args, 0, stream);
    if (e == hipSuccess && !fill) {
        const int64_t work = a->num_tokens > 64 * (int64_t)a->num_seqs ? a->num_tokens : 64 * (int64_t)a->num_seqs;
        int64_t grid = (work + kFillThreads - 1) / kFillThreads;
        grid = grid < 1 ? 1 : grid < 2048 ? grid : 2048;
        e = hipLaunchKernel((const void*)plan_fill_kernel, dim3((unsigned)grid), dim3(kFillThreads), args, 0, stream);
    }
    if (e == hipSuccess) e = hipGetLastError();
    return e == hipSuccess ? TQ_OK : (int)e;
}
