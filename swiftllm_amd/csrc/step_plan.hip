// Block tables and slot maps of one step, from request lengths (gfx950).
//
// Sequence s has cached_s tokens in the cache and brings new_s; its table holds
// the ceil(cached_s / 16) blocks in use. With have_s = ceil(cached_s / 16) and
// need_s = ceil((cached_s + new_s) / 16) - have_s:
//   a sequence is valid if cached_s, new_s >= 0 and cached_s + new_s fits its
//   table; taken_s and tokens_s are inclusive sums of need and new over the
//   valid sequences; s is planned if it is valid, its blocks are there
//   (need_s == 0 or taken_s <= num_free) and its rows are (new_s == 0 or
//   tokens_s <= num_tokens). One that is not planned keeps its length and gets no row.
//   block_tables[s, have_s + b] = free_blocks[taken_s - need_s + b], b < need_s
//   query_offsets = exclusive sums of the planned sequences' new tokens
//   row off_s + i: position cached_s + i, slot table[pos / 16] * 16 + pos % 16
// Both sums only grow, so the planned sequences' blocks are a prefix of the
// free list: no block is passed over.
//
// Bound: latency. A call of 64 sequences moves 2 KB, one of 524288 rows 4 MB.
// So it is one launch without a hand-over between workgroups: each owns 1024
// rows, scans the lengths of every sequence itself (8 bytes each, at most 512 KB
// that all of them find in the L2) 1024 at a time, keeps the ends of those in LDS and
// finds a row's sequence by bisection. A block's first row writes its table
// entry: entries that a row reads are never written in the same call.
// Measured: 64 sequences of one token each 4.8 us of the kernel, 5.4 us a call;
// 64 sequences of 169000 rows 5.5 us, the call's floor being a launch's 4.3.

#include "common.hpp"

namespace swiftllm {
namespace {

struct PlanArgs {
    int* bt;
    const int* cached;
    const int* fresh;        // new tokens
    const int* free_blocks;
    const int* num_free;     // [1]
    int* ctx;
    int* offsets;            // [S + 1]
    int* positions;
    int* slots;
    int* counts;             // [3]: blocks taken, rows in use, sequences refused
    int S;
    int T;
    int MB;
    int free_cap;
    int num_blocks;
    bool wide;               // positions and slots are 16-byte aligned
};

constexpr int kPlanThreads = 256;
constexpr int kPlanEach = 4;                           // sequences and rows per thread
constexpr int kPlanChunk = kPlanThreads * kPlanEach;
// Sums stop here, above any free list and any row count (host), so that they
// neither overflow nor come back into range.
constexpr int kPlanMost = (1 << 30) - 1;

__device__ __forceinline__ int capped(int a, int b) { return min(a + b, kPlanMost); }

// Exclusive capped prefixes of x and y over the workgroup's threads, and their
// totals. `part` is free again after the caller's next barrier.
__device__ __forceinline__ void scan2(int x, int y, int& before_x, int& before_y, int& all_x, int& all_y,
                                      int (*part)[kPlanThreads / 64]) {
    const auto op = [](int a, int b) { return capped(a, b); };
    const int lane = threadIdx.x & 63;
    const int w = threadIdx.x >> 6;
    const int ix = dpp_scan(x, 0, op);
    const int iy = dpp_scan(y, 0, op);
    if (lane == 63) {
        part[0][w] = ix;
        part[1][w] = iy;
    }
    __syncthreads();
    // A thread's exclusive prefix is the inclusive one of the lane before it.
    before_x = __shfl_up(ix, 1);
    before_y = __shfl_up(iy, 1);
    if (lane == 0) before_x = before_y = 0;
    all_x = all_y = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) {
        if (i == w) {
            before_x = capped(before_x, all_x);
            before_y = capped(before_y, all_y);
        }
        all_x = capped(all_x, part[0][i]);
        all_y = capped(all_y, part[1][i]);
    }
}

__global__ __launch_bounds__(kPlanThreads) void step_plan_kernel(const PlanArgs a) {
    __shared__ int s_part[2][2][kPlanThreads / 64];
    __shared__ int s_end[kPlanChunk];     // rows up to and with the sequence
    __shared__ int s_cached[kPlanChunk];
    __shared__ int s_new[kPlanChunk];     // planned rows
    __shared__ int s_first[kPlanChunk];   // its first place in the free list
    const int tid = threadIdx.x;
    const int num_free = min(max(a.num_free[0], 0), a.free_cap);
    const int t0 = blockIdx.x * kPlanChunk;             // this workgroup's rows
    const int t1 = min(t0 + kPlanChunk, a.T);
    int taken = 0, tokens = 0, rows = 0;                // of the chunks before
    int used = 0, refused = 0;                          // this thread's, for the counts
    const int chunks = (a.S + kPlanChunk - 1) / kPlanChunk;
    for (int c = 0; c < chunks; ++c) {
        const int s0 = c * kPlanChunk + tid * kPlanEach;
        int cached[kPlanEach], fresh[kPlanEach], need[kPlanEach];
        bool valid[kPlanEach];
        int sum_need = 0, sum_new = 0;
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            const bool in = s0 + i < a.S;
            cached[i] = in ? a.cached[s0 + i] : 0;
            fresh[i] = in ? a.fresh[s0 + i] : 0;
        }
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            // The table's tokens are below 2^31 (host), so neither side overflows.
            valid[i] = cached[i] >= 0 && fresh[i] >= 0 && cached[i] <= a.MB * kBlockTokens &&
                       fresh[i] <= a.MB * kBlockTokens - cached[i];
            const int have = (cached[i] >> kBlockShift) + ((cached[i] & (kBlockTokens - 1)) != 0);
            const int all = cached[i] + (valid[i] ? fresh[i] : 0);
            need[i] = valid[i] ? (all >> kBlockShift) + ((all & (kBlockTokens - 1)) != 0) - have : 0;
            sum_need = capped(sum_need, need[i]);
            sum_new = capped(sum_new, valid[i] ? min(fresh[i], kPlanMost) : 0);
        }
        int at_need, at_new, all_need, all_new;
        scan2(sum_need, sum_new, at_need, at_new, all_need, all_new, s_part[0]);
        at_need = capped(at_need, taken);
        at_new = capped(at_new, tokens);
        int planned[kPlanEach], first[kPlanEach];
        int sum_rows = 0, bad = 0;
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            first[i] = at_need;
            if (valid[i]) {
                at_need = capped(at_need, need[i]);
                at_new = capped(at_new, min(fresh[i], kPlanMost));
            }
            const bool fits = valid[i] && (need[i] == 0 || at_need <= num_free) && (fresh[i] == 0 || at_new <= a.T);
            planned[i] = fits ? fresh[i] : 0;
            if (fits && need[i] > 0) used = at_need;
            bad += !fits;
            sum_rows += planned[i];    // at most T in all
        }
        refused += bad;
        int at_row, none, all_rows, all_bad;
        scan2(sum_rows, bad, at_row, none, all_rows, all_bad, s_part[1]);
        at_row += rows;
        const bool writer = c % gridDim.x == blockIdx.x;
#pragma unroll
        for (int i = 0; i < kPlanEach; ++i) {
            at_row += planned[i];
            s_end[tid * kPlanEach + i] = at_row;
            s_cached[tid * kPlanEach + i] = cached[i];
            s_new[tid * kPlanEach + i] = planned[i];
            s_first[tid * kPlanEach + i] = first[i];
            if (writer && s0 + i < a.S) {
                a.ctx[s0 + i] = cached[i] + planned[i];
                a.offsets[s0 + i + 1] = at_row;
            }
        }
        __syncthreads();
        // This thread's rows that belong to the chunk.
        const int begin = rows;
        rows += all_rows;
        taken = capped(taken, all_need);
        tokens = capped(tokens, all_new);
        const int ta = max(t0 + tid * kPlanEach, begin);
        const int tb = min(min(t0 + (tid + 1) * kPlanEach, t1), rows);
        if (ta < tb) {
            const int count = min(a.S - c * kPlanChunk, kPlanChunk);
            int lo = 0, hi = count - 1;    // the first sequence that ends behind ta
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s_end[mid] > ta) hi = mid; else lo = mid + 1;
            }
            int pos[kPlanEach], slot[kPlanEach];
#pragma unroll
            for (int i = 0; i < kPlanEach; ++i) {
                const int t = ta + i;
                if (t >= tb) break;
                while (s_end[lo] <= t) ++lo;    // t < rows: some sequence of the chunk ends behind it
                const int p = s_cached[lo] + t - (s_end[lo] - s_new[lo]);
                const int j = p >> kBlockShift;
                const int have = (s_cached[lo] + kBlockTokens - 1) >> kBlockShift;
                int* const entry = a.bt + static_cast<size_t>(c * kPlanChunk + lo) * a.MB + j;
                int b;
                if (j < have) {
                    b = *entry;
                } else {
                    b = a.free_blocks[s_first[lo] + j - have];
                    if ((p & (kBlockTokens - 1)) == 0) *entry = b;
                }
                // Slots are 32 bits: a block past 2^27 has none.
                const bool known = b >= 0 && (a.num_blocks > 0 ? b < a.num_blocks : true) && b < (1 << 27);
                pos[i] = p;
                slot[i] = known ? (b << kBlockShift) + (p & (kBlockTokens - 1)) : -1;
            }
            if (a.wide && tb - ta == kPlanEach) {
                *reinterpret_cast<int4*>(a.positions + ta) = int4{pos[0], pos[1], pos[2], pos[3]};
                *reinterpret_cast<int4*>(a.slots + ta) = int4{slot[0], slot[1], slot[2], slot[3]};
            } else {
#pragma unroll
                for (int i = 0; i < kPlanEach; ++i) {
                    if (ta + i < tb) {
                        a.positions[ta + i] = pos[i];
                        a.slots[ta + i] = slot[i];
                    }
                }
            }
        }
        __syncthreads();  // the tables and s_part are free again
    }
    // Rows behind the last sequence are padding.
    for (int t = max(t0, rows) + tid; t < t1; t += kPlanThreads) {
        a.positions[t] = -1;
        a.slots[t] = -1;
    }
    if (blockIdx.x == 0) {
        const int w = tid >> 6;
        const int most = wave_max(used);
        const int none = wave_total(refused);
        if ((tid & 63) == 0) {
            s_part[0][0][w] = most;
            s_part[0][1][w] = none;
        }
        __syncthreads();
        if (tid == 0) {
            int u = 0, r = 0;
            for (int i = 0; i < kPlanThreads / 64; ++i) {
                u = max(u, s_part[0][0][i]);
                r += s_part[0][1][i];
            }
            a.offsets[0] = 0;
            a.counts[0] = u;
            a.counts[1] = rows;
            a.counts[2] = r;
        }
    }
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

int swiftllm_hip_plan_step(int32_t* block_tables, const int32_t* cached_lens, const int32_t* new_lens,
                           const int32_t* free_blocks, const int32_t* num_free, int free_capacity,
                           int num_seqs, int max_num_blocks_per_seq, int block_size, int num_tokens,
                           int num_blocks, int32_t* context_lens, int32_t* query_offsets,
                           int32_t* positions, int32_t* slot_mapping, int32_t* counts,
                           hipStream_t stream) {
    const char* who = "swiftllm_hip_plan_step";
    const int S = num_seqs, T = num_tokens, MB = max_num_blocks_per_seq;
    if (S < 0 || T < 0 || MB < 0 || free_capacity < 0 || block_size <= 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER,
                    "%s: num_seqs=%d num_tokens=%d max_num_blocks_per_seq=%d free_capacity=%d block_size=%d", who,
                    S, T, MB, free_capacity, block_size);
    }
    if (block_size != kBlockTokens) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: block_size=%d (supported: 16)", who, block_size);
    }
    if (S > 65535 || T >= kPlanMost || free_capacity >= kPlanMost || MB >= (1 << 27)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED,
                    "%s: num_seqs=%d num_tokens=%d free_capacity=%d max_num_blocks_per_seq=%d", who, S, T,
                    free_capacity, MB);
    }
    if (!num_free || !query_offsets || !counts || (S > 0 && (!cached_lens || !new_lens || !context_lens)) ||
        (S > 0 && MB > 0 && !block_tables) || (T > 0 && (!positions || !slot_mapping)) ||
        (free_capacity > 0 && !free_blocks)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    const void* all[] = {block_tables, cached_lens, new_lens, free_blocks, num_free,
                         context_lens, query_offsets, positions, slot_mapping, counts};
    for (const void* p : all) {
        if (!aligned(p, 4)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    // Every workgroup reads the lengths and the list while others write: no
    // output may lie on an input, nor on another output.
    const size_t n = sizeof(int32_t);
    const struct { const void* p; size_t bytes; } span[] = {
        {cached_lens, n * S}, {new_lens, n * S}, {free_blocks, n * free_capacity}, {num_free, n},
        {block_tables, n * S * MB}, {context_lens, n * S}, {query_offsets, n * (S + 1)},
        {positions, n * T}, {slot_mapping, n * T}, {counts, 3 * n}};
    for (int i = 4; i < 10; ++i) {
        for (int j = 0; j < i; ++j) {
            if (overlap(span[i].p, span[i].bytes, span[j].p, span[j].bytes)) {
                return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: an output overlaps another argument", who);
            }
        }
    }
    const int rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    PlanArgs a{};
    a.bt = block_tables;
    a.cached = cached_lens;
    a.fresh = new_lens;
    a.free_blocks = free_blocks;
    a.num_free = num_free;
    a.ctx = context_lens;
    a.offsets = query_offsets;
    a.positions = positions;
    a.slots = slot_mapping;
    a.counts = counts;
    a.S = S;
    a.T = T;
    a.MB = MB;
    a.free_cap = free_capacity;
    a.num_blocks = num_blocks;
    a.wide = aligned(positions, 16) && aligned(slot_mapping, 16);
    const int grid = T > 0 ? (T + kPlanChunk - 1) / kPlanChunk : 1;
    return launched(launch(step_plan_kernel, dim3(grid), dim3(kPlanThreads), 0, stream, a), who);
}

}  // extern "C"
