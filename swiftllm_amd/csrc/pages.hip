// Pages of a cache whose sequences come of one another (gfx950): forking, with
// the references of every block, and bringing a pool together.
//
// fork_pages. Row i of the new batch goes on from row p = parents[i] of the old
// one, -1 or any other number that is no row: from none. With
// used_i = ceil(context_i / 16):
//   tables_out[i, j] = tables[p, j] for j < used_p, context_out[i] = context[p]
//   refs[b] += (new rows' entries b) - (old rows' entries b)
// A partly filled last block is written by its row's next token, so that each
// row that goes on needs one of its own: of the rows that are about to write block
// b, whichever their parents, all take a copy where refs[b], as they are now, count
// a hold more than those, and all but the last where they do not. So one row keeps a
// block that nobody else holds, and every row copies one that somebody else
// holds. Copies go to the free blocks (refs[b] <= 0) in ascending order, rows in
// order; the free blocks behind those are the new list. A row whose block is
// missing ends with its whole blocks.
//
// compact_pages. The k-th highest block in use moves to the k-th lowest free one
// while it lies above it, at most max_moves. With L blocks in use, L - M of them
// stay: those below T, the lowest that moves, and ids from T on are free
// afterwards, id - L of them before id; below T the free ones but for the M lowest.
//
// Bound: latency. A step of 16 requests of 8 beams in 65536 blocks moves 0.9 MB
// (0.2 us), 1024 beams in 524288 blocks 12 MB (2.4 us). Three launches each (a fork in
// a small pool one, a compaction of few ids two), whose ends are the only order between
// workgroups: fork_pages moves references, counts the free blocks of every 4096 ids (and
// keeps them as bits) beside the copies, lists them: 3.5 + 3.6 + 3.9 us and 6.0 + 4.3 +
// 6.3 us at those sizes, each a chain of dependent reads. compact_pages counts the blocks
// in use, pairs them, renames: 3.2 + 3.8 + 3.9 us for 64 rows over 65536 blocks, 3.9 +
// 4.7 + 8.8 for 512 rows of 1000 blocks over 524288 (18 MB, 3.6 us). A block's place
// among those in use is a word of bits and the count before it; kept for every block in
// an array of its own, the last took 10.9. Where a row and its parent have the same
// block in the same place, as in a prompt that both share, nothing is counted: a
// search's reordering touches few counters.

#include <algorithm>

#include "common.hpp"

namespace swiftllm {
namespace {

constexpr int kRowThreads = 256;
constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / 64;
constexpr int kIds = 4096;               // ids of a workgroup: 64 words of 64 bits
constexpr int kWords = kIds / 64;
constexpr int kEach = kIds / kScanThreads;
constexpr int kSmallRows = 64;           // rows and entries of all, for one workgroup
constexpr int kSmallTables = 4096;
constexpr int kFewGroups = 4;            // whose ids every workgroup counts by itself
constexpr int kRowHalves = 2;            // rows of a workgroup that renames entries

struct PagesArgs {
    const int* tables;
    const int* ctx;
    const int* parents;
    int* tables_out;
    int* ctx_out;
    const int* refs;       // compact_pages: as they were
    int* refs_out;         // fork_pages: the references
    const int* taken;      // [1] or null
    int* free_blocks;
    int* num_free;         // [1]
    long long* pairs;      // [rooms][2]
    int* new_lens;         // [S] or null
    int* new_ids;
    int* counts;           // [2]
    // workspace
    int* sums;             // [groups]: blocks free (in use: compact) of a group of ids
    int* num_copies;       // [1]
    unsigned long long* bits;
    int* open;             // [S]: the block of the pool that a row is about to write, -1: none
    int* family;           // [S]: rows of its parent, where it is the last of them; 0: where it is not
    int* copies;           // [S]: rows that take a copy, in order
    int* last;             // [NB]: fork, of open blocks: the last row that is about to write it,
    int* writers;          //   and how many are
    int* from;             // [NB / 2]: compact: the blocks that move, highest first,
    int* to;               //   the free ones, lowest first,
    int* starts;           // [groups * kWords]: blocks in use before a word of ids
    int* found;            // [3]: compact: moves, blocks in use, the lowest that moves
    int S;
    int MB;
    int NB;
    int groups;            // ceil(NB / kIds)
    int rooms;             // pairs
};

__device__ __forceinline__ bool in_pool(int b, int NB) { return b >= 0 && b < NB; }

__device__ __forceinline__ int blocks_of(int ctx, int MB) {
    return min((max(ctx, 0) >> kBlockShift) + ((ctx & (kBlockTokens - 1)) != 0 && ctx > 0), MB);
}

__device__ __forceinline__ int parent_of(const PagesArgs& a, int i) {
    const int p = a.parents[i];
    return p >= 0 && p < a.S ? p : -1;
}

// The sum of x over the workgroup, in every thread.
template <int WAVES>
__device__ __forceinline__ int block_total(int x, int* part) {
    const int sum = wave_total(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) all += part[i];
    return all;
}

// Blocks that a plan took: of nobody until now.
__device__ __forceinline__ void fork_taken(const PagesArgs& a, int at, int step) {
    if (a.taken == nullptr) return;
    const int n = min(min(max(a.taken[0], 0), max(a.num_free[0], 0)), a.NB);
    for (int k = at; k < n; k += step) {
        const int b = a.free_blocks[k];
        if (in_pool(b, a.NB)) atomicAdd(a.refs_out + b, 1);
    }
}

// The last entry of a row that goes on, where it is partly filled and of the pool; -1: none.
__device__ __forceinline__ int open_entry(const PagesArgs& a, int ctx) {
    const int j = ctx >> kBlockShift;
    return (ctx & (kBlockTokens - 1)) != 0 && j < a.MB ? j : -1;
}

// Row i by THREADS threads, of which this is t: its table, the references that
// change, the block that it is about to write, its place among its siblings. part: of
// a workgroup, THREADS / 64.
template <int THREADS>
__device__ __forceinline__ void fork_row(const PagesArgs& a, int i, int t, int* part) {
    const int p = parent_of(a, i);
    const int was = blocks_of(a.ctx[i], a.MB);
    const int ctx = p < 0 ? 0 : max(a.ctx[p], 0);
    const int is = blocks_of(ctx, a.MB);
    const int* const old = a.tables + static_cast<size_t>(i) * a.MB;
    const int* const row = a.tables + static_cast<size_t>(max(p, 0)) * a.MB;
    int* const out = a.tables_out + static_cast<size_t>(i) * a.MB;
    const int open = open_entry(a, ctx);
    const int b = open < 0 ? -1 : row[open];
    for (int j = t; j < max(was, is); j += THREADS) {
        const int x = j < was ? old[j] : -1;
        const int y = j < is ? row[j] : -1;
        if (j < is) out[j] = y;
        if (x != y) {
            if (in_pool(y, a.NB)) atomicAdd(a.refs_out + y, 1);
            if (in_pool(x, a.NB)) atomicAdd(a.refs_out + x, -1);
        }
    }
    // Its siblings, itself among them, and above 16 bits those behind it.
    unsigned n = 0;
    if (p >= 0) {
        for (int k = t; k < a.S; k += THREADS) n += a.parents[k] == p ? 1u + (static_cast<unsigned>(k > i) << 16) : 0u;
    }
    if constexpr (THREADS == 64) {
        n = wave_total(static_cast<int>(n));
    } else {
        n = block_total<THREADS / 64>(static_cast<int>(n), part);
    }
    if (t == 0) {
        a.open[i] = in_pool(b, a.NB) ? b : -1;
        a.family[i] = n >> 16 ? 0 : n;
        a.ctx_out[i] = ctx;
        if (a.new_lens != nullptr) a.new_lens[i] = p >= 0;
    }
}

__global__ __launch_bounds__(kRowThreads) void fork_rows_kernel(const PagesArgs a) {
    __shared__ int s_part[kRowThreads / 64];
    fork_taken(a, blockIdx.x * kRowThreads + threadIdx.x, gridDim.x * kRowThreads);
    if (static_cast<int>(blockIdx.x) < a.S) fork_row<kRowThreads>(a, blockIdx.x, threadIdx.x, s_part);
}

// Bit b of word w of the pool: a block that nothing refers to (in use: LIVE).
template <bool LIVE>
__device__ __forceinline__ void scan_ids(const PagesArgs& a, const int* refs, int group, int* part) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int r[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int id = group * kIds + (w * kEach + k) * 64 + lane;
        r[k] = id < a.NB ? refs[id] : (LIVE ? 0 : 1);
    }
    int n = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const unsigned long long m = __ballot(LIVE ? r[k] > 0 : r[k] <= 0);
        if (lane == 0) {
            a.bits[static_cast<size_t>(group) * kWords + w * kEach + k] = m;
            n += __popcll(m);
        }
    }
    n = block_total<kScanWaves>(n, part);
    if (tid == 0) a.sums[group] = n;
}

// The rows that take a copy, in order, four rows a thread at a time. part: kScanWaves.
__device__ __forceinline__ void fork_copies(const PagesArgs& a, int* part) {
    const int tid = threadIdx.x;
    // A row with siblings behind it copies, and the last of them keeps the block where
    // nobody else refers to it. Where somebody does, those may be rows of other parents
    // that are about to write it too, as of one prompt in two requests: then all that
    // are about to write a block are counted, and the last of them found. (So in every
    // call, 1024 rows over 524288 blocks take 19.1 us and 4 over 4096 7.4, not 16.4 and 7.2.)
    int others = 0;
    for (int i = tid; i < a.S; i += kScanThreads) {
        const int b = a.open[i], family = a.family[i];
        others |= b >= 0 && family > 0 && a.refs_out[b] > family;
    }
    const bool counted = __syncthreads_or(others) != 0;
    if (counted) {
        for (int i = tid; i < a.S; i += kScanThreads) {
            const int b = a.open[i];
            if (b < 0) continue;
            a.last[b] = -1;
            a.writers[b] = 0;
        }
        __syncthreads();
        for (int i = tid; i < a.S; i += kScanThreads) {
            const int b = a.open[i];
            if (b < 0) continue;
            atomicMax(a.last + b, i);
            atomicAdd(a.writers + b, 1);
        }
        __syncthreads();
    }
    // (past the cache of this CU, as they were made)
    auto at_block = [](const int* x, int b) { return __hip_atomic_load(x + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto copies = [&](int i, int b) {
        if (counted) return i < at_block(a.last, b) || a.refs_out[b] > at_block(a.writers, b);
        const int family = a.family[i];
        return family == 0 || a.refs_out[b] > family;
    };
    int before = 0;
    for (int s0 = 0; s0 < a.S; s0 += 4 * kScanThreads) {
        bool copy[4];
        int n = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = s0 + 4 * tid + k;
            const int b = i < a.S ? a.open[i] : -1;
            copy[k] = b >= 0 && copies(i, b);
            n += copy[k];
        }
        const int incl = wave_inclusive_scan(n);
        if ((tid & 63) == 63) part[tid >> 6] = incl;
        __syncthreads();
        int at = before + incl - n;
#pragma unroll
        for (int w = 0; w < kScanWaves; ++w) {
            if (w < (tid >> 6)) at += part[w];
            before += part[w];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (copy[k]) a.copies[at++] = s0 + 4 * tid + k;
        }
    }
    if (tid == 0) a.num_copies[0] = before;
}

__global__ __launch_bounds__(kScanThreads) void fork_scan_kernel(const PagesArgs a) {
    __shared__ int s_part[kScanWaves];
    if (static_cast<int>(blockIdx.x) < a.groups) {
        scan_ids<false>(a, a.refs_out, blockIdx.x, s_part);
    } else {
        fork_copies(a, s_part);
    }
}

// What lies before this workgroup's ids, and in all: set bits. part: 2 kScanWaves.
__device__ __forceinline__ void sums_of(const PagesArgs& a, int group, int* part, int& before, int& all) {
    int x = 0, y = 0;
    for (int k = threadIdx.x; k < a.groups; k += kScanThreads) {
        const int n = a.sums[k];
        y += n;
        if (k < group) x += n;
    }
    before = block_total<kScanWaves>(x, part);
    all = block_total<kScanWaves>(y, part + kScanWaves);
}

// Set bits before each word of a group, of which lane k has word k, `before` of them
// before the group.
__device__ __forceinline__ int starts_of(unsigned long long mine, int before) {
    const int n = __popcll(mine);
    return before + wave_inclusive_scan(n) - n;
}

__device__ __forceinline__ unsigned long long word_of(const PagesArgs& a, int group) {
    return a.bits[static_cast<size_t>(group) * kWords + (threadIdx.x & 63)];
}

// For each of the thread's ids: take(id, bit, set bits before it in the pool).
// mine, start: of lane's word, as above.
template <typename F>
__device__ __forceinline__ void each_id(const PagesArgs& a, int group, unsigned long long mine, int start, F take) {
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int word = w * kEach + k;
        const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(mine), word);
        const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(mine >> 32), word);
        const unsigned long long m = static_cast<unsigned long long>(hi) << 32 | lo;
        const int id = group * kIds + word * 64 + lane;
        if (id < a.NB) {
            take(id, ((m >> lane) & 1ull) != 0,
                 __builtin_amdgcn_readlane(start, word) + __popcll(m & ((1ull << lane) - 1ull)));
        }
    }
}

// The copies and free blocks of a group's ids, one of `groups` that share the
// pairs behind the last. part: 2 kScanWaves.
__device__ __forceinline__ void fork_list(const PagesArgs& a, int group, int groups, int* part) {
    const int tid = threadIdx.x;
    int before, all;
    sums_of(a, group, part, before, all);
    const int wanted = a.num_copies[0];
    const int got = min(wanted, all);
    auto open_of = [&](int i) { return a.tables_out + static_cast<size_t>(i) * a.MB + (a.ctx_out[i] >> kBlockShift); };
    const unsigned long long mine = word_of(a, group);
    each_id(a, group, mine, starts_of(mine, before), [&](int id, bool free, int k) {
        if (!free) return;
        if (k >= got) {
            a.free_blocks[k - got] = id;
            return;
        }
        int* const entry = open_of(a.copies[k]);
        const int src = *entry;
        a.pairs[2 * static_cast<size_t>(k)] = src;
        a.pairs[2 * static_cast<size_t>(k) + 1] = id;
        *entry = id;
        a.refs_out[id] = 1;
        atomicAdd(a.refs_out + src, -1);
    });
    for (int k = got + group * kScanThreads + tid; k < a.S; k += groups * kScanThreads) {
        a.pairs[2 * static_cast<size_t>(k)] = -1;
        a.pairs[2 * static_cast<size_t>(k) + 1] = -1;
        if (k < wanted) {
            // (no other thread reads this row)
            const int i = a.copies[k];
            atomicAdd(a.refs_out + *open_of(i), -1);
            a.ctx_out[i] &= ~(kBlockTokens - 1);
            if (a.new_lens != nullptr) a.new_lens[i] = 0;
        }
    }
    if (group == 0 && tid == 0) {
        a.num_free[0] = all - got;
        a.counts[0] = got;
        a.counts[1] = wanted - got;
    }
}

__global__ __launch_bounds__(kScanThreads) void fork_list_kernel(const PagesArgs a) {
    __shared__ int s_part[2 * kScanWaves];
    fork_list(a, blockIdx.x, gridDim.x, s_part);
}

// All of it by one workgroup, a wave a row, where the pool is one group of ids and
// the tables are small. (us, three launches and one: 4 rows over 4096 blocks 9.9 and
// 7.2, 32 rows of 34 blocks 9.7 and 8.4; 4 rows over 8192 10.4 and 9.6, 32 rows of 65
// blocks over 8192 12.0 and 12.2.)
__global__ __launch_bounds__(kScanThreads) void fork_small_kernel(const PagesArgs a) {
    __shared__ int s_part[2 * kScanWaves];
    const int tid = threadIdx.x;
    fork_taken(a, tid, kScanThreads);
    for (int i = tid >> 6; i < a.S; i += kScanWaves) fork_row<64>(a, i, tid & 63, nullptr);
    __syncthreads();
    scan_ids<false>(a, a.refs_out, 0, s_part);
    __syncthreads();
    fork_copies(a, s_part);
    __syncthreads();
    fork_list(a, 0, 1, s_part);
}

__global__ __launch_bounds__(kScanThreads) void compact_scan_kernel(const PagesArgs a) {
    __shared__ int s_part[kScanWaves];
    scan_ids<true>(a, a.refs, blockIdx.x, s_part);
}

// The pairs of a group's ids, `before` of those in use before them: `live` of the first
// `all` ids are in use, of `all` in the pool, so the others move, at most the pairs' room.
__device__ __forceinline__ void compact_pairs(const PagesArgs& a, int group, unsigned long long mine, int before, int all, int live) {
    const int moves = min(all - live, a.rooms);
    if (group == 0 && threadIdx.x == 0) {
        a.found[0] = moves;
        a.found[1] = all;
        if (moves == 0) a.found[2] = a.NB;
    }
    const int start = starts_of(mine, before);
    if (threadIdx.x < kWords) a.starts[static_cast<size_t>(group) * kWords + threadIdx.x] = start;
    each_id(a, group, mine, start, [&](int id, bool used, int k) {
        const int at = used ? all - 1 - k : id - k;
        if (at >= moves) return;
        (used ? a.from : a.to)[at] = id;
        if (used && at == moves - 1) a.found[2] = id;
    });
}

__global__ __launch_bounds__(kScanThreads) void compact_pairs_kernel(const PagesArgs a) {
    __shared__ int s_part[3 * kScanWaves];
    const int tid = threadIdx.x;
    int before, all;
    sums_of(a, blockIdx.x, s_part, before, all);
    const int group = all / kIds;
    int live = 0;      // of the first `all` ids
    for (int k = tid; k < group; k += kScanThreads) live += a.sums[k];
    if (group < a.groups && tid < kWords) {
        const int n = min(max(all - group * kIds - tid * 64, 0), 64);
        const unsigned long long m = a.bits[static_cast<size_t>(group) * kWords + tid];
        live += __popcll(n == 64 ? m : m & ((1ull << n) - 1ull));
    }
    live = block_total<kScanWaves>(live, s_part + 2 * kScanWaves);
    compact_pairs(a, blockIdx.x, word_of(a, blockIdx.x), before, all, live);
}

// Both at once, where the groups are few: every workgroup counts all ids by itself, four
// neighbours of every group a thread. (us of three launches and of two, replayed: 8 rows
// over 4096 blocks 8.8 and 7.9, 32 over 16384 9.3 and 8.3; 16 groups so, 64 rows over
// 65536 blocks, 11.3 and 11.4.)
__global__ __launch_bounds__(kScanThreads) void compact_few_kernel(const PagesArgs a) {
    typedef int four __attribute__((ext_vector_type(4), aligned(4)));
    __shared__ int s_part[3 * kScanWaves];
    __shared__ unsigned long long s_bits[kWords];
    const int tid = threadIdx.x, lane = tid & 63, group = blockIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    four r[kFewGroups];
#pragma unroll
    for (int g = 0; g < kFewGroups; ++g) {
        const int id = g * kIds + 4 * tid;
        r[g] = four{0, 0, 0, 0};
        if (id + 4 <= a.NB) {
            r[g] = *reinterpret_cast<const four*>(a.refs + id);
        } else {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                if (id + k < a.NB) r[g][k] = a.refs[id + k];
            }
        }
    }
    int own[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int id = group * kIds + (w * kEach + k) * 64 + lane;
        own[k] = id < a.NB ? a.refs[id] : 0;
    }
    unsigned long long mine = 0;     // bit 4 g + k: id g kIds + 4 tid + k is in use
#pragma unroll
    for (int g = 0; g < kFewGroups; ++g) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mine |= r[g][k] > 0 ? 1ull << (4 * g + k) : 0ull;
    }
    static_assert(kFewGroups <= 16 && kIds == 4 * kScanThreads, "a word of bits");
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const unsigned long long m = __ballot(own[k] > 0);
        if (lane == 0) {
            s_bits[w * kEach + k] = m;
            a.bits[static_cast<size_t>(group) * kWords + w * kEach + k] = m;
        }
    }
    const int all = block_total<kScanWaves>(__popcll(mine), s_part);
    const int before = block_total<kScanWaves>(__popcll(mine & ((1ull << (4 * group)) - 1ull)), s_part + kScanWaves);
    // The thread's ids below `all`: four of every group before that of id `all`, and some there.
    const int last = all / kIds;
    const int some = min(max(all - last * kIds - 4 * tid, 0), 4);
    const unsigned long long lower = last >= 16 ? ~0ull : ((1ull << (4 * last)) - 1ull) | (((1ull << some) - 1ull) << (4 * last));
    const int live = block_total<kScanWaves>(__popcll(mine & lower), s_part + 2 * kScanWaves);
    compact_pairs(a, group, s_bits[lane], before, all, live);
}

__global__ __launch_bounds__(kScanThreads) void compact_apply_kernel(const PagesArgs a) {
    const int tid = threadIdx.x;
    const int moves = a.found[0], all = a.found[1], lowest = a.found[2];
    if (static_cast<int>(blockIdx.x) < a.groups) {
        const int group = blockIdx.x;
        const int start = a.starts[static_cast<size_t>(group) * kWords + (tid & 63)];
        each_id(a, group, word_of(a, group), start, [&](int id, bool live, int k) {
            const bool goes = live && id >= lowest;
            const int r = id - k;                              // free ones before this
            const bool comes = !live && r < moves;
            a.new_ids[id] = goes ? a.to[all - 1 - k] : id;
            a.refs_out[id] = goes ? 0 : a.refs[comes ? a.from[r] : id];
            if (id >= lowest) {
                a.free_blocks[id - all] = id;
            } else if (!live && !comes) {
                a.free_blocks[r - moves] = id;
            }
        });
        for (int k = group * kScanThreads + tid; k < a.rooms; k += a.groups * kScanThreads) {
            a.pairs[2 * static_cast<size_t>(k)] = k < moves ? a.from[k] : -1;
            a.pairs[2 * static_cast<size_t>(k) + 1] = k < moves ? a.to[k] : -1;
        }
        if (group == 0 && tid == 0) {
            a.num_free[0] = a.NB - all;
            a.counts[0] = moves;
            a.counts[1] = all;
        }
        return;
    }
    constexpr int kHalf = kScanThreads / kRowHalves;
    const int i = (blockIdx.x - a.groups) * kRowHalves + tid / kHalf;
    if (i >= a.S) return;
    const int used = blocks_of(a.ctx[i], a.MB);
    const size_t at = static_cast<size_t>(i) * a.MB;
    for (int j = tid % kHalf; j < used; j += kHalf) {
        const int b = a.tables[at + j];
        int to = b;
        if (b >= lowest && b < a.NB) {
            const unsigned long long m = a.bits[b >> 6], bit = 1ull << (b & 63);
            const int k = a.starts[b >> 6] + __popcll(m & (bit - 1ull));
            if ((m & bit) != 0) to = a.to[all - 1 - k];
        }
        a.tables_out[at + j] = to;
    }
}

// Offsets of the workspace.
struct Space {
    size_t sums, copies_n, found, bits, open, family, copies, last, writers, from, to, starts, bytes;
};

Space space_of(long long S, long long NB) {
    const auto up = [](long long n) { return static_cast<size_t>((n + 255) / 256 * 256); };
    const long long groups = (NB + kIds - 1) / kIds;
    Space s;
    s.sums = 0;
    s.copies_n = s.sums + up(4 * groups);
    s.found = s.copies_n + 256;
    s.bits = s.found + 256;
    s.open = s.bits + up(8 * groups * kWords);
    s.family = s.open + up(4 * S);
    s.copies = s.family + up(4 * S);
    s.last = s.copies + up(4 * S);        // a fork's,
    s.writers = s.last + up(4 * NB);
    s.from = s.last;                      // a compaction's in the same place
    s.to = s.from + up(4 * (NB / 2));
    s.starts = s.to + up(4 * (NB / 2));
    s.bytes = std::max(s.writers + up(4 * NB), s.starts + up(4 * groups * kWords));
    return s;
}

int check_sizes(const char* who, long long S, long long MB, int block_size, long long NB) {
    if (S < 0 || MB < 0 || NB <= 0 || block_size <= 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER,
                    "%s: num_seqs=%lld max_num_blocks_per_seq=%lld block_size=%d num_blocks=%lld", who, S, MB,
                    block_size, NB);
    }
    if (block_size != kBlockTokens) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: block_size=%d (supported: 16)", who, block_size);
    }
    // Slots are 32 bits, and so are a table's tokens.
    if (S > 65535 || MB >= (1 << 27) || NB >= (1 << 27)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_seqs=%lld max_num_blocks_per_seq=%lld num_blocks=%lld", who, S,
                    MB, NB);
    }
    return SWIFTLLM_OK;
}

void set_space(PagesArgs& a, void* workspace, const Space& s) {
    char* const ws = static_cast<char*>(workspace);
    a.sums = reinterpret_cast<int*>(ws + s.sums);
    a.num_copies = reinterpret_cast<int*>(ws + s.copies_n);
    a.found = reinterpret_cast<int*>(ws + s.found);
    a.bits = reinterpret_cast<unsigned long long*>(ws + s.bits);
    a.open = reinterpret_cast<int*>(ws + s.open);
    a.family = reinterpret_cast<int*>(ws + s.family);
    a.copies = reinterpret_cast<int*>(ws + s.copies);
    a.last = reinterpret_cast<int*>(ws + s.last);
    a.writers = reinterpret_cast<int*>(ws + s.writers);
    a.from = reinterpret_cast<int*>(ws + s.from);
    a.to = reinterpret_cast<int*>(ws + s.to);
    a.starts = reinterpret_cast<int*>(ws + s.starts);
}

// Whether one of the first `outputs` spans shares bytes with another span.
template <size_t N>
bool tangled(const Bytes (&span)[N], size_t outputs) {
    for (size_t i = 0; i < outputs; ++i) {
        for (size_t j = i + 1; j < N; ++j) {
            if (overlap_any(span[i], {span[j]})) return true;
        }
    }
    return false;
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

size_t swiftllm_hip_pages_workspace_size(int num_seqs, int num_blocks) {
    if (check_sizes("swiftllm_hip_pages_workspace_size", num_seqs, 0, kBlockTokens, num_blocks) != SWIFTLLM_OK) return 0;
    ok();
    return space_of(num_seqs, num_blocks).bytes;
}

int swiftllm_hip_fork_pages(int32_t* block_tables_out, int32_t* context_lens_out, const int32_t* block_tables,
                            const int32_t* context_lens, const int32_t* parents, int32_t* ref_counts,
                            int32_t* free_blocks, int32_t* num_free, const int32_t* taken, int64_t* copy_pairs,
                            int32_t* new_lens, int32_t* counts, void* workspace, size_t workspace_bytes, int num_seqs,
                            int max_num_blocks_per_seq, int block_size, int num_blocks, hipStream_t stream) {
    const char* who = "swiftllm_hip_fork_pages";
    const int S = num_seqs, MB = max_num_blocks_per_seq, NB = num_blocks;
    int rc = check_sizes(who, S, MB, block_size, NB);
    if (rc != SWIFTLLM_OK) return rc;
    if (!ref_counts || !free_blocks || !num_free || !counts || !workspace ||
        (S > 0 && (!context_lens_out || !context_lens || !parents || !copy_pairs)) ||
        (S > 0 && MB > 0 && (!block_tables_out || !block_tables))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    const Space space = space_of(S, NB);
    if (workspace_bytes < space.bytes) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, space.bytes);
    }
    const size_t n = S, word = sizeof(int32_t);
    const Bytes span[] = {{block_tables_out, word * n * MB}, {context_lens_out, word * n}, {ref_counts, word * NB},
                          {free_blocks, word * NB}, {num_free, word}, {copy_pairs, 16 * n}, {counts, 2 * word},
                          {workspace, space.bytes}, {new_lens, word * n}, {block_tables, word * n * MB}, {context_lens, word * n},
                          {parents, word * n}, {taken, word}};
    for (const Bytes& s : span) {
        if (!aligned(s.p, 4)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    if (!aligned(workspace, 256) || !aligned(copy_pairs, 8)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    if (tangled(span, 9)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: an output overlaps another argument", who);
    rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    PagesArgs a{};
    a.tables = block_tables;
    a.ctx = context_lens;
    a.parents = parents;
    a.tables_out = block_tables_out;
    a.ctx_out = context_lens_out;
    a.refs_out = ref_counts;
    a.taken = taken;
    a.free_blocks = free_blocks;
    a.num_free = num_free;
    a.pairs = reinterpret_cast<long long*>(copy_pairs);
    a.new_lens = new_lens;
    a.counts = counts;
    a.S = S;
    a.MB = MB;
    a.NB = NB;
    a.groups = (NB + kIds - 1) / kIds;
    a.rooms = S;
    set_space(a, workspace, space);
    if (a.groups == 1 && S <= kSmallRows && static_cast<long long>(S) * MB <= kSmallTables) {
        return launched(launch(fork_small_kernel, dim3(1), dim3(kScanThreads), 0, stream, a), who);
    }
    rc = launched(launch(fork_rows_kernel, dim3(std::max(S, 1)), dim3(kRowThreads), 0, stream, a), who);
    if (rc != SWIFTLLM_OK) return rc;
    rc = launched(launch(fork_scan_kernel, dim3(a.groups + 1), dim3(kScanThreads), 0, stream, a), who);
    if (rc != SWIFTLLM_OK) return rc;
    return launched(launch(fork_list_kernel, dim3(a.groups), dim3(kScanThreads), 0, stream, a), who);
}

int swiftllm_hip_compact_pages(int32_t* block_tables_out, int32_t* ref_counts_out, const int32_t* block_tables,
                               const int32_t* context_lens, const int32_t* ref_counts, int32_t* free_blocks,
                               int32_t* num_free, int64_t* copy_pairs, int32_t* new_ids, int32_t* counts,
                               void* workspace, size_t workspace_bytes, int num_seqs, int max_num_blocks_per_seq,
                               int block_size, int num_blocks, int max_moves, hipStream_t stream) {
    const char* who = "swiftllm_hip_compact_pages";
    const int S = num_seqs, MB = max_num_blocks_per_seq, NB = num_blocks;
    int rc = check_sizes(who, S, MB, block_size, NB);
    if (rc != SWIFTLLM_OK) return rc;
    if (max_moves < 0 || max_moves > NB) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: max_moves=%d of num_blocks=%d", who, max_moves, NB);
    }
    if (!ref_counts_out || !ref_counts || !free_blocks || !num_free || !new_ids || !counts || !workspace ||
        (max_moves > 0 && !copy_pairs) || (S > 0 && !context_lens) ||
        (S > 0 && MB > 0 && (!block_tables_out || !block_tables))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    const Space space = space_of(S, NB);
    if (workspace_bytes < space.bytes) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, space.bytes);
    }
    const size_t n = S, word = sizeof(int32_t);
    const Bytes span[] = {{block_tables_out, word * n * MB}, {ref_counts_out, word * NB}, {free_blocks, word * NB},
                          {num_free, word}, {copy_pairs, 16 * static_cast<size_t>(max_moves)}, {new_ids, word * NB},
                          {counts, 2 * word}, {workspace, space.bytes}, {context_lens, word * n}, {ref_counts, word * NB},
                          {block_tables_out == block_tables ? nullptr : block_tables, word * n * MB}};
    for (const Bytes& s : span) {
        if (!aligned(s.p, 4)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    if (!aligned(workspace, 256) || !aligned(copy_pairs, 8)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    if (tangled(span, 8)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: an output overlaps another argument", who);
    rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    PagesArgs a{};
    a.tables = block_tables;
    a.ctx = context_lens;
    a.tables_out = block_tables_out;
    a.refs = ref_counts;
    a.refs_out = ref_counts_out;
    a.free_blocks = free_blocks;
    a.num_free = num_free;
    a.pairs = reinterpret_cast<long long*>(copy_pairs);
    a.new_ids = new_ids;
    a.counts = counts;
    a.S = S;
    a.MB = MB;
    a.NB = NB;
    a.groups = (NB + kIds - 1) / kIds;
    a.rooms = max_moves;
    set_space(a, workspace, space);
    if (a.groups <= kFewGroups) {
        rc = launched(launch(compact_few_kernel, dim3(a.groups), dim3(kScanThreads), 0, stream, a), who);
    } else {
        rc = launched(launch(compact_scan_kernel, dim3(a.groups), dim3(kScanThreads), 0, stream, a), who);
        if (rc != SWIFTLLM_OK) return rc;
        rc = launched(launch(compact_pairs_kernel, dim3(a.groups), dim3(kScanThreads), 0, stream, a), who);
    }
    if (rc != SWIFTLLM_OK) return rc;
    const int rows = (S + kRowHalves - 1) / kRowHalves;
    return launched(launch(compact_apply_kernel, dim3(a.groups + rows), dim3(kScanThreads), 0, stream, a), who);
}

}  // extern "C"
