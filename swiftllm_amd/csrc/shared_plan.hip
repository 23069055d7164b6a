// The plan of attention over blocks that sequences share (gfx950): what a group's
// tables have in common, and the list of walks (shared_plan.hpp) that the layers of
// a step then take without looking at the tables again but for their ids.
//
// Of a group with n >= 2 sequences that have a context, the leading table entries
// that all of them use, and alike, are shared; a walk takes those that all of them
// have filled, sh blocks, so that no row sees part of one, where the (n - 1) sh that
// it saves are worth it. Rows of a group without a context count for nothing.
//
// Bound: latency. A step of 128 sequences of 256 blocks compares 131 KB, once for
// all layers. Two launches: a workgroup per sequence compares its row with its
// group's first live one; one workgroup makes the list, in scans over the sequences.
// Nothing is kept from one call for the next.

#include "shared_plan.hpp"

namespace swiftllm {
namespace {

using namespace shared;

constexpr int kMatchThreads = 256;
constexpr int kMostCounted = 1024;
constexpr int kListThreads = 512;
constexpr int kListWaves = kListThreads / 64;
constexpr int kTries = 16;          // lengths of a range that are tried
constexpr int kMostMulti = 512;
constexpr int kWindow = 2048;       // groups whose minima are in LDS at a time

struct PlanSharedArgs {
    const int* bt;
    const int* ctx;
    const int* offsets;     // [N + 1]
    int* shared;            // [N]
    Head* head;
    Start* wide;            // [ranges]
    Start* narrow;          // [ranges * kTileWaves]
    Walk* walks;
    Seq* seqs;
    int4* infos;            // [S]: group, its first live row, leading blocks alike with it, blocks shared
    int4* costs;            // [S][2]: aligned, other wide and narrow walks and their costs before it
    int S, N, MB, H, Hkv, D;
    int HC, gw, per_tile, ranges;
    int min_saved;
};

__device__ __forceinline__ int used_blocks(const PlanSharedArgs& a, int s) {
    const int L = min(max(a.ctx[s], 0), a.MB * kBlockTokens);
    return (L + kBlockTokens - 1) >> kBlockShift;
}

__global__ __launch_bounds__(kMatchThreads) void shared_match_kernel(const PlanSharedArgs a) {
    __shared__ int s_least[kMatchThreads / 64];
    const int s = blockIdx.x, tid = threadIdx.x;
    // The least of the threads' numbers, in all of them.
    auto least = [&](int x) {
        // (wave_max is of numbers >= 0)
        const int w = 0x7fffffff - wave_max(0x7fffffff - x);
        __syncthreads();
        if ((tid & 63) == 0) s_least[tid >> 6] = w;
        __syncthreads();
        int m = s_least[0];
        for (int i = 1; i < kMatchThreads / 64; ++i) m = min(m, s_least[i]);
        return m;
    };
    // The last group that begins at s or before: by counting those that do, all at
    // once, or among many by bisection. (Offsets out of order, which the list's kernel
    // refuses, give some number of a group here.)
    int lo = 0;
    if (a.N <= kMostCounted) {
        for (int i = tid; i < a.N; i += kMatchThreads) lo += a.offsets[i] <= s;
        lo = wave_total(lo);
        if ((tid & 63) == 0) s_least[tid >> 6] = lo;
        __syncthreads();
        lo = 0;
        for (int i = 0; i < kMatchThreads / 64; ++i) lo += s_least[i];
    } else {
        int hi = a.N;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.offsets[mid] <= s) lo = mid + 1; else hi = mid;
        }
    }
    const int g = lo - 1;
    int4 info = int4{-1, -1, 0, 0};
    if (g >= 0 && g < a.N && a.offsets[g + 1] > s) {
        info.x = g;
        const int b = max(a.offsets[g], 0), e = min(a.offsets[g + 1], a.S);
        int lead = 0x7fffffff;
        for (int i = b; i < e && lead == 0x7fffffff; i += kMatchThreads) {
            lead = least(i + tid < e && a.ctx[i + tid] > 0 ? i + tid : 0x7fffffff);
        }
        if (lead < a.S) {
            info.y = lead;
            const int n = min(used_blocks(a, lead), used_blocks(a, s));
            const int* const x = a.bt + static_cast<size_t>(lead) * a.MB;
            const int* const y = a.bt + static_cast<size_t>(s) * a.MB;
            info.z = n;
            constexpr int kTake = 4;
            for (int j0 = 0; j0 < n; j0 += kTake * kMatchThreads) {
                int first = n;
#pragma unroll
                for (int k = kTake - 1; k >= 0; --k) {
                    const int j = j0 + k * kMatchThreads + tid;
                    if (j < n && x[j] != y[j]) first = j;
                }
                first = least(first);
                if (first < n) {
                    info.z = first;
                    break;
                }
            }
        }
    }
    if (tid == 0) a.infos[s] = info;
}

// Exclusive prefixes of the N numbers of x over the workgroup's threads, in x, and
// their totals.
template <int N>
__device__ __forceinline__ void scan(int (&x)[N], int (&all)[N], int (*part)[kListWaves]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int upto[N];
#pragma unroll
    for (int k = 0; k < N; ++k) upto[k] = wave_inclusive_scan(x[k]);
    __syncthreads();
    if (lane == 63) {
#pragma unroll
        for (int k = 0; k < N; ++k) part[k][w] = upto[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        x[k] = upto[k] - x[k];
        all[k] = 0;
#pragma unroll
        for (int i = 0; i < kListWaves; ++i) {
            const int p = part[k][i];
            if (i < w) x[k] += p;
            all[k] += p;
        }
    }
}

// ONE: at most as many sequences as threads, each of which keeps what it knows of its own.
template <bool ONE>
__global__ __launch_bounds__(kListThreads) void shared_list_kernel(const PlanSharedArgs a) {
    __shared__ int s_least[kWindow], s_full[kWindow], s_live[kWindow];
    __shared__ int s_part[6][kListWaves];
    __shared__ int s_pad[kTries];
    __shared__ int s_multi[kMostMulti];               // costs of tiles that share with others
    __shared__ int s_tile[ONE ? kListThreads : 1];    // the walk of the tile that begins with a sequence
    __shared__ int s_bad, s_saved, s_tiles, s_most;
    const int tid = threadIdx.x;
    if (tid == 0) s_bad = s_saved = s_tiles = s_most = 0;
    if (tid < kTries) s_pad[tid] = 0;
    struct Row {
        int4 info;       // w: blocks shared
        int ctx;
        int off, end;    // its group
    };
    auto load_row = [&](int s) {
        Row r{int4{-1, -1, 0, 0}, 0, 0, 0};
        if (s < a.S) {
            r.info = a.infos[s];
            r.ctx = a.ctx[s];
            if (r.info.x >= 0) {
                r.off = a.offsets[r.info.x];
                r.end = a.offsets[r.info.x + 1];
            }
        }
        return r;
    };
    Row mine = load_row(ONE ? tid : a.S);
    auto row_of = [&](int s) { return ONE ? mine : load_row(s); };
    __syncthreads();
    for (int i = tid; i < a.N; i += kListThreads) {
        const int b = a.offsets[i], e = a.offsets[i + 1];
        if (b < 0 || e < b || e > a.S) s_bad = 1;
    }
    // What every group shares, and of that what is worth it, a window of groups at a time.
    for (int g0 = 0; g0 < max(a.N, 1); g0 += kWindow) {
        for (int i = tid; i < min(max(a.N - g0, 0), kWindow); i += kListThreads) {
            s_least[i] = s_full[i] = 0x7fffffff;
            s_live[i] = 0;
        }
        __syncthreads();
        const bool bad = s_bad != 0;
        for (int s = tid; s < a.S; s += kListThreads) {
            const Row r = row_of(s);
            const int g = r.info.x - g0;
            if (r.info.x >= 0 && g >= 0 && g < kWindow && r.ctx > 0) {
                atomicMin(&s_least[g], r.info.z);
                atomicMin(&s_full[g], r.ctx >> kBlockShift);
                atomicAdd(&s_live[g], 1);
            }
        }
        __syncthreads();
        for (int s = tid; s < a.S; s += kListThreads) {
            const Row r = row_of(s);
            const int g = r.info.x - g0;
            if (r.info.x >= 0 && g >= 0 && g < kWindow) {
                const int live = s_live[g], sh = min(s_least[g], s_full[g]);
                const bool worth = !bad && live > 1 && static_cast<long long>(live - 1) * sh >= (a.min_saved < 0 ? kLeastSaved : max(a.min_saved, 1));
                if (worth && r.info.y == s) atomicAdd(&s_saved, (live - 1) * sh);
                if (ONE) {
                    mine.info.w = worth ? sh : 0;
                } else {
                    a.infos[s].w = worth ? sh : 0;
                }
            }
        }
        for (int i = tid; i < min(a.N - g0, kWindow); i += kListThreads) {
            a.shared[g0 + i] = bad || s_live[i] == 0 ? 0 : s_least[i];
        }
        __syncthreads();
    }
    // All of it together has to be worth the joins.
    const bool share = a.min_saved >= 0 || static_cast<long long>(s_saved) * a.HC * a.D >= kLeastSavedAll;
    // A sequence's walks: a tile's, where it is the first of one, and its own.
    struct Mine {
        int sh, L, count, own;                // blocks shared; sequences of the tile; own blocks
        int wide, tile_cost, own_cost;        // (a walk's cost of 0: there is none)
        int group;                            // sequences of its group
        int lead;
    };
    auto walks_of = [&](int s) {
        Mine m{};
        if (s >= a.S) return m;
        const Row r = row_of(s);
        m.sh = share ? r.info.w : 0;
        m.lead = r.info.y;
        m.L = min(max(r.ctx, 0), a.MB * kBlockTokens);
        m.own = ((m.L + kBlockTokens - 1) >> kBlockShift) - (m.L > 0 ? m.sh : 0);
        m.own_cost = m.own > 0 ? m.own + kNarrowCost : 0;
        m.group = r.end - r.off;
        if (m.sh > 0 && (s - r.off) % a.per_tile == 0) {
            m.count = min(a.per_tile, r.end - s);
            m.wide = m.count * a.gw > kNarrowRows;
            m.tile_cost = m.sh + (m.wide ? kWideCost : kNarrowCost);
        }
        return m;
    };
    int sum[3] = {0, 0, 0}, sums[3];      // in all; what is wide, and what it takes
    for (int s = tid; s < a.S; s += kListThreads) {
        const Mine m = walks_of(s);
        sum[0] += m.tile_cost + m.own_cost;
        if (m.wide) {
            sum[1] += m.tile_cost;
            sum[2] += m.tile_cost + m.tile_cost / 12 * ((m.count * a.gw + kWaveRows - 1) / kWaveRows);
        }
        if (m.wide && m.group > a.per_tile) {
            const int at = atomicAdd(&s_tiles, 1);
            if (at < kMostMulti) s_multi[at] = m.tile_cost;
            atomicMax(&s_most, m.tile_cost);
        }
    }
    scan(sum, sums, s_part);
    const int all = sums[0];
    // The ranges of what is wide. Where that is most of all, its products bound it, and a
    // block takes a workgroup the longer the more of its waves have rows: it counts for a
    // twelfth more with each. Where it is not, HBM bounds both alike. (us a pass, counted
    // so and not: 4 x 16 questions on 30000 tokens, 64/8 heads x 128 with biases, 285 and
    // 295, 16 x 8 beams on 2500, 32/8 with a cap, 216 and 220; 128 chats on 8192 tokens
    // 306 and 288.)
    const int narrow_sum = all - sums[1];
    int wide_ranges = 0;
    if (sums[1] > 0) {
        const float takes = static_cast<float>(sums[1] > narrow_sum ? sums[2] : sums[1]);
        wide_ranges = static_cast<int>(ceilf(takes / (takes + static_cast<float>(narrow_sum)) * static_cast<float>(a.ranges)));
        wide_ranges = narrow_sum > 0 ? min(max(wide_ranges, 1), a.ranges - 1) : a.ranges;
    }
    // Where several tiles share blocks, each begins and ends with a range, so that
    // they come by the same blocks at the same time, in one L2: the first length that
    // cuts the longest tile evenly and leaves room for all. (More than kMostMulti tiles
    // are many for any cut.)
    const int tiles = s_tiles <= kMostMulti ? s_tiles : 0;
    const int len0 = wide_ranges > 0 ? max((sums[1] + wide_ranges - 1) / wide_ranges, kLeastRange) : kLeastRange;
    auto try_len = [&](int k) {
        const int cuts = s_most / len0 - k;
        return cuts > 0 ? (s_most + cuts - 1) / cuts : len0 + k * max(len0 / 16, 1);
    };
    auto padded = [](int cost, int len) { return cost > 2 * len ? (cost + len - 1) / len * len : cost; };
    for (int i = tid / kTries; i < tiles; i += kListThreads / kTries) {
        const int k = tid % kTries;
        atomicAdd(&s_pad[k], padded(s_multi[i], try_len(k)) - s_multi[i]);
    }
    __syncthreads();
    // (a lane of every wave tries a length)
    const int tried = try_len(tid % kTries);
    const unsigned long long fits = __ballot(tiles > 0 && sums[1] + static_cast<long long>(s_pad[tid % kTries]) <= static_cast<long long>(wide_ranges) * tried);
    const bool align = fits != 0;
    const int len = align ? try_len(__builtin_ctzll(fits)) : len0;
    // Aligned tiles first, other wide ones, then the narrow ones.
    auto cost_of = [&](const Mine& m, int& aligned, int& wide, int& narrow) {
        const int n = align && m.wide && m.group > a.per_tile && m.tile_cost > 2 * len ? padded(m.tile_cost, len) : 0;
        aligned = n;
        wide = m.wide && n == 0 ? m.tile_cost : 0;
        narrow = m.wide ? 0 : m.tile_cost;
    };
    int walks[3] = {0, 0, 0}, costs[3] = {0, 0, 0};     // of the chunks before
    int at_walks[3], at_costs[3];                       // of this thread's sequence, and in all at the end
    auto scan_row = [&](int s, const Mine& m) {
        int aligned, wide, narrow;
        cost_of(m, aligned, wide, narrow);
        int x[6] = {aligned > 0, aligned, wide > 0, wide, (narrow > 0) + (m.own_cost > 0), narrow + m.own_cost}, sums[6];
        scan(x, sums, s_part);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            at_walks[k] = walks[k] + x[2 * k];
            at_costs[k] = costs[k] + x[2 * k + 1];
            walks[k] += sums[2 * k];
            costs[k] += sums[2 * k + 1];
        }
        if (!ONE && s < a.S) {
            a.costs[2 * static_cast<size_t>(s)] = int4{at_walks[0], at_costs[0], at_walks[1], at_costs[1]};
            a.costs[2 * static_cast<size_t>(s) + 1] = int4{at_walks[2], at_costs[2], 0, 0};
        }
    };
    for (int s0 = 0; s0 < (ONE ? 1 : a.S); s0 += kListThreads) scan_row(s0 + tid, walks_of(s0 + tid));
    const int wide_walks = walks[0] + walks[1];
    const int wide_end = costs[0] + costs[1];
    wide_ranges = (wide_end + len - 1) / len;
    const int narrow_len = wide_ranges < a.ranges ? max((costs[2] + a.ranges - wide_ranges - 1) / (a.ranges - wide_ranges), kLeastRange) : kLeastRange;
    // A tile's walk, from the sums before its first sequence.
    auto tile_walk = [&](const Mine& m, const int (&n)[3]) {
        int aligned, wide, narrow;
        cost_of(m, aligned, wide, narrow);
        return aligned > 0 ? n[0] : wide > 0 ? walks[0] + n[1] : wide_walks + n[2];
    };
    if (ONE) s_tile[tid] = tile_walk(walks_of(tid), at_walks);
    __syncthreads();      // that, or the costs, is there for all
    int rows = 0;
    for (int s0 = 0; s0 < a.S; s0 += kListThreads) {
        const int s = s0 + tid;
        const Mine m = walks_of(s);
        if (!ONE && s < a.S) {
            const int4 x = a.costs[2 * static_cast<size_t>(s)], y = a.costs[2 * static_cast<size_t>(s) + 1];
            at_walks[0] = x.x;
            at_costs[0] = x.y;
            at_walks[1] = x.z;
            at_costs[1] = x.w;
            at_walks[2] = y.x;
            at_costs[2] = y.y;
        }
        int aligned, wide, narrow;
        cost_of(m, aligned, wide, narrow);
        const bool joins = m.sh > 0 && m.L > 0;
        const int tile_at = aligned > 0 ? at_costs[0] + kWideCost : wide > 0 ? costs[0] + at_costs[1] + kWideCost : at_costs[2] + kNarrowCost;
        const int own_at = at_costs[2] + narrow + kNarrowCost;
        int tile_rows = 0, own_rows = 0;
        if (m.count > 0) tile_rows = m.count * a.gw * pieces_of(m.wide, tile_at, m.sh, m.wide ? len : narrow_len);
        if (m.own > 0) {
            const int n = pieces_of(false, own_at, m.own, narrow_len);
            if (joins || n > 1) own_rows = a.gw * n;
        }
        int x[1] = {tile_rows + own_rows}, sums[1];
        scan(x, sums, s_part);
        if (s < a.S) {
            const int f = rows + x[0];
            // A walk, and the ranges, or waves' parts, that begin in it or in what it costs.
            auto put = [&](int v, const Walk& w, int from, int to, bool wide) {
                a.walks[v] = w;
                const unsigned scale = wide ? 1 : kTileWaves, n = wide ? len : narrow_len;
                for (unsigned r = (scale * from + n - 1) / n; r * n < scale * to; ++r) {
                    Start& begin = (wide ? a.wide : a.narrow)[r];
                    begin.walk = w;
                    begin.v = v;
                }
            };
            if (m.count > 0) {
                const Walk w{m.lead, 0, m.sh, s, m.count, tile_at, m.group <= a.per_tile, f};
                const int from = tile_at - (m.wide ? kWideCost : kNarrowCost);
                put(tile_walk(m, at_walks), w, from, aligned > 0 ? from + aligned : tile_at + m.sh, m.wide);
            }
            const int own_v = wide_walks + at_walks[2] + (narrow > 0);
            if (m.own > 0) {
                put(own_v, Walk{s, m.L > 0 ? m.sh : 0, m.own, s, 1, own_at, 1, own_rows > 0 ? f + tile_rows : -1}, own_at - kNarrowCost, own_at + m.own, false);
            }
            Seq q{m.L, m.own > 0 ? own_v : -1, -1, 0};
            if (joins) {
                // Its tile begins with another sequence of the group, or with itself.
                const Row r = row_of(s);
                q.index = (s - r.off) % a.per_tile;
                const int t = s - q.index;
                if (ONE) {
                    q.tile = s_tile[t];
                } else {
                    const int4 p = a.costs[2 * static_cast<size_t>(t)], y = a.costs[2 * static_cast<size_t>(t) + 1];
                    const int n[3] = {p.x, p.z, y.x};
                    q.tile = tile_walk(walks_of(t), n);
                }
            }
            a.seqs[s] = q;
        }
        rows += sums[0];
    }
    if (tid == 0) *a.head = Head{kMagic, a.S, a.MB, a.H, a.Hkv, a.D, wide_walks, wide_walks + walks[2], wide_end, costs[2], len, narrow_len, wide_ranges};
}

}  // namespace

namespace shared {

int check_sizes(const char* who, long long S, long long H, long long Hkv, long long D, long long BS, long long MB) {
    if (S < 0 || H <= 0 || Hkv <= 0 || D <= 0 || BS <= 0 || MB < 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER,
                    "%s: num_seqs=%lld num_heads=%lld num_kv_heads=%lld head_dim=%lld block_size=%lld "
                    "max_num_blocks_per_seq=%lld", who, S, H, Hkv, D, BS, MB);
    }
    if (H % Hkv != 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_heads %lld not a multiple of num_kv_heads %lld", who, H, Hkv);
    }
    if ((D != 64 && D != 128) || BS != kBlockTokens) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: head_dim=%lld block_size=%lld (supported: 64/128, 16)", who, D, BS);
    }
    // Token positions and the list's cost are 32-bit sums, and a fragment's row times
    // its values is too.
    if (S > 65535 || H > 65535 || MB >= (1 << 27) || 2 * S * (MB + kWideCost) >= (1LL << 30)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_seqs=%lld num_heads=%lld max_num_blocks_per_seq=%lld", who, S, H, MB);
    }
    return SWIFTLLM_OK;
}

}  // namespace shared
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

size_t swiftllm_hip_plan_shared_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim, int block_size,
                                     int max_num_blocks_per_seq) {
    if (shared::check_sizes("swiftllm_hip_plan_shared_size", num_seqs, num_heads, num_kv_heads, head_dim, block_size,
                            max_num_blocks_per_seq) != SWIFTLLM_OK) {
        return 0;
    }
    ok();
    return shared::layout_of(num_seqs, num_heads, num_kv_heads).bytes;
}

int swiftllm_hip_plan_shared(void* plan, size_t plan_bytes, int32_t* shared_blocks, const int32_t* block_tables,
                             const int32_t* context_lens, const int32_t* group_offsets, int num_groups, int num_seqs,
                             int num_heads, int num_kv_heads, int head_dim, int block_size, int max_num_blocks_per_seq,
                             int min_saved, hipStream_t stream) {
    const char* who = "swiftllm_hip_plan_shared";
    int rc = shared::check_sizes(who, num_seqs, num_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq);
    if (rc != SWIFTLLM_OK) return rc;
    if (num_groups < 0) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_groups=%d", who, num_groups);
    if (num_groups > 65535) return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_groups=%d", who, num_groups);
    if (!plan || (num_groups > 0 && (!shared_blocks || !group_offsets)) || (num_seqs > 0 && !context_lens) ||
        (num_seqs > 0 && max_num_blocks_per_seq > 0 && !block_tables)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    if (!aligned(plan, 256) || !aligned(shared_blocks, 4) || !aligned(block_tables, 4) || !aligned(context_lens, 4) ||
        !aligned(group_offsets, 4)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    const shared::Layout l = shared::layout_of(num_seqs, num_heads, num_kv_heads);
    if (plan_bytes < l.bytes) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: plan of %zu bytes, %zu needed", who, plan_bytes, l.bytes);
    }
    const size_t n = num_seqs;
    const Bytes bt{block_tables, 4 * n * max_num_blocks_per_seq}, ctx{context_lens, 4 * n};
    const Bytes off{group_offsets, num_groups > 0 ? 4 * (static_cast<size_t>(num_groups) + 1) : 0};
    const Bytes sh{shared_blocks, 4 * static_cast<size_t>(num_groups)}, out{plan, l.bytes};
    if (overlap_any(out, {sh, bt, ctx, off}) || overlap_any(sh, {bt, ctx, off})) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: an output overlaps another argument", who);
    }
    rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    const shared::Heads h = shared::heads_of(num_heads, num_kv_heads);
    char* const p = static_cast<char*>(plan);
    PlanSharedArgs a{};
    a.bt = block_tables;
    a.ctx = context_lens;
    a.offsets = group_offsets;
    a.shared = shared_blocks;
    a.head = reinterpret_cast<shared::Head*>(p);
    a.walks = reinterpret_cast<shared::Walk*>(p + l.walks);
    a.wide = reinterpret_cast<shared::Start*>(p + l.wide_starts);
    a.narrow = reinterpret_cast<shared::Start*>(p + l.narrow_starts);
    a.seqs = reinterpret_cast<shared::Seq*>(p + l.seqs);
    a.infos = reinterpret_cast<int4*>(p + l.infos);
    a.costs = reinterpret_cast<int4*>(p + l.costs);
    a.S = num_seqs;
    a.N = num_groups;
    a.MB = max_num_blocks_per_seq;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.HC = h.HC;
    a.gw = h.gw;
    a.per_tile = h.per_tile;
    a.ranges = l.ranges;
    a.min_saved = min_saved;
    if (num_seqs > 0) {
        rc = launched(launch(shared_match_kernel, dim3(num_seqs), dim3(kMatchThreads), 0, stream, a), who);
        if (rc != SWIFTLLM_OK) return rc;
    }
    return launched(launch(num_seqs <= kListThreads ? shared_list_kernel<true> : shared_list_kernel<false>, dim3(1), dim3(kListThreads), 0, stream, a), who);
}

}  // extern "C"
