// Paged attention of packed query tokens with shaped scores (gfx950): soft
// cap, distance bias, sliding window and two-sided prefix (scored_core.hpp).
// Rows query_offsets[s] .. query_offsets[s + 1] - 1 are the last tokens of
// sequence s, whose keys up to context_lens[s] are in the cache: a whole
// prompt, or a chunk of one on top of what is cached.
//
// Work. Four waves take consecutive tokens of one kv head; a wave owns 32
// query rows (32 / gw tokens x gw = min(G, 32) heads) on 32x32x16 products:
// S^T = K Q^T leaves a lane 32 scores of one row per stage of 64 keys, and P
// goes into O^T = V P^T from those registers. A stage's K and V tiles go into
// LDS once for the four waves by direct loads, two stages deep, one barrier a
// stage; V lies in the cache as the product's row operand, K comes back turned
// by ds_read_b64_tr_b16. The walk takes the stages of the prefix, then those
// from the tile's window on: hidden stages are not read. The tiles of all
// sequences are one list, longest walk first.
//
// Scores. The masks and the two-sided distance are worked out only in stages
// that some row of the wave does not see whole, and a wave leaves out the
// stages behind its last row. A capped score is c - 2 c u with
// u = 1 / (1 + e^y), y = 2 x / c: two transcendental operations, a third for
// the weight. Without a bias the score itself is not made: the largest comes
// from the least u, and the weight is exp2 of one multiply-add of u. A bias in a
// stage that is seen whole is its first key's, the same for a pair's scores, and
// a rise over them that 16 registers keep: one operation a score less, 2-4 %.
// Weights are rounded to 16 bits, to nearest, and summed as rounded: the
// output's error is that of its own rounding and a smaller one, 1.05 to 1.15
// times that of the rounding alone (8 x 2048 tokens in fp16 2.32e-4 of the
// output, not 2.07e-4). A second 16-bit part of the weights, as in decode, would
// add 16 products to a stage's 32 (D = 128).
//
// Order. What a stage costs a wave beside its 32 products (D = 128) is 115 to
// 250 vector operations for its 32 scores a lane, so the order of both is
// fixed: products of two blocks' values, both pairs' next scores, the other
// two blocks' values, each operand read two products ahead (2, 3, 4, 6 and 8
// took the same time, left to the compiler 8 x 2048 tokens with a cap took 4 %
// longer and 2048 tokens alone 14 %), with the weights still to come and the
// caps' parts of the next scores among them.
//
// Measured: 8 x 2048 tokens, 32/8 heads x 128, bfloat16, with a cap 378 us (730
// TFLOP/s; vector operations 68 % of the cycles, matrix unit 38 %, waits 23 %),
// without 308 (890; in fp16 51 %, 51 %, 31 %); chunks in a window 276 us (985 TFLOP/s;
// 1.6 GHz, matrix unit 60 % and LDS 30 % of the cycles); 24 prompts of 52-912
// tokens, 16/16 heads, with a bias and prefixes 56 us (short walks: waits 41 %).
//
// A weight of 0 times a value that is not finite is NaN. So in a stage that
// some row of the tile does not see whole, such values become zeros in LDS, and
// the sums of the rows that do see one become NaN.

#include <algorithm>
#include <type_traits>

#include "scored_core.hpp"

namespace swiftllm {
namespace {

using namespace scored;

struct ScoredPrefillArgs {
    uint16_t* out;           // [T][H][D]
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int* bt;
    const int* ctx;
    const int* qoff;
    Shape shape;             // scale > 0
    unsigned q_and, q_xor;   // on the query's bits, two values each: its sign, or zero
    int S;
    int T;
    int H;
    int Hkv;
    int G;                   // query heads per kv head
    int nhc;                 // chunks of 32 of them
    int gw;                  // heads of a chunk: min(G, 32)
    int tpw;                 // tokens per wave: 32 / gw
    int MB;
    int num_blocks;
    bool q16, out16;         // q, out 16-byte aligned
};

constexpr int kWaves = 4;
constexpr int kStage = 64;             // keys
// Sequences of the longest-first list, whose lengths fit LDS; more go in sequence
// order, by the tiles of each 64 of them (at most 65535, host). Longest first / in
// order, 32/8 heads x 128 unless said: batches that few rounds of workgroups take
// gain by the list, 2 x 2048 tokens 82 / 101 us, 40 of 1-1500 of 8/8 x 64 with a cap
// 108 / 126, 6 chunks of 1000 on up to 8000 435 / 473; those of many tiles, where an
// entry's search costs more than an even end saves, do not, 8 x 2048 320 / 312, 700 of
// 1-60 with a cap 167 / 145, 900 lognormal ones up to 4096 3950 / 3000.
constexpr int kListSeqs = 1024;
constexpr int kCountChunks = 1024;
static_assert(kCountChunks <= kListSeqs && 64 * kCountChunks >= 65535, "their sums take the list's place");
// Tiles of a lane's sequences: memory holds the rows of fewer, and sums over a
// wave stay in range where sequences share rows.
constexpr int kMostTiles = 1 << 24;
constexpr long long kCUs = 256;        // MI355X; any grid is correct
// Workgroups of a CU: as registers allow. (At D = 64 two, not three: 40 ragged
// prompts up to 1500 tokens of 8/8 heads 72 us, not 65.)
template <int D>
constexpr int kPerCU = D == 128 ? 2 : 3;

typedef __attribute__((address_space(3))) s4 lds_s4;

// LDS of one stage, in halves: four K tiles [d][16], then four V tiles in
// operand order. The second K tile of a pair sits 128 bytes off, so that the
// rows an operand read takes from both fall in different banks.
template <int D>
struct Stage {
    static constexpr int kTile = D * kBlockTokens;
    static constexpr int kOdd = kTile + 64;
    static constexpr int kPair = 2 * kTile + 128;
    static constexpr int kK = 2 * kPair;
    static constexpr int kV = 4 * kTile;
};

// A block's tile of one kv head, `off` elements into its cache; with no bytes
// there is nothing to load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const uint16_t* cache, size_t off, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(cache + off), 0, bytes, kRsrcWord3);
}

template <int D>
__device__ __forceinline__ void stage_k(const ScoredPrefillArgs& a, uint16_t* ks, int w, size_t off, int bytes, int lane) {
    const __amdgpu_buffer_rsrc_t rk = tile_rsrc(a.kc, off, bytes);
    uint16_t* const k = ks + (w >> 1) * Stage<D>::kPair + (w & 1) * Stage<D>::kOdd;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, to_lds(k + 512 * i), 16, 16u * lane, 1024u * i, 0, 0);
    }
}

// Each 32-row piece's 16-byte chunks: the rows' first 8 tokens, then their last 8.
template <int D>
__device__ __forceinline__ void stage_v(const ScoredPrefillArgs& a, uint16_t* vs, int w, size_t off, int bytes, int lane) {
    const __amdgpu_buffer_rsrc_t rv = tile_rsrc(a.vc, off, bytes);
    uint16_t* const v = vs + w * Stage<D>::kTile;
    const unsigned vo = 32u * (lane & 31) + 16u * (lane >> 5);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, to_lds(v + 512 * i), 16, vo, 1024u * i, 0, 0);
    }
}

// Row operand of K: 16 rows of a pair of blocks.
__device__ __forceinline__ s8 k_rows(const uint16_t* p) {
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(const_cast<uint16_t*>(p)));
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(const_cast<uint16_t*>(p + 64)));
    return join8(x, y);
}

// S^T of the 32 keys of a stage's pair of blocks.
template <typename T, int D>
__device__ __forceinline__ void qk_pair(f16x& sc, const uint16_t* kl, const s8 (&q)[D / 16]) {
    sc = f16x{};
#pragma unroll
    for (int J = 0; J < D / 16; ++J) {
        sc = T::mfma32(k_rows(kl + 256 * J), q[J], sc);
    }
}

// A sequence's rows and tiles of them.
struct Rows {
    int start, n;
};
__device__ __forceinline__ Rows rows_of(const ScoredPrefillArgs& a, int s) {
    const int b = as_const(a.qoff)[s], e = as_const(a.qoff)[s + 1];
    // Offsets that run backwards or out of the rows have no rows.
    return b >= 0 && e > b && e <= a.T ? Rows{b, e - b} : Rows{0, 0};
}

// The list of (tile, sequence) pairs. A tile's level is about the position of
// its last query over the tokens of a tile: sequence s has tiles at the levels
// first .. first + tiles - 1.
struct ListLds {
    int tiles[kListSeqs];
    int first[kListSeqs];
};
struct List {
    ListLds* lds;   // S > 64
    int S;
    int tiles;      // S <= 64: of sequence `lane`
    int first;
    int top;        // one past the highest level
    __device__ __forceinline__ void get(int s0, int lane, int& n, int& f) const {
        if (S <= 64) {
            n = tiles;
            f = first;
        } else {
            const bool in = s0 + lane < S;
            n = in ? lds->tiles[s0 + lane] : 0;
            f = in ? lds->first[s0 + lane] : 0;
        }
    }
    // Pairs at level i and above.
    __device__ __forceinline__ int count(int i, int lane) const {
        int sum = 0;
        for (int s0 = 0; s0 < S; s0 += 64) {
            int n, f;
            get(s0, lane, n, f);
            sum = min(sum + max(min(n, f + n - i), 0), kMostTiles);
        }
        return wave_total(sum);
    }
    // Entry e, below count(0): highest level first, sequences in order within one.
    __device__ __forceinline__ void entry(int e, int lane, int& tile, int& seq) const {
        int lo = 0, hi = top, below = 0;  // count(lo) > e >= count(hi) = below
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            const int n = count(mid, lane);
            if (n > e) {
                lo = mid;
            } else {
                hi = mid;
                below = n;
            }
        }
        int k = e - below;  // the k-th sequence with a tile at level lo
        for (int s0 = 0;; s0 += 64) {
            int n, f;
            get(s0, lane, n, f);
            const bool has = f <= lo && lo < f + n;
            const unsigned long long mask = __ballot(has);
            const int here = __popcll(mask);
            if (k < here || s0 + 64 >= S) {
                const int rank = __popcll(mask & ((1ull << lane) - 1ull));
                const int at = __ffsll(static_cast<long long>(__ballot(has && rank == k))) - 1;
                seq = max(s0 + at, 0);  // (there is one, unless sequences share rows)
                tile = lo - __builtin_amdgcn_readlane(f, at);
                return;
            }
            k -= here;
        }
    }
};

__device__ __forceinline__ List make_list(const ScoredPrefillArgs& a, int per_wg, ListLds* lds, int* part) {
    List l{lds, a.S, 0, 0, 0};
    const int lane = threadIdx.x & 63;
    const auto tiles_of = [&](int s, int& n, int& f) {
        const Rows r = rows_of(a, s);
        n = (r.n + per_wg - 1) / per_wg;
        f = (max(a.ctx[s], r.n) - r.n) / per_wg;
    };
    if (a.S <= 64) {
        if (lane < a.S) tiles_of(lane, l.tiles, l.first);
        l.top = wave_max(l.tiles > 0 ? l.first + l.tiles : 0);
        return l;
    }
    int most = 0;
    for (int s = threadIdx.x; s < a.S; s += 64 * kWaves) {
        int n, f;
        tiles_of(s, n, f);
        lds->tiles[s] = n;
        lds->first[s] = f;
        most = max(most, n > 0 ? f + n : 0);
    }
    most = wave_max(most);
    if (lane == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) l.top = max(l.top, part[i]);
    return l;
}

// Past kListSeqs: the tiles up to and with every 64 sequences, in lds->first. A
// sequence without rows, wherever its offsets lie, has no tile and changes nothing
// for the others; sums stop above the tiles of any separate rows, so those of
// shared ones do not overflow. (Found from query_offsets[s] / per_wg + s
// by bisection, where one offset out of order hides the tiles of others, 2500
// sequences of 1-30 tokens of 8/2 heads x 64 take 74 us, not 44, 1100 of 1-60 of
// 32/8 x 128 281, not 215.)
constexpr int kMostEntries = (1 << 30) - 1;   // (entries are below it, host)

__device__ __forceinline__ int capped_scan(int x) {
    return dpp_scan(x, 0, [](int a, int b) { return min(a + b, kMostEntries); });
}

__device__ __forceinline__ int tiles_at(const ScoredPrefillArgs& a, int s, int per_wg) {
    return s < a.S ? (rows_of(a, s).n + per_wg - 1) / per_wg : 0;
}

// The number of tiles.
__device__ __forceinline__ int make_counts(const ScoredPrefillArgs& a, int per_wg, ListLds* lds) {
    const int lane = threadIdx.x & 63;
    const int w = threadIdx.x >> 6;
    const int chunks = (a.S + 63) / 64;
    for (int c = w; c < chunks; c += kWaves) {
        const int sum = capped_scan(tiles_at(a, 64 * c + lane, per_wg));
        if (lane == 63) lds->tiles[c] = sum;
    }
    __syncthreads();
    if (w == 0) {
        int before = 0;
        for (int c = 0; c < chunks; c += 64) {
            const int sum = min(capped_scan(c + lane < chunks ? lds->tiles[c + lane] : 0) + before, kMostEntries);
            if (c + lane < chunks) lds->first[c + lane] = sum;
            before = __builtin_amdgcn_readlane(sum, 63);
        }
    }
    __syncthreads();
    return lds->first[chunks - 1];
}

// Entry e, below the number of tiles.
__device__ __forceinline__ void counted_entry(const ScoredPrefillArgs& a, int per_wg, const ListLds* lds, int e, int lane,
                                              int& tile, int& seq) {
    constexpr int kEach = kCountChunks / 64;
    const int last = (a.S + 63) / 64 - 1;
    // The sums ascend: the first above e, among every 16th and then among 16.
    const int g = kEach * __popcll(__ballot(lds->first[min(kEach * lane + kEach - 1, last)] <= e));
    const int c = g + __popcll(__ballot(lane < kEach && lds->first[min(g + lane, last)] <= e));
    const int k = e - (c > 0 ? lds->first[c - 1] : 0);
    const int n = tiles_at(a, 64 * c + lane, per_wg);
    const int upto = capped_scan(n);
    const int at = __popcll(__ballot(upto <= k));
    seq = 64 * c + at;
    tile = k - __builtin_amdgcn_readlane(upto - n, at);
}

// Bits 0 .. n - 1 of 8.
__device__ __forceinline__ unsigned low8(int n) { return (1u << min(max(n, 0), 8)) - 1u; }

// Zeroes the values of the wave's V tile in LDS that are not finite, once its
// loads have landed; which of its 16 keys held one.
template <typename T, int D>
__device__ __forceinline__ unsigned clean_v(uint16_t* vs, int w, int lane) {
    constexpr unsigned kExp = std::is_same<T, F16>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr unsigned kUlp = std::is_same<T, F16>::value ? 0x04000400u : 0x00800080u;
    uint16_t* const p = vs + w * Stage<D>::kTile + 8 * lane;
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const u4 u = *reinterpret_cast<const u4*>(p + 512 * i);
#pragma unroll
        for (int z = 0; z < 4; ++z) bad |= (u[z] & kExp) + kUlp;
    }
    if (!__any((bad & 0x80008000u) != 0)) return 0;
    unsigned mine = 0;
#pragma unroll 1
    for (int i = 0; i < D / 32; ++i) {
#pragma unroll 1
        for (int z = 0; z < 8; ++z) {
            if ((p[512 * i + z] & (kExp & 0xffffu)) == (kExp & 0xffffu)) {
                p[512 * i + z] = 0;
                mine |= 1u << z;
            }
        }
    }
    // Lanes 0 .. 31 hold keys 0 .. 7 of the block, the others 8 .. 15.
    unsigned keys = 0;
    for (int z = 0; z < 8; ++z) {
        const unsigned long long who = __ballot((mine >> z) & 1u);
        keys |= (static_cast<unsigned>(who) != 0 ? 1u << z : 0u) | (static_cast<unsigned>(who >> 32) != 0 ? 256u << z : 0u);
    }
    return keys;
}

// a + the two values of a packed pair.
__device__ __forceinline__ float add_pair(F16, unsigned p, float a) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), v2{1, 1}, a, false);
}
__device__ __forceinline__ float add_pair(BF16, unsigned p, float a) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0x3f803f80u), a, false);
}

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(kPerCU<D>)))
void scored_prefill_kernel(const ScoredPrefillArgs a) {
    constexpr int NJ = D / 16;   // 16-wide k steps of QK^T
    constexpr int ND = D / 32;   // 32-row pieces of the output
    using St = Stage<D>;
    __shared__ int s_part[kWaves];
    __shared__ ListLds s_list;
    __shared__ __align__(16) uint16_t s_k[2][St::kK];
    __shared__ __align__(16) uint16_t s_v[2][St::kV];
    __shared__ __align__(16) unsigned s_bad[2][4];   // keys of a stage's blocks whose values were not finite
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_wg = kWaves * a.tpw;
    const bool listed = a.S <= kListSeqs;
    List list{};
    if (listed) list = make_list(a, per_wg, &s_list, s_part);

    // Workgroups go to the XCDs round-robin, and items are heads-fastest: where
    // the heads are a multiple of 8, an XCD reads the K and V of its own ones.
    const unsigned heads = a.Hkv * a.nhc;
    // (More entries than of separate rows come of sequences that share some.)
    const int most_entries = a.T / per_wg + a.S;
    const int tiles = listed ? list.count(0, threadIdx.x & 63) : make_counts(a, per_wg, &s_list);
    const unsigned entries = max(min(tiles, most_entries), 0);
    const unsigned total = entries * heads;  // below 2^31 (host)
    // Every other round backwards: who had the longest tile gets the shortest.
    auto item_of = [&](unsigned round) {
        return round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    };
    for (unsigned round = 0; item_of(round) < total; ++round) {
    if (round > 0) __syncthreads();  // the stages are free for the next tile
    // (the lane behind an empty asm: kept over the tiles, what follows from it
    // would not leave the walk enough registers)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    // Query row r of the wave in a tile: token r / gw, head r % gw.
    const int r = lane & 31;
    const int h = lane >> 5;
    // K operand: the 16-lane group g4, lane j of it, reads 4 tokens of row
    // j / 4 of its 4-row piece; ds_read_b64_tr_b16 hands lane j the piece's 4
    // rows of one token. Groups 0 and 2 take the pair's first block, 1 and 3
    // its second, groups 2 and 3 the upper 8 of the 16 rows. The tokens of
    // j / 4 = 1 and 2 are exchanged, so the products' rows 8 a + 4 h + c hold
    // the block's tokens 8 h + 4 a + c: a lane's eight scores of a block are
    // then eight consecutive tokens, and its V operand 16 contiguous bytes.
    const int g4 = lane >> 4;
    const int j = lane & 15;
    const int swapped = ((j & 1) << 1) | ((j >> 1) & 1);
    const int koff = (g4 & 1) * St::kOdd + (8 * (g4 >> 1) + (j >> 2)) * kBlockTokens + 4 * swapped;
    const unsigned item = item_of(round);
    const unsigned e = item / heads;
    int tile, s;
    if (listed) {
        list.entry(static_cast<int>(e), lane, tile, s);
    } else {
        counted_entry(a, per_wg, &s_list, static_cast<int>(e), lane, tile, s);
    }
    s = __builtin_amdgcn_readfirstlane(s);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const Rows rows = rows_of(a, s);
    if (tile < 0 || tile * per_wg >= rows.n) continue;  // an entry without a tile
    const int yy = static_cast<int>(item - e * heads);
    const int kvh = yy / a.nhc;
    const int hc = yy - kvh * a.nhc;
    const int ctx = max(as_const(a.ctx)[s], 0);          // (below 0 as 0: no position either way)
    const int L = min(ctx, a.MB * kBlockTokens);
    const int pre = a.shape.prefix != nullptr ? min(max(as_const(a.shape.prefix)[s], 0), L) : 0;
    // A window of every key is the same as none.
    const int window = a.shape.window > 0 ? a.shape.window : 0x7fffffff;
    const int pos0 = ctx - rows.n;                       // of the sequence's first row
    const int rt = r / a.gw;
    const int rh = r - rt * a.gw;
    const int g = hc * 32 + rh;
    const int head = kvh * a.G + min(g, a.G - 1);
    const int i0 = tile * per_wg + w * a.tpw;            // the wave's first row of the sequence
    const bool ok = rt < a.tpw && g < a.G && i0 + rt < rows.n;
    const size_t qrow = (static_cast<size_t>(rows.start) + min(i0 + rt, rows.n - 1)) * a.H + head;
    const int rel = ok ? rt * a.H + head : -1;           // row among the wave's tokens
    const int pos = ok ? pos0 + i0 + rt : -1;            // negative: sees nothing
    const float slope = BIAS ? a.shape.slopes[head] * kLog2e : 0.0f;
    // Positions of the wave's first and last token, and of the tile's.
    const int wp0 = pos0 + i0;
    const int wp1 = pos0 + min(i0 + a.tpw, rows.n) - 1;  // below wp0: it has no token
    const int tp0 = pos0 + tile * per_wg;
    const int tp1 = pos0 + min((tile + 1) * per_wg, rows.n) - 1;
    // Stages: those of the prefix below the window's first, then from there on.
    const int low = max(tp0 - min(window, tp0 + 1) + 1, 0) / kStage;
    const int last = max(min(tp1, L - 1), pre - 1);      // the last key that some row sees
    const int before = min((pre + kStage - 1) / kStage, low);
    const int skip = low - before;
    const int nsteps = tp1 < 0 || last < 0 ? 0 : before + max(last / kStage - low + 1, 0);
    auto stage_of = [&](int t) { return t < before ? t : t + skip; };
    // First keys of the stages that every row of the wave sees whole, none of
    // them ahead of the row where the distance counts: w_span from w0 on, and to w2
    // in the prefix. The same for the tile's rows.
    const bool wave_rows = wp0 >= 0 && wp0 <= wp1;
    const int w0 = max(wp1 - min(window, wp1 + 1) + 1, 0);
    const unsigned w_span = wave_rows ? max(min(wp0, L - 1) - (kStage - 1) - w0 + 1, 0) : 0;
    const int w2 = wave_rows ? (BIAS ? min(pre, wp0 + 1) : pre) - kStage : -1;
    const int last_seen = max(wp1 < wp0 ? -1 : min(wp1, L - 1), pre - 1);
    const int t0 = max(tp1 - min(window, tp1 + 1) + 1, 0);
    const unsigned t_span = tp0 >= 0 ? max(min(tp0, L - 1) - (kStage - 1) - t0 + 1, 0) : 0;
    const int t2 = tp0 >= 0 ? pre - kStage : -1;

    // (zeros behind an empty asm: 16 of them would be kept over the tiles)
    float zero = 0.0f;
    asm volatile("" : "+v"(zero));
    f16x acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) {
#pragma unroll
        for (int z = 0; z < 16; ++z) acc[i][z] = zero;
    }
    float m = -INFINITY, l = 0.0f;
    if (nsteps > 0) {
    const int nblk = (L + kBlockTokens - 1) >> kBlockShift;
    const int* const row = a.bt + static_cast<size_t>(s) * a.MB;
    // Ids of 16 stages of the walk, four lanes each.
    auto chunk_ids = [&](int c) { return row[min(4 * stage_of(16 * c + (lane >> 2)) + (lane & 3), nblk - 1)]; };
    const int ids_first = chunk_ids(0);
    int ids_next = chunk_ids(1);
    // Q^T operand: lane (r, h) holds q[r][16 J + 8 h .. + 7].
    s8 q[NJ];
    {
        const uint16_t* p = a.q + qrow * D + 8 * h;
        const unsigned keep = ok ? a.q_and : 0u;
        const unsigned flip = ok ? a.q_xor : 0u;
#pragma unroll
        for (int J = 0; J < NJ; ++J) {
            u4 v;
            if (a.q16) {
                v = *reinterpret_cast<const u4*>(p + 16 * J);
            } else {
                v = __builtin_bit_cast(u4, join8(*reinterpret_cast<const s4*>(p + 16 * J),
                                                 *reinterpret_cast<const s4*>(p + 16 * J + 4)));
            }
            q[J] = __builtin_bit_cast(s8, (v & keep) ^ flip);
        }
    }
    // The chunk at hand, unknown blocks as block 0 and their bits in `known` clear.
    int ids;
    unsigned long long known;
    auto take_chunk = [&](int x) {
        const bool k = block_known(x, a.num_blocks);
        known = __ballot(k);
        ids = k ? x : 0;
    };
    take_chunk(ids_first);
    // Tile of this wave in stage t of the walk (16 stages per load of ids) and,
    // in ok4, which of the stage's four blocks are in the pool.
    auto tile_of = [&](int t, int& ok4) {
        const int at = 4 * (t & 15);
        ok4 = static_cast<int>((known >> at) & 15ull);
        return kv_tile_offset(__builtin_amdgcn_readlane(ids, at + w), kvh, a.Hkv, D);
    };
    auto bytes_of = [&](int t) { return t < nsteps ? D * kBlockTokens * 2 : 0; };
    // This wave's block of stage t of the walk has landed in its V buffer: true
    // if some row of the tile may not see the stage whole.
    auto landed = [&](int t, int ok4) {
        const int base = kStage * stage_of(t);
        if (t >= nsteps || (ok4 == 15 && (static_cast<unsigned>(base - t0) < t_span || base <= t2))) return false;
        const unsigned bad = clean_v<T, D>(s_v[t & 1], w, lane);
        if (lane == 0) s_bad[t & 1][w] = bad;
        return true;
    };
    int ok_t, ok_1;                  // of stages t and t + 1
    const size_t off = tile_of(0, ok_t);
    stage_k<D>(a, s_k[0], w, off, bytes_of(0), lane);
    stage_v<D>(a, s_v[0], w, off, bytes_of(0), lane);
    size_t off_1 = tile_of(1, ok_1);
    stage_k<D>(a, s_k[1], w, off_1, bytes_of(1), lane);
    wait_vm<0>();
    bool cleaned = landed(0, ok_t);  // stage t
    __syncthreads();
    f16x sc[2];
    qk_pair<T, D>(sc[0], s_k[0] + koff, q);
    qk_pair<T, D>(sc[1], s_k[0] + koff + St::kPair, q);
    __syncthreads();
    const float scale = a.shape.scale;
    const float cap = a.shape.cap;
    auto cap_part = [&](float x) { return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * scale) + 1.0f); };
    // Without a bias what scores are made of keeps its place: they are it times
    // mul, plus add. They fall as a cap's part grows.
    constexpr float kHidden = CAP && !BIAS ? INFINITY : -INFINITY;
    const float mul = CAP ? -2.0f * cap : scale;
    const float add = CAP ? cap : 0.0f;
    float rise[16];   // of the bias over a pair's scores
#pragma unroll
    for (int i = 0; i < 16; ++i) rise[i] = BIAS ? slope * static_cast<float>(16 * (i >> 3) + (i & 7)) : 0.0f;
    auto most = [](float x, float y) { return CAP && !BIAS ? fminf(x, y) : fmaxf(x, y); };
    if constexpr (CAP) {
#pragma unroll
        for (int i = 0; i < 32; ++i) sc[i >> 4][i & 15] = cap_part(sc[i >> 4][i & 15]);
    }
    for (int t = 0; t < nsteps; ++t) {
        int ok_2;
        stage_v<D>(a, s_v[(t + 1) & 1], w, off_1, bytes_of(t + 1), lane);
        off_1 = tile_of(t + 2, ok_2);
        stage_k<D>(a, s_k[t & 1], w, off_1, bytes_of(t + 2), lane);
        const int base = kStage * stage_of(t);
        // (The walk's stages behind the wave's last row are hidden from it.)
        if (base <= last_seen) {
        // (One copy of the stage with scalar branches: two copies, with and without
        // masks, took 100 more registers for the sums that they hand each other.)
        const bool whole = ok_t == 15 && (static_cast<unsigned>(base - w0) < w_span || base <= w2);
        // Score i of pair p: key base + 32 p + 16 (i / 8) + 8 h + i % 8; bit
        // 16 p + i of `seen` whether this row sees it.
        unsigned seen = ~0u;
        if (!whole) {
            const int first = base + 8 * h;
            const int to = min(pos, L - 1) - first + 1;         // keys first + [from, to) are seen,
            const int from = pos - min(window, pos + 1) + 1 - first;
            const int prefix = pos < 0 ? 0 : pre - first;       // and those before first + prefix
            seen = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const unsigned bits = (low8(to - 16 * b) & ~low8(from - 16 * b)) | low8(prefix - 16 * b);
                if ((ok_t >> b) & 1) seen |= bits << (8 * b);
            }
        }
        // What a pair's scores lack: in a whole stage the bias of its first key.
        float lack[2] = {add, add};
        if constexpr (BIAS) {
            // Scores in the place of what they are made of: key i lies d0 + off from
            // the row, and d0 + off <= 0 in a whole stage.
            const float d0 = static_cast<float>(base + 8 * h - pos);
            if (whole) {
                lack[0] = __builtin_fmaf(slope, d0, add);
                lack[1] = __builtin_fmaf(slope, d0 + 32.0f, add);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    sc[i >> 4][i & 15] = __builtin_fmaf(sc[i >> 4][i & 15], mul, rise[i & 15]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float bias = -slope * __builtin_fabsf(d0 + static_cast<float>(16 * (i >> 3) + (i & 7)));
                    sc[i >> 4][i & 15] = __builtin_fmaf(sc[i >> 4][i & 15], mul, bias);
                }
            }
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int keep = __builtin_amdgcn_sbfe(static_cast<int>(seen), i, 1);  // 0 or -1
                const float x = sc[i >> 4][i & 15];   // (a bit cast of the element itself takes element 0)
                const int v = __builtin_bit_cast(int, x);
                sc[i >> 4][i & 15] = __builtin_bit_cast(float, (v & keep) | (__builtin_bit_cast(int, kHidden) & ~keep));
            }
        }
        auto most_of = [&](const f16x& x) {
            float y = most(most(x[0], x[1]), x[2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) y = most(most(y, x[i]), x[i + 1]);
            return most(y, x[15]);
        };
        float bm;
        if constexpr (BIAS) {
            bm = fmaxf(most_of(sc[0]) + lack[0], most_of(sc[1]) + lack[1]);
        } else {
            bm = __builtin_fmaf(most(most_of(sc[0]), most_of(sc[1])), mul, add);
        }
        {
            const auto y = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, bm), __builtin_bit_cast(unsigned, bm), false, false);
            bm = fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(y[0])), __builtin_bit_cast(float, static_cast<unsigned>(y[1])));
        }
        if (__any(bm > m + kLag)) {
            const float m_new = fmaxf(m, bm);
            const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= alpha;
            l *= alpha;
            m = m_new;
        }
        const float c = ((m == -INFINITY) ? 0.0f : m) - weight_exp<T>;
        const float lack_c[2] = {lack[0] - c, lack[1] - c};
        if (cleaned) {
            const u4 bad = *reinterpret_cast<const u4*>(s_bad[t & 1]);
            unsigned keys = 0;   // this lane's, as `seen`
#pragma unroll
            for (int b = 0; b < 4; ++b) keys |= ((bad[b] >> (8 * h)) & 0xffu) << (8 * b);
            if (seen & keys) l = __builtin_nanf("");
        }
        // Weights, O^T += V P^T, and the next stage's scores in the place of those
        // that are used up, in a fixed order. (Behind the last stage the scores are
        // not used.)
        const uint16_t* const next = s_k[(t + 1) & 1] + koff;
        const uint16_t* const vl = s_v[t & 1] + 8 * lane;
        u4 pw[4];
        auto weights = [&](int k) {   // the k-th pair of them
            const int b = k >> 2, i = k & 3;
            float p[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const float v = sc[b >> 1][8 * (b & 1) + 2 * i + z];
                p[z] = __builtin_amdgcn_exp2f(BIAS ? v + lack_c[b >> 1] : __builtin_fmaf(v, mul, lack_c[0]));
            }
            pw[b][i] = T::down2(p[0], p[1]);
            l = add_pair(T{}, pw[b][i], l);
        };
        constexpr int kScores = 2 * ND, kBack = 2 * ND + 2 * NJ, kProducts = 4 * ND + 2 * NJ;
        constexpr int kAhead = 2;
        auto operand = [&](int n) {
            if (n >= kScores && n < kBack) {
                const int k = n - kScores;
                return k_rows(next + k / NJ * St::kPair + 256 * (k % NJ));
            }
            const int k = n < kScores ? n : n - 2 * NJ;
            return *reinterpret_cast<const s8*>(vl + k / ND * St::kTile + 512 * (k % ND));
        };
        s8 ring[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) ring[n] = operand(n);
#pragma unroll
        for (int k = 0; k < 4; ++k) weights(k);
        __builtin_amdgcn_sched_barrier(0);
        // A wave in its products goes ahead of one between them: 8 x 2048 with a bias
        // 336 us, not 348, with a cap 368, not 377; at D = 64 without a cap 54, not
        // 57, but with one 71, not 67.
        constexpr bool kAheadOf = D == 128 || !CAP;
        if constexpr (kAheadOf) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int n = 0; n < kProducts; ++n) {
            const s8 x = ring[n % kAhead];
            if (n + kAhead < kProducts) ring[n % kAhead] = operand(n + kAhead);
            if (n >= kScores && n < kBack) {
                const int k = n - kScores;
                sc[k / NJ] = T::mfma32(x, q[k % NJ], k % NJ == 0 ? f16x{} : sc[k / NJ]);
            } else {
                const int k = n < kScores ? n : n - 2 * NJ;
                acc[k % ND] = T::mfma32(x, __builtin_bit_cast(s8, pw[k / ND]), acc[k % ND]);
            }
            if (n < kScores) {
#pragma unroll
                for (int i = 4 + n * 4 / ND; i < 4 + (n + 1) * 4 / ND; ++i) weights(i);
            } else if (n < kScores + 4) {
                weights(12 + n - kScores);
            } else if (CAP && n >= kScores + NJ) {
                constexpr int kSlots = 2 * ND + NJ;
                const int k = n - kScores - NJ;
#pragma unroll
                for (int i = k * 32 / kSlots; i < (k + 1) * 32 / kSlots; ++i) sc[i >> 4][i & 15] = cap_part(sc[i >> 4][i & 15]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (kAheadOf) __builtin_amdgcn_s_setprio(0);
        }
        wait_vm<0>();
        cleaned = landed(t + 1, ok_1);
        ok_t = ok_1;
        ok_1 = ok_2;
        if (((t + 3) & 15) == 0) {
            take_chunk(ids_next);
            ids_next = chunk_ids(((t + 3) >> 4) + 1);
        }
        __syncthreads();
    }
    }

    // The wave's output rows, through its quarter of the K buffers (every
    // wave's last scores are made): chunk c (8 values) of row r at chunk
    // c ^ (r % (D / 8)), so that neither side conflicts, and back as whole rows,
    // D / 8 lanes each.
    {
        int ln = lane;
        asm volatile("" : "+v"(ln));   // nothing of it in registers through the walk
        const int er = ln & 31, eh = ln >> 5;
        const auto y = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, l), __builtin_bit_cast(unsigned, l), false, false);
        const float sum = __builtin_bit_cast(float, static_cast<unsigned>(y[0])) + __builtin_bit_cast(float, static_cast<unsigned>(y[1]));
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        constexpr int kChunks = D / 8;
        uint16_t* const o_lds = &s_k[0][0] + w * 32 * D;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u2 o = u2{T::down2(acc[i][4 * k] * inv, acc[i][4 * k + 1] * inv),
                                T::down2(acc[i][4 * k + 2] * inv, acc[i][4 * k + 3] * inv)};
                *reinterpret_cast<u2*>(o_lds + er * D + 8 * ((4 * i + k) ^ (er & (kChunks - 1))) + 4 * eh) = o;
            }
        }
        uint16_t* const op = a.out + (static_cast<size_t>(rows.start) + i0) * a.H * D + 8 * (ln & (kChunks - 1));
        int to[D / 16];
        u4 v[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int from = (64 / kChunks) * i + ln / kChunks;
            to[i] = __shfl(rel, from);
            v[i] = *reinterpret_cast<const u4*>(o_lds + from * D + 8 * ((ln ^ from) & (kChunks - 1)));
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            if (to[i] < 0) continue;
            uint16_t* const o = op + static_cast<size_t>(to[i]) * D;
            if (a.out16) {
                __builtin_nontemporal_store(v[i], reinterpret_cast<u4*>(o));
            } else {
                *reinterpret_cast<u2*>(o) = u2{v[i][0], v[i][1]};
                *reinterpret_cast<u2*>(o + 4) = u2{v[i][2], v[i][3]};
            }
        }
    }
    }
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

int swiftllm_hip_scored_prefill(void* output, const void* query, const void* key_cache, const void* value_cache,
                                const int32_t* block_tables, const int32_t* context_lens,
                                const int32_t* query_offsets, const float* alibi_slopes, const int32_t* prefix_lens,
                                float scale, float softcap, int window, int dtype, int num_tokens, int num_seqs,
                                int num_heads, int num_kv_heads, int head_dim, int block_size,
                                int max_num_blocks_per_seq, int num_blocks, hipStream_t stream) {
    const char* who = "swiftllm_hip_scored_prefill";
    const long long T = num_tokens, S = num_seqs, H = num_heads, Hkv = num_kv_heads, D = head_dim;
    const long long MB = max_num_blocks_per_seq;
    if (T < 0 || S < 0 || H <= 0 || Hkv <= 0 || D <= 0 || block_size <= 0 || MB < 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER,
                    "%s: num_tokens=%lld num_seqs=%lld num_heads=%lld num_kv_heads=%lld head_dim=%lld block_size=%d "
                    "max_num_blocks_per_seq=%lld", who, T, S, H, Hkv, D, block_size, MB);
    }
    if (H % Hkv != 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_heads %lld not a multiple of num_kv_heads %lld", who, H, Hkv);
    }
    if ((D != 64 && D != 128) || block_size != kBlockTokens) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: head_dim=%lld block_size=%d (supported: 64/128, 16)", who, D, block_size);
    }
    if (dtype != SWIFTLLM_HIP_F16 && dtype != SWIFTLLM_HIP_BF16) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: dtype=%d (supported: 0 fp16, 1 bf16)", who, dtype);
    }
    if (S > 65535 || H > 65535 || T >= (1LL << 30) || MB >= (1 << 26)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_tokens=%lld num_seqs=%lld num_heads=%lld max_num_blocks_per_seq=%lld",
                    who, T, S, H, MB);
    }
    ScoredPrefillArgs a{};
    if (!scored::make_shape(a.shape, std::fabs(scale), softcap, window, prefix_lens, alibi_slopes)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: scale=%g softcap=%g window=%d", who, scale, softcap, window);
    }
    if (softcap > scored::kMostCap) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: softcap=%g (at most %g)", who, softcap, scored::kMostCap);
    }
    if (T > 0 && S > 0 && (!output || !query || !key_cache || !value_cache || !context_lens || !query_offsets ||
                           (MB > 0 && !block_tables))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    if (!aligned(output, 8) || !aligned(query, 8) || !aligned(key_cache, 16) || !aligned(value_cache, 16) ||
        !aligned(block_tables, 4) || !aligned(context_lens, 4) || !aligned(query_offsets, 4) ||
        !aligned(alibi_slopes, 4) || !aligned(prefix_lens, 4)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    a.S = num_seqs;
    a.T = num_tokens;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.G = num_heads / num_kv_heads;
    a.nhc = (a.G + 31) / 32;
    a.gw = std::min(a.G, 32);
    a.tpw = 32 / a.gw;
    const long long heads = Hkv * a.nhc;
    const long long items = (T / (kWaves * a.tpw) + S) * heads;
    if (items >= (1LL << 30)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_tokens=%lld of %lld kv heads", who, T, Hkv);
    }
    // A wave has read its queries before it writes their rows; rows of others, and
    // what every workgroup reads, must not be among them.
    if (T > 0 && S > 0) {
        const size_t n = num_seqs;
        const Bytes out{output, static_cast<size_t>(T) * H * D * 2}, q{query, out.n};
        const Bytes kc{key_cache, cache_bytes(num_blocks, Hkv, D)}, vc{value_cache, kc.n};
        const Bytes bt{block_tables, 4 * n * max_num_blocks_per_seq}, ctx{context_lens, 4 * n};
        const Bytes off{query_offsets, 4 * (n + 1)}, pre{prefix_lens, 4 * n};
        const Bytes slopes{alibi_slopes, 4 * static_cast<size_t>(H)};
        if ((output != query && overlap_any(out, {q})) || overlap_any(out, {kc, vc, bt, ctx, off, pre, slopes})) {
            return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: output overlaps another argument", who);
        }
    }
    const int rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    if (T == 0 || S == 0) return ok();
    // The sign of the scale goes into the query, and a scale of zero makes it
    // zero: the kernel's scale is positive, so that raw products order as scores.
    // (Of products of zero any finite one does; 1 / softcap may be none.)
    a.q_and = scale == 0.0f ? 0u : 0xffffffffu;
    a.q_xor = scale < 0.0f ? 0x80008000u : 0u;
    if (scale == 0.0f) a.shape.scale = 1.0f;
    a.out = static_cast<uint16_t*>(output);
    a.q = static_cast<const uint16_t*>(query);
    a.kc = static_cast<const uint16_t*>(key_cache);
    a.vc = static_cast<const uint16_t*>(value_cache);
    a.bt = block_tables;
    a.ctx = context_lens;
    a.qoff = query_offsets;
    a.MB = max_num_blocks_per_seq;
    a.num_blocks = num_blocks;
    a.q16 = aligned(query, 16);
    a.out16 = aligned(output, 16);
    // A list in registers is made in no time, so up to four tiles per resident
    // workgroup each have one of their own, which goes where another ended; a longer
    // list is made once per resident workgroup. Four / one: 8 x 2048 tokens with a cap
    // 378 / 388 us, 40 ragged prompts of 8/8 heads x 64 with a cap 71 / 75, 700 of 1-60
    // tokens 190 / 159. (One for every tile that num_tokens has room for: 2000 tokens
    // in 65536 rows 33.5 us, not 17.6.)
    const long long resident = (S <= 64 ? 4 : 1) * kCUs * (D == 128 ? kPerCU<128> : kPerCU<64>);
    const long long grid = (std::min(items, resident) + 7) / 8 * 8;
    using K = void (*)(ScoredPrefillArgs);
#define SCORED_PREFILL(T_) \
    {{{scored_prefill_kernel<T_, 64, false, false>, scored_prefill_kernel<T_, 64, false, true>}, \
      {scored_prefill_kernel<T_, 64, true, false>, scored_prefill_kernel<T_, 64, true, true>}}, \
     {{scored_prefill_kernel<T_, 128, false, false>, scored_prefill_kernel<T_, 128, false, true>}, \
      {scored_prefill_kernel<T_, 128, true, false>, scored_prefill_kernel<T_, 128, true, true>}}}
    static const K kernels[2][2][2][2] = {SCORED_PREFILL(F16), SCORED_PREFILL(BF16)};
#undef SCORED_PREFILL
    return launched(launch(kernels[dtype == SWIFTLLM_HIP_BF16][D == 128][softcap > 0.0f][alibi_slopes != nullptr],
                           dim3(static_cast<unsigned>(grid)), dim3(64 * kWaves), 0, stream, a),
                    who);
}

}  // extern "C"
