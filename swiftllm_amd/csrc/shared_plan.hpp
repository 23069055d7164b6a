// The plan of attention over shared blocks: what swiftllm_hip_plan_shared writes
// (shared_plan.hip) and swiftllm_hip_shared_decode reads (shared_decode.hip).
//
// The work of a step is a list of walks: of a group's shared blocks by the queries
// of up to `per_tile` of its sequences, and of each sequence's other blocks by its
// own. Shared ones of more than 16 query rows are wide, a workgroup's, and
// have a list of their own; the others are narrow, a wave's. Both lists are cut into equal
// ranges of their costs, one per workgroup and chunk of heads; of what is narrow each
// wave has a quarter of one. (With one list for both, the range in which the wide ones
// end takes longest.) Every piece of a walk that does not end its rows leaves one
// fragment (maximum, sum, output) a row; those of a walk lie behind each other from row
// `frow` on.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace swiftllm {
namespace shared {

constexpr int kMagic = 0x53484152;
constexpr int kWaveRows = 32;       // query rows of a wave of a wide walk: tokens x heads
constexpr int kTileWaves = 4;
constexpr int kTileRows = kWaveRows * kTileWaves;
constexpr int kNarrowRows = 16;

// Blocks that starting and ending a walk costs. (16 and 4 or 8 are no faster.)
constexpr int kWideCost = 8;
constexpr int kNarrowCost = 2;
// Workgroups the list is cut for: two for each of the 256 CUs of an MI355X, whose
// LDS their rings of steps take.
constexpr int kResident = 2 * 256;
// Shortest range, in blocks.
constexpr int kLeastRange = 16;
// Blocks of a group that reading shared ones once has to save, and values of a head of
// all of them (blocks x chunks of heads x head_dim): below, the second launch and its
// joins cost what is saved. (4 beams on 1000 tokens, 8 kv heads x 128: 12.0 us a layer
// shared, 11.6 not; 16 x 8 beams on 2500 tokens 50.5 shared, 153 by scored_decode.)
constexpr int kLeastSaved = 16;
constexpr long long kLeastSavedAll = 2500 * 128;

struct Walk {
    int row;        // whose table names the blocks
    int first;      // its first block,
    int blocks;     //   and how many
    int seq;        // the first of its sequences
    int count;      //   and how many: more than one shares
    int at;         // its first block's place in its list
    int once;       // no other walk reads its blocks
    int frow;       // its first fragment, in rows of a chunk of heads; -1: one piece that ends its row
};

// Where a range begins: a walk, and its number.
struct Start {
    Walk walk;
    int v;
    int pad[7];
};

struct Head {
    int magic, S, MB, heads, kv_heads, head_dim;
    int wide;       // walks
    int walks;      //   in all
    int wide_end;   // of the wide walks' costs,
    int narrow_end; //   and of the narrow ones'
    int wide_len;   // of a range of the wide walks
    int narrow_len; // and of one of the narrow, of which a wave has a quarter
    int wide_ranges;
    int pad[3];
};

struct Seq {
    int L;          // keys: its context, as far as its table goes
    int own;        // its walk, -1: none
    int tile;       // the walk of its shared blocks, -1: none
    int index;      // its place in that one
};

// The range of `len` that a wide walk's block at a place of the list lies in; and the
// wave, counted over ranges, that a narrow walk's does: wave r's begin at r len / 4.
__device__ __forceinline__ int wide_range(int place, int len) { return place / len; }
__device__ __forceinline__ int narrow_range(int place, int len) {
    return static_cast<int>((kTileWaves * static_cast<unsigned>(place) + kTileWaves - 1) / static_cast<unsigned>(len));
}
__device__ __forceinline__ int narrow_begin(int range, int len) {
    return static_cast<int>(static_cast<unsigned>(range) * static_cast<unsigned>(len) / kTileWaves);
}
__device__ __forceinline__ int pieces_of(bool wide, int at, int blocks, int len) {
    return wide ? wide_range(at + blocks - 1, len) - wide_range(at, len) + 1
                : narrow_range(at + blocks - 1, len) - narrow_range(at, len) + 1;
}

// How the heads of a kv head lie in a wave's rows.
struct Heads {
    int G, nhc, gw, tpw, per_tile, HC;
};
inline Heads heads_of(int H, int Hkv) {
    Heads h;
    h.G = H / Hkv;
    h.nhc = (h.G + kWaveRows - 1) / kWaveRows;
    h.gw = std::min(h.G, kWaveRows);
    h.tpw = kWaveRows / h.gw;
    h.per_tile = h.tpw * kTileWaves;
    h.HC = Hkv * h.nhc;
    return h;
}

struct Layout {
    int ranges;
    size_t wide_starts, narrow_starts, walks, seqs, infos, costs, bytes;
    long long rows;        // fragments of a chunk of heads, at most
};

// Walks: one per sequence and, of those that share, one per tile, which has two of
// them at least. Rows: a walk has one piece and one more for every end of a range in
// it, of at most a tile's rows or, at a wave's, a sequence's heads.
inline Layout layout_of(long long S, int H, int Hkv) {
    const auto up = [](long long n) { return static_cast<size_t>((n + 255) / 256 * 256); };
    const Heads h = heads_of(H, Hkv);
    Layout l;
    l.ranges = std::max(kResident / h.HC, 2);     // (what is wide and what is narrow have ranges of their own)
    l.wide_starts = 256;
    l.narrow_starts = l.wide_starts + up(static_cast<long long>(sizeof(Start)) * l.ranges);
    l.walks = l.narrow_starts + up(static_cast<long long>(sizeof(Start)) * l.ranges * kTileWaves);
    l.seqs = l.walks + up(static_cast<long long>(sizeof(Walk)) * (2 * S + 1));
    l.infos = l.seqs + up(static_cast<long long>(sizeof(Seq)) * S);
    l.costs = l.infos + up(16 * S);
    l.bytes = l.costs + up(32 * S);
    l.rows = 2 * S * h.gw + static_cast<long long>(l.ranges) * (kTileRows + kTileWaves * std::max(h.gw, kNarrowRows));
    return l;
}

int check_sizes(const char* who, long long S, long long H, long long Hkv, long long D, long long BS, long long MB);

}  // namespace shared
}  // namespace swiftllm
