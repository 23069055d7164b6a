// The plan of attention over shared blocks: what swiftllm_hip_plan_shared writes
// (shared_plan.hip) and swiftllm_hip_shared_decode reads (shared_decode.hip).
//
// The work of a step is a list of walks: of a group's shared blocks by the queries
// of up to `per_tile` of its sequences, and of each sequence's other blocks by its
// own. The list is cut into equal ranges of its cost, one per workgroup and chunk
// of heads, and a piece of a walk that its rows are not done with leaves one
// fragment (maximum, sum, output) a row. Fragments of a walk lie behind each other,
// from row `frow` on.
#pragma once

#include <algorithm>

#include "common.hpp"

namespace swiftllm {
namespace shared {

constexpr int kMagic = 0x53484152;
constexpr int kWaveRows = 32;       // query rows of a wave: tokens x heads
constexpr int kTileWaves = 4;
constexpr int kTileRows = kWaveRows * kTileWaves;

// Blocks that starting and ending a walk costs, and one that a tile's rows cost beside.
constexpr int kWalkCost = 4;
// Workgroups the list is cut for: two for each of the 256 CUs of an MI355X, as the
// tiles' registers allow.
constexpr int kResident = 2 * 256;
// Shortest range, in blocks: a stage and what a walk costs.
constexpr int kLeastRange = 8;
// Blocks that reading shared ones once has to save.
constexpr int kLeastSaved = 16;

struct Head {
    int magic, S, MB, heads, kv_heads, head_dim;
    int walks;      // in the list
    int total;      // its cost
    int len;        // of a range
    int rows;       // fragments
    int pad[6];
};

struct Walk {
    int row;        // whose table names the blocks
    int first;      // its first block,
    int blocks;     //   and how many
    int seq;        // the first of its sequences
    int count;      //   and how many: more than one shares
    int begin;      // in the list
    int cost;
    int frow;       // its first fragment, in rows of a chunk of heads; -1: one piece that is done
};

struct Seq {
    int L;          // keys: its context, as far as its table goes
    int own;        // its walk, -1: none
    int tile;       // the walk of its shared blocks, -1: none
    int index;      // its place in that one
};

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
    int most_walks;
    size_t walks, starts, seqs, infos, costs, bytes;
    long long rows;        // fragments of a chunk of heads, at most
};

// Walks: one per sequence and, of those that share, one per tile, which has two of
// them at least. Rows: each walk has at most as many pieces as ranges touch it, and
// all of them together at most `ranges` more than there are walks.
inline Layout layout_of(long long S, int H, int Hkv) {
    const auto up = [](long long n) { return static_cast<size_t>((n + 255) / 256 * 256); };
    const Heads h = heads_of(H, Hkv);
    Layout l;
    l.ranges = std::max(kResident / h.HC, 1);
    l.most_walks = static_cast<int>(2 * S);
    l.walks = 256;
    l.starts = l.walks + up(static_cast<long long>(sizeof(Walk)) * l.most_walks);
    l.seqs = l.starts + up(4LL * l.ranges);
    l.infos = l.seqs + up(static_cast<long long>(sizeof(Seq)) * S);
    l.costs = l.infos + up(16 * S);
    l.bytes = l.costs + up(8 * S);
    l.rows = 2 * S * h.gw + l.ranges * static_cast<long long>(kTileRows + h.gw);
    return l;
}

int check_sizes(const char* who, long long S, long long H, long long Hkv, long long D, long long BS, long long MB);

}  // namespace shared
}  // namespace swiftllm
