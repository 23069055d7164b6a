// Runs of new tokens into the [num_blocks, num_kv_heads, head_dim, 16] cache:
// the part of the cache write that does not depend on where a token's row
// comes from (a copy in reshape_and_cache, a rotation in rotary_and_cache).
#pragma once

#include "common.hpp"

namespace swiftllm {
namespace cache {

// Each store is 2 bytes of a 32-byte tile row, so the memory system merges
// it into the row (a read-modify-write below the caches). Nontemporal stores
// do that inside this kernel. Cached stores leave partly dirty lines that are
// written back while the next kernel (the decode) streams the pool, and
// writes mixed into that read stream cost it more than this kernel's own
// time (config 4: 21 us here and no decode slowdown, against 9 us here and
// 10-17 us added to the decode).
__device__ __forceinline__ void put(uint16_t* p, uint16_t v) {
    __builtin_nontemporal_store(v, p);
}

// ---------------------------------------------------------------------------
// Runs of tokens (block size 16).
//
// Bound: HBM, one read of the new K/V and one write of the blocks. Column
// stores write a row's 32 bytes in 16 partial writes, each a
// read-modify-write below the caches: 16384 prompt tokens of 8 x 128 took
// 506 us (0.27 TB/s) token by token and take 21.8 us (6.2 TB/s) in runs; 600
// tokens 21.2 -> 3.9 us.
//
// A workgroup owns the runs whose first token lies in its window of W tokens,
// for 256 rows of K or of V: 16 x 512 bytes in, 8 KiB of whole lines out. The
// small piece keeps a short call parallel (a 256-token decode step is 512
// workgroups) and a long one at several workgroups per CU. Runs are cut at
// block ends only, never at a window's, so a full block is always one piece,
// wherever a prompt starts in the batch.
// ---------------------------------------------------------------------------
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4v;
typedef unsigned u4v __attribute__((ext_vector_type(4)));

constexpr int kWinRows = 256;                  // rows (h, d) of K or V per workgroup
constexpr int kWinStride = kWinRows + 16;      // halves per token in LDS (544 bytes)

// The slice of kWinRows rows from row0 of the runs of window t0, by a
// workgroup of 256 threads. W: tokens whose runs a workgroup owns, at most 16
// (one lane of 32 looks at each of the W + 15 tokens those runs can span).
// tile: (W + 15) * kWinStride halves of LDS. n: rows of a block. src gives the
// slot of token t (negative: none), and of row0's slice of it the 8 values
// from c or the one at i; before(k) comes ahead of the 8 values of token t0 + k,
// with every lane active.
template <int W, typename Src>
__device__ __forceinline__ void write_runs(const Src& src, uint16_t* const cache, uint16_t* const tile, int t0,
                                           int row0, int n, int T, long long num_slots) {
    constexpr int kMax = W + kBlockTokens - 1;
    constexpr int kLoads = (kMax + 7) / 8;     // 16-byte loads per lane, 8 tokens each
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // Lane i classifies token t0 + i: a valid token continues the run of the
    // token before it when its slot is the next one of the same block, else
    // it is a run's head.
    const int t = t0 + lane;
    int slot = -1, prev = -1;
    if (lane <= kMax && t < T) {
        slot = src.slot(t);
        if (t > 0) prev = src.slot(t - 1);
    }
    const bool valid = slot >= 0 && (num_slots <= 0 || slot < num_slots);
    const bool cont = valid && (slot & (kBlockTokens - 1)) != 0 && prev == slot - 1;
    const unsigned conts = static_cast<unsigned>(__ballot(cont));
    unsigned heads = static_cast<unsigned>(__ballot(valid && !cont)) & ((1u << W) - 1u);
    if (heads == 0) return;  // the same in every wave
    if ((conts & (heads << 1)) == 0) {
        // Every head is a lone token (a decode step): one column each, lanes
        // on consecutive rows as in the token kernel, all loads first.
        if (row0 + tid >= n) return;
        uint16_t v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = src.one(min(t0 + i, T - 1), tid);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if ((heads >> i) & 1u) {
                const int s = __builtin_amdgcn_readlane(slot, i);
                put(cache + (static_cast<size_t>(s >> kBlockShift) * n + row0 + tid) * kBlockTokens +
                        (s & (kBlockTokens - 1)),
                    v[i]);
            }
        }
        return;
    }
    const int first = __builtin_ctz(heads);
    const int last = 31 - __builtin_clz(heads);
    // A run never passes its block's end, so it has at most 16 tokens and
    // lane last + 16 <= W + 15 does not continue it.
    const int end = last + 1 + __builtin_ctz(~(conts >> (last + 1)));

    // Tokens first .. end - 1 of the window into LDS, [token][row].
    const int c = (tid & 31) * 8;
    u4v buf[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int k = first + 8 * i + (tid >> 5);
        src.before(k);
        if (k < end && row0 + c < n) {
            buf[i] = src.eight(t0 + k, c);
        }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int k = 8 * i + (tid >> 5);
        if (first + k < end) *reinterpret_cast<u4v*>(tile + k * kWinStride + c) = buf[i];
    }
    __syncthreads();

    const int r = lane & 15;
    const int kg = lane >> 4;
    for (; heads != 0; heads &= heads - 1) {
        const int i = __builtin_ctz(heads);
        const int len = 1 + __builtin_ctz(~(conts >> (i + 1)));
        const int s = __builtin_amdgcn_readlane(slot, i);
        const int o = s & (kBlockTokens - 1);
        uint16_t* const dst = cache + (static_cast<size_t>(s >> kBlockShift) * n + row0) * kBlockTokens;
        const uint16_t* const from = tile + (i - first) * kWinStride;
        if (len == 1) {
            // One column: lanes on consecutive rows (see the token kernel).
            if (row0 + tid < n) put(dst + tid * kBlockTokens + o, from[tid]);
            continue;
        }
        // Lane (r, kg) takes tokens 4 kg .. 4 kg + 3 of row r of each group
        // of 16 rows: ds_read_b64_tr_b16 hands lane i of 16 the element i % 4
        // of lanes i / 4, + 4, + 8 and + 12, so those lanes read 4 rows each
        // of 4 tokens. Columns outside the run read some staged token.
        const int col = 4 * kg + (r >> 2) - o;
        const uint16_t* const mine =
            from + min(max(col, 0), len - 1) * kWinStride + 4 * (r & 3);
        const int lo = max(o - 4 * kg, 0), hi = min(o + len - 4 * kg, 4);
#pragma unroll
        for (int g = 0; g < kWinRows / 64; ++g) {
            const int rg = 16 * (4 * g + w);
            if (row0 + rg >= n) break;
            const s4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s4v*)(const_cast<uint16_t*>(mine) + rg));
            uint16_t* const p = dst + (rg + r) * kBlockTokens + 4 * kg;
            if (lo <= 0 && hi >= 4) {
                __builtin_nontemporal_store(v, reinterpret_cast<s4v*>(p));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j >= lo && j < hi) put(p + j, static_cast<uint16_t>(v[j]));
                }
            }
        }
    }
}

// Up to here a call is a decode step or a few short prompts, and windows of 4
// tokens keep enough workgroups: 64 lone tokens of 8 x 128 take 4.5-5.1 us in
// windows of 4 and 6.4 us in windows of 16 (5.3 us token by token), 256 take
// 9.2 and 10.0 (9.5). Past it windows of 16 leave fewer workgroups that find
// no head: 1024 lone tokens take 29.0 us with them (29.6 token by token).
// A layer of few rows leaves few workgroups at any window, and short runs pay
// for it, one after the other in a window: up to kSmallPieces tokens times
// slices of 256 rows it keeps windows of 4. Measured in runs of 2 tokens,
// windows of 4 / 16 (token by token): 513 tokens of 2 x 128 5.4 / 9.8 (6.2),
// of 1 x 128 4.0 / 6.8 (4.7), 1024 of 2 x 128 6.8 / 9.9 (9.1), 2048 12.5 / 12.2
// (15.6); in one run 1024 of 2 x 128 3.8 / 4.0, of 8 x 64 4.4 / 3.9.
constexpr int kSmallTokens = 512;
constexpr long long kSmallPieces = 1024;

inline bool small_windows(long long tokens, long long slices) {
    return tokens <= kSmallTokens || tokens * slices <= kSmallPieces;
}

}  // namespace cache
}  // namespace swiftllm
