// Paged attention of one new token per sequence over blocks that sequences share
// (gfx950), with a soft cap and a distance bias (scored_core.hpp): what
// scored_decode computes, each group's shared blocks read once for all of its
// sequences. The query of sequence s is its last token, at position L_s - 1.
//
// softmax over all keys in parts: a walk over the keys [j0, j1) leaves, for every
// query row, m = max score, l = sum exp2(score - m) and o = sum exp2(score - m) v / l;
// rows are joined as sum of exp2(m - M) l o over sum of exp2(m - M) l.
//
// Work. The plan's lists (shared_plan.hpp) are cut into ranges, one workgroup per
// range and chunk of heads. A wide walk's rows are the query heads of up to
// 4 x 32 / gw sequences, gw = min(G, 32) heads each, 32 rows to a wave; its K and V
// go through LDS, a ring of four steps of 32 keys, of which two to three are on the
// way while one is used (loads the compiler does not see, counted by hand: with its
// own waits it let one be), and the products are S^T = K Q^T, O^T = V P^T, 32x32x16,
// as in scored_prefill. A narrow walk, of at most 16 rows or of one sequence, is one
// wave's as in scored_decode (scored_walk.hpp): no wave waits for another, and eight
// of them a CU keep 128 KB on the way. (One sequence's own blocks by a whole workgroup
// through LDS: 128 chats of 1-1000 own tokens behind 8192 shared ones, 32/8 heads x
// 128, 87 us a layer, not 82; 16 x 8 beams 73, not 62.)
//
// Bound: HBM, one read of the shared K and V for each tile of 128 rows and one of
// every sequence's own. At 4.92 TB/s, what a large copy reaches: 16 x 8 beams on 1000
// to 4000 tokens, 32/8 heads x 128 in bfloat16 with a cap, 44.0 us of reads, 51.3 in
// all; the 128 chats 58.1 and 67.5 (tiles share L2 for what they read); 4 x 16
// questions on 30000 tokens, 64/8 heads, with distance biases 137 and 138. What is left
// over is a range's start (its walk, ids, queries, a first step: 2.5 us), the ranges'
// unequal ends and the second launch, 4 us. One walk of 128 rows on 131072 tokens takes
// 121 us (117, and with 64 keys a step and two of them 132, with the compiler's waits
// 159, before the few other blocks had a range of their own).

#include <algorithm>
#include <cmath>

#include "scored_tiles.hpp"
#include "scored_walk.hpp"
#include "shared_plan.hpp"

namespace swiftllm {
namespace {

using namespace scored;
using namespace shared;

struct SharedArgs {
    uint16_t* out;           // [rows][H][D]
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int* bt;
    const int* qoff;         // [S + 1] or null: row s
    const Head* head;
    const Walk* walks;
    const Start* wide;
    const Start* narrow;
    const Seq* seqs;
    float2* frag_ml;         // [HC][rows]
    float* frag_o;           // [HC][rows][D]
    long long frag_rows;
    Shape shape;             // scale > 0
    unsigned q_and, q_xor;   // on the query's bits, two values each: its sign, or zero
    int T;                   // rows, where qoff is given
    int S, H, Hkv, D;
    int G;                   // query heads per kv head
    int nhc;                 // chunks of gw of them
    int gw;
    int tpw;                 // sequences of a wave's rows
    int MB;
    int num_blocks;
    bool q16, out8;          // q 16-byte, out 8-byte aligned
};

constexpr int kWaves = kTileWaves;

// The row of a sequence's query and output; negative: it has none.
__device__ __forceinline__ int row_of(const SharedArgs& a, int s) {
    if (a.qoff == nullptr) return s;
    const int b = as_const(a.qoff)[s], e = as_const(a.qoff)[s + 1];
    return b >= 0 && e > b && e <= a.T ? e - 1 : -1;
}

// Whether the plan was made for these sizes: what it names lies inside the arguments.
__device__ __forceinline__ bool plan_fits(const SharedArgs& a) {
    const const_int* const h = as_const(reinterpret_cast<const int*>(a.head));
    return h[0] == kMagic && h[1] == a.S && h[2] == a.MB && h[3] == a.H && h[4] == a.Hkv && h[5] == a.D;
}

__device__ __forceinline__ Walk walk_at(const Walk* p) {
    const const_int* const x = as_const(reinterpret_cast<const int*>(p));
    return Walk{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
}

// Four outputs of a row.
template <typename T>
__device__ __forceinline__ void put_out(uint16_t* p, f4 o, bool out8) {
    u2 x = u2{T::down2(o[0], o[1]), T::down2(o[2], o[3])};
    asm volatile("" : "+v"(x));     // rounded once, the same for any address
    if (out8) {
        *reinterpret_cast<u2*>(p) = x;
    } else {
        p[0] = x[0] & 0xffffu;
        p[1] = x[0] >> 16;
        p[2] = x[1] & 0xffffu;
        p[3] = x[1] >> 16;
    }
}

// A wave's walk for 16 query rows: blocks i0, i0 + STEP .. below i1 of the walk, for
// the heads hb .. hb + 15 of its chunk. Lane (r, kg) has query row r: sequence r / gn,
// head hb + r % gn, gn of them at hand.
template <int D>
struct Rows {
    State<D> st;
    int qrow, hd;
    int place;       // among the rows of the walk
    bool row, ok;    // there is a row for it, and a query in it
};

template <typename T, int D, bool BIAS, int STEP>
__device__ __forceinline__ void narrow_walk(const SharedArgs& a, const Walk& walk, int kvh, int hc, int hb, int i0, int i1, int lane, Rows<D>& o) {
    constexpr int NJ = D / 16;
    const int r = lane & 15;
    const int kg = lane >> 4;
    const int gn = min(a.gw - hb, kNarrowRows);
    const int rt = r / gn;
    const int rh = hb + r - rt * gn;
    const int g = hc * kWaveRows + rh;
    const int s = walk.seq + min(rt, walk.count - 1);
    const Seq sq = a.seqs[s];
    o.hd = kvh * a.G + min(g, a.G - 1);
    o.qrow = row_of(a, s);
    o.place = rt * a.gw + rh;
    o.row = rt < walk.count;
    o.ok = o.row && g < a.G && sq.L > 0 && o.qrow >= 0;
    State<D>& st = o.st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int J = 0; J < NJ; ++J) st.acc[J] = f4{0, 0, 0, 0};
    const int count = i1 > i0 ? (i1 - i0 + STEP - 1) / STEP : 0;
    if (count == 0) return;
    const int* const ids_of = a.bt + static_cast<size_t>(walk.row) * a.MB + walk.first;
    // Lane l has the id of the wave's block 64 c + l.
    auto ids_from = [&](int c) { return ids_of[min(i0 + STEP * (64 * c + lane), i1 - 1)]; };
    int ids = ids_from(0);
    s8 q[NJ / 2];
    const uint16_t* const qp = a.q + (static_cast<size_t>(max(o.qrow, 0)) * a.H + o.hd) * D + 4 * kg;
    const unsigned keep = o.ok ? a.q_and : 0u, flip = o.ok ? a.q_xor : 0u;
#pragma unroll
    for (int J = 0; J < NJ; J += 2) {
        const s8 x = join8(*reinterpret_cast<const s4*>(qp + 16 * J), *reinterpret_cast<const s4*>(qp + 16 * J + 16));
        q[J / 2] = __builtin_bit_cast(s8, (__builtin_bit_cast(u4, x) & keep) ^ flip);
    }
    const float slope = BIAS && o.ok ? a.shape.slopes[o.hd] * kLog2e : 0.0f;
    s4 ident;
#pragma unroll
    for (int i = 0; i < 4; ++i) ident[i] = 4 * kg + i == r ? static_cast<short>(T::one()) : 0;
    const int loff = kv_elem_offset(r, 4 * kg);
    // The keys of an own walk end with its sequence; shared blocks are seen whole.
    const int L = __builtin_amdgcn_readfirstlane(walk.count > 1 ? 0x7fffffff : sq.L);
    auto load = [&](int k, s4 (&kk)[NJ], s4 (&vv)[NJ], int& base, unsigned& seen) {
        if (k > 0 && (k & 63) == 0) ids = ids_from(k >> 6);
        const int b = __builtin_amdgcn_readlane(ids, k & 63);
        const bool known = block_known(b, a.num_blocks);
        base = (walk.first + i0 + STEP * k) * kBlockTokens;
        seen = known ? low_bits(L - base) : 0u;
        // A block outside the pool is read as block 0 and hidden.
        const size_t tile = kv_tile_offset(known ? b : 0, kvh, a.Hkv, D) + loff;
#pragma unroll
        for (int J = 0; J < NJ; ++J) kk[J] = load4(a.kc + tile + kv_elem_offset(16 * J, 0));
#pragma unroll
        for (int J = 0; J < NJ; ++J) vv[J] = load4(a.vc + tile + kv_elem_offset(16 * J, 0));
    };
    const int last = sq.L - 1;      // the position that a bias's distances are from
    auto take = [&](s4 (&kk)[NJ], s4 (&vv)[NJ], int base, unsigned seen) {
        attend<T, D>(st, seen, base - last, kg, kk, vv, q, ident, a.shape, slope);
    };
    // Two blocks in flight; no load of the loop depends on a condition.
    s4 kA[NJ], vA[NJ], kB[NJ], vB[NJ];
    int bA, bB;
    unsigned sA, sB;
    load(0, kA, vA, bA, sA);
    int k = 0;
    for (; k + 2 < count; k += 2) {
        load(k + 1, kB, vB, bB, sB);
        take(kA, vA, bA, sA);
        load(k + 2, kA, vA, bA, sA);
        take(kB, vB, bB, sB);
    }
    if (k + 1 < count) {
        load(k + 1, kB, vB, bB, sB);
        take(kA, vA, bA, sA);
        take(kB, vB, bB, sB);
    } else {
        take(kA, vA, bA, sA);
    }
}

// Blocks i0 .. i1 - 1 of a narrow walk, by one wave.
template <typename T, int D, bool BIAS>
__device__ __forceinline__ void narrow_piece(const SharedArgs& a, const Walk& walk, int kvh, int hc, int hb, int i0, int i1, int range, int len, int lane) {
    constexpr int NJ = D / 16;
    const int kg = lane >> 4;
    Rows<D> o;
    narrow_walk<T, D, BIAS, 1>(a, walk, kvh, hc, hb, i0, i1, lane, o);
    const float sum = sum_over_groups(o.st.l);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (walk.frow < 0) {
        if (!o.ok) return;
        uint16_t* const p = a.out + (static_cast<size_t>(o.qrow) * a.H + o.hd) * D + 4 * kg;
#pragma unroll
        for (int J = 0; J < NJ; ++J) put_out<T>(p + 16 * J, o.st.acc[J] * inv, a.out8);
    } else if (o.row) {
        const long long f = static_cast<long long>(blockIdx.x) * a.frag_rows + walk.frow +
                            static_cast<long long>(range - narrow_range(walk.at, len)) * walk.count * a.gw + o.place;
        if (kg == 0) a.frag_ml[f] = float2{o.st.m, sum};
        float* const p = a.frag_o + f * D + 4 * kg;
#pragma unroll
        for (int J = 0; J < NJ; ++J) *reinterpret_cast<f4*>(p + 16 * J) = o.st.acc[J] * inv;
    }
}

// Every sequence whole, in one launch: a workgroup per sequence and 16 heads of a
// chunk, its waves take the blocks in turn.
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(64 * kWaves) void shared_whole_kernel(const SharedArgs a) {
    constexpr int NJ = D / 16;
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    __shared__ __align__(16) float s_o[kWaves][16][D];
    if (!plan_fits(a)) return;
    const int s = blockIdx.y;
    const int parts = (a.gw + kNarrowRows - 1) / kNarrowRows;
    const int hb = static_cast<int>(blockIdx.x) % parts * kNarrowRows;
    const int sub = blockIdx.x / parts;
    const int kvh = sub / a.nhc;
    const int hc = sub - kvh * a.nhc;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int L = as_const(reinterpret_cast<const int*>(a.seqs + s))[0];
    const int row = row_of(a, s);
    if (row < 0) return;
    const int blocks = (L + kBlockTokens - 1) >> kBlockShift;
    const Walk walk{s, 0, blocks, s, 1, 0, 1, -1};
    Rows<D> o;
    narrow_walk<T, D, BIAS, kWaves>(a, walk, kvh, hc, hb, w, blocks, lane, o);
    const int r = lane & 15, kg = lane >> 4;
    const float l = sum_over_groups(o.st.l);
    if (kg == 0) {
        s_m[w][r] = o.st.m;
        s_l[w][r] = l;
    }
#pragma unroll
    for (int J = 0; J < NJ; ++J) *reinterpret_cast<f4*>(&s_o[w][r][16 * J + 4 * kg]) = o.st.acc[J];
    __syncthreads();
    const int heads = min(min(a.gw - hb, kNarrowRows), a.G - hc * kWaveRows - hb);
    for (int i = tid; i < heads * (D / 4); i += 64 * kWaves) {
        const int g = i / (D / 4);
        const int d = 4 * (i - g * (D / 4));
        float m = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) m = fmaxf(m, s_m[x][g]);
        f4 num = f4{0, 0, 0, 0};
        float den = 0.0f;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            // A wave that saw no key has zeros; one of NaN scores alone a NaN sum.
            const float f = s_m[x][g] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s_m[x][g] - m);
            num += f * *reinterpret_cast<const f4*>(&s_o[x][g][d]);
            den += f * s_l[x][g];
        }
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        const int hd = kvh * a.G + hc * kWaveRows + hb + g;
        put_out<T>(a.out + (static_cast<size_t>(row) * a.H + hd) * D + d, num * inv, a.out8);
    }
}

// The ring of steps, two blocks each, that a workgroup's loads fill ahead of its
// products.
constexpr int kRing = 4;

// 16 bytes a lane, from byte v + s of the buffer to LDS from m0 on, lanes side by
// side. In assembly, so that the compiler does not wait for all of them before any
// read of LDS: every read of what they bring comes behind wait_vm and a barrier.
// There is no register that they write; m0 holds nothing of the compiler's from one
// instruction to the next. once: what no other walk reads streams past the caches
// (8 x 32 rows on 16384 tokens, 32/8 heads x 128, 106 us, not 126; four tiles on the
// same 8192 tokens so 80, not 74).
__device__ __forceinline__ void load_lds16(u4 rsrc, unsigned lds, unsigned v, unsigned s, bool once) {
    if (once) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds" ::"s"(lds), "v"(v), "s"(rsrc), "s"(s)
                     : "memory");
    } else {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(v), "s"(rsrc), "s"(s)
                     : "memory");
    }
}

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
void shared_decode_kernel(const SharedArgs a) {
    constexpr int NJ = D / 16;   // 16-wide k steps of QK^T
    constexpr int ND = D / 32;   // 32-row pieces of the output
    using St = Stage<D>;
    constexpr int kStep = St::kPair + 2 * St::kTile;     // halves of a step: two blocks' K, then their V
    __shared__ __align__(16) uint16_t s_ring[kRing * kStep];
    __shared__ unsigned s_bad[kRing][2];                 // keys of a step's blocks whose values were not finite
    const const_int* const head = as_const(reinterpret_cast<const int*>(a.head));
    const int wide = head[6], walks = head[7], wide_end = head[8], narrow_end = head[9], len = head[10], narrow_len = head[11];
    const int wide_ranges = head[12];
    if (!plan_fits(a)) return;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kvh = blockIdx.x / a.nhc;
    const int hc = blockIdx.x - kvh * a.nhc;
    if (static_cast<int>(blockIdx.y) < wide_ranges) {
    const int start = blockIdx.y * len;
    const int end = min(start + len, wide_end);
    auto k_of = [&](int t) { return s_ring + (t & (kRing - 1)) * kStep; };
    auto v_of = [&](int t) { return k_of(t) + St::kPair; };
    const Start* const s0 = a.wide + blockIdx.y;
    Walk walk = walk_at(&s0->walk);
    int v = as_const(&s0->v)[0];
    for (;;) {
        // This range's blocks of the walk: i0 .. i1 - 1.
        const int i0 = max(start - walk.at, 0);
        const int i1 = min(end - walk.at, walk.blocks);
        const Walk next = ++v < wide ? walk_at(a.walks + v) : walk;
        if (i0 < i1) {
        // (the lane behind an empty asm: kept over the walks, what follows from it
        // would not leave them enough registers)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int r = lane & 31;
        const int h = lane >> 5;
        // K operand, as in scored_prefill: a lane's eight scores of a block are of
        // eight consecutive tokens.
        const int g4 = lane >> 4;
        const int j = lane & 15;
        const int swapped = ((j & 1) << 1) | ((j >> 1) & 1);
        const int koff = (g4 & 1) * St::kOdd + (8 * (g4 >> 1) + (j >> 2)) * kBlockTokens + 4 * swapped;
        const int first = walk.first, seq = walk.seq, count = walk.count;
        // Query row r of the wave: sequence r / gw, head r % gw.
        const int rt = r / a.gw;
        const int rh = r - rt * a.gw;
        const int g = hc * kWaveRows + rh;
        const int hd = kvh * a.G + min(g, a.G - 1);
        const int place = w * a.tpw + rt;
        const int s = seq + min(place, count - 1);
        const Seq sq = a.seqs[s];
        const int qrow = row_of(a, s);
        const bool ok = rt < a.tpw && place < count && g < a.G && sq.L > 0 && qrow >= 0;
        const bool works = __any(ok);
        const float slope = BIAS ? a.shape.slopes[hd] * kLog2e : 0.0f;
        const int* const ids_of = a.bt + static_cast<size_t>(walk.row) * a.MB + first;
        const int nsteps = (i1 - i0 + 1) >> 1;
        // Ids of a step's blocks, by scalar loads a step ahead of their use.
        auto ids_at = [&](int t) {
            return int2{as_const(ids_of)[min(i0 + 2 * t, i1 - 1)], as_const(ids_of)[min(i0 + 2 * t + 1, i1 - 1)]};
        };
        // Waves 0 and 1 load a step's K, a block each, the others its V. Which of its
        // blocks there are goes into `there`, two bits a step of the ring; others are
        // read as block 0 and hidden. (Behind the last step there is nothing to load.)
        const int mine = w & 1;
        const bool is_k = w < 2;
        const uint16_t* const cache = is_k ? a.kc : a.vc;
        const unsigned lane_at = is_k ? 16u * lane : 32u * (lane & 31) + 16u * (lane >> 5);
        const unsigned lds_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>(to_lds(
            s_ring + (is_k ? mine * St::kOdd : St::kPair + mine * St::kTile))));
        unsigned there = 0;
        auto fetch = [&](int t, int2 ids) {
            const int slot = t & (kRing - 1);
            const bool k0 = block_known(ids.x, a.num_blocks) && i0 + 2 * t < i1;
            const bool k1 = block_known(ids.y, a.num_blocks) && i0 + 2 * t + 1 < i1;
            there = (there & ~(3u << (2 * slot))) | (k0 ? 1u << (2 * slot) : 0u) | (k1 ? 2u << (2 * slot) : 0u);
            const int id = mine ? (k1 ? ids.y : 0) : (k0 ? ids.x : 0);
            const uintptr_t p = reinterpret_cast<uintptr_t>(cache + kv_tile_offset(id, kvh, a.Hkv, D));
            const u4 rsrc = u4{static_cast<unsigned>(p), static_cast<unsigned>(p >> 32) & 0xffffu,
                               t < nsteps ? D * kBlockTokens * 2u : 0u, static_cast<unsigned>(kRsrcWord3)};
            const unsigned lds = lds_at + slot * 2 * kStep;
            if (walk.once) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) load_lds16(rsrc, lds + 1024u * i, lane_at, 1024u * i, true);
            } else {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) load_lds16(rsrc, lds + 1024u * i, lane_at, 1024u * i, false);
            }
        };
#pragma unroll
        for (int t = 0; t < kRing - 1; ++t) fetch(t, ids_at(t));
        int2 ahead = ids_at(kRing - 1);
        // Q^T operand: lane (r, h) holds q[r][16 J + 8 h .. + 7].
        s8 q[NJ];
        {
            const uint16_t* p = a.q + (static_cast<size_t>(max(qrow, 0)) * a.H + hd) * D + 8 * h;
            const unsigned keep = ok ? a.q_and : 0u;
            const unsigned flip = ok ? a.q_xor : 0u;
#pragma unroll
            for (int J = 0; J < NJ; ++J) {
                u4 x;
                if (a.q16) {
                    x = *reinterpret_cast<const u4*>(p + 16 * J);
                } else {
                    x = __builtin_bit_cast(u4, join8(*reinterpret_cast<const s4*>(p + 16 * J),
                                                     *reinterpret_cast<const s4*>(p + 16 * J + 4)));
                }
                q[J] = __builtin_bit_cast(s8, (x & keep) ^ flip);
            }
        }
        f16x acc[ND];
        float zero = 0.0f;
        asm volatile("" : "+v"(zero));
#pragma unroll
        for (int i = 0; i < ND; ++i) {
#pragma unroll
            for (int z = 0; z < 16; ++z) acc[i][z] = zero;
        }
        float m = -INFINITY, l = 0.0f;
        const float scale = a.shape.scale;
        const float cap = a.shape.cap;
        // Scores are what is made of them times mul, plus add; with a cap they fall as
        // its part grows.
        constexpr float kHidden = CAP && !BIAS ? INFINITY : -INFINITY;
        const float mul = CAP ? -2.0f * cap : scale;
        const float add = CAP ? cap : 0.0f;
        auto most = [](float x, float y) { return CAP && !BIAS ? fminf(x, y) : fmaxf(x, y); };
        wait_vm<0>();      // (with the queries' loads the count of the ring's is not known)
        for (int t = 0; t < nsteps; ++t) {
            // This wave's part of step t is there: those of the next two may be on
            // their way.
            wait_vm<2 * (D / 32)>();
            const unsigned here = (there >> (2 * (t & (kRing - 1)))) & 3u;
            if (here != 3u && !is_k) {
                const unsigned bad = clean_v<T, D>(v_of(t), mine, lane);
                if (lane == 0) s_bad[t & (kRing - 1)][mine] = bad;
            }
            __syncthreads();   // and everybody's, and step t - 1 is done with
            const uint16_t* const kl = k_of(t) + koff;
            const uint16_t* const vl = v_of(t) + 8 * lane;
            // Operands are read all at once, and the next loads asked for meanwhile.
            s8 op[NJ];
#pragma unroll
            for (int J = 0; J < NJ; ++J) op[J] = k_rows(kl + 256 * J);
            __builtin_amdgcn_sched_barrier(0);
            fetch(t + kRing - 1, ahead);
            ahead = ids_at(t + kRing);
            if (!works) continue;
            // Score i: key base + 16 (i / 8) + 8 h + i % 8 of the step.
            f16x sc = f16x{};
#pragma unroll
            for (int J = 0; J < NJ; ++J) sc = T::mfma32(op[J], q[J], sc);
            __builtin_amdgcn_sched_barrier(0);
            s8 val[2 * ND];
#pragma unroll
            for (int k = 0; k < 2 * ND; ++k) val[k] = *reinterpret_cast<const s8*>(vl + k / ND * St::kTile + 512 * (k % ND));
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (CAP) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(sc[i] * scale) + 1.0f);
            }
            // What a score lacks: the bias of the step's first key.
            float lack = add;
            if constexpr (BIAS) {
                const int base = (first + i0 + 2 * t) * kBlockTokens;
                lack = __builtin_fmaf(slope, static_cast<float>(base + 8 * h - (sq.L - 1)), add);
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = __builtin_fmaf(sc[i], mul, slope * static_cast<float>(16 * (i >> 3) + (i & 7)));
            }
            if (here != 3u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (!((here >> (i >> 3)) & 1u)) sc[i] = kHidden;
                }
            }
            float bm = most(most(sc[0], sc[1]), sc[2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) bm = most(most(bm, sc[i]), sc[i + 1]);
            bm = most(bm, sc[15]);
            bm = BIAS ? bm + lack : __builtin_fmaf(bm, mul, add);
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
            const float lack_c = lack - (((m == -INFINITY) ? 0.0f : m) - weight_exp<T>);
            if (here != 3u) {
                const unsigned* const bad = s_bad[t & (kRing - 1)];
                const unsigned keys = ((here & 1u) ? (bad[0] >> (8 * h)) & 0xffu : 0u) | ((here & 2u) ? (bad[1] >> (8 * h)) & 0xffu : 0u);
                if (keys) l = __builtin_nanf("");
            }
            // A weight is rounded to the type, as in scored_prefill, and its sum is of the
            // rounded ones. The second part that a wave's walk keeps of it would be as many
            // products again: us a pass with one and with two, 16 x 8 beams with a cap 216 and
            // 217, 128 chats 287 and 305, 4 x 16 questions with biases 284 and 330, for errors
            // against 64 bits of 1.85e-3 and 1.66e-3 (bfloat16), 2.30e-4 and 2.08e-4 (fp16), of
            // which the output's own rounding is all but the difference.
            u4 pw[2];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float p[2];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float x = sc[2 * k + z];
                    p[z] = __builtin_amdgcn_exp2f(BIAS ? x + lack_c : __builtin_fmaf(x, mul, lack_c));
                }
                const unsigned both = T::down2(p[0], p[1]);
                pw[k >> 2][k & 3] = both;
                l = add_pair(T{}, both, l);
            }
#pragma unroll
            for (int k = 0; k < 2 * ND; ++k) {
                acc[k % ND] = T::mfma32(val[k], __builtin_bit_cast(s8, pw[k / ND]), acc[k % ND]);
            }
        }
        wait_vm<0>();
        // The rows' fragments: they share, and go on. Lane (r, h) has values
        // 32 i + 8 k + 4 h .. + 3 of row r.
        if (rt < a.tpw && place < count) {
            const auto y = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, l), __builtin_bit_cast(unsigned, l), false, false);
            const float sum = __builtin_bit_cast(float, static_cast<unsigned>(y[0])) + __builtin_bit_cast(float, static_cast<unsigned>(y[1]));
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const long long f = static_cast<long long>(blockIdx.x) * a.frag_rows + walk.frow +
                                static_cast<long long>(static_cast<int>(blockIdx.y) - wide_range(walk.at, len)) * count * a.gw + place * a.gw + rh;
            if (h == 0) a.frag_ml[f] = float2{m, sum};
            float* const p = a.frag_o + f * D + 4 * h;
#pragma unroll
            for (int i = 0; i < ND; ++i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    *reinterpret_cast<f4*>(p + 32 * i + 8 * k) =
                        f4{acc[i][4 * k] * inv, acc[i][4 * k + 1] * inv, acc[i][4 * k + 2] * inv, acc[i][4 * k + 3] * inv};
                }
            }
        }
        __syncthreads();       // the ring is free
        }
        if (v >= wide || next.at - kWideCost >= end) break;
        walk = next;
    }
    return;
    }
    // This wave's part of what is narrow.
    const int range = kWaves * (static_cast<int>(blockIdx.y) - wide_ranges) + w;
    const int b = narrow_begin(range, narrow_len), e = min(narrow_begin(range + 1, narrow_len), narrow_end);
    if (b >= narrow_end) return;
    const Start* const s0 = a.narrow + range;
    Walk walk = walk_at(&s0->walk);
    int v = as_const(&s0->v)[0];
    for (;;) {
        const int i0 = max(b - walk.at, 0);
        const int i1 = min(e - walk.at, walk.blocks);
        const Walk next = ++v < walks ? walk_at(a.walks + v) : walk;
        if (i0 < i1) {
            for (int hb = 0; hb < a.gw; hb += kNarrowRows) {
                int lane = threadIdx.x & 63;
                asm volatile("" : "+v"(lane));
                narrow_piece<T, D, BIAS>(a, walk, kvh, hc, hb, i0, i1, range, narrow_len, lane);
            }
        }
        if (v >= walks || next.at - kNarrowCost >= e) break;
        walk = next;
    }
}

// Joins the fragments of a sequence's rows: WAVES waves a query head, which take them
// in turn. A lane holds the maximum and the sum of a fragment, and the first rows are
// on their way before those are there: a join is bound by latency.
constexpr int kJoinRows = 8;
constexpr int kJoinWaves = 4;       // of a workgroup
// Rows below which four waves join one. (us a layer of 32/8 heads x 128, with one wave
// and with four: 4 beams on 1000 tokens 13.0 and 11.7, 4 x 4 on 8192 41.6 and 37.8,
// 32 on 32768 47.4 and 45.6; 16 x 4 on 600 25.2 and 26.7, 16 x 8 on 2500 50.3 and 55.8.)
constexpr int kFewRows = 2048;

// Tables and bytes of K and V up to which every sequence is taken whole. (us a layer of
// 2 x 4 beams, 8 heads x 64, in two launches and in one: 15 blocks each 9.2 and 5.6,
// 38 blocks 9.3 and 7.8; they meet at about 48.)
constexpr int kMostWhole = 48;
constexpr double kWholeBytes = 64e6;

template <typename T, int D, int WAVES>
__global__ __launch_bounds__(64 * kJoinWaves) void shared_join_kernel(const SharedArgs a) {
    constexpr int DL = D / 64;
    constexpr int kHeads = kJoinWaves / WAVES;
    __shared__ float s_o[WAVES > 1 ? kJoinWaves : 1][D];
    __shared__ float s_ml[WAVES > 1 ? kJoinWaves : 1][2];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = blockIdx.y * kHeads + w / WAVES;
    const int turn = w % WAVES;
    if (hd >= a.H || !plan_fits(a)) return;      // (with several waves a head, one head a workgroup)
    const int s = blockIdx.x;
    const const_int* const sq = as_const(reinterpret_cast<const int*>(a.seqs + s));
    const int own = sq[1], tile = sq[2], index = sq[3];
    const int kvh = hd / a.G;
    const int hg = hd - kvh * a.G;
    const int hc = hg / kWaveRows;
    const int rh = hg - hc * kWaveRows;
    // Fragments 0 .. n0 - 1 are of the shared blocks, the others of its own.
    int n0 = 0, n1 = 0, f0 = 0, f1 = 0, step = 0;
    const const_int* const head = as_const(reinterpret_cast<const int*>(a.head));
    auto pieces = [&](const Walk& x, int v) {
        return pieces_of(v < head[6], x.at, x.blocks, v < head[6] ? head[10] : head[11]);
    };
    if (tile >= 0) {
        const Walk x = walk_at(a.walks + tile);
        step = x.count * a.gw;
        n0 = pieces(x, tile);
        f0 = x.frow + index * a.gw + rh;
    }
    if (own >= 0) {
        const Walk x = walk_at(a.walks + own);
        if (x.frow < 0) return;      // its row is written
        n1 = pieces(x, own);
        f1 = x.frow + rh;
    }
    const long long sub = static_cast<long long>(kvh * a.nhc + hc) * a.frag_rows;
    // This wave's i-th fragment.
    const int count = max((n0 + n1 - turn + WAVES - 1) / WAVES, 0);
    auto place = [&](int i) {
        const int x = turn + WAVES * i;
        return sub + (x < n0 ? f0 + x * step : f1 + (x - n0) * a.gw);
    };
    float m = -INFINITY, l = 0.0f, o[DL];
#pragma unroll
    for (int j = 0; j < DL; ++j) o[j] = 0.0f;
    for (int c = 0; c < count; c += 64) {
        const int n = min(count - c, 64);
        float v[kJoinRows][DL];
        auto rows = [&](int i) {
#pragma unroll
            for (int k = 0; k < kJoinRows; ++k) {
                if (i + k >= n) break;
                const float* const p = a.frag_o + place(c + i + k) * D + lane * DL;
#pragma unroll
                for (int j = 0; j < DL; ++j) v[k][j] = p[j];
            }
        };
        rows(0);
        const float2 ml = a.frag_ml[place(c + min(lane, n - 1))];
        const float fm = lane < n ? ml.x : -INFINITY;
        const float fl = lane < n ? ml.y : 0.0f;
        const float top = fmaxf(m, wave_max(fm));
        const float keep = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        // An empty fragment has a sum of 0; one of NaN scores alone has NaN.
        const float weight = (fm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(fm - top)) * fl;
        l = l * keep + wave_sum(weight);
#pragma unroll
        for (int j = 0; j < DL; ++j) o[j] *= keep;
        m = top;
        for (int i = 0; i < n; i += kJoinRows) {
            if (i > 0) rows(i);
#pragma unroll
            for (int k = 0; k < kJoinRows; ++k) {
                const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), (i + k) & 63));
                if (i + k < n) {
#pragma unroll
                    for (int j = 0; j < DL; ++j) o[j] += x * v[k][j];
                }
            }
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int j = 0; j < DL; ++j) s_o[w][lane * DL + j] = o[j];
        if (lane == 0) {
            s_ml[w][0] = m;
            s_ml[w][1] = l;
        }
        __syncthreads();
        if (turn > 0) return;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) m = fmaxf(m, s_ml[x][0]);
#pragma unroll
        for (int j = 0; j < DL; ++j) o[j] = 0.0f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) {
            const float f = s_ml[x][0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s_ml[x][0] - m);
            l += f * s_ml[x][1];
#pragma unroll
            for (int j = 0; j < DL; ++j) o[j] += f * s_o[x][lane * DL + j];
        }
    }
    const int row = row_of(a, s);
    if (row < 0) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* const p = a.out + (static_cast<size_t>(row) * a.H + hd) * D + lane * DL;
#pragma unroll
    for (int j = 0; j < DL; ++j) p[j] = T::down(o[j] * inv);
}

struct Space {
    size_t o, bytes;
};
Space space_of(const Layout& l, int HC, int D) {
    const auto up = [](long long n) { return static_cast<size_t>((n + 255) / 256 * 256); };
    Space s;
    s.o = up(8LL * l.rows * HC);
    s.bytes = s.o + up(4LL * l.rows * HC * D);
    return s;
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

size_t swiftllm_hip_shared_decode_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                 int block_size, int max_num_blocks_per_seq) {
    if (shared::check_sizes("swiftllm_hip_shared_decode_workspace_size", num_seqs, num_heads, num_kv_heads, head_dim,
                            block_size, max_num_blocks_per_seq) != SWIFTLLM_OK) {
        return 0;
    }
    ok();
    return space_of(shared::layout_of(num_seqs, num_heads, num_kv_heads), shared::heads_of(num_heads, num_kv_heads).HC, head_dim).bytes;
}

int swiftllm_hip_shared_decode(void* output, void* workspace, size_t workspace_bytes, const void* plan, size_t plan_bytes,
                               const void* query, const void* key_cache, const void* value_cache,
                               const int32_t* block_tables, const int32_t* query_offsets, const float* alibi_slopes,
                               float scale, float softcap, int dtype, int num_tokens, int num_seqs, int num_heads,
                               int num_kv_heads, int head_dim, int block_size, int max_num_blocks_per_seq, int num_blocks,
                               hipStream_t stream) {
    const char* who = "swiftllm_hip_shared_decode";
    int rc = shared::check_sizes(who, num_seqs, num_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq);
    if (rc != SWIFTLLM_OK) return rc;
    if (dtype != SWIFTLLM_HIP_F16 && dtype != SWIFTLLM_HIP_BF16) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: dtype=%d (supported: 0 fp16, 1 bf16)", who, dtype);
    }
    SharedArgs a{};
    if (!scored::make_shape(a.shape, std::fabs(scale), softcap, 0, nullptr, alibi_slopes)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: scale=%g softcap=%g", who, scale, softcap);
    }
    if (softcap > scored::kMostCap) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: softcap=%g (at most %g)", who, softcap, scored::kMostCap);
    }
    if (query_offsets && num_tokens < 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_tokens=%d", who, num_tokens);
    }
    if (num_seqs > 0 && (!output || !query || !key_cache || !value_cache || !plan || !workspace ||
                         (max_num_blocks_per_seq > 0 && !block_tables))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    if (!aligned(output, 2) || !aligned(query, 8) || !aligned(key_cache, 16) || !aligned(value_cache, 16) ||
        !aligned(block_tables, 4) || !aligned(query_offsets, 4) || !aligned(alibi_slopes, 4) || !aligned(plan, 256) ||
        !aligned(workspace, 256)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    const shared::Heads h = shared::heads_of(num_heads, num_kv_heads);
    const shared::Layout l = shared::layout_of(num_seqs, num_heads, num_kv_heads);
    const Space space = space_of(l, h.HC, head_dim);
    if (num_seqs > 0 && (workspace_bytes < space.bytes || plan_bytes < l.bytes)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: workspace of %zu bytes, %zu needed; plan of %zu, %zu needed", who,
                    workspace_bytes, space.bytes, plan_bytes, l.bytes);
    }
    // Queries of one workgroup's rows are read by those of other ranges and heads'
    // outputs are written meanwhile: no output may lie on an input.
    if (num_seqs > 0) {
        const size_t n = num_seqs, rows = query_offsets ? static_cast<size_t>(num_tokens) : n;
        const Bytes out{output, rows * num_heads * head_dim * 2}, q{query, out.n}, ws{workspace, space.bytes};
        const Bytes kc{key_cache, cache_bytes(num_blocks, num_kv_heads, head_dim)}, vc{value_cache, kc.n};
        const Bytes bt{block_tables, 4 * n * max_num_blocks_per_seq}, off{query_offsets, 4 * (n + 1)};
        const Bytes slopes{alibi_slopes, 4 * static_cast<size_t>(num_heads)}, pl{plan, l.bytes};
        if (overlap_any(out, {q, kc, vc, bt, off, slopes, pl}) || overlap_any(ws, {out, q, kc, vc, bt, off, slopes, pl})) {
            return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: output or workspace overlaps another argument", who);
        }
    }
    rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    // (lanes without a query read row 0, which is there where any row is)
    if (num_seqs == 0 || (query_offsets && num_tokens == 0)) return ok();
    // The sign of the scale goes into the query, and a scale of zero makes it zero: the
    // kernel's scale is positive, so that raw products order as scores.
    a.q_and = scale == 0.0f ? 0u : 0xffffffffu;
    a.q_xor = scale < 0.0f ? 0x80008000u : 0u;
    if (scale == 0.0f) a.shape.scale = 1.0f;
    a.out = static_cast<uint16_t*>(output);
    a.q = static_cast<const uint16_t*>(query);
    a.kc = static_cast<const uint16_t*>(key_cache);
    a.vc = static_cast<const uint16_t*>(value_cache);
    a.bt = block_tables;
    a.qoff = query_offsets;
    const char* const p = static_cast<const char*>(plan);
    a.head = reinterpret_cast<const shared::Head*>(p);
    a.walks = reinterpret_cast<const shared::Walk*>(p + l.walks);
    a.wide = reinterpret_cast<const shared::Start*>(p + l.wide_starts);
    a.narrow = reinterpret_cast<const shared::Start*>(p + l.narrow_starts);
    a.seqs = reinterpret_cast<const shared::Seq*>(p + l.seqs);
    char* const ws = static_cast<char*>(workspace);
    a.frag_ml = reinterpret_cast<float2*>(ws);
    a.frag_o = reinterpret_cast<float*>(ws + space.o);
    a.frag_rows = l.rows;
    a.T = num_tokens;
    a.S = num_seqs;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.G = h.G;
    a.nhc = h.nhc;
    a.gw = h.gw;
    a.tpw = h.tpw;
    a.MB = max_num_blocks_per_seq;
    a.num_blocks = num_blocks;
    a.q16 = aligned(query, 16);
    a.out8 = aligned(output, 8);
    using K = void (*)(SharedArgs);
#define SHARED_DECODE(T_) \
    {{{shared_decode_kernel<T_, 64, false, false>, shared_decode_kernel<T_, 64, false, true>}, \
      {shared_decode_kernel<T_, 64, true, false>, shared_decode_kernel<T_, 64, true, true>}}, \
     {{shared_decode_kernel<T_, 128, false, false>, shared_decode_kernel<T_, 128, false, true>}, \
      {shared_decode_kernel<T_, 128, true, false>, shared_decode_kernel<T_, 128, true, true>}}}
    static const K kernels[2][2][2][2] = {SHARED_DECODE(F16), SHARED_DECODE(BF16)};
#undef SHARED_DECODE
    static const K joins[2][2][2] = {
        {{shared_join_kernel<F16, 64, 1>, shared_join_kernel<F16, 64, 4>}, {shared_join_kernel<F16, 128, 1>, shared_join_kernel<F16, 128, 4>}},
        {{shared_join_kernel<BF16, 64, 1>, shared_join_kernel<BF16, 64, 4>}, {shared_join_kernel<BF16, 128, 1>, shared_join_kernel<BF16, 128, 4>}}};
    const int t = dtype == SWIFTLLM_HIP_BF16;
    // Short tables of few sequences are read whole by each: less than a second launch
    // would cost. (The host knows the tables, not the contexts.)
    const int parts = (h.gw + kNarrowRows - 1) / kNarrowRows;
    const double whole = 1.0 * num_seqs * h.HC * parts * max_num_blocks_per_seq * (4.0 * kBlockTokens * head_dim);
    if (max_num_blocks_per_seq <= kMostWhole && whole <= kWholeBytes && num_seqs <= 65535) {
        static const K whole_kernel[2][2][2] = {
            {{shared_whole_kernel<F16, 64, false>, shared_whole_kernel<F16, 64, true>}, {shared_whole_kernel<F16, 128, false>, shared_whole_kernel<F16, 128, true>}},
            {{shared_whole_kernel<BF16, 64, false>, shared_whole_kernel<BF16, 64, true>}, {shared_whole_kernel<BF16, 128, false>, shared_whole_kernel<BF16, 128, true>}}};
        return launched(launch(whole_kernel[t][head_dim == 128][alibi_slopes != nullptr], dim3(h.HC * parts, num_seqs), dim3(64 * kWaves), 0, stream, a), who);
    }
    rc = launched(launch(kernels[t][head_dim == 128][softcap > 0.0f][alibi_slopes != nullptr], dim3(h.HC, l.ranges),
                         dim3(64 * kWaves), 0, stream, a), who);
    if (rc != SWIFTLLM_OK) return rc;
    // Few rows may have many fragments each, and leave the GPU to four waves of each.
    const bool few = static_cast<long long>(num_seqs) * num_heads < kFewRows;
    return launched(launch(joins[t][head_dim == 128][few], dim3(num_seqs, few ? num_heads : (num_heads + kJoinWaves - 1) / kJoinWaves),
                           dim3(64 * kJoinWaves), 0, stream, a), who);
}

}  // extern "C"
