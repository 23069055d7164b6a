// Paged attention of one new token with shaped scores (gfx950): soft cap,
// distance bias, sliding window, and a prefix that stays in sight
// (scored_core.hpp). The query of sequence s is its last token, at position
// context_lens[s] - 1: row s, or the last of its rows of a packed step.
//
// Bound: HBM, one read of the visible K and V: blocks that a window hides are
// never touched. Per 16-token block a wave has 8 KB to read at D = 128 and
// 28 small matrix products to make (8 turns of K, 4 for the scores, 16 for the
// two parts of the weights).
//
// Work. The visible blocks of all sequences form one list, each sequence with
// kPieceCost blocks of overhead on top (Q, merge, store). Short tables are
// taken whole, a workgroup per sequence and kv head; otherwise the list is cut
// into as many equal ranges as workgroups fit the GPU at once, one per kv head
// (and chunk of 16 query heads) and range, so that one long context fills the
// GPU and a ragged batch has no tail. Every workgroup finds its range in the
// lengths by itself. A sequence that a range holds whole is written at once;
// the others leave (maximum, sum, output) fragments, at most two per range,
// which a second kernel joins.
//
// A workgroup's four waves take the blocks of a piece in turn, two in flight
// per wave. A block's K comes tokens-contiguous and is turned by a product
// with the identity (exact), S^T = K Q^T and O^T = V P^T as in paged decode,
// with P in two 16-bit parts, each rounded to nearest (off by 2^-22 of a weight
// for fp16, 2^-17 for bfloat16), so that only the output is rounded. (Cut instead,
// bfloat16 outputs were 3e-6 of themselves too small in the mean and twice as many
// were not the nearest value, in the same time.)
//
// Measured, with a cap: 64 contexts of 512-4096 tokens, 32/8 heads x 128, 96 us
// (6.2 TB/s, 4.7 us of it the join), 8 x 32768 of 64/8 166 us (6.5 TB/s); 4 chats
// of 8/8 x 64 in one launch 6.2 us.

#include <algorithm>

#include "scored_walk.hpp"

namespace swiftllm {
namespace {

using namespace scored;

struct ScoredDecodeArgs {
    uint16_t* out;         // [S][H][D]
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    const int* bt;
    const int* ctx;
    const int* qoff;       // [S + 1] or null: row s
    int T;                 // rows, where qoff is given
    int4* info;            // [min(S, ranges)]: a cut sequence, its first and last range
    float* frag_ml;        // [ranges][2][HC][2][gs]
    float* frag_o;         // [ranges][2][HC][gs][D], normalised
    Shape shape;
    int S;
    int H;
    int Hkv;
    int G;                 // query heads per kv head
    int nhc;               // chunks of 16 of them
    int MB;
    int num_blocks;
    int ranges;            // 0: every sequence whole
    bool out8;             // out is 8-byte aligned
};

constexpr int kWaves = 4;
// Blocks that starting and ending a piece costs a workgroup, in its own time.
// Measured with 2 / 4 / 8 / 16: 256 lognormal contexts up to 8192 tokens 158.7 /
// 156.1 / 157.4 / 165.1 us, 128 in a window of 1024 57.0 / 56.7 / 57.0 / 60.3.
constexpr int kPieceCost = 4;
// Shortest range, in blocks: two per wave (16: 2 x 2000 tokens 13.8 us, not 12.2).
constexpr int kLeastRange = 8;

// The row of a sequence's query and output; negative: it has none.
__device__ __forceinline__ int row_of(const ScoredDecodeArgs& a, int s) {
    if (a.qoff == nullptr) return s;
    const int b = as_const(a.qoff)[s], e = as_const(a.qoff)[s + 1];
    return b >= 0 && e > b && e <= a.T ? e - 1 : -1;
}

// What the query of a sequence sees, in blocks: the walk takes blocks 0 ..
// before - 1 (the prefix) and then those from `low / 16` on. The keys end with
// the table, at L; of a longer context the query keeps its position, and a window
// of it may lie past them all (low = L). (A bias's distances are taken from key
// L - 1: what they lack is the same for every key.)
struct Sight {
    int L, low, pre, before, skip, n;
    __device__ __forceinline__ int block(int i) const { return i < before ? i : i + skip; }
    // The tokens of block j that are seen, as bits.
    __device__ __forceinline__ unsigned tokens(int j) const {
        const int base = j * kBlockTokens;
        return (low_bits(pre - base) | ~low_bits(low - base)) & low_bits(L - base);
    }
};

__device__ __forceinline__ Sight sight_of(const ScoredDecodeArgs& a, int s) {
    Sight v;
    const int ctx = row_of(a, s) < 0 ? 0 : max(as_const(a.ctx)[s], 0);
    v.L = min(ctx, a.MB * kBlockTokens);
    v.low = a.shape.window > 0 ? min(max(ctx - a.shape.window, 0), v.L) : 0;
    v.pre = a.shape.prefix != nullptr ? min(max(as_const(a.shape.prefix)[s], 0), v.L) : 0;
    const int first = v.low >> kBlockShift;
    v.before = min((v.pre + kBlockTokens - 1) >> kBlockShift, first);
    v.skip = first - v.before;
    v.n = ((v.L + kBlockTokens - 1) >> kBlockShift) - v.skip;
    return v;
}

template <int D>
__host__ __device__ constexpr int merge_floats(int gs) {
    return kWaves * 32 + kWaves * gs * D;
}

// Blocks i0 .. i1 - 1 of a sequence's walk for one kv head and chunk of query
// heads, by the whole workgroup. at: the query's row. emit(g, d, o, m, l): normalised outputs d ..
// d + 3 of head g, and its maximum and sum.
template <typename T, int D, typename Emit>
__device__ __forceinline__ void run_piece(const ScoredDecodeArgs& a, const Sight& sight, int s, int at, int kvh, int hc, int i0,
                                          int i1, Emit emit) {
    constexpr int NJ = D / 16;
    // Worked out per piece behind an empty asm: kept over the pieces, what
    // follows from it would not leave the walk enough registers.
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;
    const int kg = lane >> 4;
    const int gn = min(16, a.G - hc * 16);
    const int gs = min(16, a.G);
    const int h0 = kvh * a.G + hc * 16;
    State<D> st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int J = 0; J < NJ; ++J) st.acc[J] = f4{0, 0, 0, 0};

    const int count = i1 > i0 + w ? (i1 - i0 - w + kWaves - 1) / kWaves : 0;
    if (count > 0) {
        const int* const row = a.bt + static_cast<size_t>(s) * a.MB;
        // Lane l has the id of the wave's block 64 c + l.
        auto ids_from = [&](int c) { return row[sight.block(min(i0 + w + kWaves * (64 * c + lane), i1 - 1))]; };
        int ids = ids_from(0);
        s8 q[NJ / 2];
        const uint16_t* const qp = a.q + (static_cast<size_t>(at) * a.H + h0 + min(r, gn - 1)) * D + 4 * kg;
#pragma unroll
        for (int J = 0; J < NJ; J += 2) {
            const s8 x = join8(*reinterpret_cast<const s4*>(qp + 16 * J), *reinterpret_cast<const s4*>(qp + 16 * J + 16));
            q[J / 2] = r < gn ? x : s8{0, 0, 0, 0, 0, 0, 0, 0};
        }
        const float slope = a.shape.slopes != nullptr && r < gn ? a.shape.slopes[h0 + r] * kLog2e : 0.0f;
        s4 ident;
#pragma unroll
        for (int i = 0; i < 4; ++i) ident[i] = 4 * kg + i == r ? static_cast<short>(T::one()) : 0;
        const int loff = kv_elem_offset(r, 4 * kg);
        // The wave's k-th block, asked for in order.
        auto load = [&](int k, s4 (&kk)[NJ], s4 (&vv)[NJ], int& j, unsigned& seen) {
            if (k > 0 && (k & 63) == 0) ids = ids_from(k >> 6);
            const int b = __builtin_amdgcn_readlane(ids, k & 63);
            const bool known = block_known(b, a.num_blocks);
            j = sight.block(i0 + w + kWaves * k);
            seen = known ? sight.tokens(j) & 0xffffu : 0u;
            // A block outside the pool is read as block 0 and hidden.
            const size_t tile = kv_tile_offset(known ? b : 0, kvh, a.Hkv, D) + loff;
#pragma unroll
            for (int J = 0; J < NJ; ++J) kk[J] = load4(a.kc + tile + kv_elem_offset(16 * J, 0));
#pragma unroll
            for (int J = 0; J < NJ; ++J) vv[J] = load4(a.vc + tile + kv_elem_offset(16 * J, 0));
        };
        auto take = [&](s4 (&kk)[NJ], s4 (&vv)[NJ], int j, unsigned seen) {
            attend<T, D>(st, seen, j * kBlockTokens - (sight.L - 1), kg, kk, vv, q, ident, a.shape, slope);
        };
        // Two blocks in flight; no load of the loop depends on a condition.
        s4 kA[NJ], vA[NJ], kB[NJ], vB[NJ];
        int jA, jB;
        unsigned sA, sB;
        load(0, kA, vA, jA, sA);
        int k = 0;
        for (; k + 2 < count; k += 2) {
            load(k + 1, kB, vB, jB, sB);
            take(kA, vA, jA, sA);
            load(k + 2, kA, vA, jA, sA);
            take(kB, vB, jB, sB);
        }
        if (k + 1 < count) {
            load(k + 1, kB, vB, jB, sB);
            take(kA, vA, jA, sA);
            take(kB, vB, jB, sB);
        } else {
            take(kA, vA, jA, sA);
        }
    }
    // The four waves' states through LDS.
    const float l = sum_over_groups(st.l);
    extern __shared__ __align__(16) float smem[];
    float* const sm_m = smem;
    float* const sm_l = smem + kWaves * 16;
    float* const sm_o = smem + kWaves * 32;
    if (kg == 0) {
        sm_m[w * 16 + r] = st.m;
        sm_l[w * 16 + r] = l;
    }
    if (r < gn) {
#pragma unroll
        for (int J = 0; J < NJ; ++J) {
            *reinterpret_cast<f4*>(sm_o + static_cast<size_t>(w * gs + r) * D + 16 * J + 4 * kg) = st.acc[J];
        }
    }
    __syncthreads();
    for (int i = tid; i < gn * (D / 4); i += 64 * kWaves) {
        const int g = i / (D / 4);
        const int d = 4 * (i - g * (D / 4));
        float mx[kWaves], m = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            mx[x] = sm_m[x * 16 + g];
            m = fmaxf(m, mx[x]);
        }
        f4 num = f4{0, 0, 0, 0};
        float den = 0.0f;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            // A wave that saw no key has zeros; one of NaN scores alone a NaN sum.
            const float f = mx[x] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mx[x] - m);
            num += f * *reinterpret_cast<const f4*>(sm_o + static_cast<size_t>(x * gs + g) * D + d);
            den += f * sm_l[x * 16 + g];
        }
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        emit(g, d, num * inv, m, den);
    }
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(3)))
void scored_decode_kernel(const ScoredDecodeArgs a) {
    const int HC = a.Hkv * a.nhc;
    const int range = blockIdx.y;          // every sequence whole: the sequence
    const int sub = blockIdx.x;
    const int kvh = a.nhc == 1 ? sub : sub / a.nhc;
    const int hc = sub - kvh * a.nhc;
    const int h0 = kvh * a.G + hc * 16;
    const int gs = min(16, a.G);
    // This workgroup's part of the list, [start, end), and the sequence that
    // holds its start, which begins at `begin`.
    int start = 0, end = 1, s = range, begin = 0, len = 1;
    if (a.ranges > 0) {
        __shared__ int s_wave[kWaves];
        __shared__ int s_at[2];
        // Thread t adds up the sequences of its segment.
        const int lane = threadIdx.x & 63;
        const int w = threadIdx.x >> 6;
        const int each = (a.S + 64 * kWaves - 1) / (64 * kWaves);
        const int s0 = min(static_cast<int>(threadIdx.x) * each, a.S);
        const int s1 = min(s0 + each, a.S);
        int sum = 0;
        for (int i = s0; i < s1; ++i) sum += sight_of(a, i).n + kPieceCost;
        const int incl = wave_inclusive_scan(sum);
        if (lane == 63) s_wave[w] = incl;
        __syncthreads();
        int all = 0, before = incl - sum;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (i < w) before += s_wave[i];
            all += s_wave[i];
        }
        len = max((all + a.ranges - 1) / a.ranges, kLeastRange);
        start = range * len;    // below all + ranges * (kLeastRange + 1)
        end = min(start + len, all);
        if (start >= before && start < before + sum) {
            int i = s0, at = before;
            for (;; ++i) {
                const int cost = sight_of(a, i).n + kPieceCost;
                if (start < at + cost) break;
                at += cost;
            }
            s_at[0] = i;
            s_at[1] = at;
        }
        __syncthreads();
        s = __builtin_amdgcn_readfirstlane(s_at[0]);
        begin = __builtin_amdgcn_readfirstlane(s_at[1]);
    }
    const bool by_seq = a.S < a.ranges;   // what the entries of info belong to
    const bool teller = a.ranges > 0 && sub == 0 && threadIdx.x == 0;
    int4 cut = int4{-1, 0, 0, 0};
    for (int at = start; at < end;) {
        const Sight sight = sight_of(a, s);
        int i0 = 0, i1 = sight.n, e = end, stop = end;
        if (a.ranges > 0) {
            stop = begin + sight.n + kPieceCost;
            e = min(end, stop);
            i0 = max(at - begin - kPieceCost, 0);
            i1 = max(e - begin - kPieceCost, 0);
        }
        const bool whole = at == begin && e == stop;
        // Slot 0: the sequence began in a range before; 1: it begins here.
        const int slot = begin < start ? 0 : 1;
        if (slot == 1) {
            const int4 x = whole ? int4{-1, 0, 0, 0} : int4{s, range, (stop - 1) / len, 0};
            if (!whole) cut = x;
            if (teller && by_seq) a.info[s] = x;
        }
        const size_t f = static_cast<size_t>(2 * range + slot) * HC + sub;
        const int row = row_of(a, s);
        run_piece<T, D>(a, sight, s, row, kvh, hc, i0, i1, [&](int g, int d, f4 o, float m, float l) {
            if (whole) {
                if (row < 0) return;
                uint16_t* const p = a.out + (static_cast<size_t>(row) * a.H + h0 + g) * D + d;
                if (a.out8) {
                    *reinterpret_cast<u2*>(p) = u2{T::down2(o[0], o[1]), T::down2(o[2], o[3])};
                } else {
#pragma unroll
                    for (int z = 0; z < 4; ++z) p[z] = T::down(o[z]);
                }
                return;
            }
            *reinterpret_cast<f4*>(a.frag_o + (f * gs + g) * D + d) = o;
            if (d == 0) {
                a.frag_ml[f * 2 * gs + g] = m;
                a.frag_ml[f * 2 * gs + gs + g] = l;
            }
        });
        at = e;
        if (at >= end) break;
        __syncthreads();  // the merge's LDS is free again
        ++s;              // a piece that ends inside the range ends its sequence
        begin = stop;
    }
    if (teller && !by_seq) a.info[range] = cut;
}

// Joins the fragments of a cut sequence: one workgroup per (entry of info, query
// head), its waves take the fragments in turn. A lane holds the maximum and the
// sum of a fragment, and the first rows are on their way before those are there:
// a join is bound by latency.
constexpr int kJoinRows = 8;

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void scored_decode_join_kernel(const ScoredDecodeArgs a) {
    constexpr int DL = D / 64;
    __shared__ float s_o[kWaves][D];
    __shared__ float s_ml[kWaves][2];
    const int h = blockIdx.x;
    const const_int* const cut = as_const(reinterpret_cast<const int*>(a.info + blockIdx.y));
    const int s = cut[0], first = cut[1], last = cut[2];
    if (s < 0) return;
    const int kvh = h / a.G;
    const int hg = h - kvh * a.G;
    const int HC = a.Hkv * a.nhc;
    const int sub = kvh * a.nhc + hg / 16;
    const int g = hg % 16;
    const int gs = min(16, a.G);
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The wave's i-th fragment.
    const int count = max((last - first - w + kWaves) / kWaves, 0);
    auto place = [&](int i) {
        const int x = first + w + kWaves * i;
        return static_cast<size_t>(2 * x + (x == first)) * HC + sub;
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
                const float* const p = a.frag_o + (place(c + i + k) * gs + g) * D + lane * DL;
#pragma unroll
                for (int j = 0; j < DL; ++j) v[k][j] = p[j];
            }
        };
        rows(0);
        const float* const ml = a.frag_ml + place(c + min(lane, n - 1)) * 2 * gs + g;
        const float fm = lane < n ? ml[0] : -INFINITY;
        const float fl = lane < n ? ml[gs] : 0.0f;
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
#pragma unroll
    for (int j = 0; j < DL; ++j) s_o[w][lane * DL + j] = o[j];
    if (lane == 0) {
        s_ml[w][0] = m;
        s_ml[w][1] = l;
    }
    __syncthreads();
    if (threadIdx.x >= D) return;
    const int d = threadIdx.x;
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) M = fmaxf(M, s_ml[x][0]);
    float num = 0.0f, den = 0.0f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
        const float f = s_ml[x][0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s_ml[x][0] - M);
        num += f * s_o[x][d];
        den += f * s_ml[x][1];
    }
    const int row = row_of(a, s);
    if (row >= 0) a.out[(static_cast<size_t>(row) * a.H + h) * D + d] = T::down(den == 0.0f ? 0.0f : num / den);
}

// Workgroups the list is cut for: two for each of the 256 CUs of an MI355X, where
// three fit. Any number is correct. Measured with 512 / 768 (us per call, 32/8
// heads x 128 unless said): 64 contexts of 512-4096 tokens 104.2 / 106.2, 256
// lognormal up to 8192 154.3 / 156.1, 100 of 16/16 heads 118.9 / 120.4, 40 x 3000
// of 64/8 83.1 / 84.6, 1 x 32768 29.0 / 29.8, 1 x 7919 14.3 / 14.2.
constexpr int kResident = 2 * 256;

struct Layout {
    int ranges;
    size_t ml, o, bytes;   // offsets of the fragments, and the size
};

Layout layout_of(long long H, long long Hkv, long long D) {
    Layout l;
    const long long G = H / Hkv;
    const long long HC = Hkv * ((G + 15) / 16);
    const long long gs = std::min<long long>(G, 16);
    l.ranges = static_cast<int>(std::max<long long>(kResident / HC, 1));
    const auto up = [](long long n) { return static_cast<size_t>((n + 255) / 256 * 256); };
    l.ml = up(16LL * l.ranges);
    l.o = l.ml + up(2LL * l.ranges * HC * 2 * gs * 4);
    l.bytes = l.o + up(2LL * l.ranges * HC * gs * D * 4);
    return l;
}

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
    // Token positions and the batch's blocks are 32-bit sums.
    if (S > 65535 || H > 65535 || MB >= (1 << 27) || S * (MB + kPieceCost) >= (1LL << 30)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_seqs=%lld num_heads=%lld max_num_blocks_per_seq=%lld", who, S, H, MB);
    }
    return SWIFTLLM_OK;
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

size_t swiftllm_hip_scored_decode_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                 int block_size, int max_num_blocks_per_seq) {
    if (check_sizes("swiftllm_hip_scored_decode_workspace_size", num_seqs, num_heads, num_kv_heads, head_dim,
                    block_size, max_num_blocks_per_seq) != SWIFTLLM_OK) {
        return 0;
    }
    ok();
    return layout_of(num_heads, num_kv_heads, head_dim).bytes;
}

int swiftllm_hip_scored_decode(void* output, void* workspace, size_t workspace_bytes, const void* query,
                               const void* key_cache, const void* value_cache, const int32_t* block_tables,
                               const int32_t* context_lens, const int32_t* query_offsets, const float* alibi_slopes,
                               const int32_t* prefix_lens, float scale, float softcap, int window, int dtype,
                               int num_tokens, int num_seqs, int num_heads,
                               int num_kv_heads, int head_dim, int block_size, int max_num_blocks_per_seq,
                               int num_blocks, hipStream_t stream) {
    const char* who = "swiftllm_hip_scored_decode";
    int rc = check_sizes(who, num_seqs, num_heads, num_kv_heads, head_dim, block_size, max_num_blocks_per_seq);
    if (rc != SWIFTLLM_OK) return rc;
    if (dtype != SWIFTLLM_HIP_F16 && dtype != SWIFTLLM_HIP_BF16) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: dtype=%d (supported: 0 fp16, 1 bf16)", who, dtype);
    }
    ScoredDecodeArgs a{};
    if (!scored::make_shape(a.shape, scale, softcap, window, prefix_lens, alibi_slopes)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: scale=%g softcap=%g window=%d", who, scale, softcap, window);
    }
    if (softcap > scored::kMostCap) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: softcap=%g (at most %g)", who, softcap, scored::kMostCap);
    }
    if (query_offsets && num_tokens < 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_tokens=%d", who, num_tokens);
    }
    if (num_seqs > 0 && (!output || !query || !key_cache || !value_cache || !context_lens || !workspace ||
                         (max_num_blocks_per_seq > 0 && !block_tables))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    if (!aligned(output, 2) || !aligned(query, 8) || !aligned(key_cache, 8) || !aligned(value_cache, 8) ||
        !aligned(block_tables, 4) || !aligned(context_lens, 4) || !aligned(query_offsets, 4) ||
        !aligned(alibi_slopes, 4) || !aligned(prefix_lens, 4) || !aligned(workspace, 256)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    const Layout l = layout_of(num_heads, num_kv_heads, head_dim);
    if (num_seqs > 0 && workspace_bytes < l.bytes) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, l.bytes);
    }
    const int S = num_seqs, D = head_dim;
    const int G = num_heads / num_kv_heads;
    const int nhc = (G + 15) / 16;
    const long long HC = static_cast<long long>(num_kv_heads) * nhc;
    if (S * HC >= (1LL << 24)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_seqs=%d num_heads=%d", who, num_seqs, num_heads);
    }
    // A workgroup has read its queries before it or a later kernel writes their
    // rows; rows of others, and what every workgroup reads, must not be among them.
    if (num_seqs > 0) {
        const size_t n = num_seqs, rows = query_offsets ? static_cast<size_t>(num_tokens) : n;
        const Bytes out{output, rows * num_heads * head_dim * 2}, q{query, out.n}, ws{workspace, l.bytes};
        const Bytes kc{key_cache, cache_bytes(num_blocks, num_kv_heads, head_dim)}, vc{value_cache, kc.n};
        const Bytes bt{block_tables, 4 * n * max_num_blocks_per_seq}, ctx{context_lens, 4 * n};
        const Bytes off{query_offsets, 4 * (n + 1)}, pre{prefix_lens, 4 * n};
        const Bytes slopes{alibi_slopes, 4 * static_cast<size_t>(num_heads)};
        if ((output != query && overlap_any(out, {q})) || overlap_any(out, {kc, vc, bt, ctx, off, pre, slopes}) ||
            overlap_any(ws, {out, q, kc, vc, bt, ctx, off, pre, slopes})) {
            return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: output or workspace overlaps another argument", who);
        }
    }
    rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    if (S == 0) return ok();
    a.out = static_cast<uint16_t*>(output);
    a.q = static_cast<const uint16_t*>(query);
    a.kc = static_cast<const uint16_t*>(key_cache);
    a.vc = static_cast<const uint16_t*>(value_cache);
    a.bt = block_tables;
    a.ctx = context_lens;
    a.qoff = query_offsets;
    a.T = num_tokens;
    char* const ws = static_cast<char*>(workspace);
    a.info = reinterpret_cast<int4*>(ws);
    a.frag_ml = reinterpret_cast<float*>(ws + l.ml);
    a.frag_o = reinterpret_cast<float*>(ws + l.o);
    a.S = S;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.G = G;
    a.nhc = nhc;
    a.MB = max_num_blocks_per_seq;
    a.num_blocks = num_blocks;
    a.out8 = aligned(output, 8);
    // A sequence per workgroup, in one launch, up to `line` blocks: the longest
    // walk as far as the host knows. Whole / cut, 32/8 heads x 128: 1 sequence up
    // to 512 tokens 8.4 / 9.8 us, 1024 11.9 / 9.8; 16 up to 768 12.4 / 15.0, 1024
    // 16.4 / 16.2, 1280 19.5 / 18.6; 64 up to 1024 34.9 / 39.1, 1536 50.8 / 54.4;
    // 200 up to 1536 152.8 / 151.9, 2048 197.5 / 195.2; of 64/8 1536 155.6 / 162.3;
    // 128 ragged ones in a window of 1024 54.1 / 54.4, of 2048 77.7 / 65.9. (The host
    // does not know the contexts, only the tables: short ones in tables of 2048 blocks
    // are cut, 16 up to 256 tokens 12.0 us, not 7.5, 64 up to 1000 38.5, not 34.9.)
    const int most = window > 0 && !prefix_lens ? std::min(a.MB, window / kBlockTokens + 2) : a.MB;
    const long long items = S * HC;
    const int line = static_cast<int>(std::min<long long>(32 + items / 4, 96));
    a.ranges = most <= line || l.ranges < 4 ? 0 : l.ranges;
    const size_t lds = sizeof(float) * (D == 128 ? merge_floats<128>(std::min(G, 16)) : merge_floats<64>(std::min(G, 16)));
    using K = void (*)(ScoredDecodeArgs);
    static const K main_kernel[2][2] = {{scored_decode_kernel<F16, 64>, scored_decode_kernel<F16, 128>},
                                        {scored_decode_kernel<BF16, 64>, scored_decode_kernel<BF16, 128>}};
    static const K join_kernel[2][2] = {{scored_decode_join_kernel<F16, 64>, scored_decode_join_kernel<F16, 128>},
                                        {scored_decode_join_kernel<BF16, 64>, scored_decode_join_kernel<BF16, 128>}};
    const int t = dtype == SWIFTLLM_HIP_BF16;
    rc = launched(launch(main_kernel[t][D == 128], dim3(static_cast<unsigned>(HC), a.ranges > 0 ? a.ranges : S), dim3(64 * kWaves), lds, stream, a), who);
    if (rc != SWIFTLLM_OK || a.ranges == 0) return rc;
    return launched(launch(join_kernel[t][D == 128], dim3(num_heads, std::min(S, a.ranges)), dim3(64 * kWaves), 0, stream, a), who);
}

}  // extern "C"
