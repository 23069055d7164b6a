// A beam search's selection over beams and vocabulary (gfx950).
//
// Beam w of a request has the score c_w (a sum of log probabilities) and the
// logits x_w[v] of its next token:
//   score(w, v) = c_w + x_w[v] - lse_w,   lse_w = log sum_v exp x_w[v]
// Candidates are the C largest scores, compared in 64 bits; ties go to the lower
// beam, then the larger logit, then the lower token. Within a beam that is the
// order of (logit, token), so its C first by those hold all of its candidates: lse,
// which moves them alike, decides between beams only.
//
// First kernel, a workgroup per kChunk logits of a row: their sum of exponentials
// and a list that holds their C largest. The threads' own maxima are 256 of them,
// so the C-th largest of those is a threshold that at least C logits reach, and few
// more do: only values in threads above it can. It is found bit by bit, a ballot
// each. Second kernel, a
// workgroup per request: the rows' lse, the same threshold over all lists' scores
// rounded to 32 bits (which keeps their order), and the few that reach it ranked by
// counting. Lists that ties fill past their room are cut to C one by one.
//
// lse. exp(x - m) = 2^(x L - m L) with L = log2(e) in 32 bits and m the thread's
// maximum: one multiply-add with r, the rounded m L, and the sum times 2^(r - m L),
// that difference exact. So the roundings are those of the exponents, of exp2 and
// of the sums: 32 bits up to a chunk's, 64 bits over chunks. L's own error moves
// lse by 2e-8 of the distance from the maximum. With d the distance from the maximum in
// log2 units, whose mean under the softmax is at most log2 V + 2, all of it is less than
// 2^-24 (2 d + 2 of exp2 + 44 of sums and products) < 2^-17.
//
// Bound: HBM for 32-bit logits, for 16-bit ones as much the vector operations, 13.6
// per logit as counted, of which the exponential is four. 64 x 4 rows of 128000 bfloat16
// logits: 16.4 us, 4.0 TB/s; 9 x 32 of 100003 in 32 bits 28 us, 4.1 TB/s; 4 of 32000
// 5.2 us, as long as a chunk's way through. The second kernel is latency, of one workgroup
// a request: 5.0 us for 16 lists of 8 candidates, 6.8 for 64, 14 for 416 lists of 64 or
// more (20 with every pass over the entries in memory, their scores found again).

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "half_types.hpp"

namespace swiftllm {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 32;                  // logits of a thread
constexpr int kChunk = kThreads * kEach;
constexpr int kGroup = 8, kGroups = kEach / kGroup;
static_assert(kGroups == 4 && kEach == 32, "maxima, and a word of bits");
constexpr int kRoom = 128;                 // entries of a chunk's list
constexpr int kMostCandidates = 64;
// Up to so many, a chunk's line is the C-th largest of 128 maxima, not 256 (32 of 128
// lets 37 values pass, 64 would let 89): 64 x 4 bfloat16 rows 16.4 us, not 17.6.
constexpr int kFewCandidates = 32;
constexpr int kPickLists = 1024;           // lists that reach the first line
constexpr int kPickRoom = 1024;            // candidates that are ranked
constexpr int kFewEnough = 160;            // by one line
constexpr float kLog2e = 1.4426950408889634f;
static_assert(kMostCandidates <= kRoom && kMostCandidates <= kThreads, "a list holds the candidates");

struct Entry {
    float x;
    int token;
};

struct SelectArgs {
    const void* logits;
    const float* scores;        // [R * W]
    const int* offsets;         // [R * W + 1] or null: a row whose own are not ascending has no logits
    float* cand_scores;         // [R][C]
    int* cand_rows;
    int* cand_tokens;
    float* next_scores;         // [R][W]
    int* next_rows;
    int* next_tokens;
    // workspace
    float2* sums;               // [rows][chunks]: the maximum m, the sum of exp(x - m)
    int* fill;                  // [rows][chunks]
    Entry* lists;               // [rows][chunks][kRoom]
    long long stride;
    int W;
    int V;
    int C;
    int chunks;
    int eos;
};

struct F32 {};
template <typename T>    // the upper bits of a key that a line is found by
constexpr int key_bits = std::is_same<T, BF16>::value ? 16 : 20;
template <typename T>
constexpr int vec_of = std::is_same<T, F32>::value ? 4 : 8;    // values of 16 bytes

// Orders as the floats do (-0 below 0).
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) {
    return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// A number that n of 64 M keys reach, M of each lane, and hardly more: the
// n-th largest of them with its lower bits cleared. One ballot a key and bit: at 20
// bits a line lies at most 2^-11 of itself low.
template <int BITS, int M>
__device__ __forceinline__ unsigned nth_largest(const unsigned (&k)[M], int n) {
    unsigned t = 0;
#pragma unroll 1
    for (unsigned bit = 1u << 31; bit >= 1u << (32 - BITS); bit >>= 1) {
        const unsigned c = t | bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < M; ++i) reach += __popcll(__ballot(k[i] >= c));
        if (reach >= n) t = c;
    }
    return t;
}

// The bare instructions: fmaxf quiets its operands first, an operation each. Of
// values that are no number they make one or pass over it.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <typename T>    // -infinity, as many as fit 32 bits
constexpr unsigned kNone = std::is_same<T, F32>::value ? 0xff800000u : std::is_same<T, BF16>::value ? 0xff80ff80u : 0xfc00fc00u;

// A value that is no number counts as one that is banned.
__device__ __forceinline__ float number(float x) { return x != x ? -INFINITY : x; }

template <typename T>
__device__ __forceinline__ void unpack(u4 r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, F32>::value) {
            const unsigned u = r[i];
            v[i] = __builtin_bit_cast(float, u);
        } else {
            v[2 * i] = T::up(static_cast<uint16_t>(r[i] & 0xffffu));
            v[2 * i + 1] = T::up(static_cast<uint16_t>(r[i] >> 16));
        }
    }
}

template <typename T>
__device__ __forceinline__ float load_one(const void* row, long long i) {
    if constexpr (std::is_same<T, F32>::value) {
        return static_cast<const float*>(row)[i];
    } else {
        return T::up(static_cast<const uint16_t*>(row)[i]);
    }
}

// A sum of exp(x - m) as one of exp(x - top), top >= m.
__device__ __forceinline__ float weighed(float sum, float m, float top) {
    return m == top ? sum : sum * __builtin_amdgcn_exp2f((m - top) * kLog2e);
}

// The largest of the workgroup's keys, in every thread. part: kWaves.
__device__ __forceinline__ unsigned long long block_max(unsigned long long k, unsigned long long* part) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned lo = __shfl_xor(static_cast<int>(k), d);
        const unsigned hi = __shfl_xor(static_cast<int>(k >> 32), d);
        k = std::max(k, static_cast<unsigned long long>(hi) << 32 | lo);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = k;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) k = std::max(k, part[i]);
    return k;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void beam_chunk_kernel(const SelectArgs a) {
    constexpr int VEC = vec_of<T>;
    constexpr int NV = kEach / VEC;
    constexpr int kSize = 16 / VEC;
    __shared__ __align__(16) unsigned s_key[kThreads];
    __shared__ float s_f[kWaves], s_sum[kWaves];
    __shared__ unsigned long long s_best[kWaves];
    __shared__ Entry s_list[kRoom];
    __shared__ int s_fill;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.x / a.chunks;
    const int chunk = blockIdx.x - row * a.chunks;
    const size_t slot = static_cast<size_t>(row) * a.chunks + chunk;
    if (!(a.scores[row] > -INFINITY) || (a.offsets != nullptr && a.offsets[row + 1] <= a.offsets[row])) {
        // Nothing comes of this beam.
        if (tid == 0) {
            a.fill[slot] = 0;
            a.sums[slot] = float2{-INFINITY, 0.0f};
        }
        return;
    }
    if (tid == 0) s_fill = 0;
    // Vectors begin at 16-byte addresses, the first of them up to VEC - 1 values
    // before the row.
    const char* const base = static_cast<const char*>(a.logits) + static_cast<long long>(row) * a.stride * kSize;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15u) / kSize);
    const int first = chunk * kChunk - off;
    // All loads are on their way before the first is waited for. (Unpacked each in
    // its own branch, 64 x 4 rows of 128000 bfloat16 logits took 30 us, not 26.)
    u4 raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = first + (k * kThreads + tid) * VEC;
        raw[k] = u4{kNone<T>, kNone<T>, kNone<T>, kNone<T>};
        if (i >= 0 && i <= a.V - VEC) {
            raw[k] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(base + static_cast<long long>(i) * kSize));
        }
    }
    float v[kEach];
#pragma unroll
    for (int k = 0; k < NV; ++k) unpack<T>(raw[k], v + k * VEC);
    if (first < 0 || first + kChunk > a.V) {
        // Vectors that begin or end outside of the row.
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = first + (k * kThreads + tid) * VEC;
            if ((i < 0 && i > -VEC) || (i < a.V && i > a.V - VEC)) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (i + j >= 0 && i + j < a.V) v[k * VEC + j] = load_one<T>(base, i + j);
                }
            }
        }
    }
    // The largest of every kGroup values, and of all.
    float top[kGroups], most;
    auto maxima = [&] {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const float* const x = v + g * kGroup;
            top[g] = max3(x[0], x[1], x[2]);
#pragma unroll
            for (int k = 3; k + 1 < kGroup; k += 2) top[g] = max3(top[g], x[k], x[k + 1]);
            top[g] = max3(top[g], x[kGroup - 1], x[kGroup - 1]);
        }
        most = max3(max3(top[0], top[1], top[2]), top[3], top[3]);
    };
    maxima();
    const float r = most * kLog2e;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v[k], kLog2e, -r));
    sum *= __builtin_amdgcn_exp2f(-__builtin_fmaf(most, kLog2e, -r));
    if (__any(!(sum < INFINITY))) {
        // Values that are no number, nothing but banned ones, a product past the
        // type's range, or an infinite maximum, which has all the weight.
#pragma unroll
        for (int k = 0; k < kEach; ++k) v[k] = number(v[k]);
        maxima();
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            sum += v[k] == most ? 1.0f : __builtin_amdgcn_exp2f((v[k] - most) * kLog2e);
        }
    }
    s_key[tid] = key_of(most);
    const float wf = wave_max(most);
    const float ws = wave_sum(weighed(sum, most, wf));
    if (lane == 0) {
        s_f[w] = wf;
        s_sum[w] = ws;
    }
    __syncthreads();
    const u4 ks = *reinterpret_cast<const u4*>(s_key + 4 * lane);
    unsigned found;
    if (a.C <= kFewCandidates) {
        const unsigned keys[2] = {std::max(ks[0], ks[1]), std::max(ks[2], ks[3])};
        found = nth_largest<key_bits<T>>(keys, a.C);
    } else {
        const unsigned keys[4] = {ks[0], ks[1], ks[2], ks[3]};
        found = nth_largest<key_bits<T>>(keys, a.C);
    }
    // What is banned is no candidate. (Some keys are no number's.)
    const float line = fmaxf(of_key(found), -3.402823466e38f);
    unsigned mine = 0;     // which of the thread's values reach it
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        if (__any(top[g] >= line)) {
#pragma unroll
            for (int k = g * kGroup; k < (g + 1) * kGroup; ++k) mine |= v[k] >= line ? 1u << k : 0u;
        }
    }
    // They are few, and read again rather than held in registers by number.
    auto token_of = [&](int k) { return first + (k / VEC * kThreads + tid) * VEC + k % VEC; };
    const int count = __popc(mine);
    const int upto = wave_inclusive_scan(count);
    int at = 0;
    if (lane == 63 && upto > 0) at = atomicAdd(&s_fill, upto);
    at = __builtin_amdgcn_readlane(at, 63) + upto - count;
#pragma unroll 1
    for (unsigned left = mine; left != 0; left &= left - 1, ++at) {
        const int token = token_of(__ffs(left) - 1);
        if (at < kRoom) s_list[at] = Entry{load_one<T>(base, token), token};
    }
    __syncthreads();
    int n = s_fill;
    if (n > kRoom) {
        // Ties: the C largest one by one, each behind the last.
        n = a.C;
        unsigned long long last = ~0ull;
#pragma unroll 1
        for (int c = 0; c < n; ++c) {
            unsigned long long best = 0;
#pragma unroll 1
            for (unsigned left = mine; left != 0; left &= left - 1) {
                const int token = token_of(__ffs(left) - 1);
                const unsigned long long key = static_cast<unsigned long long>(key_of(load_one<T>(base, token) + 0.0f)) << 32 |
                                               (0xffffffffu - static_cast<unsigned>(token));
                if (key < last) best = std::max(best, key);
            }
            last = block_max(best, s_best);
            if (tid == 0) s_list[c] = Entry{of_key(static_cast<unsigned>(last >> 32)), static_cast<int>(0xffffffffu - static_cast<unsigned>(last))};
        }
        __syncthreads();
    }
    if (tid < n) a.lists[slot * kRoom + tid] = s_list[tid];
    if (tid == 0) {
        float F = -INFINITY, S = 0.0f;
        for (int i = 0; i < kWaves; ++i) F = fmaxf(F, s_f[i]);
        for (int i = 0; i < kWaves; ++i) S += weighed(s_sum[i], s_f[i], F);
        a.sums[slot] = float2{F, S};
        a.fill[slot] = n;
    }
}

// A candidate, and the order of candidates.
struct Cand {
    double score;
    float x;
    int beam;
    int token;
};
__device__ __forceinline__ bool before(const Cand& p, const Cand& q) {
    if (p.score != q.score) return p.score > q.score;
    if (p.beam != q.beam) return p.beam < q.beam;
    if (p.x != q.x) return p.x > q.x;
    return p.token < q.token;
}

// SMALL: every 16 threads have a list of their own, whose entries are on their way
// before anything else is known. Otherwise the lists' maxima give a first line, and
// only lists that reach it are read.
template <int THREADS, bool SMALL>
__global__ __launch_bounds__(THREADS) void beam_pick_kernel(const SelectArgs a) {
    constexpr int WAVES = THREADS / 64;
    constexpr int KEYS = THREADS / 128;            // a lane's, of every two threads' maxima
    __shared__ double s_base[kMostCandidates];     // of a beam: its score less log sum exp(x - top)
    __shared__ float s_top[kMostCandidates];
    __shared__ __align__(16) unsigned s_key[THREADS / 2];
    __shared__ Cand s_cand[kPickRoom];
    __shared__ Cand s_best[WAVES];
    __shared__ Cand s_order[kMostCandidates];
    __shared__ int s_list[SMALL ? 1 : kPickLists];
    __shared__ int s_fill, s_lists;
    __shared__ int s_reach[2][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = blockIdx.x;
    const int lists = a.W * a.chunks;
    const size_t slot0 = static_cast<size_t>(r) * lists;
    if (tid == 0) s_fill = s_lists = 0;
    // A thread's entries, of HELD lists. (Those past a list's fill are read and not used.)
    constexpr int kKept = kRoom / 16, kFirst = SMALL ? 2 : kKept / 2, HELD = SMALL ? 1 : 2;
    Entry kept[HELD][kKept];
    int fill[HELD] = {}, beam[HELD] = {};
    auto list_of = [&](int i) { return a.lists + (slot0 + i) * kRoom + (tid & 15); };
    if (SMALL && tid >> 4 < lists) {
        fill[0] = a.fill[slot0 + (tid >> 4)];
        beam[0] = (tid >> 4) / a.chunks;
#pragma unroll
        for (int k = 0; k < kFirst; ++k) kept[0][k] = list_of(tid >> 4)[16 * k];
    }
    // The rows' sums, by as many threads as there are chunks.
    const int span = a.chunks <= 16 ? 16 : 64, at = tid & (span - 1);
    for (int b0 = 0; b0 < a.W; b0 += THREADS / span) {
        const int b = b0 + tid / span;
        const bool real = b < a.W;
        const size_t row = static_cast<size_t>(r) * a.W + (real ? b : 0);
        const float score = a.scores[row];
        const float2* const sums = a.sums + row * a.chunks;
        const float2 mine = at < a.chunks ? sums[at] : float2{-INFINITY, 0.0f};
        float top = mine.x;
        for (int c = at + 64; c < a.chunks; c += 64) top = fmaxf(top, sums[c].x);
        for (int d = 1; d < span; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        double S = weighed(mine.y, mine.x, top);
        for (int c = at + 64; c < a.chunks; c += 64) S += weighed(sums[c].y, sums[c].x, top);
        for (int d = 1; d < span; d <<= 1) S += __shfl_xor(S, d);
        if (at == 0 && real) {
            // (a row that allows nothing is one of a beam without a score)
            const bool some = top > -INFINITY;
            s_base[b] = some ? score - log(S) : -INFINITY;
            s_top[b] = some ? top : 0.0f;
        }
    }
    auto rest_of = [&](int h, int i) {
#pragma unroll
        for (int k = kFirst; k < kKept; ++k) {
            if (16 * k < fill[h]) kept[h][k] = list_of(i)[16 * k];
        }
    };
    if (SMALL) rest_of(0, tid >> 4);
    __syncthreads();
    // (beside an infinite logit only others of its kind have a share)
    auto score_of = [&](int b, float x) { return x == s_top[b] ? s_base[b] : s_base[b] + (x - static_cast<double>(s_top[b])); };
    // A line that C candidates reach, of every two threads' maxima. Sixteen waves try
    // as many values of the next four bits, each over all keys.
    auto find_line = [&](float most) {
        most = fmaxf(most, __shfl_xor(most, 1));
        if ((tid & 1) == 0) s_key[tid >> 1] = key_of(most);
        __syncthreads();
        unsigned keys[KEYS];
        unsigned t = 0;
        if (WAVES == 16 || w == 0) {
#pragma unroll
            for (int k = 0; k < KEYS; ++k) keys[k] = s_key[64 * k + lane];
        }
        if constexpr (WAVES == 16) {
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                const unsigned c = t | static_cast<unsigned>(w) << (28 - 4 * k);
                int reach = 0;
#pragma unroll
                for (int i = 0; i < KEYS; ++i) reach += __popcll(__ballot(keys[i] >= c));
                if (lane == 0) s_reach[k & 1][w] = reach;
                __syncthreads();
                const unsigned long long on = __ballot(lane < 16 && s_reach[k & 1][lane & 15] >= a.C);
                t |= static_cast<unsigned>(__popcll(on) - 1) << (28 - 4 * k);
            }
        } else {
            if (w == 0) {
                t = nth_largest<20>(keys, a.C);
                if (lane == 0) s_reach[0][0] = static_cast<int>(t);
            }
            __syncthreads();
            t = static_cast<unsigned>(s_reach[0][0]);
        }
        return fmaxf(of_key(t), -3.402823466e38f);
    };
    int use = lists;
    bool some = false;     // the lists named in s_list
    float line = 0.0f;
    if constexpr (!SMALL) {
        // (the lists of a beam without a score are empty)
        auto list_max = [&](int i) {
            const int b = i / a.chunks;
            return s_base[b] > -INFINITY ? static_cast<float>(score_of(b, a.sums[slot0 + i].x)) : -INFINITY;
        };
        float most = -INFINITY;
        for (int i = tid; i < lists; i += THREADS) most = fmaxf(most, list_max(i));
        line = find_line(most);
        for (int i = tid; i < lists; i += THREADS) {
            if (list_max(i) >= line) {
                const int to = atomicAdd(&s_lists, 1);
                if (to < kPickLists) s_list[to] = i;
            }
        }
        __syncthreads();
        some = s_lists <= kPickLists;
        if (some) use = s_lists;
        if (use <= HELD * (THREADS / 16)) {
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                const int k = (tid >> 4) + h * (THREADS / 16);
                if (k >= use) break;
                const int i = some ? s_list[k] : k;
                fill[h] = a.fill[slot0 + i];
                beam[h] = i / a.chunks;
#pragma unroll
                for (int z = 0; z < kFirst; ++z) kept[h][z] = list_of(i)[16 * z];
            }
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                const int k = (tid >> 4) + h * (THREADS / 16);
                if (k < use) rest_of(h, some ? s_list[k] : k);
            }
        }
    }
    const bool held = SMALL || use <= HELD * (THREADS / 16);
    auto cand_of = [&](int b, const Entry& e) { return Cand{score_of(b, e.x), e.x, b, e.token}; };
    float rounded[HELD][kKept];    // scores, -infinity where there is no entry
    if (held) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
#pragma unroll
            for (int k = 0; k < kKept; ++k) {
                rounded[h][k] = -INFINITY;
                if ((tid & 15) + 16 * k < fill[h]) rounded[h][k] = static_cast<float>(score_of(beam[h], kept[h][k].x));
            }
        }
    }
    auto each = [&](auto take) {
        if (held) {
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
#pragma unroll
                for (int k = 0; k < kKept; ++k) take(rounded[h][k], beam[h], kept[h][k]);
            }
            return;
        }
        for (int k = tid >> 4; k < use; k += THREADS / 16) {
            const int i = some ? s_list[k] : k;
            const int b = i / a.chunks, n = a.fill[slot0 + i];
            for (int z = 0; (tid & 15) + z < n; z += 16) {
                const Entry e = list_of(i)[z];
                take(static_cast<float>(score_of(b, e.x)), b, e);
            }
        }
    };
    // Those that reach the line, where there is room for all of them; how many.
    auto collect = [&] {
        if constexpr (SMALL) {
            each([&](float score, int b, const Entry& e) {
                if (score >= line) {
                    const int to = atomicAdd(&s_fill, 1);
                    if (to < kPickRoom) s_cand[to] = cand_of(b, e);
                }
            });
            __syncthreads();
            return s_fill;
        }
        int count = 0;
        each([&](float score, int, const Entry&) { count += score >= line; });
        const int upto = wave_inclusive_scan(count);
        int to = 0;
        if (lane == 63 && upto > 0) to = atomicAdd(&s_fill, upto);
        to = __builtin_amdgcn_readlane(to, 63) + upto - count;
        __syncthreads();
        const int n = s_fill;
        if (n <= kPickRoom) {
            each([&](float score, int b, const Entry& e) {
                if (score >= line) s_cand[to++] = cand_of(b, e);
            });
        }
        __syncthreads();
        return n;
    };
    // The lists' line may be enough: few lie above it unless few lists hold most.
    int n = SMALL ? kPickRoom + 1 : collect();
    if (n > kPickRoom) {
        if (tid == 0) s_fill = 0;
        float most = -INFINITY;
        each([&](float score, int, const Entry&) { most = fmaxf(most, score); });
        line = find_line(most);
        n = collect();
    }
    if (THREADS == kPickRoom && n > kFewEnough && n <= kPickRoom) {
        // A closer line among these: they are ranked by n^2 comparisons.
        const Cand mine = tid < n ? s_cand[tid] : Cand{-INFINITY, 0.0f, 0, -1};
        const float closer = find_line(static_cast<float>(mine.score));
        if (tid == 0) s_fill = 0;
        __syncthreads();
        if (static_cast<float>(mine.score) >= closer) s_cand[atomicAdd(&s_fill, 1)] = mine;
        __syncthreads();
        n = s_fill;
    }
    if (n <= kPickRoom) {
        // Eight threads compare a candidate with every eighth.
        for (int i = tid >> 3; i < n; i += THREADS / 8) {
            const Cand mine = s_cand[i];
            int rank = 0;
            for (int j = tid & 7; j < n; j += 8) rank += before(s_cand[j], mine);
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) rank += __shfl_xor(rank, d);
            if ((tid & 7) == 0 && rank < a.C) s_order[rank] = mine;
        }
        n = min(n, a.C);
    } else {
        // Ties: one by one, each behind the last.
        const Cand none{-INFINITY, 0.0f, 0x7fffffff, 0x7fffffff};
        n = a.C;
        for (int k = 0; k < n; ++k) {
            Cand best = none;
            each([&](float score, int b, const Entry& e) {
                if (!(score > -INFINITY)) return;
                const Cand c = cand_of(b, e);
                if (k > 0 && !before(s_order[k - 1], c)) return;
                if (before(c, best)) best = c;
            });
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const Cand c{__shfl_xor(best.score, d), __shfl_xor(best.x, d), __shfl_xor(best.beam, d), __shfl_xor(best.token, d)};
                if (before(c, best)) best = c;
            }
            if (lane == 0) s_best[w] = best;
            __syncthreads();
            if (tid == 0) {
                for (int i = 1; i < WAVES; ++i) {
                    if (before(s_best[i], best)) best = s_best[i];
                }
                s_order[k] = best;
            }
            __syncthreads();
        }
    }
    __syncthreads();
    if (w > 0) return;
    // Lane c has candidate c.
    const bool real = lane < n;
    const Cand c = real ? s_order[lane] : Cand{-INFINITY, 0.0f, 0, -1};
    const int row = real ? r * a.W + c.beam : -1;
    const float score = static_cast<float>(c.score);
    if (lane < a.C) {
        const size_t to = static_cast<size_t>(r) * a.C + lane;
        a.cand_scores[to] = score;
        a.cand_rows[to] = row;
        a.cand_tokens[to] = c.token;
    }
    const unsigned long long on = __ballot(real && c.token != a.eos);
    const int place = __popcll(on & ((1ull << lane) - 1ull));
    const int all = __popcll(on);
    const size_t first = static_cast<size_t>(r) * a.W;
    if (((on >> lane) & 1ull) && place < a.W) {
        a.next_scores[first + place] = score;
        a.next_rows[first + place] = row;
        a.next_tokens[first + place] = c.token;
    }
    if (lane >= all && lane < a.W) {
        a.next_scores[first + lane] = -INFINITY;
        a.next_rows[first + lane] = -1;
        a.next_tokens[first + lane] = -1;
    }
}

struct Space {
    size_t sums, fill, lists, bytes;
    int chunks;
};

// A row that begins off a 16-byte address takes up to 7 values more.
Space space_of(long long rows, long long V) {
    const auto up = [](long long n) { return static_cast<size_t>((n + 255) / 256 * 256); };
    Space s;
    s.chunks = static_cast<int>((V + 7 + kChunk - 1) / kChunk);
    const long long slots = rows * s.chunks;
    s.sums = 0;
    s.fill = up(8 * slots);
    s.lists = s.fill + up(4 * slots);
    s.bytes = s.lists + up(8 * kRoom * slots) + 256;
    return s;
}

int check_sizes(const char* who, long long R, long long W, long long V, long long C) {
    if (R < 0 || W <= 0 || V <= 0 || C < W) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_requests=%lld beam_width=%lld vocab=%lld num_candidates=%lld",
                    who, R, W, V, C);
    }
    if (C > kMostCandidates || R > (1 << 20) || V > (1 << 27) || R * W * ((V + 7 + kChunk - 1) / kChunk) >= (1 << 24)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_requests=%lld beam_width=%lld vocab=%lld num_candidates=%lld (at most %d)",
                    who, R, W, V, C, kMostCandidates);
    }
    return SWIFTLLM_OK;
}

int select(const char* who, const void* logits, const float* beam_scores, const int32_t* query_offsets, float* cand_scores,
           int32_t* cand_rows, int32_t* cand_tokens, float* next_scores, int32_t* next_rows, int32_t* next_tokens,
           void* workspace, size_t workspace_bytes, int dtype, int num_requests, int beam_width, int vocab,
           int num_candidates, long long logits_stride, int eos_id, hipStream_t stream) {
    const long long R = num_requests, W = beam_width, V = vocab, C = num_candidates;
    int rc = check_sizes(who, R, W, V, C);
    if (rc != SWIFTLLM_OK) return rc;
    if (dtype != SWIFTLLM_HIP_F16 && dtype != SWIFTLLM_HIP_BF16 && dtype != SWIFTLLM_HIP_F32) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: dtype=%d (supported: 0 fp16, 1 bf16, 2 fp32)", who, dtype);
    }
    if (logits_stride < V || logits_stride > (1LL << 40)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: logits_stride=%lld of vocab=%d", who, logits_stride, vocab);
    }
    if (R > 0 && (!logits || !beam_scores || !cand_scores || !cand_rows || !cand_tokens || !next_scores || !next_rows ||
                  !next_tokens || !workspace)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    const size_t size = dtype == SWIFTLLM_HIP_F32 ? 4 : 2;
    const size_t rows = static_cast<size_t>(R * W);
    const Space space = space_of(R * W, V);
    const Bytes span[] = {{cand_scores, 4 * static_cast<size_t>(R * C)}, {cand_rows, 4 * static_cast<size_t>(R * C)},
                          {cand_tokens, 4 * static_cast<size_t>(R * C)}, {next_scores, 4 * rows}, {next_rows, 4 * rows},
                          {next_tokens, 4 * rows}, {workspace, space.bytes}, {beam_scores, 4 * rows},
                          {logits, rows == 0 ? 0 : (static_cast<size_t>(logits_stride) * (rows - 1) + V) * size},
                          {query_offsets, 4 * (rows + 1)}};
    for (const Bytes& s : span) {
        if (!aligned(s.p, s.p == logits ? size : 4)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    if (!aligned(workspace, 256)) return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    if (R > 0 && workspace_bytes < space.bytes) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, space.bytes);
    }
    for (int i = 0; i < 7; ++i) {
        for (int j = i + 1; j < 10; ++j) {
            // The next step's beams may take the place of this step's: a workgroup
            // has read its request's before it writes them.
            if (i == 3 && j == 7 && next_scores == beam_scores) continue;
            if (overlap_any(span[i], {span[j]})) {
                return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: an output overlaps another argument", who);
            }
        }
    }
    rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    if (R == 0) return ok();
    SelectArgs a{};
    a.logits = logits;
    a.scores = beam_scores;
    a.offsets = query_offsets;
    a.cand_scores = cand_scores;
    a.cand_rows = cand_rows;
    a.cand_tokens = cand_tokens;
    a.next_scores = next_scores;
    a.next_rows = next_rows;
    a.next_tokens = next_tokens;
    char* const ws = static_cast<char*>(workspace);
    a.sums = reinterpret_cast<float2*>(ws + space.sums);
    a.fill = reinterpret_cast<int*>(ws + space.fill);
    a.lists = reinterpret_cast<Entry*>(ws + space.lists);
    a.stride = logits_stride;
    a.W = beam_width;
    a.V = vocab;
    a.C = num_candidates;
    a.chunks = space.chunks;
    a.eos = eos_id >= 0 ? eos_id : -2;
    using K = void (*)(SelectArgs);
    static const K kernels[3] = {beam_chunk_kernel<F16>, beam_chunk_kernel<BF16>, beam_chunk_kernel<F32>};
    rc = launched(launch(kernels[dtype], dim3(static_cast<unsigned>(rows * space.chunks)), dim3(kThreads), 0, stream, a), who);
    if (rc != SWIFTLLM_OK) return rc;
    const long long lists = W * space.chunks;
    const K pick = lists <= 16 ? beam_pick_kernel<256, true> : lists <= 64 ? beam_pick_kernel<1024, true> : beam_pick_kernel<1024, false>;
    return launched(launch(pick, dim3(static_cast<unsigned>(R)), dim3(lists <= 16 ? 256 : 1024), 0, stream, a), who);
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

size_t swiftllm_hip_beam_select_workspace_size(int num_requests, int beam_width, int vocab, int num_candidates) {
    if (check_sizes("swiftllm_hip_beam_select_workspace_size", num_requests, beam_width, vocab, num_candidates) != SWIFTLLM_OK) {
        return 0;
    }
    ok();
    return space_of(static_cast<long long>(num_requests) * beam_width, vocab).bytes;
}

int swiftllm_hip_beam_select(const void* logits, const float* beam_scores, float* cand_scores, int32_t* cand_rows,
                             int32_t* cand_tokens, float* next_scores, int32_t* next_rows, int32_t* next_tokens,
                             void* workspace, size_t workspace_bytes, int dtype, int num_requests, int beam_width,
                             int vocab, int num_candidates, long long logits_stride, int eos_id, hipStream_t stream) {
    return select("swiftllm_hip_beam_select", logits, beam_scores, nullptr, cand_scores, cand_rows, cand_tokens, next_scores,
                  next_rows, next_tokens, workspace, workspace_bytes, dtype, num_requests, beam_width, vocab, num_candidates,
                  logits_stride, eos_id, stream);
}

int swiftllm_hip_beam_select_rows(const void* logits, const float* beam_scores, const int32_t* query_offsets,
                                  float* cand_scores, int32_t* cand_rows, int32_t* cand_tokens, float* next_scores,
                                  int32_t* next_rows, int32_t* next_tokens, void* workspace, size_t workspace_bytes,
                                  int dtype, int num_requests, int beam_width, int vocab, int num_candidates,
                                  long long logits_stride, int eos_id, hipStream_t stream) {
    return select("swiftllm_hip_beam_select_rows", logits, beam_scores, query_offsets, cand_scores, cand_rows, cand_tokens,
                  next_scores, next_rows, next_tokens, workspace, workspace_bytes, dtype, num_requests, beam_width, vocab,
                  num_candidates, logits_stride, eos_id, stream);
}

}  // extern "C"
