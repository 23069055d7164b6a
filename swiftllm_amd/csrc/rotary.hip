// Rotary positions of a step's queries and keys, fused with the cache write
// (gfx950).
//
// With a = position * inv_freq[i], i < rotary_dim / 2, and (x, y) the pair i
// of a head, elements (i, i + rotary_dim / 2) or, interleaved, (2 i, 2 i + 1):
//   (x, y) -> attn_factor * (x cos a - y sin a, y cos a + x sin a)
// for every query and key head; elements past rotary_dim stay as they are.
// Queries go to query_out, keys and values to the cache columns of the
// tokens' slots (the layout and the run handling of reshape_and_cache). A
// token with a negative position is padding and nothing of it is written; one
// without a slot in the pool keeps its queries only.
//
// Angles: at position 10^6 a 32-bit product is off by 0.06 of a radian, so
// the product and its reduction to a fraction of a turn are in 64 bits (three
// operations per angle), and sine and cosine of that fraction in 32. The
// rotation is in 32 bits and rounded once.
//
// Bound: HBM, one read of q, k and v and one write of q and of the blocks.
// One launch: a workgroup takes either a window of tokens of 256 rows of K or
// of V (see cache_runs.hpp), or the queries of four tokens. An angle's 20
// operations are made once per wave and token (per element: 123 us, not 91).
// Measured: 16384 tokens of prompts, 32/8 heads x 128, 87 us (4.6 TB/s read and
// written); 64 lone tokens of that layer 6.2 us; 2013 tokens of 8/8 x 64 6.5 us.
// 4096 lone tokens of 32/8 x 128 take 125 us: 2 bytes per 32-byte row each.

#include <algorithm>
#include <cmath>

#include "cache_runs.hpp"
#include "half_types.hpp"

namespace swiftllm {
namespace {

using namespace cache;

struct RotaryArgs {
    uint16_t* out;           // [T][H][D]
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* kc;
    uint16_t* vc;
    const int* positions;
    const int* slots;
    const double* inv_freq;
    long long q_stride;      // elements between tokens
    long long k_stride;
    long long v_stride;
    long long num_slots;     // <= 0: unknown
    float factor;
    int T;
    int H;
    int Hkv;
    int D;
    int rot;                 // rotary_dim
    int windows;             // windows of tokens of K and V
    int slices;              // of kWinRows rows
    int each;                // query heads a wave takes of a token
    int parts;               // waves per token
    bool whole;              // rotary_dim is a multiple of 16
    bool wide_q;             // 16-byte accesses of q and out, whole pieces of 8 rotated alike
    bool wide_k;
    bool wide_v;
};

constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)

// Cosine and sine, times the factor, of a pair at a position.
__device__ __forceinline__ void turn(const RotaryArgs& a, int pos, double freq, float& c, float& s) {
    const double t = static_cast<double>(pos) * freq * kPerTurn;
    const float f = static_cast<float>(__builtin_amdgcn_fract(t));
    c = __builtin_amdgcn_cosf(f) * a.factor;
    s = __builtin_amdgcn_sinf(f) * a.factor;
}

// The pair of element d < rotary_dim, where its other element is, and the sign
// of the sine for it.
template <bool INTER>
__device__ __forceinline__ void pair_of(int d, int half, int& i, int& other, float& sign) {
    if constexpr (INTER) {
        i = d >> 1;
        other = d ^ 1;
        sign = (d & 1) ? 1.0f : -1.0f;
    } else {
        const bool up = d >= half;
        i = up ? d - half : d;
        other = up ? d - half : d + half;
        sign = up ? 1.0f : -1.0f;
    }
}

// The cosines and sines of a token's pairs, one pair a lane, in LDS of the
// wave: an angle costs some 20 operations, and every head needs it.
struct TurnLds {
    float c[64], s[64];
    // The frequency of this lane's pair.
    static __device__ __forceinline__ double freq(const RotaryArgs& a) {
        const int i = threadIdx.x & 63;
        return i < a.rot >> 1 ? a.inv_freq[i] : 0.0;
    }
    __device__ __forceinline__ void make(const RotaryArgs& a, int pos, double f) {
        const int i = threadIdx.x & 63;
        float cc, ss;
        turn(a, pos, f, cc, ss);
        __builtin_amdgcn_wave_barrier();   // after the reads of the one before
        c[i] = cc;
        s[i] = ss;
        __builtin_amdgcn_wave_barrier();
    }
};

// The cosines and signed sines of elements d .. d + 7: 1 and 0 past rotary_dim.
template <bool INTER>
struct Turn8 {
    float c[8], s[8];
    __device__ __forceinline__ void take(const TurnLds& l, int d, int rot, bool whole) {
        const int half = rot >> 1;
        if (whole) {   // (rotary_dim a multiple of 16: 8 elements lie in one half)
            if (d >= rot) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    c[e] = 1.0f;
                    s[e] = 0.0f;
                }
            } else if constexpr (INTER) {
                const f4 cc = *reinterpret_cast<const f4*>(l.c + (d >> 1));
                const f4 ss = *reinterpret_cast<const f4*>(l.s + (d >> 1));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    c[e] = cc[e >> 1];
                    s[e] = e & 1 ? ss[e >> 1] : -ss[e >> 1];
                }
            } else {
                const bool up = d >= half;
                const int i = up ? d - half : d;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const f4 cc = *reinterpret_cast<const f4*>(l.c + i + e);
                    const f4 ss = *reinterpret_cast<const f4*>(l.s + i + e);
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        c[e + z] = cc[z];
                        s[e + z] = up ? ss[z] : -ss[z];
                    }
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            c[e] = 1.0f;
            s[e] = 0.0f;
            if (d + e < rot) {
                int i, other;
                float sign;
                pair_of<INTER>(d + e, half, i, other, sign);
                c[e] = l.c[i];
                s[e] = l.s[i] * sign;
            }
        }
    }
};

// Elements d .. d + 7 of a head at p, and the other elements of their pairs.
template <bool INTER>
__device__ __forceinline__ void load8(const uint16_t* p, int d, int rot, bool wide, uint16_t (&x)[8], uint16_t (&y)[8]) {
    if (wide) {
        // rotary_dim is a multiple of 16, so a piece of 8 lies in one half.
        const u4v u = *reinterpret_cast<const u4v*>(p + d);
        __builtin_memcpy(x, &u, 16);
        if constexpr (INTER) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
        } else {
            const int half = rot >> 1;
            const u4v z = *reinterpret_cast<const u4v*>(p + (d >= rot ? d : d >= half ? d - half : d + half));
            __builtin_memcpy(y, &z, 16);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        int i, other = d + e;
        float sign;
        if (d + e < rot) pair_of<INTER>(d + e, rot >> 1, i, other, sign);
        x[e] = p[d + e];
        y[e] = p[other];
    }
}

template <typename T, bool INTER>
__device__ __forceinline__ u4v rotate8(const Turn8<INTER>& t, const uint16_t (&x)[8], const uint16_t (&y)[8], int d,
                                       int rot) {
    uint16_t r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // A copy past rotary_dim: a value that is not finite stays what it is.
        const float z = __builtin_fmaf(T::up(x[e]), t.c[e], T::up(y[e]) * t.s[e]);
        r[e] = d + e < rot ? T::down(z) : x[e];
    }
    u4v u;
    __builtin_memcpy(&u, r, 16);
    return u;
}

// Rows of K, rotated, or of V, as they are, for write_runs.
template <typename T, bool INTER>
struct RowSrc {
    const RotaryArgs& a;
    const uint16_t* rows;     // row 0 of the block, not of the slice
    long long stride;
    int row0;
    bool is_v;
    bool wide;
    TurnLds* lds;             // two of this wave: the tokens of its lower and upper lanes
    int pos;                  // of token t0 + lane
    double freq;              // of pair `lane`
    __device__ __forceinline__ int slot(int t) const { return a.positions[t] < 0 ? -1 : a.slots[t]; }
    __device__ __forceinline__ void before(int k) const {
        if (is_v) return;
        lds[0].make(a, __builtin_amdgcn_readlane(pos, __builtin_amdgcn_readlane(k, 0) & 63), freq);
        lds[1].make(a, __builtin_amdgcn_readlane(pos, __builtin_amdgcn_readlane(k, 63) & 63), freq);
    }
    __device__ __forceinline__ uint16_t one(int t, int i) const {
        const uint16_t* const p = rows + t * stride + row0 + i;
        const int d = (row0 + i) & (a.D - 1);
        if (is_v || d >= a.rot) return *p;
        int pair, other;
        float sign, c, s;
        pair_of<INTER>(d, a.rot >> 1, pair, other, sign);
        turn(a, a.positions[t], a.inv_freq[pair], c, s);
        return T::down(__builtin_fmaf(T::up(*p), c, T::up(p[other - d]) * (s * sign)));
    }
    __device__ __forceinline__ u4v eight(int t, int i) const {
        const uint16_t* const p = rows + t * stride + row0 + i;
        uint16_t x[8], y[8];
        if (is_v) {
            if (wide) return *reinterpret_cast<const u4v*>(p);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[e];
            u4v u;
            __builtin_memcpy(&u, x, 16);
            return u;
        }
        const int d = (row0 + i) & (a.D - 1);
        Turn8<INTER> r;
        r.take(lds[(threadIdx.x >> 5) & 1], d, a.rot, a.whole);
        load8<INTER>(p - d, d, a.rot, wide, x, y);
        return rotate8<T, INTER>(r, x, y, d, a.rot);
    }
};

template <typename T, bool INTER, int W>
__global__ __launch_bounds__(256) void rotary_and_cache_kernel(const RotaryArgs a) {
    __shared__ __align__(16) uint16_t tile[(W + kBlockTokens - 1) * kWinStride];
    __shared__ __align__(16) TurnLds s_turn[4][2];
    TurnLds* const lds = s_turn[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
    const int lane = threadIdx.x & 63;
    const int pieces = 2 * a.slices;   // of a window: its slices of K, then of V
    const int kv = a.windows * pieces;
    if (blockIdx.x < static_cast<unsigned>(kv)) {
        const int piece = blockIdx.x / a.windows;
        const int t0 = (blockIdx.x - piece * a.windows) * W;
        const bool is_v = piece >= a.slices;
        const int row0 = (is_v ? piece - a.slices : piece) * kWinRows;
        const int pos = a.positions[min(t0 + lane, a.T - 1)];
        const RowSrc<T, INTER> src{a, is_v ? a.v : a.k, is_v ? a.v_stride : a.k_stride, row0, is_v,
                                   is_v ? a.wide_v : a.wide_k, lds, pos, is_v ? 0.0 : TurnLds::freq(a)};
        write_runs<W>(src, is_v ? a.vc : a.kc, tile, t0, row0, a.Hkv * a.D, a.T, a.num_slots);
        return;
    }
    // Queries. A wave takes `each` heads of one token, 1 KB of its row at a
    // time. The lanes of one head are lanes of one wave, and each has its loads
    // back before any stores: query_out may be query.
    const int unit = (blockIdx.x - kv) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = unit / a.parts;
    if (t >= a.T) return;
    const int pos = a.positions[t];
    const double freq = TurnLds::freq(a);
    const int lanes = a.D >> 3;                 // of one head
    const int d = 8 * (lane & (lanes - 1));
    const int step = 64 / lanes;
    const int h0 = (unit - t * a.parts) * a.each + lane / lanes;
    const int h1 = min(a.H, (unit - t * a.parts + 1) * a.each);
    const uint16_t* const src = a.q + t * a.q_stride;
    uint16_t* const dst = a.out + static_cast<size_t>(t) * a.H * a.D + d;
    Turn8<INTER> r;
    if (pos < 0) return;
    lds->make(a, pos, freq);
    r.take(*lds, d, a.rot, a.whole);
    if (a.wide_q) {
#pragma unroll 8
        for (int h = h0; h < h1; h += step) {
            uint16_t x[8], y[8];
            load8<INTER>(src + h * a.D, d, a.rot, true, x, y);
            *reinterpret_cast<u4v*>(dst + h * a.D) = rotate8<T, INTER>(r, x, y, d, a.rot);
        }
        return;
    }
    for (int h = h0; h < h1; h += step) {
        uint16_t x[8], y[8], w[8];
        load8<INTER>(src + h * a.D, d, a.rot, false, x, y);
        const u4v u = rotate8<T, INTER>(r, x, y, d, a.rot);
        __builtin_memcpy(w, &u, 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[h * a.D + e] = w[e];
    }
}

// The bytes of `tokens` rows of n values, `stride` values apart.
Bytes rows_of(const void* p, long long tokens, long long n, long long stride) {
    return Bytes{p, 2 * static_cast<size_t>((tokens - 1) * stride + n)};
}

}  // namespace
}  // namespace swiftllm

using namespace swiftllm;

extern "C" {

int swiftllm_hip_rotary_and_cache(void* query_out, const void* query, const void* key, const void* value,
                                  void* key_cache, void* value_cache, const int32_t* positions,
                                  const int32_t* slot_mapping, const void* inv_freq, float attn_factor,
                                  int interleaved, int dtype, int num_tokens, int num_heads, int num_kv_heads,
                                  int head_dim, int rotary_dim, int block_size, long long query_stride,
                                  long long key_stride, long long value_stride, int num_blocks,
                                  hipStream_t stream) {
    const char* who = "swiftllm_hip_rotary_and_cache";
    const long long T = num_tokens, H = num_heads, Hkv = num_kv_heads, D = head_dim;
    if (T < 0 || H <= 0 || Hkv <= 0 || D <= 0 || block_size <= 0 || !std::isfinite(attn_factor)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER,
                    "%s: num_tokens=%d num_heads=%d num_kv_heads=%d head_dim=%d block_size=%d attn_factor=%g", who,
                    num_tokens, num_heads, num_kv_heads, head_dim, block_size, attn_factor);
    }
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: rotary_dim=%d of head_dim=%d (even, at most head_dim)", who,
                    rotary_dim, head_dim);
    }
    if ((D != 64 && D != 128) || block_size != kBlockTokens) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: head_dim=%d block_size=%d (supported: 64/128, 16)", who, head_dim,
                    block_size);
    }
    if (dtype != SWIFTLLM_HIP_F16 && dtype != SWIFTLLM_HIP_BF16) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: dtype=%d (supported: 0 fp16, 1 bf16)", who, dtype);
    }
    if (H > 65535 || Hkv > 65535) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_heads=%d num_kv_heads=%d", who, num_heads, num_kv_heads);
    }
    // Elements between tokens, and from the first to the last: 2^47 bytes hold any
    // tensor, so offsets and the sums of one with a pointer stay below 2^63.
    const long long most = 1LL << 40, most_all = 1LL << 46;
    if (query_stride < H * D || key_stride < Hkv * D || value_stride < Hkv * D || query_stride > most ||
        key_stride > most || value_stride > most ||
        (T > 1 && std::max({query_stride, key_stride, value_stride}) > most_all / (T - 1))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: num_tokens=%d query_stride=%lld key_stride=%lld value_stride=%lld",
                    who, num_tokens, query_stride, key_stride, value_stride);
    }
    if (T > 0 && (!query_out || !query || !key || !value || !key_cache || !value_cache || !positions ||
                  !slot_mapping || (rotary_dim > 0 && !inv_freq))) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: null pointer", who);
    }
    if (!aligned(query_out, 2) || !aligned(query, 2) || !aligned(key, 2) || !aligned(value, 2) ||
        !aligned(key_cache, 8) || !aligned(value_cache, 8) || !aligned(positions, 4) || !aligned(slot_mapping, 4) ||
        !aligned(inv_freq, 8)) {
        return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: misaligned pointer", who);
    }
    if (T > 0) {
        // In place is fine; any other overlap would be read, or written again, after
        // it is written. (Of caches, where their size is known.)
        const Bytes o = rows_of(query_out, T, H * D, H * D), q = rows_of(query, T, H * D, query_stride);
        const Bytes k = rows_of(key, T, Hkv * D, key_stride), v = rows_of(value, T, Hkv * D, value_stride);
        const Bytes pos{positions, 4 * static_cast<size_t>(T)}, slots{slot_mapping, 4 * static_cast<size_t>(T)};
        const Bytes freq{inv_freq, 4 * static_cast<size_t>(rotary_dim)};
        const Bytes kc{key_cache, cache_bytes(num_blocks, Hkv, D)}, vc{value_cache, kc.n};
        const bool in_place = query_out == query && query_stride == H * D;
        if ((!in_place && overlap_any(o, {q})) || overlap_any(o, {k, v, pos, slots, freq, kc, vc})) {
            return fail(SWIFTLLM_ERR_INVALID_PARAMETER, "%s: query_out overlaps another argument", who);
        }
    }
    RotaryArgs a{};
    a.out = static_cast<uint16_t*>(query_out);
    a.q = static_cast<const uint16_t*>(query);
    a.k = static_cast<const uint16_t*>(key);
    a.v = static_cast<const uint16_t*>(value);
    a.kc = static_cast<uint16_t*>(key_cache);
    a.vc = static_cast<uint16_t*>(value_cache);
    a.positions = positions;
    a.slots = slot_mapping;
    a.inv_freq = static_cast<const double*>(inv_freq);
    a.q_stride = query_stride;
    a.k_stride = key_stride;
    a.v_stride = value_stride;
    a.num_slots = num_blocks > 0 ? static_cast<long long>(num_blocks) * kBlockTokens : 0;
    a.factor = attn_factor;
    a.T = num_tokens;
    a.H = num_heads;
    a.Hkv = num_kv_heads;
    a.D = head_dim;
    a.rot = rotary_dim;
    a.whole = rotary_dim % 16 == 0;
    a.wide_q = a.whole && aligned(query, 16) && aligned(query_out, 16) && query_stride % 8 == 0;
    a.wide_k = a.whole && aligned(key, 16) && key_stride % 8 == 0;
    a.wide_v = aligned(value, 16) && value_stride % 8 == 0;
    a.slices = static_cast<int>((Hkv * D + kWinRows - 1) / kWinRows);
    const int W = small_windows(T, a.slices) ? 4 : 16;
    a.windows = static_cast<int>((T + W - 1) / W);
    // Long calls have a wave per token, which makes its angles once; in others a
    // wave takes 1 KB of it. Split / whole: 64/8 heads x 128 64 tokens 5.8 / 9.0 us,
    // 1024 10.1 / 12.4, 2048 16.9 / 16.8, 4096 30.3 / 29.1; 32/8 512 6.1 / 7.6, 1024
    // 7.4 / 7.3, 2048 11.3 / 11.0, 4096 20.1 / 19.0. (A first row asked for with the
    // position, so that padding is read too: 2048 tokens 10.4 and 15.5 us, 64 in 1024
    // rows 11.5, not 9.9.)
    const int step = static_cast<int>(512 / D);
    a.each = T > 1024 ? num_heads : std::min(num_heads, step);
    a.parts = (num_heads + a.each - 1) / a.each;
    const long long grid = 2LL * a.windows * a.slices + (T * a.parts + 3) / 4;
    if (grid >= (1LL << 24)) {
        return fail(SWIFTLLM_ERR_NOT_SUPPORTED, "%s: num_tokens=%d of %d + 2 * %d heads", who, num_tokens, num_heads,
                    num_kv_heads);
    }
    const int rc = require_device();
    if (rc != SWIFTLLM_OK) return rc;
    if (T == 0) return ok();
    using K = void (*)(RotaryArgs);
    static const K kernels[2][2][2] = {
        {{rotary_and_cache_kernel<F16, false, 4>, rotary_and_cache_kernel<F16, false, 16>},
         {rotary_and_cache_kernel<F16, true, 4>, rotary_and_cache_kernel<F16, true, 16>}},
        {{rotary_and_cache_kernel<BF16, false, 4>, rotary_and_cache_kernel<BF16, false, 16>},
         {rotary_and_cache_kernel<BF16, true, 4>, rotary_and_cache_kernel<BF16, true, 16>}}};
    return launched(launch(kernels[dtype == SWIFTLLM_HIP_BF16][interleaved != 0][W == 16],
                           dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, a),
                    who);
}

}  // extern "C"
