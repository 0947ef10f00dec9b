// The next token of each row drawn from its logits: temperature, top-k, top-p,
// min-p and one given random number.
//
// Per row, with m the largest logit: w(v) = exp((x(v) - m) / temperature), held as
// a whole number of units of 2^-43, so that sums of weights are exact in 64 bits
// and the same in any order.  Tokens are ranked by logit, equal ones by index.
// Kept are the first top_k; of those the first ones whose weights come to top_p of
// their total; of those the ones with w >= min_p, and always the first.  The token
// is, in index order, the first whose running sum of kept weights exceeds uniform *
// their sum.
//
// Where a running sum stands beside uniform * total, or beside top_p * total, the
// last bits of the weights decide a whole number, so they are formed in fp64: 2^-43
// a weight, against some 2^-24 in fp32, which over a flat vocabulary of 200000 would
// move the token in some of every thousand draws.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "abi_util.hpp"
#include "device_common.hpp"

namespace asdsl {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 1024;            // tokens of a wave's step, whose kept weight is noted
constexpr int kBins = 256;             // of log2 weights, between the row's largest and smallest
constexpr double kDepth = 44.0;        // or 2^-kDepth, from which on there is no weight
constexpr int kListMost = 4096;        // tokens of the bins that a cut runs through, of a row
constexpr int kSliceMost = 1024;       // and of a slice
constexpr int kMaxSlices = 64;
constexpr int kMaxVocab = 1 << 20;     // 2^20 weights of 2^43 stay below 2^64
constexpr double kLog2eWide = 1.4426950408889634074;

// What a row's cuts leave open once its bins are counted.
struct RowState {
    unsigned long long total;   // weight of all
    unsigned long long base_p;  // weight of the bins before the first that the cut of top-p may run through
    unsigned long long base_k;  // weight and tokens of those before the one that the cut of top-k runs through
    uint32_t count_k;
    int bin_k;                  // that bin, kBins without a cut
    int p_lo, p_hi;             // and those of top-p, p_lo kBins without a cut
};

struct SampleArgs {
    const float* logits;
    const float* uniform;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* tokens;
    float* probs;
    unsigned long long* best;  // [rows][slices] largest logit and its first token
    uint32_t* low;             // [rows][slices] a small logit that may have a weight
    unsigned long long* mass;  // [rows][slices][kBins]
    uint32_t* count;           // [rows][slices][kBins]
    unsigned long long* tile;  // [rows][tiles]
    RowState* state;           // [rows]
    uint32_t* listed;          // [rows][slices], more than kSliceMost where the list does not hold them
    uint2* list;               // [rows][slices][kSliceMost] (logit, token)
    int vocab, slices, slice, tiles;
};

// Larger for a larger logit, equal for both zeros; 0 for none.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.0f ? 0.0f : x);
    return (b >> 31) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t order) {
    return __builtin_bit_cast(float, (order >> 31) ? order & 0x7FFFFFFFu : ~order);
}

// What a row's slices found.
struct Ends {
    unsigned long long best;  // order_of the largest logit, and below it ~ its first token; 0: nothing to draw from
    uint32_t low;             // order_of the logit at which the last bin begins; smaller ones may have weights
};

// Logits so far below another have no weight.
__device__ __forceinline__ float reach_of(const SampleArgs& a, int row) {
    return static_cast<float>(kDepth / kLog2eWide) * (a.temperature ? a.temperature[row] : 1.0f);
}

// A row's weights.  Every kernel forms them with the same roundings (none is
// contracted), so that what one counts is what the next one finds.
struct Scale {
    double m, c;      // largest logit, log2(e) / temperature
    double per_bin;   // bins a unit of log2
    bool infinite;    // the largest is +inf
    bool greedy;      // only the first is kept

    __device__ __forceinline__ Scale(const SampleArgs& a, int row, const Ends& e) {
#pragma clang fp contract(off)
        const float t = a.temperature ? a.temperature[row] : 1.0f, top = logit_of(static_cast<uint32_t>(e.best >> 32));
        greedy = !(t > 0.0f) || (a.top_k && a.top_k[row] == 1) || (a.top_p && a.top_p[row] <= 0.0f) ||
                 (a.min_p && a.min_p[row] > 1.0f);
        infinite = top == INFINITY;
        m = top;
        c = kLog2eWide / static_cast<double>(t);
        const double depth = infinite ? 0.0 : fmin((m - static_cast<double>(logit_of(e.low))) * c, kDepth);
        per_bin = depth > 0.0 ? (kBins - 1) / depth : 0.0;
    }
    // log2 of a token's weight; any() is false where it has none (NaN and -inf among them)
    __device__ __forceinline__ double log2w(float x) const {
#pragma clang fp contract(off)
        if (infinite) return x == INFINITY ? 0.0 : -2.0 * kDepth;
        return (static_cast<double>(x) - m) * c;
    }
    static __device__ __forceinline__ bool any(double y) { return y > -kDepth; }
    // 2^y in units of 2^-43 where any(y): 2^n for the nearest whole number n times a
    // polynomial for 2^f, |f| <= 1/2, through its values at 10 Chebyshev nodes (2^-45
    // off at most); both sums with 2^52 round to a whole number.
    static __device__ __forceinline__ unsigned long long weight(double y) {
#pragma clang fp contract(off)
        const double shifted = y + 0x1.8p52;
        const double f = y - (shifted - 0x1.8p52);
        double p = 1.0205905686697933e-07;
        p = fma(p, f, 1.325964524635787e-06);
        p = fma(p, f, 1.525267292316862e-05);
        p = fma(p, f, 0.0001540343375124206);
        p = fma(p, f, 0.0013333558200798077);
        p = fma(p, f, 0.00961812919393433);
        p = fma(p, f, 0.05550410866465164);
        p = fma(p, f, 0.2402265069564034);
        p = fma(p, f, 0.6931471805599462);
        p = fma(p, f, 1.0000000000000135);
        const uint32_t n = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, shifted));
        const uint64_t power = static_cast<uint64_t>((1023u + 43u + n) << 20) << 32;
        return __builtin_bit_cast(uint64_t, fma(p, __builtin_bit_cast(double, power), 0x1p52)) & 0xFFFFFFFFFFFFFull;
    }
    // The same for any y, 0 where any(y) is false, without a branch, so that several run
    // side by side: 64 rows of 200064 to their sums 19.5 us, 23.0 behind a branch each.
    static __device__ __forceinline__ unsigned long long weight_or_none(double y) {
        const unsigned long long w = weight(fmax(y, -2.0 * kDepth));
        return any(y) ? w : 0ull;
    }
    // 0 .. kBins - 1, rising as weights fall; the sum with 2^52 rounds to a whole number.
    // The last bin takes in all that is smaller.  Held to it before the bits are taken:
    // the bins may end a bit of a float below the largest logit (Ends::low), and 44
    // doublings in units of such bins are past 32 bits and past 2^52.
    __device__ __forceinline__ int bin(double y) const {
        return static_cast<int>(__builtin_bit_cast(uint64_t, fmin(fma(y, -per_bin, 0x1p52), 0x1p52 + (kBins - 1))));
    }
};

__device__ __forceinline__ unsigned long long share_of(float part, unsigned long long total) {
    const double x = ceil(static_cast<double>(part) * static_cast<double>(total));
    return !(x > 1.0) ? 1ull : x < static_cast<double>(total) ? static_cast<unsigned long long>(x) : total;
}

// min_p in units: tokens of at least that weight are kept.
__device__ __forceinline__ unsigned long long least_weight(const SampleArgs& a, int row) {
    const float p = a.min_p ? a.min_p[row] : 0.0f;
    return p > 0.0f ? static_cast<unsigned long long>(ceil(static_cast<double>(fminf(p, 1.0f)) * 0x1p43)) : 1ull;
}

// How many tokens are kept at most.
__device__ __forceinline__ uint32_t most_kept(const SampleArgs& a, int row) {
    const int k = a.top_k ? a.top_k[row] : 0;
    return k > 0 ? static_cast<uint32_t>(k) : 0xFFFFFFFFu;
}

// Running f over the lanes of a wave, all of them here: lane i's takes in lanes 0 ..
// i.  Within rows of 16 lanes by shifts, then the last lane of a row for the next
// row or two; moves between registers, some 150 cycles where exchanges through LDS
// take 700.
template <int CTRL, int kRows16, typename T>
__device__ __forceinline__ T moved(T v, T none) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, none);
        const uint32_t lo = __builtin_amdgcn_update_dpp(static_cast<uint32_t>(b), static_cast<uint32_t>(a), CTRL, kRows16, 0xF, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(static_cast<uint32_t>(b >> 32), static_cast<uint32_t>(a >> 32), CTRL, kRows16,
                                                        0xF, false);
        return __builtin_bit_cast(T, (static_cast<uint64_t>(hi) << 32) | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(uint32_t, none),
                                                                 __builtin_bit_cast(uint32_t, v), CTRL, kRows16, 0xF, false));
    }
}

template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T v, T none, F f) {
    constexpr int kRowShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;
    v = f(v, moved<kRowShr + 1, 0xF>(v, none));
    v = f(v, moved<kRowShr + 2, 0xF>(v, none));
    v = f(v, moved<kRowShr + 4, 0xF>(v, none));
    v = f(v, moved<kRowShr + 8, 0xF>(v, none));
    v = f(v, moved<kBcast15, 0xA>(v, none));
    return f(v, moved<kBcast31, 0xC>(v, none));
}

template <typename T>
__device__ __forceinline__ T last_lane(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t a = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(a), kWave - 1);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(a >> 32), kWave - 1);
        return __builtin_bit_cast(T, (static_cast<uint64_t>(hi) << 32) | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, v), kWave - 1));
    }
}

template <typename T>
__device__ __forceinline__ T running_sum(T v) { return wave_scan(v, T(0), [](T p, T q) { return p + q; }); }
template <typename T>
__device__ __forceinline__ T wave_sum(T v) { return last_lane(running_sum(v)); }
template <typename T>
__device__ __forceinline__ T wave_max(T v) { return last_lane(wave_scan(v, T(0), [](T p, T q) { return p > q ? p : q; })); }
template <typename T>
__device__ __forceinline__ T wave_min(T v) { return last_lane(wave_scan(v, static_cast<T>(~T(0)), [](T p, T q) { return p < q ? p : q; })); }

// The logits of a slice as a wave takes them, 4 neighbouring tokens a lane and chunk,
// -inf past the slice's end; the first chunks are requested where it is made.  kVec:
// rows lie in whole 16-byte units.  kTiles: whole tiles of 4 chunks a wave, the first
// one of another wave in each workgroup, so that the compute unit's four SIMDs come
// out even; else every fourth chunk.
constexpr int kChunk = 4 * kWave;
template <bool kVec, bool kTiles>
struct Stream {
    static constexpr int kWaves = kThreads / kWave;
    static_assert(kTile == 4 * kChunk && kWaves == 4, "chunks of a tile, and of the registers below");
    const float* x;
    int begin, end, lane;
    float4 b0, b1, b2, b3;

    __device__ __forceinline__ Stream(const SampleArgs& a, int row, int slice)
        : x(a.logits + static_cast<size_t>(row) * a.vocab), end(min(a.vocab, (slice + 1) * a.slice)),
          lane(static_cast<int>(threadIdx.x) % kWave) {
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
        begin = slice * a.slice + (kTiles ? (wave + row + slice) % kWaves * kTile : wave * kChunk);
        b0 = load(0);
        b1 = load(1);
        b2 = load(2);
        b3 = load(3);
    }
    __device__ __forceinline__ int at(int c) const {
        return begin + (kTiles ? c / 4 * (kWaves * kTile) + c % 4 * kChunk : c * (kWaves * kChunk));
    }
    __device__ __forceinline__ float4 load(int c) const {
        const int v = at(c) + 4 * lane;
        if constexpr (kVec) {
            return v < end ? *reinterpret_cast<const float4*>(x + v)
                           : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        } else {
            return make_float4(v < end ? x[v] : -INFINITY, v + 1 < end ? x[v + 1] : -INFINITY,
                               v + 2 < end ? x[v + 2] : -INFINITY, v + 3 < end ? x[v + 3] : -INFINITY);
        }
    }
    // f(token, 4 logits) of every chunk, and with kTiles after(tile) behind each tile, by
    // all lanes of a wave
    template <typename F, typename G>
    __device__ __forceinline__ void each(F f, G after) {
#pragma unroll 1
        for (int c = 0; at(kTiles ? c / 4 * 4 : c) < end; ++c) {
            const float q[4] = {b0.x, b0.y, b0.z, b0.w};
            b0 = b1;
            b1 = b2;
            b2 = b3;
            b3 = load(c + 4);
            f(at(c) + 4 * lane, q);
            if (kTiles && c % 4 == 3) after(at(c) / kTile);
        }
    }
};

// ------------------------------------------------------------- largest logit
// And, for the bins, a small one of those that may have a weight beside it: logits of
// -10000 for tokens that do not exist or are not allowed would leave the others few
// bins.  It is some such logit, not the least: a lane forgets what it has when its
// largest one rises out of reach of it, and lanes and slices whose small one is out of
// the largest one's reach do not count, also where others of theirs are in it.  What
// lies below goes into the last bin.
//
// Bound by memory: 64 rows of 200064 (51 MB) 10.8 us, 4.7 TB/s; one row 3.6.
template <bool kVec, bool kLow>
__global__ __launch_bounds__(kThreads) void sample_best_kernel(const SampleArgs a) {
    __shared__ unsigned long long red[kThreads / kWave];
    __shared__ uint32_t lows[kThreads / kWave];
    const int row = static_cast<int>(blockIdx.x) / a.slices, slice = static_cast<int>(blockIdx.x) % a.slices;
    const float reach = reach_of(a, row);
    float top = -INFINITY, low = INFINITY, from = INFINITY;  // from: the smallest in reach
    int token = 0;
    Stream<kVec, false>(a, row, slice).each([&](int v, const float (&x)[4]) {
        const float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));  // of numbers, whatever NaN are beside them
        if (most > top) {
            top = most;
            token = v + (x[0] == most ? 0 : x[1] == most ? 1 : x[2] == most ? 2 : 3);
            from = fmaxf(top - reach, -FLT_MAX);
            if (low < from) low = top;
        }
        if constexpr (kLow) {
#pragma unroll
            for (int i = 0; i < 4; ++i) low = fminf(low, x[i] >= from ? x[i] : INFINITY);
        }
    }, [](int) {});
    unsigned long long best =
        top > -INFINITY ? (static_cast<unsigned long long>(order_of(top)) << 32) | (0xFFFFFFFFu - token) : 0ull;
    best = wave_max(best);
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) best = red[i] > best ? red[i] : best;
    const float most = logit_of(static_cast<uint32_t>(best >> 32));
    const uint32_t mine = wave_min(best != 0ull && low < INFINITY && !(low < most - reach) ? order_of(low) : 0xFFFFFFFFu);
    if (threadIdx.x % kWave == 0) lows[threadIdx.x / kWave] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        a.best[blockIdx.x] = best;
        a.low[blockIdx.x] = min(min(lows[0], lows[1]), min(lows[2], lows[3]));
    }
}

// The row's ends from its slices', by every wave for itself.
__device__ __forceinline__ Ends row_ends(const SampleArgs& a, int row) {
    static_assert(kMaxSlices <= kWave, "a lane a slice");
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    const size_t at = static_cast<size_t>(row) * a.slices + lane;
    Ends e{0ull, 0xFFFFFFFFu};
    if (lane < a.slices) e = Ends{a.best[at], a.low[at]};
    e.best = wave_max(e.best);
    const float most = logit_of(static_cast<uint32_t>(e.best >> 32));
    const bool near = e.low != 0xFFFFFFFFu && !(logit_of(e.low) < most - reach_of(a, row));
    e.low = min(wave_min(near ? e.low : 0xFFFFFFFFu), static_cast<uint32_t>(e.best >> 32));
    return e;
}

// ------------------------------------------------------- weights by their size
// kCount, kMass: what the cuts that the call asks for need (top-k, top-p).  Bound by
// the weights, some 25 instructions in fp64 each: 64 rows of 200064 with top-p 21.6 us
// (19.0 go to the weights' sum alone), with top-k, which asks for none, 11.3; one row
// with both 6.1.
template <bool kVec, bool kCount, bool kMass>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs a) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    const int row = static_cast<int>(blockIdx.x) / a.slices, slice = static_cast<int>(blockIdx.x) % a.slices;
    Stream<kVec, false> in(a, row, slice);
    static_assert(kBins == kThreads, "a thread a bin");
    mass[threadIdx.x] = 0ull;
    count[threadIdx.x] = 0u;
    const Ends ends = row_ends(a, row);
    const Scale s(a, row, ends);
    if (ends.best == 0ull || s.greedy) return;
    __syncthreads();
    in.each([&](int, const float (&x)[4]) {
        bool any[4];
        int b[4];
        unsigned long long w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double y = s.log2w(x[i]);
            any[i] = Scale::any(y);
            b[i] = s.bin(y);
            if constexpr (kMass) w[i] = Scale::weight(y);  // of any(y) only is used
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!any[i]) continue;
            if constexpr (kMass) atomicAdd(&mass[b[i]], w[i]);
            if constexpr (kCount) atomicAdd(&count[b[i]], 1u);
        }
    }, [](int) {});
    __syncthreads();
    const size_t at = static_cast<size_t>(blockIdx.x) * kBins + threadIdx.x;
    if constexpr (kMass) a.mass[at] = mass[threadIdx.x];
    if constexpr (kCount) a.count[at] = count[threadIdx.x];
}

// --------------------------------------------- kept weights, and the cut's bins
struct Bins {
    unsigned long long mass[kBins + 1];  // before bin b
    uint32_t count[kBins + 1];
    union {
        struct {
            unsigned long long mass[kThreads / kWave][kBins];
            uint32_t count[kThreads / kWave][kBins];
        } part;
        struct {
            unsigned long long mass[kThreads / kWave];
            uint32_t count[kThreads / kWave];
        } wave;
    };
    int first[3];
};

// The row's bins from its slices': a wave takes every fourth slice, 4 bins a lane.
template <bool kCount, bool kMass>
__device__ __forceinline__ void count_bins(const SampleArgs& a, int row, Bins& s) {
    const int t = static_cast<int>(threadIdx.x), lane = t % kWave, wave = t / kWave;
    unsigned long long ms[4] = {};
    uint32_t ns[4] = {};
#pragma unroll 4
    for (int i = wave; i < a.slices; i += kThreads / kWave) {
        const size_t at = (static_cast<size_t>(row) * a.slices + i) * kBins + 4 * lane;
        if constexpr (kMass) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(a.mass + at);
            const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(a.mass + at + 2);
            ms[0] += x.x; ms[1] += x.y; ms[2] += y.x; ms[3] += y.y;
        }
        if constexpr (kCount) {
            const uint4 x = *reinterpret_cast<const uint4*>(a.count + at);
            ns[0] += x.x; ns[1] += x.y; ns[2] += x.z; ns[3] += x.w;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s.part.mass[wave][4 * lane + i] = ms[i];
        s.part.count[wave][4 * lane + i] = ns[i];
    }
    if (t < 3) s.first[t] = kBins;
    __syncthreads();
    unsigned long long m = 0ull;
    uint32_t n = 0u;
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) {
        m += s.part.mass[i][t];
        n += s.part.count[i][t];
    }
    __syncthreads();
    m = running_sum(m);
    n = running_sum(n);
    if (lane == kWave - 1) {
        s.wave.mass[wave] = m;
        s.wave.count[wave] = n;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / kWave - 1; ++i)
        if (i < wave) {
            m += s.wave.mass[i];
            n += s.wave.count[i];
        }
    s.mass[t + 1] = m;
    s.count[t + 1] = n;
    if (t == 0) {
        s.mass[0] = 0ull;
        s.count[0] = 0u;
    }
    __syncthreads();
}

// Thread b's bin is the first whose end reaches what is asked.
__device__ __forceinline__ RowState find_bins(const SampleArgs& a, int row, Bins& s) {
    const int t = static_cast<int>(threadIdx.x);
    const uint32_t k = most_kept(a, row);
    if (s.count[t] < k && s.count[t + 1] >= k) s.first[0] = t;
    __syncthreads();
    RowState r{};
    r.total = s.mass[kBins];
    r.bin_k = k < s.count[kBins] ? s.first[0] : kBins;
    const bool cut = r.bin_k < kBins;
    r.base_k = cut ? s.mass[r.bin_k] : 0ull;
    r.count_k = cut ? s.count[r.bin_k] : 0u;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const bool part = p < 1.0f;
    const unsigned long long lo = share_of(p, cut ? s.mass[r.bin_k] : r.total);
    const unsigned long long hi = share_of(p, cut ? s.mass[r.bin_k + 1] : r.total);
    if (part && s.mass[t] < lo && s.mass[t + 1] >= lo) s.first[1] = t;
    if (part && s.mass[t] < hi && s.mass[t + 1] >= hi) s.first[2] = t;
    __syncthreads();
    r.p_lo = part ? s.first[1] : kBins;
    r.p_hi = part ? s.first[2] : kBins;
    r.base_p = part ? s.mass[r.p_lo] : 0ull;
    return r;
}

// One wave's tokens on their way to their weights, 64 at a time.
constexpr int kQueue = 2 * kChunk;
// From so many of a chunk's tokens on they are weighed where they are.  us for 64 rows
// of 200064 with top-p of 0.9 / 0.999, a quarter of a chunk: 23.9 / 32.8, a half: 23.7 /
// 35.2, always in the queue: 23.7 / 37.5.
constexpr int kDense = kChunk / 4;
struct Queue {
    float x[kQueue];
    int v[kQueue];
};

// kCount, kMass: top-k or top-p may cut; kLeast: min_p may drop tokens.  Without
// any a token goes straight to its weight, else those that a comparison of floats
// cannot rule out go through a queue, so that the others cost no fp64 work.  64 rows
// of 200064 take 19.0 us without cuts, with top-p of 0.5 / 0.9 / 0.999 18.7 / 23.8 /
// 33.1, of which the row's bins, summed by every workgroup for itself, are some 5; one
// row 8.3 with every filter.
template <bool kVec, bool kCount, bool kMass, bool kLeast>
__global__ __launch_bounds__(kThreads) void sample_keep_kernel(const SampleArgs a) {
    constexpr bool kCuts = kCount || kMass, kDirect = !kCuts && !kLeast;
    __shared__ std::conditional_t<kCuts, Bins, char> bins;
    __shared__ Queue queues[kDirect ? 1 : kThreads / kWave];
    __shared__ uint2 list[kCuts ? kSliceMost : 1];
    __shared__ uint32_t listed;
    const int row = static_cast<int>(blockIdx.x) / a.slices, slice = static_cast<int>(blockIdx.x) % a.slices;
    const int lane = static_cast<int>(threadIdx.x) % kWave, wave = static_cast<int>(threadIdx.x) / kWave;
    Stream<kVec, true> in(a, row, slice);
    const Ends ends = row_ends(a, row);
    const Scale s(a, row, ends);
    if (ends.best == 0ull || s.greedy) return;
    RowState r{};
    r.bin_k = r.p_lo = r.p_hi = kBins;
    if constexpr (kCuts) {
        if (threadIdx.x == 0) listed = 0u;
        count_bins<kCount, kMass>(a, row, bins);
        r = find_bins(a, row, bins);
        if (slice == 0 && threadIdx.x == 0) a.state[row] = r;
    }
    const unsigned long long least = least_weight(a, row);
    unsigned long long sum = 0ull;
    const auto store = [&](int tile) {
        const unsigned long long all = wave_sum(sum);
        if (lane == 0) a.tile[static_cast<size_t>(row) * a.tiles + tile] = all;
        sum = 0ull;
    };
    if constexpr (kDirect) {
        in.each([&](int, const float (&x)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += Scale::weight_or_none(s.log2w(x[i]));
        }, store);
        return;
    }
    // The bins that are kept whatever the cuts, and the last that may be touched by one.
    const int before = min(r.p_lo, r.bin_k);
    const int last = before == kBins ? kBins - 1 : max(r.p_lo < kBins ? r.p_hi : -1, r.bin_k < kBins ? r.bin_k : -1);
    // No logit below `from` is in them: the bin's end, or min_p where nothing cuts, some 2^-22 lower.
    double reach = s.per_bin > 0.0 && last < kBins - 1 ? (last + 1) / s.per_bin : kDepth;
    if (before == kBins && least > 1ull) reach = fmin(reach, 43.0 - log2(static_cast<double>(least)));
    const double edge = s.m - (reach + 0x1p-20) / s.c;
    const float from = s.infinite ? INFINITY
                                  : static_cast<float>(edge - (fabs(edge) + fabs(s.m)) * 0x1p-22 - 0x1p-140);
    volatile Queue& queue = queues[wave];
    int head = 0, held = 0;  // the same in every lane
    const auto in_cut = [&](int b) { return kCuts & ((b == r.bin_k) | ((b >= r.p_lo) & (b <= r.p_hi))); };
    const auto note = [&](float x, int v) {
        const uint32_t i = atomicAdd(&listed, 1u);
        if (i < kSliceMost) list[i] = make_uint2(__builtin_bit_cast(uint32_t, x), v);
    };
    const auto weigh = [&](int n) {
        if (lane >= n) return;
        const int at = (head + lane) % kQueue;
        const float x = queue.x[at];
        const double y = s.log2w(x);
        if (!Scale::any(y)) return;
        const int b = kCuts ? s.bin(y) : 0;
        const unsigned long long w = Scale::weight(y);
        sum += (b < before && w >= least) ? w : 0ull;
        if (b >= before && in_cut(b)) note(x, kCuts ? queue.v[at] : 0);
    };
    in.each([&](int v, const float (&x)[4]) {
        uint64_t mask[4];
        int taken = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mask[i] = __builtin_amdgcn_ballot_w64(x[i] >= from);
            taken += __builtin_popcountll(mask[i]);
        }
        if (taken >= kDense) {
            uint32_t cut = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double y = s.log2w(x[i]);
                const unsigned long long w = Scale::weight_or_none(y);
                const int b = kCuts ? s.bin(y) : 0;
                const bool any = Scale::any(y);
                sum += (any & (b < before) & (w >= least)) ? w : 0ull;
                cut |= (any & (b >= before) & in_cut(b)) ? 1u << i : 0u;
            }
            if (kCuts && cut != 0u) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((cut >> i) & 1u) note(x[i], v + i);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (x[i] >= from) {
                const int at = (head + held + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask[i] >> 32),
                                              __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask[i]), 0u))) % kQueue;
                queue.x[at] = x[i];
                if constexpr (kCuts) queue.v[at] = v + i;
            }
            held += __builtin_popcountll(mask[i]);
        }
#pragma unroll 1
        for (; held >= kWave; held -= kWave) {
            weigh(kWave);
            head = (head + kWave) % kQueue;
        }
    }, [&](int tile) {
        weigh(held);
        head = held = 0;
        store(tile);
    });
    if constexpr (kCuts) {
        __syncthreads();
        if (threadIdx.x == 0) a.listed[blockIdx.x] = listed;
        for (int i = static_cast<int>(threadIdx.x); i < static_cast<int>(min(listed, 1u * kSliceMost)); i += kThreads)
            a.list[static_cast<size_t>(blockIdx.x) * kSliceMost + i] = list[i];
    }
}

// ------------------------------------------------------------------ the token
constexpr int kLast = 1024;   // threads
constexpr int kPartBits = 8;
constexpr int kParts = 1 << kPartBits;  // of one level of a selection, 4 a lane of one wave
constexpr int kRankBits = 20;
static_assert(kTile == kLast && kMaxVocab / kTile <= kLast, "a thread a token, a tile");

// A token's place in the ranking: larger comes first, no two alike.
__device__ __forceinline__ unsigned long long rank_of(float x, int v) {
    return (static_cast<unsigned long long>(order_of(x)) << kRankBits) | static_cast<unsigned long long>(kMaxVocab - 1 - v);
}
__device__ __forceinline__ int token_of(unsigned long long rank) {
    return kMaxVocab - 1 - static_cast<int>(rank & (kMaxVocab - 1));
}

struct Last {
    unsigned long long mass[kParts];
    uint32_t count[kParts];
    unsigned long long wave_mass[kLast / kWave];
    unsigned long long key[kWave], weight[kWave];
    unsigned long long found, found_mass, total, target, before, low, high;
    uint32_t found_count, found_held, few, upto[kMaxSlices];
    int found_part, tile;
    unsigned long long tiles[kMaxVocab / kTile];
    unsigned long long rank[kListMost], held[kListMost];  // held: weight, and the bin above kBinShift
};
constexpr int kBinShift = 48;

// Running sums over the block: thread t's inclusive one.
__device__ __forceinline__ unsigned long long block_scan(Last& s, unsigned long long m) {
    const int t = static_cast<int>(threadIdx.x), wave = t / kWave;
    m = running_sum(m);
    if (t % kWave == kWave - 1) s.wave_mass[wave] = m;
    __syncthreads();
    m += wave_sum(t % kWave < wave ? s.wave_mass[t % kWave] : 0ull);
    __syncthreads();
    return m;
}

// Tokens of a step: one a lane, or (N = 4) four neighbouring ones a lane, all of the
// wave's `mine` of one logit and so of one weight w.
template <int N>
struct Some {
    unsigned long long key[N], w;
    bool mine[N];

    // Their weights, and with kCount their number, to mass[place] and count[place], place =
    // f(key): as one sum where a wave's lie in one place, or lane by lane.
    template <bool kCount, typename F>
    __device__ __forceinline__ void add(unsigned long long* mass, uint32_t* count, F f) const {
        int at[N], here = -1;
        bool alike = true;  // this lane's
#pragma unroll
        for (int i = 0; i < N; ++i) {
            at[i] = f(key[i]);
            alike = alike && (!mine[i] || here < 0 || at[i] == here);
            here = mine[i] ? at[i] : here;
        }
        const uint64_t any = __builtin_amdgcn_ballot_w64(here >= 0);
        if (any == 0ull) return;
        const int first = __builtin_ctzll(any), there = __builtin_amdgcn_readlane(here, first);
        if (__builtin_amdgcn_ballot_w64(!alike || (here >= 0 && here != there)) == 0ull) {
            uint32_t n = 0u;
#pragma unroll
            for (int i = 0; i < N; ++i) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine[i]));
            const unsigned long long sum = N > 1 ? w * n : wave_sum(mine[0] ? w : 0ull);
            if (static_cast<int>(threadIdx.x) % kWave == first) {
                atomicAdd(&mass[there], sum);
                if constexpr (kCount) atomicAdd(&count[there], n);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (mine[i]) {
                    atomicAdd(&mass[at[i]], w);
                    if constexpr (kCount) atomicAdd(&count[at[i]], 1u);
                }
        }
    }
};

// The tokens that a cut may fall on: the list, or where it did not hold them all the
// row.
struct Source {
    const SampleArgs& a;
    const Scale& scale;
    Last& s;
    int row, n;
    bool whole;

    // f(Some) of the tokens of bins [lo, hi] with ranks [low, low + span), by whole waves
    // that hold any.  kRanksOnly: whatever their bins, no weights.
    template <bool kRanksOnly, typename F>
    __device__ __forceinline__ void each(int lo, int hi, unsigned long long low, unsigned long long span, F f) const {
        const int t = static_cast<int>(threadIdx.x);
        if (!whole) {
#pragma unroll 1
            for (int i = t; i - t % kWave < n; i += kLast) {
                const unsigned long long w = i < n ? s.held[i] : 0ull, key = i < n ? s.rank[i] : 0ull;
                const int b = static_cast<int>(w >> kBinShift);
                const bool mine = i < n && b >= lo && b <= hi && key - low < span;
                if (__builtin_amdgcn_ballot_w64(mine) != 0ull)
                    f(Some<1>{{key}, w & ((1ull << kBinShift) - 1), {mine}});
            }
            return;
        }
        // A comparison of floats first, and of one logit's equals only those in range: a
        // vector instruction a token is 1.3 us of a row of 200064 by one workgroup.
        // The range's end is held to the first token of +inf: the topmost of a selection's
        // equal parts may reach past it, into ranks of no logit.
        const unsigned long long first = (static_cast<unsigned long long>(order_of(INFINITY)) << kRankBits) | (kMaxVocab - 1);
        const unsigned long long end = low + span - 1 < first ? low + span - 1 : first;
        const uint32_t o0 = static_cast<uint32_t>(low >> kRankBits), o1 = static_cast<uint32_t>(end >> kRankBits);
        const float x0 = logit_of(o0), x1 = logit_of(o1);
        const int v0 = o0 == o1 ? token_of(end) & ~3 : 0, v1 = o0 == o1 ? min(n, token_of(low) + 1) : n;
        // four neighbouring tokens a thread, the next ones on their way
        const float* x = a.logits + static_cast<size_t>(row) * a.vocab;
        const auto load = [&](int v) {
            return make_float4(v < v1 ? x[v] : -INFINITY, v + 1 < v1 ? x[v + 1] : -INFINITY,
                               v + 2 < v1 ? x[v + 2] : -INFINITY, v + 3 < v1 ? x[v + 3] : -INFINITY);
        };
        constexpr int kStep = 4 * kLast;
        float4 next = load(v0 + 4 * t), then = load(v0 + 4 * t + kStep), last = load(v0 + 4 * t + 2 * kStep);
#pragma unroll 1
        for (int v = v0 + 4 * t; v - 4 * (t % kWave) < v1; v += kStep) {
            float4 q = next;
            next = then;
            then = last;
            last = load(v + 3 * kStep);
            const float z[4] = {q.x, q.y, q.z, q.w};
            float here = 0.0f;  // a logit of this lane's that is in range
            bool in[4], alike = true, any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                in[i] = z[i] >= x0 && z[i] <= x1;
                alike = alike && (!in[i] || !any || z[i] == here);
                here = in[i] ? z[i] : here;
                any = any || in[i];
            }
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(any);
            if (lanes == 0ull) continue;
            const float there = __builtin_bit_cast(
                float, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, here), __builtin_ctzll(lanes)));
            if (__builtin_amdgcn_ballot_w64(!alike || (any && here != there)) == 0ull) {
                Some<4> some;
                some.w = 0ull;
                if constexpr (!kRanksOnly) {
                    const double y = scale.log2w(there);
                    const int b = scale.bin(y);
                    if (!Scale::any(y) || b < lo || b > hi) continue;
                    some.w = Scale::weight(y);
                }
                const unsigned long long top = rank_of(there, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    some.key[i] = top - static_cast<uint32_t>(v + i);
                    some.mine[i] = in[i] && some.key[i] - low < span;
                }
                f(some);
                continue;
            }
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
                const float x = q.x;
                q = make_float4(q.y, q.z, q.w, 0.0f);
                const unsigned long long key = rank_of(x, v + j);
                bool mine = x >= x0 && x <= x1 && key - low < span;
                if (__builtin_amdgcn_ballot_w64(mine) == 0ull) continue;
                unsigned long long w = 0ull;
                if constexpr (!kRanksOnly) {
                    const double y = scale.log2w(x);
                    const int b = scale.bin(y);
                    mine = mine && Scale::any(y) && b >= lo && b <= hi;
                    if (__builtin_amdgcn_ballot_w64(mine) == 0ull) continue;
                    w = Scale::weight_or_none(y);
                }
                f(Some<1>{{key}, w, {mine}});
            }
        }
    }
};

// The rank of the last kept token among those of bins [lo, hi], of which `mass` and
// `count` come before: the first whose running count reaches `want_count` or
// whose running weight reaches `want_mass`.  Level by level over a range of ranks
// [s.low, s.high] in kParts equal parts, until a part holds no more than a wave;
// returns its rank and, in `mass`, the weight up to and with it.  s.mass, s.count
// and s.few are zero before and after.
__device__ __forceinline__ unsigned long long select_rank(const Source& src, int lo, int hi, uint32_t want_count,
                                                          unsigned long long want_mass, uint32_t count,
                                                          unsigned long long& mass) {
    Last& s = src.s;
    const int t = static_cast<int>(threadIdx.x), lane = t % kWave;
    const auto reached = [&](uint32_t cn, unsigned long long cm) { return cn >= want_count || cm >= want_mass; };
    unsigned long long low = s.low, span = s.high - low + 1;
    int shift = max(0, 64 - __builtin_clzll((span - 1) | 1ull) - kPartBits);
#pragma unroll 1
    for (;;) {
        src.each<false>(lo, hi, low, span, [&](const auto& some) {
            some.template add<true>(s.mass, s.count, [&](unsigned long long key) {
                return kParts - 1 - static_cast<int>((key - low) >> shift);
            });
        });
        __syncthreads();
        if (t < kWave) {
            unsigned long long m[4], all = 0ull;
            uint32_t n[4], held = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                all += m[i] = s.mass[4 * t + i];
                held += n[i] = s.count[4 * t + i];
                s.mass[4 * t + i] = 0ull;
                s.count[4 * t + i] = 0u;
            }
            unsigned long long upto = mass + running_sum(all) - all;
            uint32_t upto_n = count + running_sum(held) - held;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!reached(upto_n, upto) && reached(upto_n + n[i], upto + m[i])) {
                    s.found_part = 4 * t + i;
                    s.found_mass = upto;
                    s.found_count = upto_n;
                    s.found_held = n[i];
                }
                upto += m[i];
                upto_n += n[i];
            }
        }
        __syncthreads();
        const uint32_t held = s.found_held;
        mass = s.found_mass;
        count = s.found_count;
        low += static_cast<unsigned long long>(kParts - 1 - s.found_part) << shift;
        span = 1ull << shift;
        if (held <= kWave || shift == 0) break;
        shift = shift > kPartBits ? shift - kPartBits : 0;
    }
    src.each<false>(lo, hi, low, span, [&](const auto& some) {
#pragma unroll
        for (size_t j = 0; j < sizeof(some.mine); ++j) {
            if (!some.mine[j]) continue;
            const uint32_t i = atomicAdd(&s.few, 1u);
            if (i < kWave) {
                s.key[i] = some.key[j];
                s.weight[i] = some.w;
            }
        }
    });
    __syncthreads();
    if (t < kWave) {
        const int held = static_cast<int>(min(s.few, 1u * kWave));
        const bool mine = t < held;
        const unsigned long long key = mine ? s.key[t] : 0ull, w = mine ? s.weight[t] : 0ull;
        uint32_t n = count + 1;
        unsigned long long m = mass + w;
        for (int i = 0; i < held; ++i)
            if (s.key[i] > key) {
                ++n;
                m += s.weight[i];
            }
        if (mine && reached(n, m) && !reached(n - 1, m - w)) {
            s.found = key;
            s.found_mass = m;
        }
        if (t == 0) s.few = 0u;
    }
    __syncthreads();
    mass = s.found_mass;
    return s.found;
}

// One workgroup a row.  A chain of loads (the slices' ends, their lists, the token's
// tile), scans and barriers: 3.7 us without cuts for one row, 4.2 for 64.  With cuts it
// goes by the longest row's list, 1024 tokens a step of each pass over it: 7.9 / 9.2 for
// one row / 64 with top-k of 50, 9.8 / 12.5 with top-p of 0.95; 64 rows with top-p of 0.5 /
// 0.95 / 0.999, some 30 / 1100 / 2800 tokens in a list (N(0, 3) logits), 9.5 / 12.5 / 17.3.
// Where the lists did not hold the cut's bins it goes through the row for each level of
// a selection, bound by the vector instructions of one compute unit: a call for one row of
// 200064 equal logits takes 170 us with top-k of 1000 and 226 with top-p of 0.9, with a
// weight and a sum for each token instead of one for a wave's 299 and 411.
template <bool kCuts>
__global__ __launch_bounds__(kLast) void sample_token_kernel(const SampleArgs a) {
    __shared__ Last s;
    const int row = static_cast<int>(blockIdx.x), t = static_cast<int>(threadIdx.x);
    // every load whose place is known, before the first is waited for
    const int lane = t % kWave;
    const float u = a.uniform[row], p = a.top_p ? a.top_p[row] : 1.0f;
    const uint32_t k = most_kept(a, row);
    const uint32_t own = kCuts && lane < a.slices ? a.listed[static_cast<size_t>(row) * a.slices + lane] : 0u;
    RowState r{};
    if (kCuts) r = a.state[row];
    const unsigned long long weight_here = t < a.tiles ? a.tile[static_cast<size_t>(row) * a.tiles + t] : 0ull;
    const Ends ends = row_ends(a, row);
    const Scale scale(a, row, ends);
    if (ends.best == 0ull || scale.greedy) {
        if (t == 0) {
            a.tokens[row] = ends.best == 0ull ? -1 : static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(ends.best));
            a.probs[row] = ends.best == 0ull ? 0.0f : 1.0f;
        }
        return;
    }
    const unsigned long long least = least_weight(a, row);
    s.tiles[t] = weight_here;
    unsigned long long cut = 0ull;  // the last kept rank
    if (kCuts && (r.bin_k < kBins || r.p_lo < kBins)) {
        const uint32_t upto = running_sum(own);
        const uint32_t listed = last_lane(upto);
        const bool whole = listed > kListMost || __builtin_amdgcn_ballot_w64(own > kSliceMost) != 0ull;
        const Source src{a, scale, s, row, whole ? a.vocab : static_cast<int>(listed), whole};
        if (t < kParts) {
            s.mass[t] = 0ull;
            s.count[t] = 0u;
        }
        if (t < kMaxSlices) s.upto[t] = upto;
        if (t == 0) {
            s.low = ~0ull;
            s.high = 0ull;
            s.few = 0u;
            s.found_part = 0;
            s.found_held = 0u;
        }
        __syncthreads();
        if (!whole) {
            // the slices' lists behind each other, an entry a thread
            for (uint32_t i = t; i < listed; i += kLast) {
                int slice = 0;  // whose entries hold i
#pragma unroll
                for (int o = kMaxSlices / 2; o >= 1; o >>= 1)
                    if (s.upto[slice + o - 1] <= i) slice += o;
                const uint32_t first = slice > 0 ? s.upto[slice - 1] : 0u;
                const uint2 e = a.list[(static_cast<size_t>(row) * a.slices + slice) * kSliceMost + (i - first)];
                const float x = __builtin_bit_cast(float, e.x);
                const double y = scale.log2w(x);
                s.rank[i] = rank_of(x, static_cast<int>(e.y));
                s.held[i] = Scale::weight(y) | (static_cast<unsigned long long>(scale.bin(y)) << kBinShift);
            }
            __syncthreads();
        }
        // The range of their ranks: by the ends of the bins, some 2^-22 wider; of the last bin
        // and of a whole row, where levels are dear, by the tokens.
        const int lo = min(r.p_lo, r.bin_k), hi = max(r.p_lo < kBins ? r.p_hi : 0, r.bin_k < kBins ? r.bin_k : 0);
        const float top = logit_of(static_cast<uint32_t>(ends.best >> 32));
        float x0 = -FLT_MAX, x1 = top;
        if (scale.per_bin > 0.0) {
            const double wide = 1.0 / (scale.per_bin * scale.c), e0 = scale.m - (hi + 1) * wide, e1 = scale.m - (lo - 1) * wide;
            const double more = fabs(scale.m) * 0x1p-22 + 0x1p-140;
            if (hi < kBins - 1) x0 = fmaxf(static_cast<float>(e0 - fabs(e0) * 0x1p-22 - more), x0);
            x1 = fminf(static_cast<float>(e1 + fabs(e1) * 0x1p-22 + more), x1);
        }
        unsigned long long low = static_cast<unsigned long long>(order_of(x0)) << kRankBits;
        unsigned long long high = (static_cast<unsigned long long>(order_of(x1)) << kRankBits) | (kMaxVocab - 1);
        if (whole || x0 == -FLT_MAX) {
            const unsigned long long from = low, span = high - low + 1;
            low = ~0ull;
            high = 0ull;
            src.each<true>(lo, hi, from, span, [&](const auto& some) {
#pragma unroll
                for (size_t j = 0; j < sizeof(some.mine); ++j) {
                    low = some.mine[j] && some.key[j] < low ? some.key[j] : low;
                    high = some.mine[j] && some.key[j] > high ? some.key[j] : high;
                }
            });
            low = wave_min(low);
            high = wave_max(high);
        }
        if (lane == 0 && high != 0ull) {
            atomicMin(&s.low, low);
            atomicMax(&s.high, high);
        }
        __syncthreads();
        unsigned long long total = r.total;
#pragma unroll 1
        for (int by_p = 0; by_p < 2; ++by_p) {  // top-k, then top-p of what it leaves
            const int from = by_p ? r.p_lo : r.bin_k, upto = by_p ? r.p_hi : r.bin_k;
            if (from == kBins) continue;
            unsigned long long mass = by_p ? r.base_p : r.base_k;
            cut = select_rank(src, from, upto, by_p ? 0xFFFFFFFFu : k, by_p ? share_of(p, total) : ~0ull,
                              by_p ? 0u : r.count_k, mass);
            total = mass;
        }
        // the kept ones of the cut's bins join their tiles
        src.each<false>(lo, kBins - 1, cut, s.high - cut + 1, [&](auto some) {
#pragma unroll
            for (size_t j = 0; j < sizeof(some.mine); ++j) some.mine[j] = some.mine[j] && some.w >= least;
            some.template add<false>(s.tiles, nullptr, [&](unsigned long long key) { return token_of(key) / kTile; });
        });
        __syncthreads();
    }
    // the tile that the random number falls into
    const unsigned long long here = s.tiles[t];
    unsigned long long m = block_scan(s, here);
    if (t == kLast - 1) {
        const double at = u > 0.0f ? static_cast<double>(u) * static_cast<double>(m) : 0.0;
        s.total = m;
        s.target = at < static_cast<double>(m) ? min(static_cast<unsigned long long>(at), m - 1) : m - 1;
    }
    __syncthreads();
    const unsigned long long target = s.target;
    if (m > target && m - here <= target) {
        s.tile = t;
        s.before = m - here;
    }
    __syncthreads();
    // and its token
    const int v = s.tile * kTile + t;
    const float x = v < a.vocab ? a.logits[static_cast<size_t>(row) * a.vocab + v] : -INFINITY;
    const double y = scale.log2w(x);
    unsigned long long w = Scale::any(y) ? Scale::weight(y) : 0ull;
    if (w < least || (kCuts && rank_of(x, v) < cut)) w = 0ull;
    m = s.before + block_scan(s, w);
    if (m > target && m - w <= target) {
        a.tokens[row] = v;
        a.probs[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(s.total));
    }
}

// ----------------------------------------------------------------------- host
// Tiles of a slice at most, so that the tokens of the bin that a cut runs through,
// some 1.4 % of a row of normally distributed logits whatever their spread, stay
// within the slice's list: without a list the token's workgroup looks the row through.
constexpr int kSliceTiles = 48;

// Slices of a row: so many that the launch fills the chip, of whole steps.  What only
// top-k and top-p use (bins and lists, 11 KB a slice) has no place without them.
struct Plan {
    int slices, slice, tiles;
    size_t best, low, tile, mass, count, state, listed, list, bytes;  // where each begins
};

Plan plan_for(int n_rows, int vocab, bool cuts) {
    Plan p;
    p.tiles = (vocab + kTile - 1) / kTile;
    const int want = std::min((1024 + n_rows - 1) / n_rows, kMaxSlices);
    const int per = std::min((p.tiles + want - 1) / want, kSliceTiles);
    p.slice = per * kTile;
    p.slices = (p.tiles + per - 1) / per;
    size_t at = 0;
    auto place = [&](size_t& field, size_t bytes) {
        field = at;
        at += (bytes + 255) / 256 * 256;
    };
    const size_t rows = static_cast<size_t>(n_rows), pieces = rows * p.slices;
    place(p.best, pieces * sizeof(unsigned long long));
    place(p.low, pieces * sizeof(uint32_t));
    place(p.tile, rows * p.tiles * sizeof(unsigned long long));
    const size_t cut = cuts ? pieces : 0;
    place(p.mass, cut * kBins * sizeof(unsigned long long));
    place(p.count, cut * kBins * sizeof(uint32_t));
    place(p.state, cuts ? rows * sizeof(RowState) : 0);
    place(p.listed, cut * sizeof(uint32_t));
    place(p.list, cut * kSliceMost * sizeof(uint2));
    p.bytes = at;
    return p;
}

}  // namespace
}  // namespace asdsl

using namespace asdsl;

extern "C" size_t asdsl_sample_logits_work_bytes_cuts(int n_rows, int vocab, int cuts) {
    if (n_rows <= 0 || vocab <= 0 || vocab > kMaxVocab) return 0;
    return plan_for(n_rows, vocab, cuts != 0).bytes;
}

extern "C" size_t asdsl_sample_logits_work_bytes(int n_rows, int vocab) {
    return asdsl_sample_logits_work_bytes_cuts(n_rows, vocab, 1);
}

extern "C" asdsl_status asdsl_sample_logits(const float* logits, const float* uniform, const float* temperature,
                                            const int* top_k, const float* top_p, const float* min_p, int* tokens,
                                            float* probs, int n_rows, int vocab, void* work, size_t work_bytes,
                                            asdsl_stream_t stream) {
    const char* what = "sample_logits";
    ASDSL_CHECK_ARG(logits && uniform && tokens && probs, "%s: null pointer", what);
    ASDSL_CHECK_ARG(n_rows > 0 && vocab > 0, "%s: n_rows and vocab must be positive", what);
    ASDSL_CHECK_ARG(vocab <= kMaxVocab, "%s: vocab must be at most 2^20", what);
    const bool cuts = top_k || top_p;
    const Plan p = plan_for(n_rows, vocab, cuts);
    ASDSL_CHECK_ARG(fits_launch(static_cast<long long>(n_rows) * p.slices, kThreads) && fits_launch(n_rows, kLast),
                    "%s: too many rows: more than 2^32 work items", what);
    ASDSL_CHECK_ARG(work, "%s: needs a work buffer of %zu bytes", what, p.bytes);
    void* ws = nullptr;
    asdsl_status st = work_buffer(as_hip(stream), work, work_bytes, p.bytes, &ws, what);
    if (st != ASDSL_OK) return st;
    char* at = static_cast<char*>(ws);
    const SampleArgs a{logits, uniform, temperature, top_k, top_p, min_p, tokens, probs,
                       reinterpret_cast<unsigned long long*>(at + p.best),
                       reinterpret_cast<uint32_t*>(at + p.low),
                       reinterpret_cast<unsigned long long*>(at + p.mass),
                       reinterpret_cast<uint32_t*>(at + p.count),
                       reinterpret_cast<unsigned long long*>(at + p.tile),
                       reinterpret_cast<RowState*>(at + p.state),
                       reinterpret_cast<uint32_t*>(at + p.listed),
                       reinterpret_cast<uint2*>(at + p.list),
                       vocab, p.slices, p.slice, p.tiles};
    const bool vec = vocab % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0;
    const dim3 grid(static_cast<unsigned>(n_rows * p.slices)), block(kThreads);
    const hipStream_t hs = as_hip(stream);
    auto with = [&](auto is_vec, auto count, auto mass, auto drops) {
        constexpr bool kVec = decltype(is_vec)::value, kCount = decltype(count)::value, kMass = decltype(mass)::value;
        asdsl_status res = launch("sample_best_kernel", sample_best_kernel<kVec, kCount || kMass>, grid, block, 0, hs, a);
        if constexpr (kCount || kMass)
            if (res == ASDSL_OK)
                res = launch("sample_bins_kernel", sample_bins_kernel<kVec, kCount, kMass>, grid, block, 0, hs, a);
        if (res != ASDSL_OK) return res;
        return launch("sample_keep_kernel", sample_keep_kernel<kVec, kCount, kMass, decltype(drops)::value>, grid, block,
                      0, hs, a);
    };
    const std::true_type yes{};
    const std::false_type no{};
    auto by_cuts = [&](auto is_vec) {
        return top_k   ? top_p ? with(is_vec, yes, yes, yes) : with(is_vec, yes, no, yes)
               : top_p ? with(is_vec, no, yes, yes)
               : min_p ? with(is_vec, no, no, yes)
                       : with(is_vec, no, no, no);
    };
    st = vec ? by_cuts(yes) : by_cuts(no);
    if (st != ASDSL_OK) return st;
    return launch("sample_token_kernel", cuts ? sample_token_kernel<true> : sample_token_kernel<false>, dim3(n_rows),
                  dim3(kLast), 0, hs, a);
}
