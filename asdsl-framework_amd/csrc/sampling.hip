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
// last bits of the weights decide a whole number, so exponents are formed in fp64
// (full rate here): 2^-43 a weight, against some 2^-24 in fp32, which over a flat
// vocabulary of 200000 would move the token in some of every thousand draws.
#include "abi_util.hpp"
#include "device_common.hpp"

namespace asdsl {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 256;             // tokens of a wave's step, whose kept weight is noted
constexpr int kStep = kThreads * 4;    // tokens of a workgroup's step
constexpr int kBins = 256;             // of log2 weights in (-kDepth, 0]
constexpr double kDepth = 44.0;
constexpr int kListMost = 8192;        // tokens of the bins that a cut runs through
constexpr int kMaxSlices = 64;
constexpr int kMaxVocab = 1 << 20;     // 2^20 weights of 2^43 stay below 2^64
constexpr double kLog2eWide = 1.4426950408889634074;

// What a row's cuts leave open once its bins are counted.
struct RowState {
    unsigned long long total;   // weight of all
    unsigned long long base_p;  // weight of the bins before the first that the cut of top-p may run through
    unsigned long long base_k;  // weight and tokens of those before the one that the cut of top-k runs through
    int count_k;
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
    unsigned long long* mass;  // [rows][slices][kBins]
    uint32_t* count;           // [rows][slices][kBins]
    unsigned long long* tile;  // [rows][tiles]
    RowState* state;           // [rows]
    uint32_t* listed;          // [rows]
    uint2* list;               // [rows][list_cap] (logit, token)
    int vocab, slices, slice, tiles, list_cap;
};

// Larger for a larger logit, equal for both zeros; 0 for none.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x == 0.0f ? 0.0f : x);
    return (b >> 31) ? ~b : b | 0x80000000u;
}

// A row's weights.
struct Scale {
    float m;
    double c;  // log2(e) / temperature
    bool greedy;  // only the first is kept

    __device__ __forceinline__ Scale(const SampleArgs& a, int row, float top) : m(top) {
        const float t = a.temperature ? a.temperature[row] : 1.0f;
        greedy = !(t > 0.0f) || (a.top_k && a.top_k[row] == 1) || (a.top_p && a.top_p[row] <= 0.0f) ||
                 (a.min_p && a.min_p[row] > 1.0f);
        c = kLog2eWide / static_cast<double>(t);
    }
    // log2 of a token's weight, -kDepth or less where it has none (NaN and -inf among them)
    __device__ __forceinline__ double log2w(float x) const {
        if (x == m) return 0.0;
        const double d = static_cast<double>(x) - static_cast<double>(m);
        return x > -INFINITY && d > -INFINITY ? d * c : -2.0 * kDepth;
    }
    // 2^y in units of 2^-43, y in (-kDepth, 0]: a series of 2^f about 0 for |f| <= 1/2
    // (its 13th term is below 2^-52), times a power of two; 2^52 + w is rounded to a
    // whole number as it is added.
    static __device__ __forceinline__ unsigned long long weight(double y) {
        const double n = rint(y), f = (y - n) * 0.69314718055994530942;
        double p = 1.0 / 479001600.0;
        p = fma(p, f, 1.0 / 39916800.0);
        p = fma(p, f, 1.0 / 3628800.0);
        p = fma(p, f, 1.0 / 362880.0);
        p = fma(p, f, 1.0 / 40320.0);
        p = fma(p, f, 1.0 / 5040.0);
        p = fma(p, f, 1.0 / 720.0);
        p = fma(p, f, 1.0 / 120.0);
        p = fma(p, f, 1.0 / 24.0);
        p = fma(p, f, 1.0 / 6.0);
        p = fma(p, f, 0.5);
        p = fma(p, f, 1.0);
        p = fma(p, f, 1.0);
        const long long e = 1023 + 43 + static_cast<int>(n);
        const double r = fma(p, __builtin_bit_cast(double, e << 52), 0x1p52);
        return __builtin_bit_cast(unsigned long long, r) & 0xFFFFFFFFFFFFFull;
    }
    static __device__ __forceinline__ int bin(double y) {  // rising as weights fall
        return min(static_cast<int>(y * (-kBins / kDepth)), kBins - 1);
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

template <typename T, typename F>
__device__ __forceinline__ T wave_all(T v, F f) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = f(v, __shfl_xor(v, o, kWave));
    return v;
}

// f(token, logit) for a lane's 4 neighbouring tokens of every step of a slice, and
// after(tile) by all lanes of a wave behind each; kVec: rows lie in whole 16-byte
// units.
template <bool kVec, typename F, typename G>
__device__ __forceinline__ void over_slice(const SampleArgs& a, int row, int slice, F f, G after) {
    const float* x = a.logits + static_cast<size_t>(row) * a.vocab;
    const int end = min(a.vocab, (slice + 1) * a.slice);
    for (int v0 = slice * a.slice; v0 < end; v0 += kStep) {
        const int v = v0 + 4 * static_cast<int>(threadIdx.x);
        if constexpr (kVec) {
            if (v < end) {
                const float4 q = *reinterpret_cast<const float4*>(x + v);
                f(v, q.x); f(v + 1, q.y); f(v + 2, q.z); f(v + 3, q.w);
            }
        } else {
            float q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = v + i < end ? x[v + i] : -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v + i < end) f(v + i, q[i]);
        }
        after(v0 / kTile + static_cast<int>(threadIdx.x) / kWave);
    }
}

// ------------------------------------------------------------- largest logit
template <bool kVec>
__global__ __launch_bounds__(kThreads) void sample_best_kernel(const SampleArgs a) {
    __shared__ unsigned long long red[kThreads / kWave];
    const int row = static_cast<int>(blockIdx.x) / a.slices, slice = static_cast<int>(blockIdx.x) % a.slices;
    unsigned long long best = 0ull;
    over_slice<kVec>(a, row, slice, [&](int v, float x) {
        if (x > -INFINITY) {
            const unsigned long long key = (static_cast<unsigned long long>(order_of(x)) << 32) | (0xFFFFFFFFu - v);
            best = key > best ? key : best;
        }
    }, [](int) {});
    best = wave_all(best, [](auto p, auto q) { return p > q ? p : q; });
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kThreads / kWave; ++i) best = red[i] > best ? red[i] : best;
        a.best[blockIdx.x] = best;
        if (slice == 0) a.listed[row] = 0u;
    }
}

// The row's largest logit, by every wave for itself (0: nothing to draw from).
__device__ __forceinline__ unsigned long long row_best(const SampleArgs& a, int row) {
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    unsigned long long best = lane < a.slices ? a.best[static_cast<size_t>(row) * a.slices + lane] : 0ull;
    static_assert(kMaxSlices <= kWave, "a lane a slice");
    return wave_all(best, [](auto p, auto q) { return p > q ? p : q; });
}

__device__ __forceinline__ float logit_of(unsigned long long best) {
    const uint32_t o = static_cast<uint32_t>(best >> 32);
    return __builtin_bit_cast(float, (o >> 31) ? o & 0x7FFFFFFFu : ~o);
}

// ------------------------------------------------------- weights by their size
template <bool kVec>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs a) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t count[kBins];
    const int row = static_cast<int>(blockIdx.x) / a.slices, slice = static_cast<int>(blockIdx.x) % a.slices;
    static_assert(kBins == kThreads, "a thread a bin");
    mass[threadIdx.x] = 0ull;
    count[threadIdx.x] = 0u;
    __syncthreads();
    const unsigned long long best = row_best(a, row);
    const Scale s(a, row, logit_of(best));
    if (best == 0ull || s.greedy) return;
    over_slice<kVec>(a, row, slice, [&](int, float x) {
        const double y = s.log2w(x);
        if (y > -kDepth) {
            const int b = Scale::bin(y);
            atomicAdd(&mass[b], Scale::weight(y));
            atomicAdd(&count[b], 1u);
        }
    }, [](int) {});
    __syncthreads();
    const size_t at = static_cast<size_t>(blockIdx.x) * kBins + threadIdx.x;
    a.mass[at] = mass[threadIdx.x];
    a.count[at] = count[threadIdx.x];
}

// --------------------------------------------- kept weights, and the cut's bins
struct Bins {
    unsigned long long mass[kBins + 1];  // before bin b
    uint32_t count[kBins + 1];
    unsigned long long wave_mass[kThreads / kWave];
    uint32_t wave_count[kThreads / kWave];
    int first[3];
};

__device__ __forceinline__ void count_bins(const SampleArgs& a, int row, Bins& s) {
    const int t = static_cast<int>(threadIdx.x), lane = t % kWave;
    unsigned long long m = 0ull;
    uint32_t n = 0u;
    for (int i = 0; i < a.slices; ++i) {
        const size_t at = (static_cast<size_t>(row) * a.slices + i) * kBins + t;
        m += a.mass[at];
        n += a.count[at];
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const unsigned long long mo = __shfl_up(m, o, kWave);
        const uint32_t no = __shfl_up(n, o, kWave);
        if (lane >= o) {
            m += mo;
            n += no;
        }
    }
    if (lane == kWave - 1) {
        s.wave_mass[t / kWave] = m;
        s.wave_count[t / kWave] = n;
    }
    if (t < 3) s.first[t] = kBins;
    __syncthreads();
    for (int i = 0; i < t / kWave; ++i) {
        m += s.wave_mass[i];
        n += s.wave_count[i];
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
    RowState r;
    r.total = s.mass[kBins];
    r.bin_k = k < s.count[kBins] ? s.first[0] : kBins;
    const bool cut = r.bin_k < kBins;
    r.base_k = cut ? s.mass[r.bin_k] : 0ull;
    r.count_k = cut ? static_cast<int>(s.count[r.bin_k]) : 0;
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

// Whether a bin's tokens are all kept by the cuts, or the cut may run through it.
__device__ __forceinline__ bool before_cuts(const RowState& r, int b) { return b < min(r.p_lo, r.bin_k); }
__device__ __forceinline__ bool in_cut(const RowState& r, int b) {
    return b == r.bin_k || (b >= r.p_lo && b <= r.p_hi);
}

// kCuts: top-k or top-p may cut.
template <bool kVec, bool kCuts>
__global__ __launch_bounds__(kThreads) void sample_keep_kernel(const SampleArgs a) {
    __shared__ Bins bins;
    const int row = static_cast<int>(blockIdx.x) / a.slices, slice = static_cast<int>(blockIdx.x) % a.slices;
    const unsigned long long best = row_best(a, row);
    const Scale s(a, row, logit_of(best));
    if (best == 0ull || s.greedy) return;
    RowState r{};
    r.bin_k = r.p_lo = r.p_hi = kBins;
    if constexpr (kCuts) {
        count_bins(a, row, bins);
        r = find_bins(a, row, bins);
    }
    if (slice == 0 && threadIdx.x == 0) a.state[row] = r;
    const unsigned long long least = least_weight(a, row);
    const int lane = static_cast<int>(threadIdx.x) % kWave;
    unsigned long long sum = 0ull;
    over_slice<kVec>(a, row, slice, [&](int v, float x) {
        const double y = s.log2w(x);
        if (!(y > -kDepth)) return;
        const int b = Scale::bin(y);
        if (before_cuts(r, b)) {
            const unsigned long long w = Scale::weight(y);
            if (w >= least) sum += w;
        } else if (kCuts && in_cut(r, b)) {
            const uint32_t at = atomicAdd(&a.listed[row], 1u);
            if (at < static_cast<uint32_t>(a.list_cap))
                a.list[static_cast<size_t>(row) * a.list_cap + at] = make_uint2(__builtin_bit_cast(uint32_t, x), v);
        }
    }, [&](int tile) {
        const unsigned long long all = wave_all(sum, [](auto p, auto q) { return p + q; });
        if (lane == 0 && tile < a.tiles) a.tile[static_cast<size_t>(row) * a.tiles + tile] = all;
        sum = 0ull;
    });
}

// ------------------------------------------------------------------ the token
constexpr int kLast = 1024;   // threads
constexpr int kSub = 2048;    // bins of one level of a selection
constexpr int kRankBits = 20;

// A token's place in the ranking: larger comes first, no two alike.
__device__ __forceinline__ unsigned long long rank_of(float x, int v) {
    return (static_cast<unsigned long long>(order_of(x)) << kRankBits) | static_cast<unsigned long long>(kMaxVocab - 1 - v);
}

struct Last {
    unsigned long long mass[kSub];
    uint32_t count[kSub];
    unsigned long long wave_mass[kLast / kWave];
    uint32_t wave_count[kLast / kWave];
    unsigned long long key[kWave], weight[kWave];
    unsigned long long found, found_mass, total, target, before;
    int found_bin;
    uint32_t few;
    int tile, token;
    unsigned long long tiles[kMaxVocab / kTile];
    uint2 list[kListMost];
};

// Running sums over the block: thread t's inclusive ones.
__device__ __forceinline__ void block_scan(Last& s, unsigned long long& m, uint32_t& n) {
    const int t = static_cast<int>(threadIdx.x), lane = t % kWave;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const unsigned long long mo = __shfl_up(m, o, kWave);
        const uint32_t no = __shfl_up(n, o, kWave);
        if (lane >= o) {
            m += mo;
            n += no;
        }
    }
    if (lane == kWave - 1) {
        s.wave_mass[t / kWave] = m;
        s.wave_count[t / kWave] = n;
    }
    __syncthreads();
    for (int i = 0; i < t / kWave; ++i) {
        m += s.wave_mass[i];
        n += s.wave_count[i];
    }
    __syncthreads();
}

// The tokens that a cut may fall on: the list, or where it did not hold them all the row.
struct Source {
    const SampleArgs& a;
    const RowState& r;
    const Scale& scale;
    Last& s;
    int row, n;
    bool whole;
    // f(rank, weight) for those of bins [lo, hi]
    template <typename F>
    __device__ __forceinline__ void each(int lo, int hi, F f) const {
        const float* x = a.logits + static_cast<size_t>(row) * a.vocab;
        for (int i = static_cast<int>(threadIdx.x); i < n; i += kLast) {
            const float q = whole ? x[i] : __builtin_bit_cast(float, s.list[i].x);
            const int v = whole ? i : static_cast<int>(s.list[i].y);
            const double y = scale.log2w(q);
            if (!(y > -kDepth)) continue;
            const int b = Scale::bin(y);
            if (b >= lo && b <= hi) f(rank_of(q, v), Scale::weight(y));
        }
    }
};

// The rank of the last kept token among those of bins [lo, hi], of which `mass` and
// `count` come before: the first whose running count reaches `want_count` or
// whose running weight reaches `want_mass`.  Level by level over a range of ranks in
// kSub equal parts, until a part holds few; returns its rank and, in `mass`, the
// weight up to and with it.
__device__ unsigned long long select_rank(const Source& src, int lo, int hi, uint32_t want_count,
                                          unsigned long long want_mass, uint32_t count, unsigned long long& mass) {
    Last& s = src.s;
    const int t = static_cast<int>(threadIdx.x);
    unsigned long long low = 0ull, span = 1ull << (32 + kRankBits);  // ranks [low, low + span) in parts of 2^shift
    int shift = 32 + kRankBits - 11;
    static_assert(kSub == 1 << 11, "11 bits a level");
    for (;;) {
        for (int i = t; i < kSub; i += kLast) {
            s.mass[i] = 0ull;
            s.count[i] = 0u;
        }
        if (t == 0) {
            s.few = 0u;
            s.found_bin = 0;
        }
        __syncthreads();
        src.each(lo, hi, [&](unsigned long long key, unsigned long long w) {
            if (key >= low && key - low < span) {
                const int at = static_cast<int>((key - low) >> shift);
                atomicAdd(&s.mass[kSub - 1 - at], w);
                atomicAdd(&s.count[kSub - 1 - at], 1u);
            }
        });
        __syncthreads();
        // two neighbouring parts a thread
        const unsigned long long m0 = s.mass[2 * t], m1 = s.mass[2 * t + 1];
        const uint32_t n0 = s.count[2 * t], n1 = s.count[2 * t + 1];
        unsigned long long m = m0 + m1;
        uint32_t n = n0 + n1;
        block_scan(s, m, n);
        m += mass;
        n += count;
        const auto reached = [&](uint32_t cn, unsigned long long cm) { return cn >= want_count || cm >= want_mass; };
        const bool before = reached(n - n0 - n1, m - m0 - m1), after = reached(n, m);
        if (!before && after) {
            const bool first = reached(n - n1, m - m1);
            s.found_bin = first ? 2 * t : 2 * t + 1;
            s.found_mass = first ? m - m0 - m1 : m - m1;
            s.wave_count[0] = first ? n - n0 - n1 : n - n1;
        }
        __syncthreads();
        const int part = s.found_bin;
        mass = s.found_mass;
        count = s.wave_count[0];
        const uint32_t held = s.count[part];
        low += static_cast<unsigned long long>(kSub - 1 - part) << shift;
        span = 1ull << shift;
        if (held <= kWave || shift == 0) {
            src.each(lo, hi, [&](unsigned long long key, unsigned long long w) {
                if (key >= low && key - low < span) {
                    const uint32_t i = atomicAdd(&s.few, 1u);
                    s.key[i] = key;
                    s.weight[i] = w;
                }
            });
            __syncthreads();
            if (t < kWave) {
                const bool mine = t < static_cast<int>(held);
                const unsigned long long key = mine ? s.key[t] : 0ull, w = mine ? s.weight[t] : 0ull;
                uint32_t n = count + 1;
                unsigned long long m = mass + w;
                for (int i = 0; i < static_cast<int>(held); ++i) {
                    const unsigned long long ko = s.key[i];
                    if (ko > key) {
                        ++n;
                        m += s.weight[i];
                    }
                }
                if (mine && reached(n, m) && !reached(n - 1, m - w)) {
                    s.found = key;
                    s.found_mass = m;
                }
            }
            __syncthreads();
            mass = s.found_mass;
            return s.found;
        }
        shift = shift > 11 ? shift - 11 : 0;
        __syncthreads();
    }
}

template <bool kCuts>
__global__ __launch_bounds__(kLast) void sample_token_kernel(const SampleArgs a) {
    __shared__ Last s;
    const int row = static_cast<int>(blockIdx.x), t = static_cast<int>(threadIdx.x);
    const unsigned long long best = row_best(a, row);
    const Scale scale(a, row, logit_of(best));
    if (best == 0ull || scale.greedy) {
        if (t == 0) {
            a.tokens[row] = best == 0ull ? -1 : static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best));
            a.probs[row] = best == 0ull ? 0.0f : 1.0f;
        }
        return;
    }
    const unsigned long long least = least_weight(a, row);
    const RowState r = a.state[row];
    for (int i = t; i < a.tiles; i += kLast) s.tiles[i] = a.tile[static_cast<size_t>(row) * a.tiles + i];
    unsigned long long cut = 0ull;  // the last kept rank
    if (kCuts && (r.bin_k < kBins || r.p_lo < kBins)) {
        const uint32_t listed = a.listed[row];
        const bool whole = listed > static_cast<uint32_t>(a.list_cap);
        const Source src{a, r, scale, s, row, whole ? a.vocab : static_cast<int>(listed), whole};
        if (!whole)
            for (int i = t; i < src.n; i += kLast) s.list[i] = a.list[static_cast<size_t>(row) * a.list_cap + i];
        __syncthreads();
        unsigned long long total = r.total;
        if (r.bin_k < kBins) {
            total = r.base_k;
            cut = select_rank(src, r.bin_k, r.bin_k, most_kept(a, row), ~0ull,
                              static_cast<uint32_t>(r.count_k), total);
        }
        if (r.p_lo < kBins) {
            unsigned long long mass = r.base_p;
            cut = select_rank(src, r.p_lo, r.p_hi, 0xFFFFFFFFu, share_of(a.top_p[row], total), 0u, mass);
        }
        // the kept ones of the cut's bins join their tiles
        const int lo = min(r.p_lo, r.bin_k);
        src.each(lo, kBins - 1, [&](unsigned long long key, unsigned long long w) {
            if (key >= cut && w >= least)
                atomicAdd(&s.tiles[(kMaxVocab - 1 - static_cast<int>(key & (kMaxVocab - 1))) / kTile], w);
        });
    }
    __syncthreads();
    // the tile that the random number falls into, a thread a run of tiles
    const int per = (a.tiles + kLast - 1) / kLast;
    unsigned long long m = 0ull;
    uint32_t none = 0u;
    for (int i = t * per; i < min(a.tiles, (t + 1) * per); ++i) m += s.tiles[i];
    const unsigned long long own = m;
    block_scan(s, m, none);
    if (t == kLast - 1) {
        const float u = a.uniform[row];
        const double at = u > 0.0f ? static_cast<double>(u) * static_cast<double>(m) : 0.0;
        s.total = m;
        s.target = at < static_cast<double>(m) ? min(static_cast<unsigned long long>(at), m - 1) : m - 1;
    }
    __syncthreads();
    const unsigned long long target = s.target;
    if (m > target && m - own <= target) {
        unsigned long long before = m - own;
        int i = t * per;
        while (before + s.tiles[i] <= target) before += s.tiles[i++];
        s.tile = i;
        s.before = before;
    }
    __syncthreads();
    // and its token, 4 of a lane of one wave
    if (t >= kWave) return;
    const float* x = a.logits + static_cast<size_t>(row) * a.vocab;
    unsigned long long w[4], sum = 0ull;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = s.tile * kTile + 4 * t + i;
        const float q = v < a.vocab ? x[v] : -INFINITY;
        const double y = scale.log2w(q);
        w[i] = y > -kDepth ? Scale::weight(y) : 0ull;
        if (w[i] < least || rank_of(q, v) < cut) w[i] = 0ull;
        sum += w[i];
    }
    unsigned long long upto = sum;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const unsigned long long other = __shfl_up(upto, o, kWave);
        if (t >= o) upto += other;
    }
    unsigned long long run = s.before + upto - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (run <= target && run + w[i] > target) {
            a.tokens[row] = s.tile * kTile + 4 * t + i;
            a.probs[row] = static_cast<float>(static_cast<double>(w[i]) / static_cast<double>(s.total));
        }
        run += w[i];
    }
}

// ----------------------------------------------------------------------- host
// Slices of a row: so many that the launch fills the chip, of whole steps.
struct Plan {
    int slices, slice, tiles, list_cap;
    size_t best, mass, count, tile, state, listed, list, bytes;  // where each begins
};

Plan plan_for(int n_rows, int vocab) {
    Plan p;
    const int steps = (vocab + kStep - 1) / kStep;
    int want = (512 + n_rows - 1) / n_rows;
    want = want < kMaxSlices ? want : kMaxSlices;
    const int per = (steps + want - 1) / want;
    p.slice = per * kStep;
    p.slices = (steps + per - 1) / per;
    p.tiles = (vocab + kTile - 1) / kTile;
    p.list_cap = vocab < kListMost ? vocab : kListMost;
    size_t at = 0;
    auto place = [&](size_t& field, size_t bytes) {
        field = at;
        at += (bytes + 255) / 256 * 256;
    };
    const size_t rows = static_cast<size_t>(n_rows), pieces = rows * p.slices;
    place(p.best, pieces * sizeof(unsigned long long));
    place(p.mass, pieces * kBins * sizeof(unsigned long long));
    place(p.count, pieces * kBins * sizeof(uint32_t));
    place(p.tile, rows * p.tiles * sizeof(unsigned long long));
    place(p.state, rows * sizeof(RowState));
    place(p.listed, rows * sizeof(uint32_t));
    place(p.list, rows * p.list_cap * sizeof(uint2));
    p.bytes = at;
    return p;
}

}  // namespace
}  // namespace asdsl

using namespace asdsl;

extern "C" size_t asdsl_sample_logits_work_bytes(int n_rows, int vocab) {
    if (n_rows <= 0 || vocab <= 0 || vocab > kMaxVocab) return 0;
    return plan_for(n_rows, vocab).bytes;
}

extern "C" asdsl_status asdsl_sample_logits(const float* logits, const float* uniform, const float* temperature,
                                            const int* top_k, const float* top_p, const float* min_p, int* tokens,
                                            float* probs, int n_rows, int vocab, void* work, size_t work_bytes,
                                            asdsl_stream_t stream) {
    const char* what = "sample_logits";
    ASDSL_CHECK_ARG(logits && uniform && tokens && probs, "%s: null pointer", what);
    ASDSL_CHECK_ARG(n_rows > 0 && vocab > 0, "%s: n_rows and vocab must be positive", what);
    ASDSL_CHECK_ARG(vocab <= kMaxVocab, "%s: vocab must be at most 2^20", what);
    const Plan p = plan_for(n_rows, vocab);
    ASDSL_CHECK_ARG(fits_launch(static_cast<long long>(n_rows) * p.slices, kThreads) && fits_launch(n_rows, kLast),
                    "%s: too many rows: more than 2^32 work items", what);
    ASDSL_CHECK_ARG(work, "%s: needs a work buffer of %zu bytes", what, p.bytes);
    void* ws = nullptr;
    asdsl_status st = work_buffer(as_hip(stream), work, work_bytes, p.bytes, &ws, what);
    if (st != ASDSL_OK) return st;
    char* at = static_cast<char*>(ws);
    const SampleArgs a{logits, uniform, temperature, top_k, top_p, min_p, tokens, probs,
                       reinterpret_cast<unsigned long long*>(at + p.best),
                       reinterpret_cast<unsigned long long*>(at + p.mass),
                       reinterpret_cast<uint32_t*>(at + p.count),
                       reinterpret_cast<unsigned long long*>(at + p.tile),
                       reinterpret_cast<RowState*>(at + p.state),
                       reinterpret_cast<uint32_t*>(at + p.listed),
                       reinterpret_cast<uint2*>(at + p.list),
                       vocab, p.slices, p.slice, p.tiles, p.list_cap};
    const bool vec = vocab % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0;
    const bool cuts = top_k || top_p;
    const dim3 grid(static_cast<unsigned>(n_rows * p.slices)), block(kThreads);
    const hipStream_t hs = as_hip(stream);
    st = launch("sample_best_kernel", vec ? sample_best_kernel<true> : sample_best_kernel<false>, grid, block, 0, hs, a);
    if (st == ASDSL_OK && cuts)
        st = launch("sample_bins_kernel", vec ? sample_bins_kernel<true> : sample_bins_kernel<false>, grid, block, 0, hs,
                    a);
    if (st == ASDSL_OK)
        st = launch("sample_keep_kernel",
                    cuts ? (vec ? sample_keep_kernel<true, true> : sample_keep_kernel<false, true>)
                         : (vec ? sample_keep_kernel<true, false> : sample_keep_kernel<false, false>),
                    grid, block, 0, hs, a);
    if (st != ASDSL_OK) return st;
    return launch("sample_token_kernel", cuts ? sample_token_kernel<true> : sample_token_kernel<false>, dim3(n_rows),
                  dim3(kLast), 0, hs, a);
}
