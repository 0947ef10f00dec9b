// Attention of many tokens and sequences over KV caches, beside the decode
// step's single-sequence kernels: the cache append (RoPE of queries and keys,
// the new K/V rows), attention with a sliding window and first tokens that
// stay visible, and attention of sequences that share a prefix.
//
// Caches are [sequence][kv head][row][head_dim], fp16, or int8 codes with one
// fp32 scale per 64 dims (the decode step's two forms); queries and outputs
// are fp32.
#include <hip/hip_fp16.h>

#include <climits>
#include <type_traits>

#include "abi_util.hpp"
#include "device_common.hpp"

namespace asdsl {
namespace {

constexpr int kBlockDims = 64;  // dims per scale of an int8 cache
constexpr float kInv127 = 1.0f / 127.0f;
constexpr float kLog2e = 1.44269504088896340736f;

// One cache: K and V rows, and the scales of the int8 form.
struct Cache {
    const void* k;
    const void* v;
    const float* ks;
    const float* vs;
};

// ------------------------------------------------------------------ append
// Four dims of one head of one token per lane, so that loads and stores are 16
// neighbouring bytes a lane (8 of an fp16 row).  A rotated pair is (fmaf(a, c,
// -(b * s)), fmaf(a, s, b * c)), as in the decode step's attention, and the
// stored forms are its too: fp16 rounded to nearest, or per 64 dims scale =
// amax * (1/127) (1e-12 when amax <= 1e-12) and code = round-half-even(x * (1 /
// scale)) clamped to [-127, 127].
//
// Bound by memory: 2045 tokens of 24 + 2 * 8 heads of 128 dims move 76 MB in 18.1 us
// where nothing of a call is in the caches (24 calls' buffers in turn; 4.2 TB/s, a
// copy of 1 GiB gets 5.15) and in 14.8 where the last call's are; into int8 caches
// 18.8 and 15.1.  A head per workgroup of scalar lanes took 47.  16 tokens take 3.0
// us (int8 3.1), of which the launch and one chain of loads (position, then
// tables) are nearly all.
struct AppendArgs {
    const float* qkv;
    void* k;
    void* v;
    float* ks;
    float* vs;
    const float* cos;
    const float* sin;
    const int* pos;
    float* q_out;
    int n_tokens, n_heads, n_kv, rot_half, rows, offset, rope_rows;
    int chunks;  // workgroups a token
};
constexpr int kAppendThreads = 256;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }

// kVec: rotary pairs and table rows lie in whole 16-byte units.
template <int D, bool Q8, bool kVec>
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(const AppendArgs a) {
    constexpr int kUnits = D / 4;  // per head
    const int heads = a.n_heads + 2 * a.n_kv;
    const int row = static_cast<int>(blockIdx.x) / a.chunks;  // token row of the call
    const int u = static_cast<int>(blockIdx.x) % a.chunks * kAppendThreads + static_cast<int>(threadIdx.x);
    const int head = u / kUnits, d = u % kUnits * 4;
    if (head >= heads) return;  // whole heads: the lanes of a 64-dim block leave together
    const int seq = row / a.n_tokens;
    const float* src = a.qkv + (static_cast<size_t>(row) * heads + head) * D;
    const float4 own = load4(src + d);
    const long long r = static_cast<long long>(a.pos[seq]) + row % a.n_tokens;  // cache row
    const long long p = r + a.offset;                                           // rotary position
    const bool inside = r >= 0 && r < a.rows && p >= 0 && p < a.rope_rows;
    if (!inside && head >= a.n_heads) return;
    float x[4] = {own.x, own.y, own.z, own.w};
    const int half = a.rot_half;
    if (!inside) {
        x[0] = x[1] = x[2] = x[3] = 0.0f;
    } else if (head < a.n_heads + a.n_kv && d < 2 * half) {
        const float* cs = a.cos + p * half;
        const float* sn = a.sin + p * half;
        if constexpr (kVec) {
            const bool first = d < half;
            const int j = first ? d : d - half;
            const float4 o = load4(src + (first ? d + half : j)), c4 = load4(cs + j), s4 = load4(sn + j);
            const float y[4] = {o.x, o.y, o.z, o.w}, c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = first ? fmaf(x[i], c[i], -(y[i] * s[i])) : fmaf(y[i], s[i], x[i] * c[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (d + i >= 2 * half) continue;
                const bool first = d + i < half;
                const int j = first ? d + i : d + i - half;
                const float lo = src[j], hi = src[j + half];
                x[i] = first ? fmaf(lo, cs[j], -(hi * sn[j])) : fmaf(lo, sn[j], hi * cs[j]);
            }
        }
    }
    if (head < a.n_heads) {
        *reinterpret_cast<float4*>(a.q_out + (static_cast<size_t>(row) * a.n_heads + head) * D + d) =
            make_float4(x[0], x[1], x[2], x[3]);
        return;
    }
    const bool key = head < a.n_heads + a.n_kv;
    const int kvh = head - a.n_heads - (key ? 0 : a.n_kv);
    const size_t crow = (static_cast<size_t>(seq) * a.n_kv + kvh) * a.rows + static_cast<size_t>(r);
    void* base = key ? a.k : a.v;
    if constexpr (Q8) {
        const float m = group_max<16>(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        const float scale = m > 1e-12f ? m * kInv127 : 1e-12f;
        const float inv = 1.0f / scale;
        int q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = static_cast<int>(fminf(fmaxf(__builtin_rintf(x[i] * inv), -127.0f), 127.0f));
        *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(base) + crow * D + d) = pack4_i8(q[0], q[1], q[2], q[3]);
        if (d % kBlockDims == 0) (key ? a.ks : a.vs)[crow * (D / kBlockDims) + d / kBlockDims] = scale;
    } else {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[2 * i]))) |
                   (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[2 * i + 1]))) << 16);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + crow * D + d) = make_uint2(w[0], w[1]);
    }
}

// --------------------------------------------------------------- attention
// Scores and weights are fp32 in the definition, and K and V are fp16 numbers
// (or int8 codes, exact in fp16), so only the query and the weights have to be
// cut for the matrix instructions: each is held as the sum of two fp16 numbers,
// a first part of 11 bits and the rest (2^-22 off at most), at twice the
// products.  One part alone would leave 2^-12 a weight, 1e-4 of an output.
// The parts keep clear of fp16's small numbers: a query row is scaled by a power
// of two to 2^12..2^13, the weights are 2^kShift times theirs or more (the first
// part is then whole down to 2^-22 of the largest weight, the second to 2^-11 of
// it, and off by 2^-33 of it below; more costs bits of the exponent's argument).
//
// A wave takes 16 query rows (the columns of its tiles) and 32 keys a step:
//   S' = K Q'  two 16x16 tiles; a lane gets 8 scores of the one row it holds, so
//              the running maximum and sum need two lane exchanges a step
//   O' = V' P' the lane's 8 weights are its operand as they stand when V's is
//              read for the same 8 keys: every lane loads its D / 16 dims of those
//              keys and turns the block in registers; no transposition in memory.
// This form for few rows streams: 32 sequences of one token (24 heads of 128, 8 KV
// heads, int8 caches, about 3300 rows each seen, 232 MB) take 52.6 us and 4.8 of
// join, 4.4 TB/s, bound by HBM and by the bytes its waves keep on the way.  For
// small calls a workgroup's chain of position, first keys and join in LDS counts:
// 6.3 us at 128 keys, where a compute unit then draws 32 bytes a ns.  Keys of many
// rows, read once per 16 of them, are left to the other form.
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRows = 16;      // query rows of a wave's tile
constexpr int kKeys = 32;      // keys of a wave's step
constexpr float kShift = 8.0f;
constexpr float kMost = 14.0f;
constexpr int kFewWaves = 4;

// The keys of one KV head that a workgroup's rows see between them: rows [0, na)
// and then [na + db, N + db) of the cache, counted 0 .. N - 1.  `masked`: which
// of them a token t sees goes by its position p = p0 + t (rows [max(0, p -
// window + 1), p] and rows below sinks; window 0: all up to p).
struct Keys {
    const void* k;
    const void* v;
    const float* ks;
    const float* vs;
    int na, db, n;
    bool masked;
    int p_first;  // smallest position of the workgroup's tokens that is in the cache
    int lo_last;  // first row of the last such token's window
    int sinks;
};

// One query row as a lane holds it: what it sees, and whether it sees anything.
struct RowSight {
    int p, lo;
    bool any;
};

struct AttnArgs {
    const float* q;
    float* out;
    float* part;    // [q row][slots][D] then, at ml, [q row][slots] (maximum, sum)
    float2* ml;
    Cache a, b;
    const int* pos;
    int n_seq, n_tokens, n_heads, n_kv, rows_a, rows_b;
    int prefix;  // shared prefix: its rows; -1 with a window
    int window, sinks;
    int splits, slots;  // key splits of this launch's jobs, partials kept per row
    float scale;        // log2(e) / sqrt(D)
};

// f over the lanes that hold one row: lane % kStep is the same (16: four lanes,
// 32: two).  A swap exchanges one half (or odd rows of 16) of a register with
// the other half of a second one, so with two copies of v the results hold
// both lanes' values.  The copy is kept apart from v: given one register twice,
// the swap leaves it as it is.
template <int kStep, typename F>
__device__ __forceinline__ float lanes(float v, F f) {
    uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
    asm("" : "+v"(b));
    auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    v = f(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
    if constexpr (kStep == 16) {
        a = b = __builtin_bit_cast(uint32_t, v);
        asm("" : "+v"(b));
        r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        v = f(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
              __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
    }
    return v;
}
template <int kStep>
__device__ __forceinline__ float lanes_max(float v) {
    return lanes<kStep>(v, [](float x, float y) { return fmaxf(x, y); });
}
template <int kStep>
__device__ __forceinline__ float lanes_sum(float v) {
    return lanes<kStep>(v, [](float x, float y) { return x + y; });
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float pow2(int e) {  // 2^e, -126 <= e <= 127
    return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ int exponent(float x) {
    return static_cast<int>((__builtin_bit_cast(uint32_t, x) >> 23) & 0xFFu) - 127;
}

constexpr float kLeast = 0x1p-126f;
// The factor 2^x of what was accumulated where a larger base comes, x <= 0: never
// zero, so that an infinite value of next to no weight stays one.
__device__ __forceinline__ float factor(float x) { return fmaxf(exp2_fast(x), kLeast); }

// x = hi + lo with fp16 parts, two at a time.
__device__ __forceinline__ void two_parts(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const half2v h = __builtin_convertvector((f32x2{x0, x1}), half2v);
    hi = __builtin_bit_cast(uint32_t, h);
    f32x2 d;  // x - h, exactly; the compiler converts h back in an instruction of its own
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d.x) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d.y) : "v"(hi), "v"(x1));
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(d, half2v));
}

__device__ __forceinline__ half8 as_half8(const uint32_t (&w)[4]) {
    return __builtin_bit_cast(half8, make_uint4(w[0], w[1], w[2], w[3]));
}

// Two int8 codes at bits 0-7 and 16-23 of w as fp16 numbers: with the top bit
// flipped a code is u = code + 128, and 0x6400 | u is 1024 + u, exactly.
__device__ __forceinline__ uint32_t codes_half2(uint32_t w) {
    const half2v h = __builtin_bit_cast(half2v, w ^ 0x64806480u) - half2v{_Float16(1152.0f), _Float16(1152.0f)};
    return __builtin_bit_cast(uint32_t, h);
}

// Eight int8 codes as the K operand's eight fp16 numbers.
__device__ __forceinline__ half8 codes_half8(uint2 c) {
    uint32_t w[4];
    w[0] = codes_half2(__builtin_amdgcn_perm(0u, c.x, 0x0C010C00u));
    w[1] = codes_half2(__builtin_amdgcn_perm(0u, c.x, 0x0C030C02u));
    w[2] = codes_half2(__builtin_amdgcn_perm(0u, c.y, 0x0C010C00u));
    w[3] = codes_half2(__builtin_amdgcn_perm(0u, c.y, 0x0C030C02u));
    return as_half8(w);
}

// A query row's operands: dims kDims * s + 8 * part .. + 8 in step s, part =
// lane / (512 / kDims): kDims 32 for 16x16 tiles, 16 for 32x32 tiles.
template <int D, int kDims>
struct Query {
    half8 hi[D / kDims], lo[D / kDims];
    float c;  // score = product * c, in powers of two

    __device__ __forceinline__ void load(const float* row, int part, float scale) {
        float x[D / kDims][8];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < D / kDims; ++s) {
            if (row) {
                const float4 a = *reinterpret_cast<const float4*>(row + kDims * s + 8 * part);
                const float4 b = *reinterpret_cast<const float4*>(row + kDims * s + 8 * part + 4);
                x[s][0] = a.x; x[s][1] = a.y; x[s][2] = a.z; x[s][3] = a.w;
                x[s][4] = b.x; x[s][5] = b.y; x[s][6] = b.z; x[s][7] = b.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[s][i]));
        }
        top = lanes_max<512 / kDims>(top);
        int e = 12 - exponent(top);  // a query that is not finite stays as it is
        e = e < -115 ? 0 : (e > 120 ? 120 : e);
        const float f = pow2(e);
        c = scale * pow2(-e);
#pragma unroll
        for (int s = 0; s < D / kDims; ++s) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) two_parts(x[s][2 * i] * f, x[s][2 * i + 1] * f, h[i], l[i]);
            hi[s] = as_half8(h);
            lo[s] = as_half8(l);
        }
    }
};

// The D / 16 operands of V for 8 keys, key i in half i: operand j has row
// lane % 16 = r for dim fp16_dim(r, j) or code_dim(r, j).
template <int D>
__device__ __forceinline__ int fp16_dim(int r, int j) { return D / 16 * r + j; }
__device__ __forceinline__ int code_dim(int r, int j) { return 64 * (j >> 2) + 4 * r + (j & 3); }

template <int D, bool Q8>
struct VRaw;
template <int D>
struct VRaw<D, false> {
    uint32_t w[8][D / 32];
    __device__ __forceinline__ void load(const char* row, int key, int r) {
        const char* src = row + D / 8 * r;
        if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(src);
            w[key][0] = x.x; w[key][1] = x.y; w[key][2] = x.z; w[key][3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            w[key][0] = x.x; w[key][1] = x.y;
        }
    }
    __device__ __forceinline__ half8 operand(int j) const {
        uint32_t o[4];
#pragma unroll
        for (int p = 0; p < 4; ++p)
            o[p] = __builtin_amdgcn_perm(w[2 * p + 1][j >> 1], w[2 * p][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        return as_half8(o);
    }
};
template <int D>
struct VRaw<D, true> {
    uint32_t w[8][D / 64];
    __device__ __forceinline__ void load(const char* row, int key, int r) {
        const char* src = row + 4 * r;
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
            w[key][b] = *reinterpret_cast<const uint32_t*>(src + 64 * b);
    }
    __device__ __forceinline__ half8 operand(int j) const {
        uint32_t o[4];
        const uint32_t sel = 0x0C040C00u + 0x00010001u * static_cast<uint32_t>(j & 3);
#pragma unroll
        for (int p = 0; p < 4; ++p)
            o[p] = codes_half2(__builtin_amdgcn_perm(w[2 * p + 1][j >> 2], w[2 * p][j >> 2], sel));
        return as_half8(o);
    }
};

// Running state of one query row, held by the lanes of equal lane % kStep: the
// base m of its weights exp2(score - m) and their sum over the lane's share of
// the keys.  A base is set kShift below the row's largest score so far and
// stays while the scores keep kTop above it at most: nearly always after a
// row's first keys, so that a step then needs no exchange between lanes and no
// scaling of what was accumulated.  Over int8 caches bases are whole numbers
// (Scaled).
template <bool Q8, int kStep>
struct Softmax {
    static constexpr float kTop = Q8 ? 12.9f : kMost;
    float m = -INFINITY, l = 0.0f;

    // Whether a step's products (score = s * c) ask for a new base in this lane;
    // top: the largest score.
    template <int N>
    __device__ __forceinline__ bool rises(const float (&s)[N], float c, float& top) const {
        top = s[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, s[i]);
        top *= c;
        return top - m > kTop;
    }
    // The new base where any lane of the wave asks for one: how far it rose.
    __device__ __forceinline__ float rebase(float top) {
        top = lanes_max<kStep>(top);
        const float m1 = top - m > kTop ? (Q8 ? ceilf(top) : top) - kShift : m;
        const float up = m == m1 ? 0.0f : m1 - m;
        m = m1;
        l *= exp2_fast(-up);
        return up;
    }
    // The weights of N keys from their products, in place.
    template <int N>
    __device__ __forceinline__ void weigh(float (&s)[N], float c) {
        const float base = m == -INFINITY ? 0.0f : m;
        float sum[4] = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = exp2_fast(fmaf(s[i], c, -base));
            sum[i & 3] += s[i];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
};

// An int8 cache's value scales go into a row's weights before those are cut into
// fp16 parts: products of weight and scale, times a power of two 2^-ev of the
// row's own, which puts the largest product so far at 2^8 or more, so that each is
// held to 2^-22 of itself or 2^-33 of the largest one, however far the scales are
// from each other and whatever weight the loud values have.  (By the largest
// scale, a loud value of small weight takes the bits of all others.)  The
// accumulators are 2^-ev times O'.  The base of the weights is a whole number:
// where it rises the accumulators stay and ev falls.  A step whose weights, 2^12.9
// at most, times scales stay below 2^15.9 by the scales' exponents alone needs no
// look at its products: nearly every one whose scales are within 4 of the others'.
// 4096 tokens over as many rows take 249 us, 245 by the largest scale (24 heads of
// 128, 8 KV heads); of 64 dims 235 and 246.
struct Scaled {
    static constexpr int kNone = 127;  // no keys yet: no scale asks for more
    static constexpr int kLow = -100;  // products below 2^-92 keep fewer bits
    static constexpr int kLook = -1000;
    int ev = kNone;

    // Whether a value scale, seen or not, asks for a look at the products.
    static __device__ __forceinline__ bool asks(float scale, int ev) { return exponent(fabsf(scale)) > ev + 2; }
    // The row's base has risen, from no keys (first) or by `rose`.
    __device__ __forceinline__ void rebase(bool first, float rose, bool keys) {
        ev = !first ? ev - static_cast<int>(fminf(rose, 1000.0f)) : keys ? kLow : kNone;
    }
    // The power for a step whose largest product in this lane is `most`: the factor
    // of the accumulators.
    template <int kStep>
    __device__ __forceinline__ float raise(float most) {
        const int held = ev;
        ev = max(max(held, exponent(lanes_max<kStep>(most)) - 8), kLow);
        return pow2(max(held - ev, -126));
    }
};

// A product of a weight and a scale where the scale is of any use (others make
// their weights infinite); zero for a key that the row does not see.
__device__ __forceinline__ float use(float weight, float scale) {
    const float a = fabsf(scale);
    return a < 1e30f ? weight * a : 0.0f;
}

// O' of 16 rows: element i of acc[j] at dim *_dim(4 * (lane / 16) + i, j).
template <int D, bool Q8>
struct State : Softmax<Q8, 16> {
    f32x4 acc[D / 16];
    std::conditional_t<Q8, Scaled, char> sc;

    __device__ __forceinline__ State() {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void step(float (&s)[8], float c, const float (&vs)[8][D / 64]) {
        float top;
        bool look = __builtin_amdgcn_ballot_w64(this->rises(s, c, top)) != 0ull;
        if (look) {
            const bool first = this->m == -INFINITY;
            const float rose = this->rebase(top);
            if constexpr (Q8) {
                sc.rebase(first, rose, this->m != -INFINITY);
            } else {
                const float alpha = factor(-rose);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) acc[j] *= alpha;
            }
        }
        this->weigh(s, c);
        if constexpr (Q8) {
            float any = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int b = 0; b < D / 64; ++b) any = fmaxf(any, fabsf(vs[i][b]));
            if (look || __builtin_amdgcn_ballot_w64(Scaled::asks(any, sc.ev)) != 0ull) {
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int b = 0; b < D / 64; ++b) most = fmaxf(most, use(s[i], vs[i][b]));
                const float f = sc.template raise<16>(most);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) acc[j] *= f;
            }
        }
    }
};

// A value that is the same in every lane, in a scalar register.  Every condition
// around a matrix instruction has to be one: the instruction writes all lanes,
// also where the compiler has masked them off for the other side of a branch.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int cache_row(const Keys& K, int i) { return i < K.na ? i : i + K.db; }

// Whether the rows of keys [i0, i0 + kKeys) follow each other in the cache.
__device__ __forceinline__ bool rows_follow(const Keys& K, int i0) {
    return i0 + kKeys <= K.n && (i0 >= K.na || i0 + kKeys <= K.na);
}

// Whether every one of the workgroup's tokens sees all the keys [i0, i0 + n).
__device__ __forceinline__ bool all_seen(const Keys& K, int i0, int n) {
    if (i0 + n > K.n) return false;
    if (!K.masked) return true;
    return cache_row(K, i0 + n - 1) <= K.p_first && (i0 + n <= K.na || cache_row(K, max(i0, K.na)) >= K.lo_last);
}

// P' of 8 keys as two fp16 operands per scale block (one without scales).
template <int D, bool Q8>
struct Weights {
    static constexpr int kBlocks = Q8 ? D / 64 : 1;
    uint32_t h[kBlocks][4], l[kBlocks][4];

    // vs: the keys' value scales; one of a key that the row does not see may be
    // anything (all: the row sees them all).  ev: the row's Scaled::ev.
    __device__ __forceinline__ void cut(const float* s, const float (*vs)[D / 64], bool all, uint32_t seen, int ev) {
        if constexpr (Q8) {
            const float f = pow2(-ev);
            if (all) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s0 = s[2 * i] * f, s1 = s[2 * i + 1] * f;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b) two_parts(s0 * vs[2 * i][b], s1 * vs[2 * i + 1][b], h[b][i], l[b][i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s0 = s[2 * i] * f, s1 = s[2 * i + 1] * f;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b)
                        two_parts((seen >> (2 * i)) & 1u ? s0 * vs[2 * i][b] : 0.0f,
                                  (seen >> (2 * i + 1)) & 1u ? s1 * vs[2 * i + 1][b] : 0.0f, h[b][i], l[b][i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) two_parts(s[2 * i], s[2 * i + 1], h[0][i], l[0][i]);
        }
    }
    __device__ __forceinline__ half8 first(int b) const { return as_half8(h[Q8 ? b : 0]); }
    __device__ __forceinline__ half8 rest(int b) const { return as_half8(l[Q8 ? b : 0]); }
    // acc += V' P' for an operand of V in scale block b
    template <typename T>
    __device__ __forceinline__ T add(half8 o, int b, T acc) const {
        b = Q8 ? b : 0;
        return mfma(o, as_half8(l[b]), mfma(o, as_half8(h[b]), acc));
    }
};

// Which of N keys a row sees (bit i: the key with index at(i)); the products of
// the others become -inf.
template <int N, typename F>
__device__ __forceinline__ uint32_t mask_keys(const Keys& K, const RowSight& see, float* s, F at) {
    uint32_t seen = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int k = at(i);
        const int row = cache_row(K, k);
        const bool ok = (k < K.n) & ((row <= see.p) & ((row >= see.lo) | (row < K.sinks)));
        s[i] = ok ? s[i] : -INFINITY;
        seen |= ok ? 1u << i : 0u;
    }
    return seen;
}

// ------------------------------------------------- few rows: waves over keys
// Steps t0, t0 + stride, ... below t1 of 32 keys each, K and V straight from
// the cache into the operands' registers: 16 lanes read a V row's 256 bytes, 4
// lanes 64 bytes of a K row.  A step's loads are issued one phase ahead.
template <int D, bool Q8>
struct Step {
    uint4 k16[2][D / 32];
    uint2 k8[2][D / 32];
    VRaw<D, Q8> v;
    float ks[8][D / 64], vs[8][D / 64];

    // Key i's row is at(i) rows past `first`; kFollow: at(i) = i, so that the
    // addresses are one scalar and constants, and a lane's scales lie together.
    template <bool kFollow, typename F>
    __device__ __forceinline__ void k_rows(const Keys& K, size_t first, F at, int lane) {
        constexpr int kBytes = Q8 ? 1 : 2;
        const int r = lane & 15, gq = lane >> 4;
        const char* src = static_cast<const char*>(K.k) + first * (D * kBytes);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const char* x = src + (at(16 * kt + r) * (D * kBytes) + 8 * gq * kBytes);
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                if constexpr (Q8)
                    k8[kt][s] = *reinterpret_cast<const uint2*>(x + 32 * s);
                else
                    k16[kt][s] = *reinterpret_cast<const uint4*>(x + 64 * s);
            }
        }
        if constexpr (Q8) scale_rows<kFollow>(K.ks, first, at, gq, ks);
    }
    template <bool kFollow, typename F>
    __device__ __forceinline__ void v_rows(const Keys& K, size_t first, F at, int lane) {
        constexpr int kBytes = Q8 ? 1 : 2;
        const int r = lane & 15, gq = lane >> 4;
        const char* src = static_cast<const char*>(K.v) + first * (D * kBytes);
#pragma unroll
        for (int i = 0; i < 8; ++i) v.load(src + at((i & 4) * 4 + 4 * gq + (i & 3)) * (D * kBytes), i, r);
        if constexpr (Q8) scale_rows<kFollow>(K.vs, first, at, gq, vs);
    }
    // The scales of the lane's 8 keys.
    template <bool kFollow, typename F>
    __device__ __forceinline__ void scale_rows(const float* src, size_t first, F at, int gq, float (&dst)[8][D / 64]) {
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // a row's scales start anywhere
        src += first * (D / 64);
        if constexpr (kFollow) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4 * (D / 64); i += 4) {
                    const f4 x = *reinterpret_cast<const f4*>(src + (16 * h + 4 * gq) * (D / 64) + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dst[4 * h + (i + e) / (D / 64)][(i + e) % (D / 64)] = x[e];
                }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int b = 0; b < D / 64; ++b) dst[i][b] = src[at((i & 4) * 4 + 4 * gq + (i & 3)) * (D / 64) + b];
        }
    }
    // Step t: where its rows do not follow each other (at a range's end) every
    // row is looked up by itself.
    __device__ __forceinline__ void load_k(const Keys& K, int t, int lane) {
        const int i0 = t * kKeys;
        if (rows_follow(K, i0))
            k_rows<true>(K, static_cast<size_t>(cache_row(K, i0)), [](int i) { return i; }, lane);
        else
            k_rows<false>(K, 0, [&](int i) { return static_cast<long long>(cache_row(K, min(i0 + i, K.n - 1))); }, lane);
    }
    __device__ __forceinline__ void load_v(const Keys& K, int t, int lane) {
        const int i0 = t * kKeys;
        if (rows_follow(K, i0))
            v_rows<true>(K, static_cast<size_t>(cache_row(K, i0)), [](int i) { return i; }, lane);
        else
            v_rows<false>(K, 0, [&](int i) { return static_cast<long long>(cache_row(K, min(i0 + i, K.n - 1))); }, lane);
    }
    __device__ __forceinline__ half8 k_operand(int kt, int s) const {
        if constexpr (Q8)
            return codes_half8(k8[kt][s]);
        else
            return __builtin_bit_cast(half8, k16[kt][s]);
    }
    __device__ __forceinline__ void scores(const Query<D, 32>& q, float (&s)[8]) const {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            if constexpr (Q8) {
                f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < D / 64; ++b) {
                    f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int x = 2 * b; x < 2 * b + 2; ++x) {
                        const half8 k = k_operand(kt, x);
                        a = mfma(k, q.hi[x], a);
                        a = mfma(k, q.lo[x], a);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = fmaf(a[i], ks[4 * kt + i][b], sum[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * kt + i] = sum[i];
            } else {
                f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    const half8 k = k_operand(kt, x);
                    a = mfma(k, q.hi[x], a);
                    a = mfma(k, q.lo[x], a);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * kt + i] = a[i];
            }
        }
    }
};

template <int D, bool Q8>
__device__ __forceinline__ void few_rows(const Keys& K, const Query<D, 32>& q, const RowSight& see, int t0, int t1,
                                         int stride, int lane, State<D, Q8>& st) {
    if (t0 >= t1) return;
    const int gq = lane >> 4;
    Step<D, Q8> x;
    x.load_k(K, t0, lane);
    x.load_v(K, t0, lane);
    for (int t = t0; t < t1; t += stride) {
        float s[8];
        x.scores(q, s);
        const int next = t + stride;
        if (next < t1) x.load_k(K, next, lane);
        const bool all = all_seen(K, t * kKeys, kKeys);  // the same in every lane
        uint32_t seen = 0xFFu;
        if (!all) seen = mask_keys<8>(K, see, s, [&](int i) { return t * kKeys + (i & 4) * 4 + 4 * gq + (i & 3); });
        st.step(s, q.c, x.vs);
        Weights<D, Q8> w;
        int ev = 0;
        if constexpr (Q8) ev = st.sc.ev;
        w.cut(s, x.vs, all, seen, ev);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st.acc[j] = w.add(x.v.operand(j), j >> 2, st.acc[j]);
        if (next < t1) x.load_v(K, next, lane);
    }
}

// Infinities and NaN at keys that a row sees.  The loops take the products as they
// come: an infinite key times a second part of the query that is zero or of the
// other sign is NaN there, and so is an infinite value times a second part of a
// weight, or times the zero of a row that does not see it.  All of it leaves a sum
// or an accumulator that is not finite, and finite fp16 rows never do; such a row is
// taken again here, in fp32 and with the definition's own products: a score of
// +inf or NaN makes the row NaN, a key of score -inf has no weight, and an infinite
// value is its dim's at any weight above none.  A row at a time: the keys of steps
// t0, t0 + stride, ... below t1 over the lanes, then the dims: 5.9 ms for a prompt of
// 2048 whose every value is NaN (99 us without), 0.77 for 32 tokens over 4000 rows
// (0.099).  O' (or, without ml, the output of a row that the call has whole) to dst,
// base and sum to ml.
template <int D>
__device__ __forceinline__ void strict_row(const Keys& K, const float* row, float scale, const RowSight& see, int t0, int t1,
                                           int stride, int lane, float* dst, float2* ml) {
    constexpr int kDims = D / kWave;  // of a lane
    float m = -INFINITY, l = 0.0f, acc[kDims] = {};
#pragma unroll 1
    for (int t = t0; t < t1; t += 2 * stride) {
        const int step = t + (lane >> 5) * stride, key = step * kKeys + (lane & 31);
        const int r = cache_row(K, min(key, K.n - 1));
        const bool ok = step < t1 && key < K.n && r <= see.p && (r >= see.lo || r < K.sinks);
        float s = 0.0f;
        if (ok) {
            const char* src = static_cast<const char*>(K.k) + static_cast<size_t>(r) * (2 * D);
#pragma unroll 1
            for (int d0 = 0; d0 < D; d0 += 64) {
                half8 k[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) k[j] = *reinterpret_cast<const half8*>(src + 2 * d0 + 16 * j);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) s = fmaf(static_cast<float>(k[j][i]), row[d0 + 8 * j + i], s);
            }
        }
        s = ok ? s * scale : -INFINITY;
        float top = s;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
        const float m1 = fmaxf(m, top), alpha = m == m1 ? 1.0f : factor(m - m1);
        m = m1;
        float p = exp2_fast(s - (m == -INFINITY ? 0.0f : m));
        p = s == -INFINITY ? 0.0f : p < kLeast ? kLeast : p;
        l = l * alpha + p;
#pragma unroll
        for (int e = 0; e < kDims; ++e) acc[e] *= alpha;
        const uint64_t seen = __builtin_amdgcn_ballot_w64(ok);
#pragma unroll 1
        for (int i0 = 0; i0 < kWave; i0 += 16) {
            float v[16][kDims];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const _Float16* src = static_cast<const _Float16*>(K.v) +
                                      static_cast<size_t>(__builtin_amdgcn_readlane(r, i0 + i)) * D + kDims * lane;
#pragma unroll
                for (int e = 0; e < kDims; ++e) v[i][e] = static_cast<float>(src[e]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (((seen >> (i0 + i)) & 1ull) == 0ull) continue;
                const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), i0 + i));
#pragma unroll
                for (int e = 0; e < kDims; ++e) acc[e] = fmaf(w, v[i][e], acc[e]);
            }
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, kWave);
    if (ml && lane == 0) *ml = make_float2(m, l);
#pragma unroll
    for (int e = 0; e < kDims; ++e) dst[kDims * lane + e] = ml ? acc[e] : l != 0.0f ? acc[e] / l : 0.0f;
}

// The workgroup's waves joined: their (maximum, sum) and O' through LDS, then
// each thread forms its share of the 16 rows: as out rows where the job has all
// the keys (final), else as partials for attention_join_kernel.
template <int D, int W>
struct JoinArea {
    float acc[W][kRows][D + 4];
    float2 ml[W][kRows];
};

// The factor of a part (base, sum) under the common base m: 0 without keys, NaN
// for a sum that is NaN.
__device__ __forceinline__ float share(float2 ml, float m) {
    return ml.y == 0.0f ? 0.0f : ml.y == ml.y ? factor(ml.x - m) : ml.y;
}

// A state's O' to a row of D floats; over int8 caches operand j's dims are code_dim's.
template <int D, bool Q8>
__device__ __forceinline__ void store_row(float* dst, const State<D, Q8>& st, int gq) {
    const auto& acc = st.acc;
    float f = 1.0f;
    if constexpr (Q8) f = pow2(st.sc.ev);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * gq + i;
#pragma unroll
        for (int j = 0; j < D / 16; j += 4) {
            const int d = Q8 ? code_dim(r, j) : fp16_dim<D>(r, j);
            *reinterpret_cast<float4*>(dst + d) =
                make_float4(acc[j][i] * f, acc[j + 1][i] * f, acc[j + 2][i] * f, acc[j + 3][i] * f);
        }
    }
}

// Query rows of one workgroup: row n is token n / g of n_tokens, head n % g of
// the KV head's group, q and out row base + token * n_heads + n % g.
struct RowMap {
    long long base;
    int g, n_heads, total;
    __device__ __forceinline__ long long at(int n) const {
        return base + static_cast<long long>(n / g) * n_heads + n % g;
    }
};

// What a row sees: any = false gives a row of zeros.
__device__ __forceinline__ RowSight sight(const Keys& K, long long p, int rows, int window) {
    RowSight s;
    s.any = !K.masked || (p >= 0 && p < rows);
    s.p = !K.masked ? INT_MAX : s.any ? static_cast<int>(p) : -1;
    s.lo = K.masked && window > 0 ? s.p - window + 1 : 0;
    return s;
}

template <int D, bool Q8>
__device__ __forceinline__ void few_job(const AttnArgs& g, const Keys& K, const RowMap& map, int row0, long long p0,
                                        int rows, int split, int splits, int slot, JoinArea<D, kFewWaves>& area) {
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = uniform(tid >> 6);
    const int n = row0 + (lane & 15), gq = lane >> 4;
    const bool real = n < map.total;
    Query<D, 32> q;
    q.load(real ? g.q + map.at(n) * D : nullptr, gq, g.scale);
    const RowSight see = sight(K, p0 + n / map.g, rows, g.window);
    State<D, Q8> st;
    const int steps = (K.n + kKeys - 1) / kKeys;
    // a split's steps, a multiple of the waves'
    const int per = ((steps + splits - 1) / splits + kFewWaves - 1) / kFewWaves * kFewWaves;
    few_rows<D, Q8>(K, q, see, split * per + wave, min(steps, (split + 1) * per), kFewWaves, lane, st);
    st.l = lanes_sum<16>(st.l);
    store_row<D, Q8>(area.acc[wave][lane & 15], st, gq);
    if (gq == 0) area.ml[wave][lane & 15] = make_float2(st.m, st.l);
    __syncthreads();
    constexpr int kPer = kRows * D / (kFewWaves * 64);  // values a thread, 16 threads a row: 8 (D 128) or 4
    const int r = tid * kPer / D, d = tid * kPer % D;
    if (row0 + 4 * wave >= map.total) return;
    const bool mine = row0 + r < map.total;
    const bool any = mine && sight(K, p0 + (row0 + r) / map.g, rows, g.window).any;
    const long long at = mine ? map.at(row0 + r) : 0;
    float m = -INFINITY, l = 0.0f, w[kFewWaves];
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) m = fmaxf(m, area.ml[i][r].x);
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) {
        w[i] = share(area.ml[i][r], m);
        l += area.ml[i][r].y * w[i];
    }
    float o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i)
        if (w[i] != 0.0f) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) o[e] = fmaf(area.acc[i][r][d + e], w[i], o[e]);
        }
    if constexpr (!Q8) {
        float none = l * 0.0f;  // 0, or NaN
#pragma unroll
        for (int e = 0; e < kPer; ++e) none = fmaf(o[e], 0.0f, none);
        uint64_t odd = __builtin_amdgcn_ballot_w64(none != 0.0f && any);
        if (__builtin_expect(odd != 0ull, 0)) {
            const bool again = ((odd >> (lane & 48)) & 0xFFFFull) != 0ull;
            for (int i = 0; i < 4; ++i) {
                if (((odd >> (16 * i)) & 0xFFFFull) == 0ull) continue;
                const int n1 = row0 + 4 * wave + i;
                const long long at1 = map.at(n1);
                strict_row<D>(K, g.q + at1 * D, g.scale, sight(K, p0 + n1 / map.g, rows, g.window), split * per,
                              min(steps, (split + 1) * per), 1, lane,
                              g.slots == 1 ? g.out + at1 * D : g.part + (at1 * g.slots + slot) * D,
                              g.slots == 1 ? nullptr : g.ml + at1 * g.slots + slot);
            }
            if (again) return;
        }
    }
    if (!mine) return;
    float* dst;
    if (g.slots == 1) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] = any && l != 0.0f ? o[e] / l : 0.0f;
        dst = g.out + at * D + d;
    } else {
        if (d == 0) g.ml[at * g.slots + slot] = make_float2(m, l);
        if (l == 0.0f) return;
        dst = g.part + (at * g.slots + slot) * D + d;
    }
#pragma unroll
    for (int e = 0; e < kPer; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
}

template <int D, bool Q8>
__device__ __forceinline__ Keys head_keys(const Cache& c, long long head, int rows) {
    Keys K{};
    const size_t row = static_cast<size_t>(head) * rows;
    const size_t bytes = row * D * (Q8 ? 1 : 2);
    K.k = static_cast<const char*>(c.k) + bytes;
    K.v = static_cast<const char*>(c.v) + bytes;
    if constexpr (Q8) {
        K.ks = c.ks + row * (D / 64);
        K.vs = c.vs + row * (D / 64);
    }
    return K;
}

// The keys that tokens [t0, t1) of a sequence see with a window.
template <int D, bool Q8>
__device__ __forceinline__ Keys window_keys(const AttnArgs& g, int seq, int kvh, int t0, int t1) {
    Keys K = head_keys<D, Q8>(g.b, static_cast<long long>(seq) * g.n_kv + kvh, g.rows_b);
    const long long p0 = g.pos[seq];
    const long long first = p0 + t0 > 0 ? p0 + t0 : 0;
    const long long last = p0 + t1 - 1 < g.rows_b ? p0 + t1 - 1 : g.rows_b - 1;
    K.masked = true;
    K.sinks = g.sinks;
    if (first > last) return K;  // no token in the cache: no keys
    const int lo = g.window > 0 ? max(0, static_cast<int>(first) - g.window + 1) : 0;
    K.na = min(g.sinks, lo);
    K.db = lo - K.na;
    K.n = K.na + static_cast<int>(last) - lo + 1;
    K.p_first = static_cast<int>(first);
    K.lo_last = g.window > 0 ? static_cast<int>(last) - g.window + 1 : 0;
    return K;
}

// ---------------------------------------------- many rows: waves over rows
// A wave takes 32 query rows (columns of 32x32 tiles: half the operand reads a
// product of 16x16 ones, and one lane exchange a step), the workgroup's four
// waves share each 32 keys through LDS, where K and V lie as the operands are
// read, 16 bytes a lane; int8 codes are turned into fp16 on the way.  Waves 0 and
// 1 bring 64 dims of V each (turned in registers), waves 2 and 3 16 keys of K.
// Four buffers in a ring: a tile's loads are started two tiles ahead, run during
// its products and are written behind them, so that waves may be two tiles
// apart and one barrier does for two tiles.
//
// 4096 tokens with a window of 2048 over up to 6000 rows (24 heads of 128, 8 KV
// heads, fp16): 215 us, 480 TFLOP/s of the definition's products and twice that
// in the matrix cores, which are busy 48 % of the time; two products in fp16
// parts at the rate of a large library product would take 189.  Of 227 us in one
// run, without the tiles' loads 198 were left, without their stores to LDS 211,
// without the softmax 213, without all three 174: none alone bounds it.  Two
// buffers and a barrier a tile took 260 us, the form for few rows 816.  Over int8
// caches 4096 tokens take 253 us with all of 4096 rows to see.
//
// A lane holds one row n = lane % 32 and, with h = lane / 32, the keys
// wide_key(i, h) of a tile's score registers i = 0..15; operand step s of the
// weighted values takes i = 8 s .. 8 s + 7.
constexpr int kManyWaves = 4;
constexpr int kWideRows = 32;
constexpr int kStages = 4;

__device__ __forceinline__ int wide_key(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// Operand row m of V's dim tile u is dim 64 (u / 2) + 4 (m % 16) + 2 (u % 2) + m / 16:
// a lane that brings 4 neighbouring dims of 8 keys writes beside its neighbours.
template <int D, bool Q8>
struct Stage {
    half8 k[D / 8][kKeys + 1];     // [8 dims][key]: the odd stride spreads a key's dims over the banks
    half8 v[D / 32][2][2][32];     // [dim tile][step][h][m]
    float ks[Q8 ? D / 64 : 1][Q8 ? kKeys : 4], vs[Q8 ? D / 64 : 1][Q8 ? kKeys : 4];
};

// A wave's share of a tile on its way, 8 or 16 dwords.
template <int D, bool Q8>
struct Bring {
    static constexpr int kV = Q8 ? 1 : 2;   // dwords of 4 dims of V
    static constexpr int kK = Q8 ? 2 : 4;   // dwords of 8 dims of K
    static constexpr int kLoads = D / 32;   // 16 keys of K
    uint32_t w[8 * kV];
    float scale;

    // Key i of the 8 that lane group q = lane / 16 brings of V.
    static __device__ __forceinline__ int v_key(int i, int q) {
        return 16 * (q >> 1) + 4 * (q & 1) + 8 * (i >> 2) + (i & 3);
    }
    static __device__ __forceinline__ int k_key(int i, int wave, int lane) {
        return 16 * (wave - 2) + (16 / kLoads) * i + lane / (D / 8);
    }
    // Key i's row is at(i) rows past `first`.
    template <typename F>
    __device__ __forceinline__ void load_rows(const Keys& K, size_t first, F at, int wave, int lane) {
        constexpr int kBytes = Q8 ? 1 : 2;
        if (wave < 2) {
            if (wave < D / 64) {
                const char* src = static_cast<const char*>(K.v) + first * (D * kBytes);
                const int lane_at = (64 * wave + 4 * (lane & 15)) * kBytes;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const char* x = src + (at(v_key(i, lane >> 4)) * (D * kBytes) + lane_at);
                    if constexpr (Q8) {
                        w[i] = *reinterpret_cast<const uint32_t*>(x);
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(x);
                        w[2 * i] = v.x;
                        w[2 * i + 1] = v.y;
                    }
                }
            }
        } else {
            const char* src = static_cast<const char*>(K.k) + first * (D * kBytes);
            const int lane_at = 8 * (lane % (D / 8)) * kBytes;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const char* x = src + (at(k_key(i, wave, lane)) * (D * kBytes) + lane_at);
                if constexpr (Q8) {
                    const uint2 v = *reinterpret_cast<const uint2*>(x);
                    w[2 * i] = v.x;
                    w[2 * i + 1] = v.y;
                } else {
                    const uint4 v = *reinterpret_cast<const uint4*>(x);
                    w[4 * i] = v.x;
                    w[4 * i + 1] = v.y;
                    w[4 * i + 2] = v.z;
                    w[4 * i + 3] = v.w;
                }
            }
        }
        if constexpr (Q8) {
            const int e = wave * 64 + lane;
            if (e < 2 * kKeys * (D / 64)) {
                const int i = e % (kKeys * (D / 64));
                const float* src = (e < kKeys * (D / 64) ? K.ks : K.vs) + first * (D / 64);
                scale = src[at(i / (D / 64)) * (D / 64) + i % (D / 64)];
            }
        }
    }
    // Tile t.  Where its rows follow each other its addresses are one scalar and
    // constants; at a range's end every row is looked up by itself.
    __device__ __forceinline__ void load(const Keys& K, int t, int wave, int lane) {
        const int i0 = t * kKeys;
        if (rows_follow(K, i0))
            load_rows(K, static_cast<size_t>(cache_row(K, i0)), [](int i) { return i; }, wave, lane);
        else
            load_rows(K, 0, [&](int i) { return static_cast<long long>(cache_row(K, min(i0 + i, K.n - 1))); }, wave, lane);
    }
    __device__ __forceinline__ void store(Stage<D, Q8>& s, int wave, int lane) {
        if (wave < 2) {
            if (wave < D / 64) {
                const int q = lane >> 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t o[4];
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        if constexpr (Q8)
                            o[p] = codes_half2(__builtin_amdgcn_perm(w[2 * p + 1], w[2 * p],
                                                                     0x0C040C00u + 0x00010001u * static_cast<uint32_t>(j)));
                        else
                            o[p] = __builtin_amdgcn_perm(w[2 * (2 * p + 1) + (j >> 1)], w[2 * (2 * p) + (j >> 1)],
                                                         (j & 1) ? 0x07060302u : 0x05040100u);
                    }
                    s.v[2 * wave + (j >> 1)][q >> 1][q & 1][16 * (j & 1) + (lane & 15)] = as_half8(o);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                half8 x;
                if constexpr (Q8)
                    x = codes_half8(make_uint2(w[2 * i], w[2 * i + 1]));
                else
                    x = __builtin_bit_cast(half8, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
                s.k[lane % (D / 8)][k_key(i, wave, lane)] = x;
            }
        }
        if constexpr (Q8) {
            const int e = wave * 64 + lane;
            if (e < 2 * kKeys * (D / 64)) {
                const int at = e % (kKeys * (D / 64));
                (e < kKeys * (D / 64) ? s.ks : s.vs)[at % (D / 64)][at / (D / 64)] = scale;
            }
        }
    }
};

template <int D, bool Q8>
__device__ __forceinline__ void many_job(const AttnArgs& g, const Keys& K, const RowMap& map, int row0, long long p0,
                                         int rows, int split, int splits, int slot, Stage<D, Q8> (&stage)[kStages]) {
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = uniform(tid >> 6);
    const int n = row0 + wave * kWideRows + (lane & 31), h = lane >> 5;
    const int tiles = (K.n + kKeys - 1) / kKeys;
    const int per = (tiles + splits - 1) / splits;
    const int t0 = split * per, t1 = min(tiles, t0 + per);
    Query<D, 16> q;
    q.load(n < map.total ? g.q + map.at(n) * D : nullptr, h, g.scale);
    const RowSight see = sight(K, p0 + n / map.g, rows, g.window);
    Softmax<Q8, 32> st;
    f32x16 acc[D / 32];
    Scaled sc;  // int8; and the least power of the wave's rows that have keys
    int ev_low = Scaled::kNone;
#pragma unroll
    for (int u = 0; u < D / 32; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[u][i] = 0.0f;
    Bring<D, Q8> next;
    if (t0 < t1) {
        next.load(K, t0, wave, lane);
        next.store(stage[0], wave, lane);
        if (t0 + 1 < t1) {
            next.load(K, t0 + 1, wave, lane);
            next.store(stage[1], wave, lane);
        }
    }
    for (int t = t0; t < t1; ++t) {
        const int at = t - t0;
        if (at % 2 == 0) __syncthreads();
        const Stage<D, Q8>& s = stage[at % kStages];
        half8 o[D / 16];  // the tile's K operands, then V's
#pragma unroll
        for (int x = 0; x < D / 16; ++x) o[x] = s.k[2 * x + h][lane & 31];
        if (t + 2 < t1) next.load(K, t + 2, wave, lane);
        __builtin_amdgcn_sched_barrier(0);
        float p[16];
#pragma unroll
        for (int b = 0; b < (Q8 ? D / 64 : 1); ++b) {
            f32x16 a;
#pragma unroll
            for (int i = 0; i < 16; ++i) a[i] = 0.0f;
#pragma unroll
            for (int x = b * 4; x < (Q8 ? b * 4 + 4 : D / 16); ++x) {
                a = mfma(o[x], q.hi[x], a);
                a = mfma(o[x], q.lo[x], a);
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                if constexpr (Q8) {
                    const float4 sc = *reinterpret_cast<const float4*>(&s.ks[b][wide_key(i, h)]);
                    p[i] = b ? fmaf(a[i], sc.x, p[i]) : a[i] * sc.x;
                    p[i + 1] = b ? fmaf(a[i + 1], sc.y, p[i + 1]) : a[i + 1] * sc.y;
                    p[i + 2] = b ? fmaf(a[i + 2], sc.z, p[i + 2]) : a[i + 2] * sc.z;
                    p[i + 3] = b ? fmaf(a[i + 3], sc.w, p[i + 3]) : a[i + 3] * sc.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[i + e] = a[i + e];
                }
            }
        }
        constexpr bool kBoth = !Q8;  // registers for both of V's steps (with int8 codes they would spill)
        if constexpr (kBoth) {
#pragma unroll
            for (int u = 0; u < D / 16; ++u) o[u] = s.v[u % (D / 32)][u / (D / 32)][h][lane & 31];
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool all = all_seen(K, t * kKeys, kKeys);
        uint32_t seen = 0xFFFFu;
        if (!all) seen = mask_keys<16>(K, see, p, [&](int i) { return t * kKeys + wide_key(i, h); });
        float high;
        if (__builtin_amdgcn_ballot_w64(st.rises(p, q.c, high)) != 0ull) {
            const bool first = st.m == -INFINITY;
            const float rose = st.rebase(high);
            if constexpr (Q8) {
                sc.rebase(first, rose, st.m != -INFINITY);
                ev_low = Scaled::kLook;
            } else {
                const float alpha = factor(-rose);
#pragma unroll
                for (int u = 0; u < D / 32; ++u) acc[u] *= alpha;
            }
        }
        st.weigh(p, q.c);
        if constexpr (Q8) {
            // A value scale a lane; then each row by its products.
            const float any = s.vs[lane % (D / 64)][lane / (D / 64) % kKeys];
            if (__builtin_amdgcn_ballot_w64(Scaled::asks(any, ev_low)) != 0ull) {
                float most = 0.0f;
#pragma unroll 1
                for (int b = 0; b < D / 64; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = fmaxf(most, use(p[i], s.vs[b][wide_key(i, h)]));
                const float f = sc.template raise<32>(most);
#pragma unroll
                for (int u = 0; u < D / 32; ++u) acc[u] *= f;
                ev_low = sc.ev;
#pragma unroll
                for (int x = 16; x >= 1; x >>= 1) ev_low = min(ev_low, __shfl_xor(ev_low, x, kWave));
                ev_low = uniform(ev_low);
            }
        }
        Weights<D, Q8> w;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (!kBoth) {
#pragma unroll
                for (int u = 0; u < D / 32; ++u) o[u] = s.v[u][e][h][lane & 31];
            }
            float vs[8][D / 64];
            if constexpr (Q8) {
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        const float4 sc = *reinterpret_cast<const float4*>(&s.vs[b][wide_key(8 * e + i, h)]);
                        vs[i][b] = sc.x;
                        vs[i + 1][b] = sc.y;
                        vs[i + 2][b] = sc.z;
                        vs[i + 3][b] = sc.w;
                    }
            }
            w.cut(p + 8 * e, vs, all, seen >> (8 * e), sc.ev);
            const half8* v = &o[kBoth ? e * (D / 32) : 0];
#pragma unroll
            for (int u = 0; u < D / 32; ++u) acc[u] = mfma(v[u], w.first(u >> 1), acc[u]);
#pragma unroll
            for (int u = 0; u < D / 32; ++u) acc[u] = mfma(v[u], w.rest(u >> 1), acc[u]);
        }
        if (t + 2 < t1) next.store(stage[(at + 2) % kStages], wave, lane);
    }
    const float l = lanes_sum<32>(st.l);
    if constexpr (!Q8) {
        float none[4] = {l * 0.0f, 0.0f, 0.0f, 0.0f};  // 0, or NaN
#pragma unroll
        for (int u = 0; u < D / 32; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) none[i & 3] = fmaf(acc[u][i], 0.0f, none[i & 3]);
        const bool odd = (none[0] + none[1]) + (none[2] + none[3]) != 0.0f;
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(odd && n < map.total && see.any);
        uint32_t again = static_cast<uint32_t>(lanes) | static_cast<uint32_t>(lanes >> 32);
        if (__builtin_expect(again != 0u, 0)) {
            const bool mine = ((again >> (lane & 31)) & 1u) == 0u;
            for (; again != 0u; again &= again - 1u) {
                const int m = row0 + wave * kWideRows + __builtin_ctz(again);
                const long long at = map.at(m);
                const bool whole = g.slots == 1;
                strict_row<D>(K, g.q + at * D, g.scale, sight(K, p0 + m / map.g, rows, g.window), t0, t1, 1, lane,
                              whole ? g.out + at * D : g.part + (at * g.slots + slot) * D,
                              whole ? nullptr : g.ml + at * g.slots + slot);
            }
            if (!mine) return;
        }
    }
    if (n >= map.total) return;
    const long long at = map.at(n);
    float f = Q8 ? pow2(sc.ev) : 1.0f;
    float* dst;
    if (g.slots == 1) {
        const bool any = see.any && l != 0.0f;
        f = any ? f / l : 0.0f;
        if (!any) {
#pragma unroll
            for (int u = 0; u < D / 32; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[u][i] = 0.0f;
        }
        dst = g.out + at * D;
    } else {
        if (h == 0) g.ml[at * g.slots + slot] = make_float2(st.m, l);
        if (l == 0.0f) return;
        dst = g.part + (at * g.slots + slot) * D;
    }
#pragma unroll
    for (int u = 0; u < D / 32; u += 2)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 o = make_float4(acc[u][i] * f, acc[u][i + 8] * f, acc[u + 1][i] * f, acc[u + 1][i + 8] * f);
            *reinterpret_cast<float4*>(dst + 32 * u + 4 * wide_key(i, h)) = o;
        }
}

// Row tiles from the last one down: with no window its tokens see the most.
template <int D, bool Q8>
__global__ __launch_bounds__(kManyWaves * 64, 2) void window_many_kernel(const AttnArgs g) {
    __shared__ Stage<D, Q8> stage[kStages];
    constexpr int kWgRows = kManyWaves * kWideRows;
    const int group = g.n_heads / g.n_kv;
    const int total = g.n_tokens * group;
    const int tiles = (total + kWgRows - 1) / kWgRows;
    int b = static_cast<int>(blockIdx.x);
    const int kvh = b % g.n_kv;
    b /= g.n_kv;
    const int split = b % g.splits;
    b /= g.splits;
    const int row0 = (tiles - 1 - b % tiles) * kWgRows;
    const int seq = b / tiles;
    const RowMap map{static_cast<long long>(seq) * g.n_tokens * g.n_heads + static_cast<long long>(kvh) * group, group,
                     g.n_heads, total};
    const Keys K = window_keys<D, Q8>(g, seq, kvh, row0 / group, (min(row0 + kWgRows, total) - 1) / group + 1);
    many_job<D, Q8>(g, K, map, row0, g.pos[seq], g.rows_b, split, g.splits, split, stage);
}

// ------------------------------------------------------- few rows: kernels
// blockIdx.x = ((sequence * row tiles + tile) * splits + split) * n_kv + kv head:
// with 8 KV heads one head's workgroups share an XCD's L2.
template <int D, bool Q8>
__global__ __launch_bounds__(kFewWaves * 64, 2) void window_few_kernel(const AttnArgs g) {
    __shared__ JoinArea<D, kFewWaves> area;
    const int group = g.n_heads / g.n_kv;
    const int total = g.n_tokens * group;
    const int tiles = (total + kRows - 1) / kRows;
    int b = static_cast<int>(blockIdx.x);
    const int kvh = b % g.n_kv;
    b /= g.n_kv;
    const int split = b % g.splits;
    b /= g.splits;
    const int row0 = b % tiles * kRows;
    const int seq = b / tiles;
    const RowMap map{static_cast<long long>(seq) * g.n_tokens * g.n_heads + static_cast<long long>(kvh) * group, group,
                     g.n_heads, total};
    const Keys K = window_keys<D, Q8>(g, seq, kvh, row0 / group, (min(row0 + kRows, total) - 1) / group + 1);
    few_job<D, Q8>(g, K, map, row0, g.pos[seq], g.rows_b, split, g.splits, split, area);
}

// Shared prefix: the first `jobs` workgroups take rows of a KV head, 16 or 128
// of all sequences' (sequence, head) rows, and a split of the prefix, the others
// a sequence's own keys.
template <int D, bool Q8, bool kMany>
__global__ __launch_bounds__(kFewWaves * 64, 2) void prefix_kernel(const AttnArgs g, int prefix_splits, int jobs) {
    static_assert(kFewWaves == kManyWaves, "one workgroup size");
    constexpr int kWgRows = kMany ? kManyWaves * kWideRows : kRows;
    __shared__ union Lds {
        JoinArea<D, kFewWaves> area;
        Stage<D, Q8> stage[kMany ? kStages : 1];
        __device__ Lds() {}
    } lds;
    const int group = g.n_heads / g.n_kv;
    int b = static_cast<int>(blockIdx.x);
    if (b < jobs) {
        const int total = g.n_seq * group;
        const int tiles = (total + kWgRows - 1) / kWgRows;
        const int kvh = b % g.n_kv;
        b /= g.n_kv;
        const int row0 = b % tiles * kWgRows;
        const int split = b / tiles;
        const RowMap map{static_cast<long long>(kvh) * group, group, g.n_heads, total};
        Keys K = head_keys<D, Q8>(g.a, kvh, g.rows_a);
        K.n = g.prefix;
        if constexpr (kMany)
            many_job<D, Q8>(g, K, map, row0, 0, 0, split, prefix_splits, split, lds.stage);
        else
            few_job<D, Q8>(g, K, map, row0, 0, 0, split, prefix_splits, split, lds.area);
        return;
    }
    b -= jobs;
    const int kvh = b % g.n_kv;
    b /= g.n_kv;
    const int own_splits = g.slots - prefix_splits;
    const int split = b % own_splits;
    b /= own_splits;
    const int tiles = (group + kRows - 1) / kRows;
    const int row0 = b % tiles * kRows;
    const int seq = b / tiles;
    const RowMap map{static_cast<long long>(seq) * g.n_heads + static_cast<long long>(kvh) * group, group, g.n_heads,
                     group};
    Keys K = head_keys<D, Q8>(g.b, static_cast<long long>(seq) * g.n_kv + kvh, g.rows_b);
    const int p = g.pos[seq];
    K.n = p >= 0 && p < g.rows_b ? p + 1 : 0;
    few_job<D, Q8>(g, K, map, row0, 0, 0, split, own_splits, prefix_splits + split, lds.area);
}

// One wave per query row: its partials in slot order, so that the result does not
// depend on the order in which the pieces end.  2.7 us at 24 rows, which is its
// launch and two dependent loads; 5.6 us at 8272 rows of 128 dims in 4 pieces
// (17 MB).
constexpr int kJoinRows = 4;  // rows (waves) of a workgroup
constexpr int kMaxSlots = 64;
template <int D>
__global__ __launch_bounds__(kJoinRows * 64) void attention_join_kernel(const AttnArgs g, long long q_rows) {
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const long long row = static_cast<long long>(blockIdx.x) * kJoinRows + (threadIdx.x >> 6);
    if (row >= q_rows) return;
    const long long tok = row / g.n_heads;
    const int seq = static_cast<int>(tok / g.n_tokens);
    const long long p = static_cast<long long>(g.pos[seq]) + tok % g.n_tokens;
    const bool any = p >= (g.prefix >= 0 ? -1 : 0) && p < g.rows_b;
    const float2 ml = lane < g.slots ? g.ml[row * g.slots + lane] : make_float2(-INFINITY, 0.0f);
    float m = ml.x;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
    const float w = share(ml, m);
    float l = ml.y * w;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, kWave);
    // Slots with keys, four at a time: their loads are independent.
    float acc[D / 64] = {};
    const float* part = g.part + row * g.slots * D + lane * (D / 64);
    uint64_t left = __builtin_amdgcn_ballot_w64(w != 0.0f);
    while (left != 0ull) {
        int s[4];
        float ws[4], x[4][D / 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = left != 0ull ? __builtin_ctzll(left) : s[0];
            ws[i] = left != 0ull ? __shfl(w, s[i], kWave) : 0.0f;
            left &= left - 1;
#pragma unroll
            for (int e = 0; e < D / 64; ++e) x[i][e] = part[s[i] * D + e];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (ws[i] != 0.0f) {
#pragma unroll
                for (int e = 0; e < D / 64; ++e) acc[e] = fmaf(x[i][e], ws[i], acc[e]);
            }
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) g.out[row * D + lane * (D / 64) + i] = any && l != 0.0f ? acc[i] / l : 0.0f;
}

// ------------------------------------------------------------- host checks
// f(head_dim, int8) as compile-time constants.
template <typename F>
asdsl_status with_form(int head_dim, bool q8, F f) {
    using std::integral_constant;
    if (head_dim == 128)
        return q8 ? f(integral_constant<int, 128>{}, std::true_type{}) : f(integral_constant<int, 128>{}, std::false_type{});
    return q8 ? f(integral_constant<int, 64>{}, std::true_type{}) : f(integral_constant<int, 64>{}, std::false_type{});
}

constexpr int kMaxRows = 1 << 30;  // rows seen, so that a tile past the last of them is an int

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

asdsl_status check_heads(const char* what, int n_seq, int n_tokens, int n_heads, int n_kv_heads, int head_dim) {
    ASDSL_CHECK_ARG(n_seq > 0 && n_tokens > 0, "%s: n_seq and n_tokens must be positive", what);
    ASDSL_CHECK_ARG(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0,
                    "%s: n_heads must be a multiple of n_kv_heads", what);
    ASDSL_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128", what);
    ASDSL_CHECK_ARG(n_heads <= 65536 && n_kv_heads <= 65536, "%s: more than 65536 heads", what);
    // query rows, and with them every grid and work buffer index, in 31 bits
    ASDSL_CHECK_ARG(static_cast<long long>(n_seq) * n_tokens <= INT_MAX / (n_heads + 2LL * n_kv_heads),
                    "%s: n_seq * n_tokens * heads exceeds 2^31", what);
    return ASDSL_OK;
}

asdsl_status append(const char* what, bool q8, const float* qkv, void* k, void* v, float* ks, float* vs,
                    const float* rope_cos, const float* rope_sin, const int* pos, float* q_out, int n_seq,
                    int n_tokens, int n_heads, int n_kv_heads, int head_dim, int rotary_dim, int rows, int pos_offset,
                    int rope_rows, asdsl_stream_t stream) {
    ASDSL_CHECK_ARG(qkv && k && v && rope_cos && rope_sin && pos && q_out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(!q8 || (ks && vs), "%s: null scale array", what);
    const asdsl_status st = check_heads(what, n_seq, n_tokens, n_heads, n_kv_heads, head_dim);
    if (st != ASDSL_OK) return st;
    ASDSL_CHECK_ARG(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
                    "%s: rotary_dim must be even and <= head_dim", what);
    ASDSL_CHECK_ARG(rows > 0 && rope_rows > 0 && pos_offset >= 0,
                    "%s: rows and rope_rows must be positive, pos_offset not negative", what);
    ASDSL_CHECK_ARG(aligned16(qkv) && aligned16(k) && aligned16(v) && aligned16(q_out),
                    "%s: qkv, caches and q_out must be 16-byte aligned", what);
    const int chunks = ((n_heads + 2 * n_kv_heads) * (head_dim / 4) + kAppendThreads - 1) / kAppendThreads;
    const long long grid = static_cast<long long>(n_seq) * n_tokens * chunks;
    ASDSL_CHECK_ARG(fits_launch(grid, kAppendThreads), "%s: n_seq * n_tokens * heads: more than 2^32 work items", what);
    const AppendArgs a{qkv, k, v, ks, vs, rope_cos, rope_sin, pos, q_out, n_tokens, n_heads, n_kv_heads,
                       rotary_dim / 2, rows, pos_offset, rope_rows, chunks};
    const bool vec = rotary_dim % 8 == 0 && aligned16(rope_cos) && aligned16(rope_sin);
    return with_form(head_dim, q8, [&](auto dim, auto codes) {
        constexpr int kD = decltype(dim)::value;
        constexpr bool kQ8 = decltype(codes)::value;
        return launch("kv_append_kernel", vec ? kv_append_kernel<kD, kQ8, true> : kv_append_kernel<kD, kQ8, false>,
                      dim3(static_cast<unsigned>(grid)), dim3(kAppendThreads), 0, as_hip(stream), a);
    });
}

// How many key splits get a launch of `jobs` workgroups to `fill` of them when
// each split keeps at least kLeastKeys of at most n keys.
constexpr int kLeastKeys = kFewWaves * kKeys;

int splits_for(long long fill, long long jobs, long long n, int most) {
    long long s = (fill + jobs - 1) / jobs;
    const long long by_keys = (n + kLeastKeys - 1) / kLeastKeys;
    s = s < by_keys ? s : by_keys;
    s = s < most ? s : most;
    return s > 1 ? static_cast<int>(s) : 1;
}

// Which form takes `total` rows of each of `heads` KV heads over about `keys` keys
// each.  The few-rows form reads the keys once per 16 rows and streams better, the
// many-rows form once per 128, whole or not, and is some 6 us slower to start: it
// pays where the steps of the one, 16 rows by 128 keys, exceed those of the other,
// 128 rows by 128 keys, by more than `margin` when one of these counts as `worth`
// of those.  Int8 keys are half the bytes, and their conversion, which the many-rows
// form saves, is cheap beside 64 dims' softmax.  us few / many in a graph, 8 KV
// heads, rows x keys (s: for each of s sequences, p: of a causal prompt):
//   128 dims fp16  36 x 5000 19.9 / 19.1, 48 x 2000 15.0 / 14.9, 144 x 16000 102 / 49,
//                  p 768 x 256 11.6 / 18.7, p 6144 x 2048 232 / 86
//   128 dims int8  96 x 5000 23.7 / 29.5, 192 x 5000 41.6 / 35.3, 144 x 16000 76 / 63,
//                  p 1551 x 517 23.9 / 31.7, p 6144 x 2048 158 / 114
//   64 dims fp16   64 x 16000 22.4 / 27.7, 108 x 16000 36.6 / 30.6, 64 s 32 x 1000
//                  32.1 / 54.6, p 2068 x 517 16.1 / 22.8, p 16384 x 4096 436 / 184
//   64 dims int8   256 x 16000 43.8 / 46.5, 8 s 160 x 8000 104 / 138, 64 s 32 x 1000
//                  25.6 / 72.9, p 8192 x 2048 82 / 107, p 16384 x 4096 269 / 235
// One rule by steps does not fit all: 4 s 4096 rows of 64 dims over int8 caches with
// a window of 256 take 74 in the form for few, 54 in the other.
bool takes_many(long long total, long long heads, long long keys, int head_dim, bool q8) {
    if (total <= kRows) return false;
    const int wide = kManyWaves * kWideRows;
    const long long pieces = heads * ((keys + kLeastKeys - 1) / kLeastKeys);
    const long long few = (total + kRows - 1) / kRows * pieces, many = (total + wide - 1) / wide * pieces;
    const int worth = head_dim == 128 ? (q8 ? 3 : 2) : (q8 ? 5 : 3);
    const int margin = head_dim == 128 ? (q8 ? 1900 : 300) : (q8 ? 40000 : 3900);
    return few - worth * many > margin;
}

// Workgroups a launch is split up to: two a compute unit.  The many-rows form's
// partials are 16 times as large a job, so with 128 dims it is split to one a
// compute unit where those of two would come to a quarter of the keys' bytes (2068
// rows over 1000 keys, 4 KV heads: 29 us, 38 with two; 16 sequences of 36 rows over
// 2000 keys, 8 KV heads: 46 us, 41 with two).  With 64 dims a tile is shorter and
// more of its waves fit: two pay (4096 rows over 4096 keys, 8 KV heads: 141 us, 101
// with two) but where they alone would ask for a join of short pieces (16
// sequences of 256 rows over 500 keys: 27 us, 35 with two).
constexpr long long kFillFew = 512;

long long fill_many(long long jobs, long long rows, long long heads, long long n, int head_dim) {
    if (head_dim == 64)
        return n <= 4 * kLeastKeys && splits_for(kFillFew / 2, jobs, n, kMaxSlots) == 1 ? kFillFew / 2 : kFillFew;
    const long long splits = splits_for(kFillFew, jobs, n, kMaxSlots);
    return rows * splits * 4 <= heads * n ? kFillFew : kFillFew / 2;
}

// Values of a KV head's keys that few rows take in one piece: a second launch
// for the join costs more than the pieces save.  us a call in a graph (queued
// one by one), whole / in pieces of 128 keys, 8 KV heads of 128 dims: 200 keys
// 7.9 (9.5) / 9.2 (13.6), 256 8.5 (9.5) / 9.3 (13.1), 400 11.6 (11.6) / 9.3
// (13.1); a compute unit alone draws some 32 bytes a ns.  64 dims: 512 keys 7.1
// (9.5) / 7.1 (13.1), 1024 10.2 / 7.3.
constexpr long long kAlone = 256 * 128;

// How a call is laid out; the same for the work buffer's size and the launch.
struct Plan {
    bool many;          // the many-rows form
    int splits;         // of the window's keys, or of the prefix
    int slots;          // partials a query row (1: none kept)
    int wg_rows;        // query rows of a workgroup
    long long jobs;     // workgroups
    long long own_jobs; // and those of the sequences' own keys behind a prefix
    size_t rows, work;  // query rows, bytes
};

Plan finish(Plan p, int head_dim) {
    p.work = 0;
    if (p.slots > 1) {
        const size_t n = p.rows * p.slots;
        p.work = (n * head_dim * sizeof(float) + 255) / 256 * 256 + (n * sizeof(float2) + 255) / 256 * 256;
    }
    return p;
}

Plan plan_window(int n_seq, int n_tokens, int n_heads, int n_kv, int head_dim, bool q8, int rows, int window,
                 int sinks) {
    Plan p{};
    p.rows = static_cast<size_t>(n_seq) * n_tokens * n_heads;
    long long n = rows;
    if (window > 0 && static_cast<long long>(window) + sinks + n_tokens - 1 < n)
        n = static_cast<long long>(window) + sinks + n_tokens - 1;
    const long long total = static_cast<long long>(n_tokens) * (n_heads / n_kv);
    // keys of a row tile: half of the call's own tokens' on average, or the window's
    long long keys = n - (n_tokens < n ? n_tokens : n) / 2;
    if (window > 0) {
        const long long near = static_cast<long long>(window) + sinks + kManyWaves * kWideRows / (n_heads / n_kv);
        keys = near < keys ? near : keys;
    }
    p.many = takes_many(total, static_cast<long long>(n_seq) * n_kv, keys, head_dim, q8);
    p.wg_rows = p.many ? kManyWaves * kWideRows : kRows;
    p.jobs = n_seq * ((total + p.wg_rows - 1) / p.wg_rows) * n_kv;
    if (!p.many && n * head_dim <= kAlone)
        p.splits = 1;
    else
        p.splits = splits_for(p.many ? fill_many(p.jobs, p.rows, static_cast<long long>(n_seq) * n_kv, n, head_dim)
                                     : kFillFew,
                              p.jobs, n, kMaxSlots);
    p.slots = p.splits;
    p.jobs *= p.splits;
    return finish(p, head_dim);
}

Plan plan_prefix(int n_seq, int n_heads, int n_kv, int head_dim, bool q8, int prefix_len, int own_rows) {
    Plan p{};
    p.rows = static_cast<size_t>(n_seq) * n_heads;
    const int group = n_heads / n_kv;
    const long long total = static_cast<long long>(n_seq) * group;
    p.many = prefix_len > 0 && takes_many(total, n_kv, prefix_len, head_dim, q8);
    p.wg_rows = p.many ? kManyWaves * kWideRows : kRows;
    p.own_jobs = static_cast<long long>(n_seq) * ((group + kRows - 1) / kRows) * n_kv;
    const int own_splits = splits_for(kFillFew, p.own_jobs, own_rows, kMaxSlots / 4);
    const long long jobs = (total + p.wg_rows - 1) / p.wg_rows * n_kv;
    if (prefix_len > 0)
        p.splits = splits_for(p.many ? fill_many(jobs, p.rows, n_kv, prefix_len, head_dim) : kFillFew, jobs, prefix_len,
                              kMaxSlots - own_splits);
    p.jobs = jobs * p.splits;
    p.own_jobs *= own_splits;
    p.slots = p.splits + own_splits;
    return finish(p, head_dim);
}

// The grids of the call's launches: the keys' pieces, and the join's.
asdsl_status check_launches(const char* what, const Plan& p) {
    static_assert(kFewWaves == kManyWaves, "one workgroup size");
    const long long join = p.slots > 1 ? static_cast<long long>((p.rows + kJoinRows - 1) / kJoinRows) : 0;
    ASDSL_CHECK_ARG(fits_launch(p.jobs + p.own_jobs, kFewWaves * 64) && fits_launch(join, kJoinRows * 64),
                    "%s: too many query rows: more than 2^32 work items", what);
    return ASDSL_OK;
}

void place_work(AttnArgs& g, const Plan& p, void* work, int head_dim) {
    if (p.work == 0) return;
    g.part = static_cast<float*>(work);
    g.ml = reinterpret_cast<float2*>(static_cast<char*>(work) +
                                     (p.rows * p.slots * head_dim * sizeof(float) + 255) / 256 * 256);
}

asdsl_status join(const AttnArgs& g, const Plan& p, int head_dim, asdsl_stream_t stream) {
    if (p.slots == 1) return ASDSL_OK;
    return launch("attention_join_kernel", head_dim == 128 ? attention_join_kernel<128> : attention_join_kernel<64>,
                  dim3(static_cast<unsigned>((p.rows + kJoinRows - 1) / kJoinRows)), dim3(kJoinRows * 64), 0,
                  as_hip(stream), g, static_cast<long long>(p.rows));
}

asdsl_status work_of(const char* what, const Plan& p, void* work, size_t work_bytes, asdsl_stream_t stream) {
    if (p.work == 0) return ASDSL_OK;
    ASDSL_CHECK_ARG(work, "%s: needs a work buffer of %zu bytes", what, p.work);
    void* out = nullptr;
    return work_buffer(as_hip(stream), work, work_bytes, p.work, &out, what);
}

asdsl_status window(const char* what, bool q8, const float* q, const Cache& c, const int* pos, float* out, int n_seq,
                    int n_tokens, int n_heads, int n_kv_heads, int head_dim, int rows, int window, int sinks,
                    void* work, size_t work_bytes, asdsl_stream_t stream) {
    ASDSL_CHECK_ARG(q && c.k && c.v && pos && out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(!q8 || (c.ks && c.vs), "%s: null scale array", what);
    asdsl_status st = check_heads(what, n_seq, n_tokens, n_heads, n_kv_heads, head_dim);
    if (st != ASDSL_OK) return st;
    ASDSL_CHECK_ARG(rows > 0 && rows <= kMaxRows, "%s: rows must be positive and at most 2^30", what);
    ASDSL_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window and sinks must not be negative", what);
    ASDSL_CHECK_ARG(aligned16(q) && aligned16(c.k) && aligned16(c.v) && aligned16(out),
                    "%s: q, caches and out must be 16-byte aligned", what);
    const Plan p = plan_window(n_seq, n_tokens, n_heads, n_kv_heads, head_dim, q8, rows, window, sinks);
    st = check_launches(what, p);
    if (st != ASDSL_OK) return st;
    st = work_of(what, p, work, work_bytes, stream);
    if (st != ASDSL_OK) return st;
    AttnArgs g{q, out, nullptr, nullptr, c, c, pos, n_seq, n_tokens, n_heads, n_kv_heads, rows, rows, -1, window,
               sinks, p.splits, p.slots, kLog2e / sqrtf(static_cast<float>(head_dim))};
    place_work(g, p, work, head_dim);
    const dim3 grid(static_cast<unsigned>(p.jobs));
    auto with = [&](auto dim, auto codes) {
        constexpr int kD = decltype(dim)::value;
        constexpr bool kQ8 = decltype(codes)::value;
        if (!p.many)
            return launch("window_few_kernel", window_few_kernel<kD, kQ8>, grid, dim3(kFewWaves * 64), 0,
                          as_hip(stream), g);
        return launch("window_many_kernel", window_many_kernel<kD, kQ8>, grid, dim3(kManyWaves * 64), 0,
                      as_hip(stream), g);
    };
    st = with_form(head_dim, q8, with);
    return st != ASDSL_OK ? st : join(g, p, head_dim, stream);
}

asdsl_status prefix(const char* what, bool q8, const float* q, const Cache& shared, const Cache& own,
                    const int* own_pos, float* out, int n_seq, int n_heads, int n_kv_heads, int head_dim,
                    int prefix_len, int prefix_rows, int own_rows, void* work, size_t work_bytes,
                    asdsl_stream_t stream) {
    ASDSL_CHECK_ARG(q && own.k && own.v && own_pos && out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(prefix_len >= 0 && prefix_len <= prefix_rows && prefix_len <= kMaxRows,
                    "%s: prefix_len must be in [0, prefix_rows] and at most 2^30", what);
    ASDSL_CHECK_ARG(prefix_len == 0 || (shared.k && shared.v), "%s: null pointer", what);
    ASDSL_CHECK_ARG(!q8 || (own.ks && own.vs && (prefix_len == 0 || (shared.ks && shared.vs))),
                    "%s: null scale array", what);
    asdsl_status st = check_heads(what, n_seq, 1, n_heads, n_kv_heads, head_dim);
    if (st != ASDSL_OK) return st;
    ASDSL_CHECK_ARG(own_rows > 0 && own_rows <= kMaxRows, "%s: own_rows must be positive and at most 2^30", what);
    ASDSL_CHECK_ARG(aligned16(q) && aligned16(shared.k) && aligned16(shared.v) && aligned16(own.k) &&
                        aligned16(own.v) && aligned16(out),
                    "%s: q, caches and out must be 16-byte aligned", what);
    const Plan p = plan_prefix(n_seq, n_heads, n_kv_heads, head_dim, q8, prefix_len, own_rows);
    st = check_launches(what, p);
    if (st != ASDSL_OK) return st;
    st = work_of(what, p, work, work_bytes, stream);
    if (st != ASDSL_OK) return st;
    AttnArgs g{q, out, nullptr, nullptr, shared, own, own_pos, n_seq, 1, n_heads, n_kv_heads, prefix_rows, own_rows,
               prefix_len, 0, 0, 0, p.slots, kLog2e / sqrtf(static_cast<float>(head_dim))};
    place_work(g, p, work, head_dim);
    st = with_form(head_dim, q8, [&](auto dim, auto codes) {
        constexpr int kD = decltype(dim)::value;
        constexpr bool kQ8 = decltype(codes)::value;
        return launch("prefix_kernel", p.many ? prefix_kernel<kD, kQ8, true> : prefix_kernel<kD, kQ8, false>,
                      dim3(static_cast<unsigned>(p.jobs + p.own_jobs)), dim3(kFewWaves * 64), 0, as_hip(stream), g,
                      p.splits, static_cast<int>(p.jobs));
    });
    return st != ASDSL_OK ? st : join(g, p, head_dim, stream);
}

}  // namespace
}  // namespace asdsl

using namespace asdsl;

extern "C" asdsl_status asdsl_kv_append_f16(const float* qkv, uint16_t* k_cache, uint16_t* v_cache,
                                            const float* rope_cos, const float* rope_sin, const int* pos,
                                            float* q_out, int n_seq, int n_tokens, int n_heads, int n_kv_heads,
                                            int head_dim, int rotary_dim, int rows, int pos_offset, int rope_rows,
                                            asdsl_stream_t stream) {
    return append("kv_append_f16", false, qkv, k_cache, v_cache, nullptr, nullptr, rope_cos, rope_sin, pos, q_out,
                  n_seq, n_tokens, n_heads, n_kv_heads, head_dim, rotary_dim, rows, pos_offset, rope_rows, stream);
}

extern "C" asdsl_status asdsl_kv_append_q8(const float* qkv, int8_t* k_cache, int8_t* v_cache, float* k_scale,
                                           float* v_scale, const float* rope_cos, const float* rope_sin,
                                           const int* pos, float* q_out, int n_seq, int n_tokens, int n_heads,
                                           int n_kv_heads, int head_dim, int rotary_dim, int rows, int pos_offset,
                                           int rope_rows, asdsl_stream_t stream) {
    return append("kv_append_q8", true, qkv, k_cache, v_cache, k_scale, v_scale, rope_cos, rope_sin, pos, q_out,
                  n_seq, n_tokens, n_heads, n_kv_heads, head_dim, rotary_dim, rows, pos_offset, rope_rows, stream);
}

extern "C" size_t asdsl_attention_window_work_bytes(int n_seq, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                                    int rows, int window_size, int sinks) {
    if (check_heads("attention_window", n_seq, n_tokens, n_heads, n_kv_heads, head_dim) != ASDSL_OK || rows <= 0 ||
        rows > kMaxRows || window_size < 0 || sinks < 0)
        return 0;
    size_t most = 0;  // of the two cache types
    for (const bool q8 : {false, true}) {
        const Plan p = plan_window(n_seq, n_tokens, n_heads, n_kv_heads, head_dim, q8, rows, window_size, sinks);
        most = p.work > most ? p.work : most;
    }
    return most;
}

extern "C" asdsl_status asdsl_attention_window_f16kv(const float* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                                     const int* pos, float* out, int n_seq, int n_tokens, int n_heads,
                                                     int n_kv_heads, int head_dim, int rows, int window_size,
                                                     int sinks, void* work, size_t work_bytes,
                                                     asdsl_stream_t stream) {
    return window("attention_window_f16kv", false, q, Cache{k_cache, v_cache, nullptr, nullptr}, pos, out, n_seq,
                  n_tokens, n_heads, n_kv_heads, head_dim, rows, window_size, sinks, work, work_bytes, stream);
}

extern "C" asdsl_status asdsl_attention_window_q8kv(const float* q, const int8_t* k_cache, const int8_t* v_cache,
                                                    const float* k_scale, const float* v_scale, const int* pos,
                                                    float* out, int n_seq, int n_tokens, int n_heads, int n_kv_heads,
                                                    int head_dim, int rows, int window_size, int sinks, void* work,
                                                    size_t work_bytes, asdsl_stream_t stream) {
    return window("attention_window_q8kv", true, q, Cache{k_cache, v_cache, k_scale, v_scale}, pos, out, n_seq,
                  n_tokens, n_heads, n_kv_heads, head_dim, rows, window_size, sinks, work, work_bytes, stream);
}

extern "C" size_t asdsl_attention_prefix_work_bytes(int n_seq, int n_heads, int n_kv_heads, int head_dim,
                                                    int prefix_len, int own_rows) {
    if (check_heads("attention_prefix", n_seq, 1, n_heads, n_kv_heads, head_dim) != ASDSL_OK || prefix_len < 0 ||
        prefix_len > kMaxRows || own_rows <= 0 || own_rows > kMaxRows)
        return 0;
    size_t most = 0;  // of the two cache types
    for (const bool q8 : {false, true}) {
        const Plan p = plan_prefix(n_seq, n_heads, n_kv_heads, head_dim, q8, prefix_len, own_rows);
        most = p.work > most ? p.work : most;
    }
    return most;
}

extern "C" asdsl_status asdsl_attention_prefix_f16kv(const float* q, const uint16_t* k_prefix,
                                                     const uint16_t* v_prefix, const uint16_t* k_own,
                                                     const uint16_t* v_own, const int* own_pos, float* out, int n_seq,
                                                     int n_heads, int n_kv_heads, int head_dim, int prefix_len,
                                                     int prefix_rows, int own_rows, void* work, size_t work_bytes,
                                                     asdsl_stream_t stream) {
    return prefix("attention_prefix_f16kv", false, q, Cache{k_prefix, v_prefix, nullptr, nullptr},
                  Cache{k_own, v_own, nullptr, nullptr}, own_pos, out, n_seq, n_heads, n_kv_heads, head_dim,
                  prefix_len, prefix_rows, own_rows, work, work_bytes, stream);
}

extern "C" asdsl_status asdsl_attention_prefix_q8kv(const float* q, const int8_t* k_prefix, const int8_t* v_prefix,
                                                    const float* k_prefix_scale, const float* v_prefix_scale,
                                                    const int8_t* k_own, const int8_t* v_own, const float* k_own_scale,
                                                    const float* v_own_scale, const int* own_pos, float* out,
                                                    int n_seq, int n_heads, int n_kv_heads, int head_dim,
                                                    int prefix_len, int prefix_rows, int own_rows, void* work,
                                                    size_t work_bytes, asdsl_stream_t stream) {
    return prefix("attention_prefix_q8kv", true, q, Cache{k_prefix, v_prefix, k_prefix_scale, v_prefix_scale},
                  Cache{k_own, v_own, k_own_scale, v_own_scale}, own_pos, out, n_seq, n_heads, n_kv_heads, head_dim,
                  prefix_len, prefix_rows, own_rows, work, work_bytes, stream);
}
