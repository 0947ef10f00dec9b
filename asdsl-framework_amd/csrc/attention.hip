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
// Eight dims of one head of one token per lane.  A rotated pair is
// (fmaf(a, c, -(b * s)), fmaf(a, s, b * c)), as in the decode step's
// attention, and the stored forms are its too: fp16 rounded to nearest, or
// per 64 dims scale = amax * (1/127) (1e-12 when amax <= 1e-12) and code =
// round-half-even(x * (1 / scale)) clamped to [-127, 127].
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
    long long units;  // 8-dim units of the call
};

template <int D, bool Q8>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
    constexpr int kUnits = D / 8;  // per head
    const long long e = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (e >= a.units) return;  // units are a multiple of 8: the lanes of a 64-dim block leave together
    const int heads = a.n_heads + 2 * a.n_kv;
    const int dc = static_cast<int>(e % kUnits);
    const long long hr = e / kUnits;
    const int head = static_cast<int>(hr % heads);
    const long long row = hr / heads;  // token row of the call
    const int seq = static_cast<int>(row / a.n_tokens);
    const long long r = static_cast<long long>(a.pos[seq]) + row % a.n_tokens;  // cache row
    const long long p = r + a.offset;                                           // rotary position
    const bool inside = r >= 0 && r < a.rows && p >= 0 && p < a.rope_rows;
    if (!inside && head >= a.n_heads) return;
    const float* src = a.qkv + (row * heads + head) * D;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = 8 * dc + i;
        if (!inside) {
            x[i] = 0.0f;
        } else if (head >= a.n_heads + a.n_kv || d >= 2 * a.rot_half) {
            x[i] = src[d];
        } else {
            const int j = d < a.rot_half ? d : d - a.rot_half;
            const float lo = src[j], hi = src[j + a.rot_half];
            const float c = a.cos[p * a.rot_half + j], s = a.sin[p * a.rot_half + j];
            x[i] = d < a.rot_half ? fmaf(lo, c, -(hi * s)) : fmaf(lo, s, hi * c);
        }
    }
    if (head < a.n_heads) {
        float4* dst = reinterpret_cast<float4*>(a.q_out + (row * a.n_heads + head) * D + 8 * dc);
        dst[0] = make_float4(x[0], x[1], x[2], x[3]);
        dst[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    const bool key = head < a.n_heads + a.n_kv;
    const int kvh = head - a.n_heads - (key ? 0 : a.n_kv);
    const long long crow = (static_cast<long long>(seq) * a.n_kv + kvh) * a.rows + r;
    void* base = key ? a.k : a.v;
    if constexpr (Q8) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
        m = group_max<8>(m);
        const float scale = m > 1e-12f ? m * kInv127 : 1e-12f;
        const float inv = 1.0f / scale;
        int q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            q[i] = static_cast<int>(fminf(fmaxf(__builtin_rintf(x[i] * inv), -127.0f), 127.0f));
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(base) + crow * D + 8 * dc) =
            make_uint2(pack4_i8(q[0], q[1], q[2], q[3]), pack4_i8(q[4], q[5], q[6], q[7]));
        if ((dc & 7) == 0) (key ? a.ks : a.vs)[crow * (D / kBlockDims) + (dc >> 3)] = scale;
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[2 * i]))) |
                   (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[2 * i + 1]))) << 16);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + crow * D + 8 * dc) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// --------------------------------------------------------------- attention
// Scores and weights are fp32 in the definition, and K and V are fp16 numbers
// (or int8 codes, exact in fp16), so only the query and the weights have to be
// cut for the matrix instructions: each is held as the sum of two fp16 numbers,
// a first part of 11 bits and the rest (2^-22 off at most), at twice the
// products.  One part alone would leave 2^-12 a weight, 1e-4 of an output.
// The parts keep clear of fp16's small numbers: a query row is scaled by a power
// of two to 2^12..2^13, the weights are 2^kShift times theirs (the first part is
// then whole down to 2^-22 of the largest weight, the second to 2^-11 of it, and
// off by 2^-33 of it below; a larger shift costs the exponent's argument bits).
//
// A wave takes 16 query rows (the columns of its tiles) and 32 keys a step:
//   S' = K Q'  two 16x16 tiles; a lane gets 8 scores of the one row it holds, so
//              the running maximum and sum need two lane exchanges a step
//   O' = V' P' the lane's 8 weights are its operand as they stand when V's is
//              read for the same 8 keys: every lane loads its D / 16 dims of those
//              keys and turns the block in registers; no transposition in memory.
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;      // query rows of a wave's tile
constexpr int kKeys = 32;      // keys of a wave's step
constexpr float kShift = 8.0f;
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

// The other operand's value from lane ^ 32 and lane ^ 16: the swap exchanges one
// half (rows of 16) of a register with the other half of a second one, so with
// two copies of v the results hold both lanes' values.  The copy is kept
// apart from v: given one register twice, the swap leaves it as it is.
template <typename F>
__device__ __forceinline__ float lanes16(float v, F f) {
    uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
    asm("" : "+v"(b));
    auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    v = f(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
    a = b = __builtin_bit_cast(uint32_t, v);
    asm("" : "+v"(b));
    r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return f(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

// Over the four lanes of equal lane % 16.
__device__ __forceinline__ float lanes16_max(float v) {
    return lanes16(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float lanes16_sum(float v) {
    return lanes16(v, [](float x, float y) { return x + y; });
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float pow2(int e) {  // 2^e, -126 <= e <= 127
    return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ int exponent(float x) {
    return static_cast<int>((__builtin_bit_cast(uint32_t, x) >> 23) & 0xFFu) - 127;
}

// x = hi + lo with fp16 parts, two at a time.
__device__ __forceinline__ void two_parts(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const half2v h = {static_cast<_Float16>(x0), static_cast<_Float16>(x1)};
    const half2v l = {static_cast<_Float16>(x0 - static_cast<float>(h.x)),
                      static_cast<_Float16>(x1 - static_cast<float>(h.y))};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ half8 as_half8(const uint32_t (&w)[4]) {
    return __builtin_bit_cast(half8, make_uint4(w[0], w[1], w[2], w[3]));
}

// Two bytes c0 at bits 0-7 and c1 at bits 16-23 of w, int8 codes with their top
// bit flipped, as fp16 numbers: 0x6400 | u is 1024 + u, exactly.
__device__ __forceinline__ uint32_t codes_half2(uint32_t w) {
    const half2v h = __builtin_bit_cast(half2v, w | 0x64006400u) - half2v{_Float16(1152.0f), _Float16(1152.0f)};
    return __builtin_bit_cast(uint32_t, h);
}

// Eight int8 codes as the K operand's eight fp16 numbers.
__device__ __forceinline__ half8 codes_half8(uint2 c) {
    uint32_t w[4];
    c.x ^= 0x80808080u;
    c.y ^= 0x80808080u;
    w[0] = codes_half2(__builtin_amdgcn_perm(0u, c.x, 0x0C010C00u));
    w[1] = codes_half2(__builtin_amdgcn_perm(0u, c.x, 0x0C030C02u));
    w[2] = codes_half2(__builtin_amdgcn_perm(0u, c.y, 0x0C010C00u));
    w[3] = codes_half2(__builtin_amdgcn_perm(0u, c.y, 0x0C030C02u));
    return as_half8(w);
}

// A query row's operands: dims 32 * s + 8 * (lane / 16) .. + 8 in step s.
template <int D>
struct Query {
    half8 hi[D / 32], lo[D / 32];
    float c;  // score = product * c, in powers of two

    __device__ __forceinline__ void load(const float* row, int gq, float scale) {
        float x[D / 32][8];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            if (row) {
                const float4 a = *reinterpret_cast<const float4*>(row + 32 * s + 8 * gq);
                const float4 b = *reinterpret_cast<const float4*>(row + 32 * s + 8 * gq + 4);
                x[s][0] = a.x; x[s][1] = a.y; x[s][2] = a.z; x[s][3] = a.w;
                x[s][4] = b.x; x[s][5] = b.y; x[s][6] = b.z; x[s][7] = b.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[s][i]));
        }
        top = lanes16_max(top);
        int e = 12 - exponent(top);  // a query that is not finite stays as it is
        e = e < -115 ? 0 : (e > 120 ? 120 : e);
        const float f = pow2(e);
        c = scale * pow2(-e);
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
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
    __device__ __forceinline__ void load(const void* v, int key, size_t row, int r) {
        const uint16_t* src = static_cast<const uint16_t*>(v) + row * D + D / 16 * r;
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
    // whether any value is an infinity or NaN (an exponent of all ones)
    __device__ __forceinline__ bool odd() const {
        uint32_t any = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) any |= (w[i][d] & 0x7C007C00u) + 0x04000400u;
        return (any & 0x80008000u) != 0u;
    }
};
template <int D>
struct VRaw<D, true> {
    uint32_t w[8][D / 64];
    __device__ __forceinline__ void load(const void* v, int key, size_t row, int r) {
        const int8_t* src = static_cast<const int8_t*>(v) + row * D + 4 * r;
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
            w[key][b] = *reinterpret_cast<const uint32_t*>(src + 64 * b) ^ 0x80808080u;
    }
    __device__ __forceinline__ half8 operand(int j) const {
        uint32_t o[4];
        const uint32_t sel = 0x0C040C00u + 0x00010001u * static_cast<uint32_t>(j & 3);
#pragma unroll
        for (int p = 0; p < 4; ++p) o[p] = codes_half2(__builtin_amdgcn_perm(w[2 * p + 1][j >> 2], w[2 * p][j >> 2], sel));
        return as_half8(o);
    }
};

// Running state of one query row (column lane % 16): the base m of its weights
// exp2(score - m), kShift below the largest score so far, their sum over the
// lane's share of the keys, and O' with element i of acc[j] at dim
// *_dim(4 * (lane / 16) + i, j).  An int8 cache's value scales go into the
// weights before they are cut; ev is the power of two that keeps those in
// fp16's range (the accumulator is 2^-ev times O').
template <int D, bool Q8>
struct State {
    float m = -INFINITY, l = 0.0f;
    int ev = -126;
    f32x4 acc[D / 16];

    __device__ __forceinline__ State() {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // The weights of N keys from their products s (score = s * c; -inf where not
    // seen), in place.  vs_max: the largest finite value scale among the keys
    // of this step that the row sees.
    template <int N>
    __device__ __forceinline__ void weigh(float (&s)[N], float c, float vs_max) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, s[i]);
        const float m1 = fmaxf(m, lanes16_max(top) * c - kShift);
        const float base = m1 == -INFINITY ? 0.0f : m1;
        float alpha = exp2_fast(m - base);
        l *= alpha;
        if constexpr (Q8) {
            const int e1 = max(ev, exponent(lanes16_max(vs_max)));
            alpha *= pow2(max(ev - e1, -126));
            ev = e1;
        }
        m = m1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = exp2_fast(fmaf(s[i], c, -base));
            l += s[i];
        }
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0ull) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) acc[j] *= alpha;
        }
    }
};

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int cache_row(const Keys& K, int i) { return i < K.na ? i : i + K.db; }

// Whether every one of the workgroup's tokens sees all the keys [i0, i0 + n).
__device__ __forceinline__ bool all_seen(const Keys& K, int i0, int n) {
    if (i0 + n > K.n) return false;
    if (!K.masked) return true;
    return cache_row(K, i0 + n - 1) <= K.p_first && (i0 + n <= K.na || cache_row(K, max(i0, K.na)) >= K.lo_last);
}

// P' of 8 keys (s) as two fp16 operands, and O' += V' P'.
template <int D, bool Q8>
__device__ __forceinline__ void add_values(State<D, Q8>& st, const VRaw<D, Q8>& v, const float (&s)[8],
                                           const float (&vs)[8][D / 64], uint32_t seen, bool all) {
    if constexpr (Q8) {
        const float f = pow2(min(max(-st.ev, -126), 126));
#pragma unroll
        for (int b = 0; b < D / 64; ++b) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // a scale of a key that the row does not see may be anything
                const float x0 = (seen >> (2 * i)) & 1u ? s[2 * i] * (vs[2 * i][b] * f) : 0.0f;
                const float x1 = (seen >> (2 * i + 1)) & 1u ? s[2 * i + 1] * (vs[2 * i + 1][b] * f) : 0.0f;
                two_parts(x0, x1, h[i], l[i]);
            }
#pragma unroll
            for (int j = 4 * b; j < 4 * b + 4; ++j) {
                const half8 o = v.operand(j);
                st.acc[j] = mfma(o, as_half8(h), st.acc[j]);
                st.acc[j] = mfma(o, as_half8(l), st.acc[j]);
            }
        }
    } else {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) two_parts(s[2 * i], s[2 * i + 1], h[i], l[i]);
        // Infinities and NaN among the values of keys that not every row sees:
        // a weight of zero would make them NaN in every row.  They are taken
        // out, and NaN goes to the outputs of the rows that see them.
        if (!all && __builtin_amdgcn_ballot_w64(v.odd()) != 0ull) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = ((seen >> (2 * i)) & 1u ? 0x3C00u : 0u) | ((seen >> (2 * i + 1)) & 1u ? 0x3C000000u : 0u);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const uint4 o = __builtin_bit_cast(uint4, v.operand(j));
                uint32_t clean[4] = {o.x, o.y, o.z, o.w}, bad[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t t = ((clean[i] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
                    const uint32_t mask = (t & 0x8000u ? 0xFFFFu : 0u) | (t & 0x80000000u ? 0xFFFF0000u : 0u);
                    bad[i] = mask & 0x3C003C00u;
                    clean[i] &= ~mask;
                }
                const f32x4 hit = mfma(as_half8(bad), as_half8(w), f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                st.acc[j] = mfma(as_half8(clean), as_half8(h), st.acc[j]);
                st.acc[j] = mfma(as_half8(clean), as_half8(l), st.acc[j]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (hit[i] > 0.0f) st.acc[j][i] = __builtin_nanf("");
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            const half8 o = v.operand(j);
            st.acc[j] = mfma(o, as_half8(h), st.acc[j]);
            st.acc[j] = mfma(o, as_half8(l), st.acc[j]);
        }
    }
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

    __device__ __forceinline__ void load_k(const Keys& K, int t, int lane) {
        const int r = lane & 15, gq = lane >> 4;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const size_t row = cache_row(K, min(t * kKeys + 16 * kt + r, K.n - 1));
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                if constexpr (Q8)
                    k8[kt][s] = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(K.k) + row * D + 32 * s + 8 * gq);
                else
                    k16[kt][s] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(K.k) + row * D + 32 * s + 8 * gq);
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t row = cache_row(K, min(t * kKeys + (i & 4) * 4 + 4 * gq + (i & 3), K.n - 1));
#pragma unroll
                for (int b = 0; b < D / 64; ++b) ks[i][b] = K.ks[row * (D / 64) + b];
            }
        }
    }
    __device__ __forceinline__ void load_v(const Keys& K, int t, int lane) {
        const int r = lane & 15, gq = lane >> 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t row = cache_row(K, min(t * kKeys + (i & 4) * 4 + 4 * gq + (i & 3), K.n - 1));
            v.load(K.v, i, row, r);
            if constexpr (Q8) {
#pragma unroll
                for (int b = 0; b < D / 64; ++b) vs[i][b] = K.vs[row * (D / 64) + b];
            }
        }
    }
    __device__ __forceinline__ void scores(const Query<D>& q, float (&s)[8]) const {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            if constexpr (Q8) {
                f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < D / 64; ++b) {
                    f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int x = 2 * b; x < 2 * b + 2; ++x) {
                        const half8 k = codes_half8(k8[kt][x]);
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
                    const half8 k = __builtin_bit_cast(half8, k16[kt][x]);
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
__device__ __forceinline__ void few_rows(const Keys& K, const Query<D>& q, const RowSight& see, int t0, int t1,
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
        if (!all) {
            seen = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = t * kKeys + (i & 4) * 4 + 4 * gq + (i & 3);
                const int row = cache_row(K, at);
                const bool ok = at < K.n && (!K.masked || (row <= see.p && (row >= see.lo || row < K.sinks)));
                s[i] = ok ? s[i] : -INFINITY;
                seen |= ok ? 1u << i : 0u;
            }
        }
        float vs_max = 0.0f;
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int b = 0; b < D / 64; ++b) {
                    const float a = fabsf(x.vs[i][b]);
                    vs_max = (seen >> i) & 1u && a < 1e30f ? fmaxf(vs_max, a) : vs_max;
                }
        }
        st.weigh(s, q.c, vs_max);
        add_values<D, Q8>(st, x.v, s, x.vs, seen, all);
        if (next < t1) x.load_v(K, next, lane);
    }
}

// The workgroup's waves joined: their (maximum, sum) and O' through LDS, then
// each thread forms its share of the 16 rows: as out rows where the job has all
// the keys (final), else as partials for attention_join_kernel.
template <int D, int W>
struct JoinArea {
    float acc[W][kRows][D + 4];
    float2 ml[W][kRows];
};

// The factor of a part (base, sum) under the common base m: none without keys,
// NaN for a sum that is NaN.
__device__ __forceinline__ float share(float2 ml, float m) {
    return ml.y == 0.0f ? 0.0f : ml.y == ml.y ? exp2_fast(ml.x - m) : ml.y;
}

template <int D, bool Q8>
__device__ __forceinline__ float out_scale(const State<D, Q8>& st) {
    if constexpr (Q8) return pow2(min(max(st.ev, -126), 127));
    return 1.0f;
}

template <int D, bool Q8>
__device__ __forceinline__ void store_row(float* dst, const State<D, Q8>& st, int gq, float f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * gq + i;
#pragma unroll
        for (int j = 0; j < D / 16; j += 4) {
            const int d = Q8 ? code_dim(r, j) : fp16_dim<D>(r, j);
            *reinterpret_cast<float4*>(dst + d) =
                make_float4(st.acc[j][i] * f, st.acc[j + 1][i] * f, st.acc[j + 2][i] * f, st.acc[j + 3][i] * f);
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
    s.p = s.any ? static_cast<int>(p) : -1;
    s.lo = window > 0 ? s.p - window + 1 : 0;
    return s;
}

template <int D, bool Q8>
__device__ __forceinline__ void few_job(const AttnArgs& g, const Keys& K, const RowMap& map, int row0, long long p0,
                                        int rows, int split, int splits, int slot, JoinArea<D, kFewWaves>& area) {
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int n = row0 + (lane & 15), gq = lane >> 4;
    const bool real = n < map.total;
    Query<D> q;
    q.load(real ? g.q + map.at(n) * D : nullptr, gq, g.scale);
    const RowSight see = sight(K, p0 + n / map.g, rows, g.window);
    State<D, Q8> st;
    const int steps = (K.n + kKeys - 1) / kKeys;
    // a split's steps, a multiple of the waves'
    const int per = ((steps + splits - 1) / splits + kFewWaves - 1) / kFewWaves * kFewWaves;
    few_rows<D, Q8>(K, q, see, split * per + wave, min(steps, (split + 1) * per), kFewWaves, lane, st);
    st.l = lanes16_sum(st.l);
    store_row<D, Q8>(area.acc[wave][lane & 15], st, gq, out_scale(st));
    if (gq == 0) area.ml[wave][lane & 15] = make_float2(st.m, st.l);
    __syncthreads();
    constexpr int kPer = kRows * D / (kFewWaves * 64);  // values a thread: 8 (D 128) or 4
    const int r = tid * kPer / D, d = tid * kPer % D;
    if (row0 + r >= map.total) return;
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
    const long long at = map.at(row0 + r);
    float* dst;
    if (g.slots == 1) {
        const bool any = sight(K, p0 + (row0 + r) / map.g, rows, g.window).any && l != 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] = any ? o[e] / l : 0.0f;
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

// blockIdx.x = ((sequence * row tiles + tile) * splits + split) * n_kv + kv head:
// with 8 KV heads one head's workgroups share an XCD's L2.
template <int D, bool Q8>
__global__ __launch_bounds__(kFewWaves * 64) void window_few_kernel(const AttnArgs g) {
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

// Shared prefix: the first jobs take 16 (sequence, head) rows of a KV head and a
// split of the prefix, the others a sequence's own keys.
template <int D, bool Q8>
__global__ __launch_bounds__(kFewWaves * 64) void prefix_few_kernel(const AttnArgs g, int prefix_splits, int jobs) {
    __shared__ JoinArea<D, kFewWaves> area;
    const int group = g.n_heads / g.n_kv;
    int b = static_cast<int>(blockIdx.x);
    if (b < jobs) {
        const int total = g.n_seq * group;
        const int tiles = (total + kRows - 1) / kRows;
        const int kvh = b % g.n_kv;
        b /= g.n_kv;
        const int row0 = b % tiles * kRows;
        const int split = b / tiles;
        const RowMap map{static_cast<long long>(kvh) * group, group, g.n_heads, total};
        Keys K = head_keys<D, Q8>(g.a, kvh, g.rows_a);
        K.n = g.prefix;
        few_job<D, Q8>(g, K, map, row0, 0, 0, split, prefix_splits, split, area);
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
    few_job<D, Q8>(g, K, map, row0, 0, 0, split, own_splits, prefix_splits + split, area);
}

// One wave per query row: its partials in slot order.
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
    float acc[D / 64] = {};
    const float* part = g.part + row * g.slots * D + lane * (D / 64);
    for (int s = 0; s < g.slots; ++s) {
        const float ws = __shfl(w, s, kWave);
        if (ws == 0.0f) continue;  // the same in every lane
#pragma unroll
        for (int i = 0; i < D / 64; ++i) acc[i] = fmaf(part[s * D + i], ws, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) g.out[row * D + lane * (D / 64) + i] = any && l != 0.0f ? acc[i] / l : 0.0f;
}

// ------------------------------------------------------------- host checks
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
    AppendArgs a{qkv, k, v, ks, vs, rope_cos, rope_sin, pos, q_out, n_tokens, n_heads, n_kv_heads, rotary_dim / 2,
                 rows, pos_offset, rope_rows, 0};
    a.units = static_cast<long long>(n_seq) * n_tokens * (n_heads + 2 * n_kv_heads) * (head_dim / 8);
    auto kern = head_dim == 128 ? (q8 ? kv_append_kernel<128, true> : kv_append_kernel<128, false>)
                                : (q8 ? kv_append_kernel<64, true> : kv_append_kernel<64, false>);
    return launch("kv_append_kernel", kern, dim3(static_cast<unsigned>((a.units + 255) / 256)), dim3(256), 0,
                  as_hip(stream), a);
}

// Workgroups that fill the device (256 compute units), and how many key splits
// get a launch of `jobs` workgroups there when each split keeps at least
// `least` of at most n keys.
constexpr long long kFill = 512;

int splits_for(long long jobs, long long n, int least, int most) {
    long long s = (kFill + jobs - 1) / jobs;
    const long long by_keys = (n + least - 1) / least;
    s = s < by_keys ? s : by_keys;
    s = s < most ? s : most;
    return s > 1 ? static_cast<int>(s) : 1;
}

// How a call is laid out; the same for the work buffer's size and the launch.
struct Plan {
    int splits;         // of the window's keys, or of the prefix
    int slots;          // partials a query row (1: none kept)
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

Plan plan_window(int n_seq, int n_tokens, int n_heads, int n_kv, int head_dim, int rows, int window, int sinks) {
    Plan p{};
    p.rows = static_cast<size_t>(n_seq) * n_tokens * n_heads;
    long long n = rows;
    if (window > 0 && static_cast<long long>(window) + sinks + n_tokens - 1 < n)
        n = static_cast<long long>(window) + sinks + n_tokens - 1;
    const long long tiles = (static_cast<long long>(n_tokens) * (n_heads / n_kv) + kRows - 1) / kRows;
    p.splits = p.slots = splits_for(n_seq * tiles * n_kv, n, kFewWaves * kKeys, kMaxSlots);
    return finish(p, head_dim);
}

Plan plan_prefix(int n_seq, int n_heads, int n_kv, int head_dim, int prefix_len, int own_rows) {
    Plan p{};
    p.rows = static_cast<size_t>(n_seq) * n_heads;
    const int group = n_heads / n_kv;
    const long long tiles = (static_cast<long long>(n_seq) * group + kRows - 1) / kRows;
    const long long own_jobs = static_cast<long long>(n_seq) * ((group + kRows - 1) / kRows) * n_kv;
    p.splits = prefix_len > 0 ? splits_for(tiles * n_kv, prefix_len, kFewWaves * kKeys, kMaxSlots / 2) : 0;
    p.slots = p.splits + splits_for(own_jobs, own_rows, kFewWaves * kKeys, kMaxSlots / 2);
    return finish(p, head_dim);
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
    ASDSL_CHECK_ARG(rows > 0, "%s: rows must be positive", what);
    ASDSL_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window and sinks must not be negative", what);
    ASDSL_CHECK_ARG(aligned16(q) && aligned16(c.k) && aligned16(c.v) && aligned16(out),
                    "%s: q, caches and out must be 16-byte aligned", what);
    const Plan p = plan_window(n_seq, n_tokens, n_heads, n_kv_heads, head_dim, rows, window, sinks);
    st = work_of(what, p, work, work_bytes, stream);
    if (st != ASDSL_OK) return st;
    AttnArgs g{q, out, nullptr, nullptr, c, c, pos, n_seq, n_tokens, n_heads, n_kv_heads, rows, rows, -1, window,
               sinks, p.splits, p.slots, kLog2e / sqrtf(static_cast<float>(head_dim))};
    place_work(g, p, work, head_dim);
    const long long tiles = (static_cast<long long>(n_tokens) * (n_heads / n_kv_heads) + kRows - 1) / kRows;
    const long long grid = n_seq * tiles * p.splits * n_kv_heads;
    ASDSL_CHECK_ARG(grid <= INT_MAX, "%s: too many query rows", what);
    auto kern = head_dim == 128 ? (q8 ? window_few_kernel<128, true> : window_few_kernel<128, false>)
                                : (q8 ? window_few_kernel<64, true> : window_few_kernel<64, false>);
    st = launch("window_few_kernel", kern, dim3(static_cast<unsigned>(grid)), dim3(kFewWaves * 64), 0, as_hip(stream),
                g);
    return st != ASDSL_OK ? st : join(g, p, head_dim, stream);
}

asdsl_status prefix(const char* what, bool q8, const float* q, const Cache& shared, const Cache& own,
                    const int* own_pos, float* out, int n_seq, int n_heads, int n_kv_heads, int head_dim,
                    int prefix_len, int prefix_rows, int own_rows, void* work, size_t work_bytes,
                    asdsl_stream_t stream) {
    ASDSL_CHECK_ARG(q && own.k && own.v && own_pos && out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(prefix_len >= 0 && prefix_len <= prefix_rows,
                    "%s: prefix_len must be in [0, prefix_rows]", what);
    ASDSL_CHECK_ARG(prefix_len == 0 || (shared.k && shared.v), "%s: null pointer", what);
    ASDSL_CHECK_ARG(!q8 || (own.ks && own.vs && (prefix_len == 0 || (shared.ks && shared.vs))),
                    "%s: null scale array", what);
    asdsl_status st = check_heads(what, n_seq, 1, n_heads, n_kv_heads, head_dim);
    if (st != ASDSL_OK) return st;
    ASDSL_CHECK_ARG(own_rows > 0, "%s: own_rows must be positive", what);
    ASDSL_CHECK_ARG(aligned16(q) && aligned16(shared.k) && aligned16(shared.v) && aligned16(own.k) &&
                        aligned16(own.v) && aligned16(out),
                    "%s: q, caches and out must be 16-byte aligned", what);
    const Plan p = plan_prefix(n_seq, n_heads, n_kv_heads, head_dim, prefix_len, own_rows);
    st = work_of(what, p, work, work_bytes, stream);
    if (st != ASDSL_OK) return st;
    AttnArgs g{q, out, nullptr, nullptr, shared, own, own_pos, n_seq, 1, n_heads, n_kv_heads, prefix_rows, own_rows,
               prefix_len, 0, 0, 0, p.slots, kLog2e / sqrtf(static_cast<float>(head_dim))};
    place_work(g, p, work, head_dim);
    const int group = n_heads / n_kv_heads;
    const long long jobs = (static_cast<long long>(n_seq) * group + kRows - 1) / kRows * p.splits * n_kv_heads;
    const long long own_jobs = static_cast<long long>(n_seq) * ((group + kRows - 1) / kRows) * (p.slots - p.splits) *
                               n_kv_heads;
    ASDSL_CHECK_ARG(jobs + own_jobs <= INT_MAX, "%s: too many query rows", what);
    auto kern = head_dim == 128 ? (q8 ? prefix_few_kernel<128, true> : prefix_few_kernel<128, false>)
                                : (q8 ? prefix_few_kernel<64, true> : prefix_few_kernel<64, false>);
    st = launch("prefix_few_kernel", kern, dim3(static_cast<unsigned>(jobs + own_jobs)), dim3(kFewWaves * 64), 0,
                as_hip(stream), g, p.splits, static_cast<int>(jobs));
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
        window_size < 0 || sinks < 0)
        return 0;
    return plan_window(n_seq, n_tokens, n_heads, n_kv_heads, head_dim, rows, window_size, sinks).work;
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
        own_rows <= 0)
        return 0;
    return plan_prefix(n_seq, n_heads, n_kv_heads, head_dim, prefix_len, own_rows).work;
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
