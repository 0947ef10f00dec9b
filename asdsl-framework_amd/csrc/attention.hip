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
// The keys a row sees are two ranges: rows [0, na) of cache A, then rows
// [b0, b0 + nb) of cache B.  With a window A is the cache's first tokens and B
// its window; with a shared prefix A is the prefix and B the sequence's rows.
struct AttnArgs {
    const float* q;
    float* out;
    Cache a, b;
    const int* pos;
    int n_tokens, n_heads, n_kv, rows_a, rows_b;
    int prefix;           // shared prefix: rows of A that all see; -1 with a window
    int window, sinks;
    long long q_rows;     // n_seq * n_tokens * n_heads
    float scale;
};

struct Ranges {
    long long na, b0, nb;
};

__device__ __forceinline__ Ranges visible(const AttnArgs& g, int seq, int t) {
    const long long p = static_cast<long long>(g.pos[seq]) + t;
    if (g.prefix >= 0) {
        if (p < -1 || p >= g.rows_b) return {0, 0, 0};
        return {g.prefix, 0, p + 1};
    }
    if (p < 0 || p >= g.rows_b) return {0, 0, 0};
    const long long lo = g.window > 0 && p - g.window + 1 > 0 ? p - g.window + 1 : 0;
    const long long na = lo < g.sinks ? lo : g.sinks;
    return {na, lo, p + 1 - lo};
}

template <int D, bool Q8>
__device__ __forceinline__ float kv_at(const void* x, const float* scales, long long row, int d) {
    if constexpr (Q8)
        return static_cast<float>(static_cast<const int8_t*>(x)[row * D + d]) *
               scales[row * (D / kBlockDims) + d / kBlockDims];
    else
        return __half2float(__ushort_as_half(static_cast<const uint16_t*>(x)[row * D + d]));
}

// One wave per query row, 64 keys a step: a lane forms its key's score, the
// wave's running maximum and sum follow, then each lane adds its dims.
template <int D, bool Q8>
__global__ __launch_bounds__(64) void attention_row_kernel(const AttnArgs g) {
    __shared__ float qs[D];
    __shared__ float ps[64];
    const long long row = blockIdx.x;
    const int lane = static_cast<int>(threadIdx.x);
    const int head = static_cast<int>(row % g.n_heads);
    const long long tok = row / g.n_heads;
    const int seq = static_cast<int>(tok / g.n_tokens);
    const int kvh = head / (g.n_heads / g.n_kv);
    const Ranges v = visible(g, seq, static_cast<int>(tok % g.n_tokens));
    for (int d = lane; d < D; d += 64) qs[d] = g.q[row * D + d] * g.scale;
    __syncthreads();
    const long long base_a = (g.prefix >= 0 ? kvh : static_cast<long long>(seq) * g.n_kv + kvh) * g.rows_a;
    const long long base_b = (static_cast<long long>(seq) * g.n_kv + kvh) * g.rows_b + v.b0;
    float m = -INFINITY, l = 0.0f, acc[D / 64] = {};
    const long long n = v.na + v.nb;
    for (long long k0 = 0; k0 < n; k0 += 64) {
        const long long k = k0 + lane;
        float s = -INFINITY;
        if (k < n) {
            const bool in_a = k < v.na;
            const Cache& c = in_a ? g.a : g.b;
            const long long crow = in_a ? base_a + k : base_b + (k - v.na);
            s = 0.0f;
            for (int d = 0; d < D; ++d) s = fmaf(qs[d], kv_at<D, Q8>(c.k, c.ks, crow, d), s);
        }
        float top = s;
        for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float m1 = fmaxf(m, top);
        const float base = m1 == -INFINITY ? 0.0f : m1;
        const float p = k < n ? expf(s - base) : 0.0f;
        const float alpha = expf(m - base);
        float sum = p;
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        l = l * alpha + sum;
        m = m1;
        ps[lane] = p;
        __syncthreads();
        for (int i = 0; i < D / 64; ++i) acc[i] *= alpha;
        const int cnt = static_cast<int>(n - k0 < 64 ? n - k0 : 64);
        for (int j = 0; j < cnt; ++j) {
            const bool in_a = k0 + j < v.na;
            const Cache& c = in_a ? g.a : g.b;
            const long long crow = in_a ? base_a + k0 + j : base_b + (k0 + j - v.na);
            for (int i = 0; i < D / 64; ++i)
                acc[i] = fmaf(ps[j], kv_at<D, Q8>(c.v, c.vs, crow, lane + 64 * i), acc[i]);
        }
        __syncthreads();
    }
    for (int i = 0; i < D / 64; ++i) g.out[row * D + lane + 64 * i] = n > 0 ? acc[i] / l : 0.0f;
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

asdsl_status attend(const char* what, bool q8, AttnArgs g, int n_seq, int head_dim, asdsl_stream_t stream) {
    g.scale = 1.0f / sqrtf(static_cast<float>(head_dim));
    g.q_rows = static_cast<long long>(n_seq) * g.n_tokens * g.n_heads;
    auto kern = head_dim == 128 ? (q8 ? attention_row_kernel<128, true> : attention_row_kernel<128, false>)
                                : (q8 ? attention_row_kernel<64, true> : attention_row_kernel<64, false>);
    return launch("attention_row_kernel", kern, dim3(static_cast<unsigned>(g.q_rows)), dim3(64), 0, as_hip(stream), g);
}

asdsl_status window(const char* what, bool q8, const float* q, const Cache& c, const int* pos, float* out, int n_seq,
                    int n_tokens, int n_heads, int n_kv_heads, int head_dim, int rows, int window, int sinks,
                    void* work, size_t work_bytes, asdsl_stream_t stream) {
    ASDSL_CHECK_ARG(q && c.k && c.v && pos && out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(!q8 || (c.ks && c.vs), "%s: null scale array", what);
    const asdsl_status st = check_heads(what, n_seq, n_tokens, n_heads, n_kv_heads, head_dim);
    if (st != ASDSL_OK) return st;
    ASDSL_CHECK_ARG(rows > 0, "%s: rows must be positive", what);
    ASDSL_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window and sinks must not be negative", what);
    ASDSL_CHECK_ARG(aligned16(q) && aligned16(c.k) && aligned16(c.v) && aligned16(out),
                    "%s: q, caches and out must be 16-byte aligned", what);
    AttnArgs g{q, out, c, c, pos, n_tokens, n_heads, n_kv_heads, rows, rows, -1, window, sinks, 0, 0.0f};
    return attend(what, q8, g, n_seq, head_dim, stream);
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
    const asdsl_status st = check_heads(what, n_seq, 1, n_heads, n_kv_heads, head_dim);
    if (st != ASDSL_OK) return st;
    ASDSL_CHECK_ARG(own_rows > 0, "%s: own_rows must be positive", what);
    ASDSL_CHECK_ARG(aligned16(q) && aligned16(shared.k) && aligned16(shared.v) && aligned16(own.k) &&
                        aligned16(own.v) && aligned16(out),
                    "%s: q, caches and out must be 16-byte aligned", what);
    AttnArgs g{q, out, shared, own, own_pos, 1, n_heads, n_kv_heads, prefix_rows, own_rows, prefix_len, 0, 0, 0, 0.0f};
    return attend(what, q8, g, n_seq, head_dim, stream);
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
    return 0;
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
    return 0;
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
