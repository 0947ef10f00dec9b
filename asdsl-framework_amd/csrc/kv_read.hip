// Rows of int8 or 4-bit caches read back as the values they stand for, fp16 or
// fp32: code * scale (int8, in fp32, rounded once more to fp16) or (code - z) *
// scale (4-bit, exact in both).
#include <hip/hip_fp16.h>

#include <type_traits>

#include "abi_util.hpp"
#include "device_common.hpp"
#include "kv_int4.hpp"

namespace asdsl {
namespace {

constexpr int kReadThreads = 256;
constexpr int kBlockDims8 = 64;  // dims per scale of an int8 cache

struct ReadArgs {
    const void* in[2];  // K, V
    const void* scale[2];
    void* out[2];
    const int* pos;  // null: row 0
    int n_kv, rows, n_rows, chunks;
};

// 16 bytes of output a lane: 8 fp16 or 4 fp32 values of one row, so that a wave
// writes 1 KB in a row; its codes are the 2 to 8 bytes a lane beside each other.  A
// lane takes kPer rows, whose loads it requests together.
//
// Bound by memory and, for small calls, by the chain of position, codes and stores:
// 4001 rows of 8 KV heads of 128 dims from 4 bits to fp16 (21 MB) take 6.6 us and to
// fp32 (37 MB) 8.9 (4.2 TB/s), from int8 to fp16 (25 MB) 7.2; 701 rows of 12 sequences
// of 8 heads of 64 dims from int8 to fp32 (44 MB) 10.2 (4.3 TB/s).  A row a lane took
// 1.5 us more at the first and the last of these.
constexpr int kPer = 4;
template <int D, bool kFour, typename T>
__global__ __launch_bounds__(kReadThreads) void kv_read_kernel(const ReadArgs a) {
    constexpr int kDims = 16 / sizeof(T), kUnits = D / kDims;  // dims a lane, lanes a row
    constexpr int kRowsAtOnce = kReadThreads / kUnits;
    const int chunk = static_cast<int>(blockIdx.x) % a.chunks;
    const long long job = static_cast<long long>(blockIdx.x) / a.chunks;
    const int side = static_cast<int>(job & 1);
    const long long head = job >> 1;  // sequence * n_kv + KV head
    const int t0 = chunk * (kPer * kRowsAtOnce) + static_cast<int>(threadIdx.x) / kUnits;
    const int d = static_cast<int>(threadIdx.x) % kUnits * kDims;
    const long long first = a.pos ? a.pos[head / a.n_kv] : 0;
    uint32_t c[kPer][2];
    uint32_t scale[kPer];  // the word, or the bits of the fp32 scale; 0 reads as zeros
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int t = t0 + j * kRowsAtOnce;
        const long long r = first + t;
        c[j][0] = c[j][1] = scale[j] = 0u;
        if (t >= a.n_rows || r < 0 || r >= a.rows) continue;
        const size_t row = static_cast<size_t>(head) * a.rows + static_cast<size_t>(r);
        if constexpr (kFour) {
            scale[j] = static_cast<const uint16_t*>(a.scale[side])[row * (D / kGroup4) + d / kGroup4];
            const char* src = static_cast<const char*>(a.in[side]) + (row * D + d) / 2;
            if constexpr (kDims == 8)
                c[j][0] = *reinterpret_cast<const uint32_t*>(src);
            else
                c[j][0] = *reinterpret_cast<const uint16_t*>(src);
        } else {
            scale[j] = static_cast<const uint32_t*>(a.scale[side])[row * (D / kBlockDims8) + d / kBlockDims8];
            const char* src = static_cast<const char*>(a.in[side]) + row * D + d;
            if constexpr (kDims == 8) {
                const uint2 x = *reinterpret_cast<const uint2*>(src);
                c[j][0] = x.x;
                c[j][1] = x.y;
            } else {
                c[j][0] = *reinterpret_cast<const uint32_t*>(src);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int t = t0 + j * kRowsAtOnce;
        if (t >= a.n_rows) return;
        T y[kDims];
#pragma unroll
        for (int i = 0; i < kDims; ++i) {
            if constexpr (kFour)
                y[i] = static_cast<T>(value4((c[j][0] >> (4 * i)) & 15u, scale[j]));
            else
                y[i] = static_cast<T>(static_cast<float>(static_cast<int8_t>(c[j][i / 4] >> (8 * (i % 4)))) *
                                      __builtin_bit_cast(float, scale[j]));
        }
        uint4 o;
        static_assert(sizeof(y) == sizeof(o), "one store a lane");
        __builtin_memcpy(&o, y, sizeof(o));
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out[side]) + (static_cast<size_t>(head) * a.n_rows + t) * D + d) = o;
    }
}

bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

asdsl_status read_rows(const char* what, bool four, const void* k, const void* v, const void* ks, const void* vs,
                       const int* pos, void* k_out, void* v_out, int out_fp32, int n_seq, int n_kv_heads, int head_dim,
                       int rows, int n_rows, asdsl_stream_t stream) {
    ASDSL_CHECK_ARG(k && v && k_out && v_out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(ks && vs, "%s: null scale array", what);
    ASDSL_CHECK_ARG(n_seq > 0 && n_kv_heads > 0, "%s: n_seq and n_kv_heads must be positive", what);
    ASDSL_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128", what);
    ASDSL_CHECK_ARG(rows > 0 && n_rows > 0, "%s: rows and n_rows must be positive", what);
    ASDSL_CHECK_ARG(aligned(k, 16) && aligned(v, 16) && aligned(k_out, 16) && aligned(v_out, 16),
                    "%s: caches and outputs must be 16-byte aligned", what);
    ASDSL_CHECK_ARG(aligned(ks, 4) && aligned(vs, 4), "%s: scales must be 4-byte aligned", what);
    const int per = kPer * (kReadThreads / (head_dim / (out_fp32 ? 4 : 8)));  // rows of a workgroup
    const long long chunks = (static_cast<long long>(n_rows) + per - 1) / per, heads = static_cast<long long>(n_seq) * n_kv_heads;
    ASDSL_CHECK_ARG(heads <= (1LL << 31) && fits_launch(2 * heads * chunks, kReadThreads),
                    "%s: too many rows: more than 2^32 work items", what);
    ASDSL_CHECK_ARG(k_out != v_out, "%s: keys and values need an output each", what);
    const ReadArgs a{{k, v}, {ks, vs}, {k_out, v_out}, pos, n_kv_heads, rows, n_rows, static_cast<int>(chunks)};
    auto with = [&](auto dim, auto is_four) {
        constexpr int kD = decltype(dim)::value;
        constexpr bool kFour = decltype(is_four)::value;
        return launch("kv_read_kernel", out_fp32 ? kv_read_kernel<kD, kFour, float> : kv_read_kernel<kD, kFour, _Float16>,
                      dim3(static_cast<unsigned>(2 * heads * chunks)), dim3(kReadThreads), 0, as_hip(stream), a);
    };
    auto by_form = [&](auto dim) { return four ? with(dim, std::true_type{}) : with(dim, std::false_type{}); };
    return head_dim == 128 ? by_form(std::integral_constant<int, 128>{}) : by_form(std::integral_constant<int, 64>{});
}

}  // namespace
}  // namespace asdsl

using namespace asdsl;

extern "C" asdsl_status asdsl_kv_read_q8(const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                                         const float* v_scale, const int* pos, void* k_out, void* v_out, int out_fp32,
                                         int n_seq, int n_kv_heads, int head_dim, int rows, int n_rows,
                                         asdsl_stream_t stream) {
    return read_rows("kv_read_q8", false, k_cache, v_cache, k_scale, v_scale, pos, k_out, v_out, out_fp32, n_seq,
                     n_kv_heads, head_dim, rows, n_rows, stream);
}

extern "C" asdsl_status asdsl_kv_read_q4(const uint8_t* k_cache, const uint8_t* v_cache, const uint16_t* k_scale,
                                         const uint16_t* v_scale, const int* pos, void* k_out, void* v_out,
                                         int out_fp32, int n_seq, int n_kv_heads, int head_dim, int rows, int n_rows,
                                         asdsl_stream_t stream) {
    return read_rows("kv_read_q4", true, k_cache, v_cache, k_scale, v_scale, pos, k_out, v_out, out_fp32, n_seq,
                     n_kv_heads, head_dim, rows, n_rows, stream);
}
