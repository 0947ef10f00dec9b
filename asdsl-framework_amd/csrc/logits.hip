// Control of the next token: penalties for tokens that occurred, biases and a
// grammar's mask on logits, and the greedy token of what is left.
//
// Per row, with seen(v) = token v is in the row's history, n(v) = its
// occurrences past the prompt, each step rounded to fp32:
//   y = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   y = y - frequency * n;  y = n > 0 ? y - presence : y;  y = y + bias
//   out = allowed ? y : -inf;  token = the first largest allowed y (-1: none)
#include "abi_util.hpp"
#include "device_common.hpp"

namespace asdsl {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;  // a slice's word per token: seen, and the count past the prompt

struct ControlArgs {
    const float* logits;
    float* out;
    unsigned long long* keys;  // [rows][slices], null without tokens
    const int* history;
    const int* prompt_len;
    const int* history_len;
    const float* repetition;
    const float* frequency;
    const float* presence;
    const float* bias;
    const uint32_t* allowed;
    int cap, vocab, slices;
    long long bias_stride, allowed_stride;
};

// A workgroup takes kPer tokens a thread of one row.  Their logits are requested
// first; while they come, the slice's words are counted in LDS from the row's
// whole history (integer atomics: any order gives the same).  kVec: the rows of
// logits, out and bias lie in whole 16-byte units.
//
// 64 rows of 200064 read and write 104 MB (20.2 us at a copy's 5.15 TB/s).  With
// histories of 4000, masks and one bias they take 37.8 us where nothing of a call is
// in the caches (16 calls' buffers in turn) and 33.1 where the last call's are, some
// 4 of them the tokens' launch; with histories of 500 33.5 and 28.5: beside memory
// each of a row's 49 workgroups counts the row's ids.  One pass per step of the
// definition took 59.  Stores past the caches save 1.3 us here and cost as much in
// the kernel that reads the result.  One row: 4.6 us and 2.2, launches and the chain
// of history length, ids and counts.
template <int kPer, bool kVec>
__global__ __launch_bounds__(kThreads) void logits_control_kernel(const ControlArgs a) {
#pragma clang fp contract(off)  // each step of the definition rounds by itself
    constexpr int kSlice = kThreads * kPer;
    constexpr int kWide = kVec ? 4 : 1;  // tokens of one load
    __shared__ __align__(16) uint32_t word[kSlice];
    __shared__ unsigned long long red[kThreads / kWave];
    const int tid = static_cast<int>(threadIdx.x);
    const int row = static_cast<int>(blockIdx.x / a.slices);
    const int v0 = static_cast<int>(blockIdx.x % a.slices) * kSlice;
    const int n = min(kSlice, a.vocab - v0);
    const long long base = static_cast<long long>(row) * a.vocab + v0;
    const float* bias = a.bias ? a.bias + row * a.bias_stride + v0 : nullptr;
    const uint32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
    float y[kPer], b[kPer];
    uint32_t mask[kPer / kWide];
#pragma unroll
    for (int i = 0; i < kPer / kWide; ++i) {
        const int at = (i * kThreads + tid) * kWide;
        mask[i] = ~0u;
        if (at >= n) continue;
        if constexpr (kVec) {
            const float4 x = *reinterpret_cast<const float4*>(a.logits + base + at);
            y[4 * i] = x.x; y[4 * i + 1] = x.y; y[4 * i + 2] = x.z; y[4 * i + 3] = x.w;
            if (bias) {
                const float4 z = *reinterpret_cast<const float4*>(bias + at);
                b[4 * i] = z.x; b[4 * i + 1] = z.y; b[4 * i + 2] = z.z; b[4 * i + 3] = z.w;
            }
        } else {
            y[i] = a.logits[base + at];
            if (bias) b[i] = bias[at];
        }
        if (allowed) mask[i] = allowed[(v0 + at) >> 5] >> ((v0 + at) & 31);
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.history) {
#pragma unroll
        for (int i = 0; i < kPer; i += 4)
            *reinterpret_cast<uint4*>(word + (i * kThreads + 4 * tid)) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        const int told = min(max(a.history_len ? a.history_len[row] : a.cap, 0), a.cap);
        const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
        const int* ids = a.history + static_cast<long long>(row) * a.cap;
        constexpr int kIds = 8;  // of a thread at a time, all requested before one is counted
        for (int i0 = tid; i0 < told; i0 += kIds * kThreads) {
            int id[kIds];
#pragma unroll
            for (int j = 0; j < kIds; ++j) id[j] = i0 + j * kThreads < told ? ids[i0 + j * kThreads] : -1;
#pragma unroll
            for (int j = 0; j < kIds; ++j) {
                const uint32_t at = static_cast<uint32_t>(id[j]) - static_cast<uint32_t>(v0);
                if (id[j] >= 0 && at < static_cast<uint32_t>(n)) {
                    atomicOr(&word[at], kSeen);
                    if (i0 + j * kThreads >= prompt) atomicAdd(&word[at], 1u);
                }
            }
        }
        if (a.repetition) rep = a.repetition[row];
        if (a.frequency) freq = a.frequency[row];
        if (a.presence) pres = a.presence[row];
        __syncthreads();
    }
    // A thread meets its tokens in rising order: only a larger one replaces the best.
    float top = -INFINITY;
    int top_at = -1;
#pragma unroll
    for (int i = 0; i < kPer / kWide; ++i) {
        const int at = (i * kThreads + tid) * kWide;
        if (at >= n) continue;
        uint32_t w[kWide];
#pragma unroll
        for (int e = 0; e < kWide; ++e) w[e] = a.history ? word[at + e] : 0u;
#pragma unroll
        for (int e = 0; e < kWide; ++e) {
            float x = y[kWide * i + e];
            if (w[e] != 0u) {
                x = x > 0.0f ? x / rep : x * rep;
                const uint32_t c = w[e] & ~kSeen;
                x = x - freq * static_cast<float>(c);
                if (c != 0u) x = x - pres;
            }
            if (bias) x = x + b[kWide * i + e];
            const bool ok = ((mask[i] >> e) & 1u) != 0u;
            y[kWide * i + e] = ok ? x : -INFINITY;
            if (ok & ((x > top) | ((top_at < 0) & (x == x)))) {
                top = x;
                top_at = at + e;
            }
        }
        if constexpr (kVec)
            *reinterpret_cast<float4*>(a.out + base + at) =
                make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
        else
            a.out[base + at] = y[i];
    }
    if (!a.keys) return;
    // equal values of either sign of zero are one
    unsigned long long best = top_at < 0 ? 0ull : argmax_key(top == 0.0f ? 0.0f : top, v0 + top_at);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const unsigned long long other = __shfl_xor(best, o, kWave);
        best = other > best ? other : best;
    }
    if ((tid & (kWave - 1)) == 0) red[tid / kWave] = best;
    __syncthreads();
    if (tid == 0) {
        for (int q = 1; q < kThreads / kWave; ++q) best = red[q] > best ? red[q] : best;
        a.keys[blockIdx.x] = best;
    }
}

// One wave per row: the largest of its slices' keys (0: nothing was allowed).
__global__ __launch_bounds__(kWave) void logits_token_kernel(const unsigned long long* __restrict__ keys, int slices,
                                                             int* __restrict__ tokens) {
    unsigned long long best = 0ull;
    for (int i = static_cast<int>(threadIdx.x); i < slices; i += kWave) {
        const unsigned long long k = keys[static_cast<long long>(blockIdx.x) * slices + i];
        best = k > best ? k : best;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const unsigned long long other = __shfl_xor(best, o, kWave);
        best = other > best ? other : best;
    }
    if (threadIdx.x == 0)
        tokens[blockIdx.x] = best != 0ull ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best)) : -1;
}

// Tokens a thread: 16, or 4 where 16 leave compute units without a workgroup (every
// workgroup reads its row's whole history).  us in a graph with 16 / 4: 64 rows of
// 200064 26.3 / 29.5, 256 of 32000 18.8 / 20.6, 8 of 200064 8.5 / 9.0; 4 of 200064
// 8.0 / 7.3, one 7.5 / 6.2, 16 of 32000 8.0 / 6.4, 7 of 50257 10.8 / 6.9.
int per_thread(int n_rows, int vocab) {
    const long long slices = (vocab + 16LL * kThreads - 1) / (16 * kThreads);
    return n_rows * slices < 256 ? 4 : 16;
}
long long slices_of(int n_rows, int vocab) {
    const long long slice = static_cast<long long>(per_thread(n_rows, vocab)) * kThreads;
    return (vocab + slice - 1) / slice;
}

}  // namespace
}  // namespace asdsl

using namespace asdsl;

extern "C" size_t asdsl_logits_control_work_bytes(int n_rows, int vocab) {
    if (n_rows <= 0 || vocab <= 0) return 0;
    return (static_cast<size_t>(n_rows) * slices_of(n_rows, vocab) * sizeof(unsigned long long) + 255) / 256 * 256;
}

extern "C" asdsl_status asdsl_logits_control(const float* logits, float* out, int* tokens, const int* history,
                                             const int* prompt_len, const int* history_len, int history_cap,
                                             const float* repetition, const float* frequency, const float* presence,
                                             const float* bias, long long bias_stride, const uint32_t* allowed,
                                             long long allowed_stride, int n_rows, int vocab, void* work,
                                             size_t work_bytes, asdsl_stream_t stream) {
    const char* what = "logits_control";
    ASDSL_CHECK_ARG(logits && out, "%s: null pointer", what);
    ASDSL_CHECK_ARG(n_rows > 0 && vocab > 0, "%s: n_rows and vocab must be positive", what);
    ASDSL_CHECK_ARG(history_cap >= 0 && history_cap <= 1 << 30, "%s: history_cap must be in [0, 2^30]", what);
    ASDSL_CHECK_ARG(history || (!prompt_len && !history_len && !repetition && !frequency && !presence),
                    "%s: lengths or penalties without a history", what);
    ASDSL_CHECK_ARG(!bias || bias_stride == 0 || bias_stride >= vocab,
                    "%s: bias_stride must be 0 or at least vocab", what);
    ASDSL_CHECK_ARG(!allowed || allowed_stride == 0 || allowed_stride >= (vocab + 31LL) / 32,
                    "%s: allowed_stride must be 0 or at least (vocab + 31) / 32", what);
    ASDSL_CHECK_ARG(fits_launch(n_rows * slices_of(n_rows, vocab), kThreads),
                    "%s: too many rows: more than 2^32 work items", what);
    void* ws = nullptr;
    if (tokens) {
        ASDSL_CHECK_ARG(work, "%s: tokens need a work buffer", what);
        const asdsl_status st = work_buffer(as_hip(stream), work, work_bytes,
                                            asdsl_logits_control_work_bytes(n_rows, vocab), &ws, what);
        if (st != ASDSL_OK) return st;
    }
    const int slices = static_cast<int>(slices_of(n_rows, vocab));
    const ControlArgs a{logits, out, static_cast<unsigned long long*>(ws), history_cap > 0 ? history : nullptr,
                        prompt_len, history_len, repetition, frequency, presence, bias, allowed, history_cap, vocab,
                        slices, bias_stride, allowed_stride};
    auto whole = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool vec = vocab % 4 == 0 && whole(logits) && whole(out) && whole(bias) && bias_stride % 4 == 0;
    const bool four = per_thread(n_rows, vocab) == 4;
    asdsl_status st = launch("logits_control_kernel",
                             four ? (vec ? logits_control_kernel<4, true> : logits_control_kernel<4, false>)
                                  : (vec ? logits_control_kernel<16, true> : logits_control_kernel<16, false>),
                             dim3(static_cast<unsigned>(n_rows * slices)), dim3(kThreads), 0, as_hip(stream), a);
    if (st != ASDSL_OK || !tokens) return st;
    return launch("logits_token_kernel", logits_token_kernel, dim3(n_rows), dim3(kWave), 0, as_hip(stream),
                  static_cast<const unsigned long long*>(ws), slices, tokens);
}
