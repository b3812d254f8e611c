// Rotary positions of the q and k heads of packed rows.
//
//   y_i = a (x_i cos t - x_j sin t),  y_j = a (x_i sin t + x_j cos t),  t = position * frequency
//
// for the pairs (i, j) = (i, i + R/2) or (2i, 2i + 1) of the first R elements of a head; the others pass.
// Angles are reduced to a part of one turn in 64 bits (position * frequency has up to 2^31 radians, of which fp32
// holds none of the fraction) and only then go through sin and cos in fp32; products and sums in fp32, one rounding.
//
// Bound by memory: every element is read once and written once.  A workgroup takes a few tokens, puts
// the cos and sin of their pairs into LDS once (one evaluation serves all heads of the token) and then walks over
// their elements in order, a unit -- V elements and their V partners, or V elements that pass -- per thread.
// Four tokens to a workgroup (one for small batches, where workgroups are what is missing): 32768 rows of 32 + 8 heads of 128 in
// 16 bits, 671 MB, 127 us, 5.3 TB/s (8 tokens 133, 16 136; a large copy 5.2); half of each head turned, 16384 rows, 71 us;
// 32 rows 3.3 us, most of it the launch.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"

#include <math.h>

namespace lg {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxUnits = 65536;   // (token, unit) of a workgroup: divided by multiplication
constexpr int kRopeAngles = 512;      // angles of a workgroup

struct RopeParams {
    const void* q_in;
    const void* k_in;
    void* q_out;
    void* k_out;
    const int32_t* positions;
    const double* inv_freq;
    int64_t q_in_stride, k_in_stride, q_out_stride, k_out_stride;  // elements
    int tokens, hq, hkv, d, half;  // half: pairs of a head
    int tok;                       // tokens per workgroup
    int units, unit_magic;         // units of a token; ceil(2^32 / units)
    int turn, head_units, head_magic;  // units of a head that turn, all of them, ceil(2^32 / head_units)
    float amplitude;
};

// n / d for n < 65536, d <= 65536 and magic = ceil(2^32 / d)
__device__ __forceinline__ int small_div(int n, int magic, int d) {
    return d == 1 ? n : (int)__umulhi((unsigned)n, (unsigned)magic);
}

template <typename E, int V>
struct alignas(sizeof(E) * V) RopeVec {
    E e[V];
};

template <typename E, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kRopeThreads) void rope_packed_kernel(const RopeParams p) {
    __shared__ float cs[kRopeAngles], sn[kRopeAngles];
    const int t0 = blockIdx.x * p.tok;
    const int n_tok = p.tokens - t0 < p.tok ? p.tokens - t0 : p.tok;
    for (int i = threadIdx.x; i < n_tok * p.half; i += kRopeThreads) {
        const int t = i / p.half, f = i - t * p.half;
        double turns = (double)p.positions[t0 + t] * p.inv_freq[f] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        cs[i] = c * p.amplitude;
        sn[i] = s * p.amplitude;
    }
    __syncthreads();
    typedef RopeVec<E, V> vec;
    for (int i = threadIdx.x; i < n_tok * p.units; i += kRopeThreads) {
        const int t = small_div(i, p.unit_magic, p.units), u = i - t * p.units;
        const int head = small_div(u, p.head_magic, p.head_units), at = u - head * p.head_units;
        const bool is_k = head >= p.hq;
        const int64_t row = t0 + t;
        const E* src = is_k ? static_cast<const E*>(p.k_in) + row * p.k_in_stride + (int64_t)(head - p.hq) * p.d
                            : static_cast<const E*>(p.q_in) + row * p.q_in_stride + (int64_t)head * p.d;
        E* dst = is_k ? static_cast<E*>(p.k_out) + row * p.k_out_stride + (int64_t)(head - p.hq) * p.d
                      : static_cast<E*>(p.q_out) + row * p.q_out_stride + (int64_t)head * p.d;
        if (at >= p.turn) {
            const int e = 2 * p.half + (at - p.turn) * V;
            *reinterpret_cast<vec*>(dst + e) = *reinterpret_cast<const vec*>(src + e);
            continue;
        }
        const float* c = cs + t * p.half;
        const float* s = sn + t * p.half;
        const int a0 = INTERLEAVED ? 2 * V * at : V * at, b0 = INTERLEAVED ? a0 + V : a0 + p.half;
        const vec a = *reinterpret_cast<const vec*>(src + a0), b = *reinterpret_cast<const vec*>(src + b0);
        vec x, y;
        const int f = V * at;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            // interleaved: element 2e of the 2V behind one another pairs with 2e + 1
            const float one = INTERLEAVED ? (float)(2 * e < V ? a.e[2 * e % V] : b.e[2 * e % V]) : (float)a.e[e];
            const float two = INTERLEAVED ? (float)(2 * e + 1 < V ? a.e[(2 * e + 1) % V] : b.e[(2 * e + 1) % V]) : (float)b.e[e];
            const float cv = c[f + e], sv = s[f + e];
            const E n1 = (E)(one * cv - two * sv), n2 = (E)(one * sv + two * cv);
            if constexpr (INTERLEAVED) {
                (2 * e < V ? x : y).e[2 * e % V] = n1;
                (2 * e + 1 < V ? x : y).e[(2 * e + 1) % V] = n2;
            } else {
                x.e[e] = n1;
                y.e[e] = n2;
            }
        }
        *reinterpret_cast<vec*>(dst + a0) = x;
        *reinterpret_cast<vec*>(dst + b0) = y;
    }
}

template <typename E, int V>
static hipError_t rope_launch_v(const RopeParams& p, bool interleaved, hipStream_t stream) {
    const unsigned grid = (unsigned)((p.tokens + p.tok - 1) / p.tok);
    if (interleaved) rope_packed_kernel<E, V, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else rope_packed_kernel<E, V, false><<<grid, kRopeThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename E>
static logismos_status_t rope_launch(RopeParams p, bool interleaved, hipStream_t stream) {
    // elements per access: what divides the pairs, the width, and the strides and addresses in bytes
    const int rest = p.d - 2 * p.half;
    uint64_t all = (uint64_t)p.half | (uint64_t)rest | (uint64_t)p.d | (uint64_t)p.q_in_stride |
                   (uint64_t)p.q_out_stride | (reinterpret_cast<uintptr_t>(p.q_in) / sizeof(E)) |
                   (reinterpret_cast<uintptr_t>(p.q_out) / sizeof(E));
    if (p.hkv > 0)
        all |= (uint64_t)p.k_in_stride | (uint64_t)p.k_out_stride |
               (reinterpret_cast<uintptr_t>(p.k_in) / sizeof(E)) |
               (reinterpret_cast<uintptr_t>(p.k_out) / sizeof(E));
    int v = 16 / (int)sizeof(E);
    while (v > 1 && all % (unsigned)v != 0) v /= 2;
    p.turn = p.half / v;
    p.head_units = p.turn + rest / v;
    p.units = (p.hq + p.hkv) * p.head_units;
    auto magic = [](int d) { return (int)(unsigned)(((1ull << 32) + (unsigned)d - 1) / (unsigned)d); };
    p.head_magic = magic(p.head_units);
    p.unit_magic = magic(p.units);
    int tok = 4;
    while (tok > 1 && (tok * p.half > kRopeAngles || (int64_t)tok * p.units > kRopeMaxUnits ||
                       p.tokens < 1024 * tok))
        tok /= 2;
    p.tok = tok;
    hipError_t rc = hipSuccess;
    if constexpr (sizeof(E) == 2)
        if (v == 8) rc = rope_launch_v<E, 8>(p, interleaved, stream);
    if (v == 4) rc = rope_launch_v<E, 4>(p, interleaved, stream);
    if (v == 2) rc = rope_launch_v<E, 2>(p, interleaved, stream);
    if (v == 1) rc = rope_launch_v<E, 1>(p, interleaved, stream);
    return static_cast<logismos_status_t>(rc);
}

static logismos_status_t rope_packed(int elem_bytes, int type, const void* q_in, const void* k_in, void* q_out,
                                     void* k_out, const int32_t* positions, const double* inv_freq, int tokens,
                                     int hq, int hkv, int d, int rotary, int q_in_stride, int k_in_stride,
                                     int q_out_stride, int k_out_stride, float amplitude, int interleaved,
                                     logismos_stream_t stream) {
    if (logismos_check_rope_packed_shape(tokens, hq, hkv, d, rotary, q_in_stride, k_in_stride, q_out_stride,
                                         k_out_stride, nullptr, 0) != 0)
        return static_cast<logismos_status_t>(hipErrorInvalidValue);
    const uintptr_t at = reinterpret_cast<uintptr_t>(q_in) | reinterpret_cast<uintptr_t>(q_out) |
                         (hkv > 0 ? reinterpret_cast<uintptr_t>(k_in) | reinterpret_cast<uintptr_t>(k_out) : 0);
    if (!q_in || !q_out || (hkv > 0 && (!k_in || !k_out)) || !positions || !inv_freq || !isfinite(amplitude) ||
        at % (uintptr_t)elem_bytes != 0 || reinterpret_cast<uintptr_t>(inv_freq) % 8 != 0 ||
        reinterpret_cast<uintptr_t>(positions) % 4 != 0)
        return static_cast<logismos_status_t>(hipErrorInvalidValue);
    // (one address with two strides: rows would be read after others were written over them)
    if (tokens > 1 && ((q_in == q_out && q_in_stride != q_out_stride) ||
                       (hkv > 0 && k_in == k_out && k_in_stride != k_out_stride)))
        return static_cast<logismos_status_t>(hipErrorInvalidValue);
    RopeParams p = {};
    p.q_in = q_in;
    p.k_in = k_in;
    p.q_out = q_out;
    p.k_out = k_out;
    p.positions = positions;
    p.inv_freq = inv_freq;
    p.q_in_stride = q_in_stride;
    p.k_in_stride = k_in_stride;
    p.q_out_stride = q_out_stride;
    p.k_out_stride = k_out_stride;
    p.tokens = tokens;
    p.hq = hq;
    p.hkv = hkv;
    p.d = d;
    p.half = rotary / 2;
    p.amplitude = amplitude;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == 0) return rope_launch<_Float16>(p, interleaved != 0, st);
    if (type == 1) return rope_launch<__bf16>(p, interleaved != 0, st);
    return rope_launch<float>(p, interleaved != 0, st);
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_rope_packed_shape(int tokens, int num_q_heads, int num_kv_heads, int head_dim,
                                                   int rotary_dim, int q_in_stride, int k_in_stride,
                                                   int q_out_stride, int k_out_stride, char* msg, size_t cap) {
    using lg::reject;
    if (tokens <= 0 || num_q_heads <= 0 || head_dim <= 0)
        return reject(msg, cap, "tokens, num_q_heads and head_dim must be positive (%d, %d, %d)", tokens, num_q_heads,
                      head_dim);
    if (tokens > lg::kPackedMaxRows) return reject(msg, cap, "tokens exceeds %d (%d)", lg::kPackedMaxRows, tokens);
    if (num_kv_heads < 0) return reject(msg, cap, "num_kv_heads must not be negative (%d)", num_kv_heads);
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
        return reject(msg, cap, "rotary_dim must be even, positive and at most head_dim (%d of %d)", rotary_dim,
                      head_dim);
    if (head_dim > 1024) return reject(msg, cap, "head_dim must be at most 1024 (%d)", head_dim);
    if (((int64_t)num_q_heads + num_kv_heads) * head_dim > lg::kRopeMaxUnits)
        return reject(msg, cap, "(num_q_heads + num_kv_heads) * head_dim = %lld exceeds %d",
                      (long long)(((int64_t)num_q_heads + num_kv_heads) * head_dim), lg::kRopeMaxUnits);
    if (q_in_stride < num_q_heads * head_dim || q_out_stride < num_q_heads * head_dim)
        return reject(msg, cap, "a q stride is smaller than a row of %d elements", num_q_heads * head_dim);
    if (num_kv_heads > 0 && (k_in_stride < num_kv_heads * head_dim || k_out_stride < num_kv_heads * head_dim))
        return reject(msg, cap, "a k stride is smaller than a row of %d elements", num_kv_heads * head_dim);
    return 0;
}

logismos_status_t logismos_rope_frequencies(double* inv_freq, float* amplitude, int rotary_dim, double base,
                                            int scaling, double factor, int original_positions, double turns_fast,
                                            double turns_slow) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (!inv_freq || !amplitude || rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > 1024) return bad;
    if (!(base > 0.0) || !isfinite(base)) return bad;
    if (scaling < LOGISMOS_ROPE_SCALE_NONE || scaling > LOGISMOS_ROPE_SCALE_PARTS) return bad;
    if (scaling != LOGISMOS_ROPE_SCALE_NONE && !(factor >= 1.0 && isfinite(factor))) return bad;
    if (scaling == LOGISMOS_ROPE_SCALE_BASE && rotary_dim <= 2) return bad;
    if (scaling == LOGISMOS_ROPE_SCALE_PARTS &&
        (original_positions <= 0 || !(turns_slow >= 0.0) || !(turns_fast > turns_slow) || !isfinite(turns_fast)))
        return bad;
    const double r = rotary_dim;
    if (scaling == LOGISMOS_ROPE_SCALE_BASE) base *= pow(factor, r / (r - 2.0));
    // (the largest frequency is base^0 or, for a base below 1, that of the last pair)
    if (!isfinite(base) || !isfinite(pow(base, -2.0 * (rotary_dim / 2 - 1) / r))) return bad;
    *amplitude = 1.0f;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = pow(base, -2.0 * i / r);
        if (scaling == LOGISMOS_ROPE_SCALE_LINEAR) f /= factor;
        if (scaling == LOGISMOS_ROPE_SCALE_PARTS) {
            const double turns = original_positions * f * 0.15915494309189533577;
            const double keep = fmin(1.0, fmax(0.0, (turns - turns_slow) / (turns_fast - turns_slow)));
            f = keep * f + (1.0 - keep) * (f / factor);
        }
        inv_freq[i] = f;
    }
    if (scaling == LOGISMOS_ROPE_SCALE_PARTS) *amplitude = (float)(0.1 * log(factor) + 1.0);
    return 0;
}

#define LOGISMOS_ROPE_PACKED(name, bytes, type)                                                                       \
    logismos_status_t logismos_launch_rope_packed_##name(                                                             \
        const void* q_in, const void* k_in, void* q_out, void* k_out, const int32_t* positions,                       \
        const double* inv_freq, int tokens, int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim,          \
        int q_in_stride, int k_in_stride, int q_out_stride, int k_out_stride, float amplitude, int interleaved,       \
        logismos_stream_t stream) {                                                                                   \
        return lg::rope_packed(bytes, type, q_in, k_in, q_out, k_out, positions, inv_freq, tokens, num_q_heads,       \
                               num_kv_heads, head_dim, rotary_dim, q_in_stride, k_in_stride, q_out_stride,            \
                               k_out_stride, amplitude, interleaved, stream);                                         \
    }
LOGISMOS_ROPE_PACKED(fp16, 2, 0)
LOGISMOS_ROPE_PACKED(bf16, 2, 1)
LOGISMOS_ROPE_PACKED(f32, 4, 2)
#undef LOGISMOS_ROPE_PACKED

}  // extern "C"
