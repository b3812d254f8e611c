// RMS norm of every q and k head of packed rows and rotary positions in the same pass.
//
//   z_i = x_i * gain_i / sqrt(mean(x^2) + eps)                       (no gains: z = x)
//   y_i = a (z_i cos t - z_j sin t),  y_j = a (z_i sin t + z_j cos t),  t = positions[axis(pair)][row] * frequency
//
// for the pairs (i, j) = (i, i + R/2) or (2i, 2i + 1) of the first R elements of a head; the others are z as they are.  Squares and
// their sum, the norm and the products in fp32, one rounding; angles reduced to a part of one turn in 64 bits as in rope_packed.hip.
//
// Bound by memory: every element is read once and written once.  A head belongs to a power of two of lanes that hold all of it (a
// lane V elements and their V partners, or V that pass), so that the sum of squares is a few lane exchanges; heads with more pieces than
// a wave has lanes are walked twice, the second time out of the cache.  A workgroup takes a few tokens, whose cos and sin, evaluated once,
// serve all heads.
//
// 32768 rows of 32 + 8 heads of 128, bf16, 671 MB: 132 us, 5.1 TB/s, of the 5.2 of a copy (the rotation alone, rope_packed.hip, 126); 8190 rows of
// 12 + 2 heads, three axes, pairs side by side 14.4; 24 rows of 14 + 2 heads of 64, fp32, 3.6.  Gains kept in registers took 162 us of the first, the next
// head's elements asked for ahead 150, eight tokens to a workgroup 145; two 132.6, but more of the small calls.  An access is the greatest power of two that
// divides pairs, rest, width, strides and addresses: with 120 of 128 elements turning (8 bytes) 250 us, with 126 (2 bytes, heads walked twice) 649.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"

#include <math.h>

namespace lg {

constexpr int kNormRopeThreads = 256;
constexpr int kNormRopeAngles = 512;  // angles of a workgroup

struct NormRopeParams {
    const void* q_in;
    const void* k_in;
    void* q_out;
    void* k_out;
    const int32_t* positions;
    const uint8_t* axis_of_pair;
    const double* inv_freq;
    const float* q_gain;
    const float* k_gain;
    int64_t q_in_stride, k_in_stride, q_out_stride, k_out_stride, position_stride;  // elements
    int tokens, hq, hkv, d, half, axes;  // half: pairs of a head
    int tok;                             // tokens per workgroup
    int turn, units;                     // pieces of a head that turn, and all of them
    float eps, amplitude;
};

template <typename E, int V>
struct alignas(sizeof(E) * V) NormRopeVec {
    E e[V];
};

// Sum over the LANES lanes of a head.
template <int LANES>
__device__ __forceinline__ float head_lanes_sum(float v) {
    if constexpr (LANES > 1) v += lane_xor_f32<1>(v);
    if constexpr (LANES > 2) v += lane_xor_f32<2>(v);
    if constexpr (LANES > 4) v += lane_xor_f32<4>(v);
    if constexpr (LANES > 8) v += lane_xor_f32<8>(v);
    if constexpr (LANES > 16) v += lane_xor_f32<16>(v);
    if constexpr (LANES > 32) v += lane_xor_f32<32>(v);
    return v;
}

// 1 / sqrt(sum / d + eps).  Rows whose squares leave the range of fp32 (bf16 and fp32 values beyond 2^59) are summed again in units of
// 2^70, and their elements taken in units of 2^30: the reciprocal of a large root, and a small gain times it, would be below fp32's range.
constexpr float kNormDown = 0x1p-70f, kNormUnit = 0x1p-30f;
__device__ __forceinline__ float inv_rms(float sum, float d, float eps) { return 1.0f / sqrtf(sum / d + eps); }
__device__ __forceinline__ float inv_rms_down(float sum, float d, float eps) {
    return kNormDown / kNormUnit / sqrtf(sum / d + eps * kNormDown * kNormDown);
}

template <typename E, int V, bool INTERLEAVED, int LANES>
__global__ __launch_bounds__(kNormRopeThreads) void norm_rope_packed_kernel(const NormRopeParams p) {
    __shared__ float cs[kNormRopeAngles], sn[kNormRopeAngles];
    typedef NormRopeVec<E, V> vec;
    constexpr int kGroups = kNormRopeThreads / LANES;
    const int t0 = blockIdx.x * p.tok;
    const int n_tok = p.tokens - t0 < p.tok ? p.tokens - t0 : p.tok;
    for (int i = threadIdx.x; i < n_tok * p.half; i += kNormRopeThreads) {
        const int t = i / p.half, f = i - t * p.half;
        const int axis = p.axis_of_pair ? p.axis_of_pair[f] : 0;
        const int at = axis < p.axes ? p.positions[axis * p.position_stride + t0 + t] : 0;
        double turns = (double)at * p.inv_freq[f] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        cs[i] = c * p.amplitude;
        sn[i] = s * p.amplitude;
    }
    __syncthreads();
    const int heads = p.hq + p.hkv;
    const int lane = threadIdx.x % LANES;
    for (int item = threadIdx.x / LANES; item < n_tok * heads; item += kGroups) {
        const int t = item / heads, head = item - t * heads;
        const bool is_k = head >= p.hq;
        const int64_t row = t0 + t;
        const E* src = is_k ? static_cast<const E*>(p.k_in) + row * p.k_in_stride + (int64_t)(head - p.hq) * p.d
                            : static_cast<const E*>(p.q_in) + row * p.q_in_stride + (int64_t)head * p.d;
        E* dst = is_k ? static_cast<E*>(p.k_out) + row * p.k_out_stride + (int64_t)(head - p.hq) * p.d
                      : static_cast<E*>(p.q_out) + row * p.q_out_stride + (int64_t)head * p.d;
        const float* gain = is_k ? p.k_gain : p.q_gain;
        const float* c = cs + t * p.half;
        const float* s = sn + t * p.half;
        // piece u of the head: where its V elements and the V that they turn with lie (one that passes: itself twice)
        auto first = [&](int u) LG_INLINE {
            return u >= p.turn ? 2 * p.half + (u - p.turn) * V : INTERLEAVED ? 2 * V * u : V * u;
        };
        auto second = [&](int u, int a0) LG_INLINE { return u >= p.turn ? a0 : INTERLEAVED ? a0 + V : a0 + p.half; };
        vec a, b;
        auto load = [&](int u) LG_INLINE {
            const int a0 = first(u);
            a = *reinterpret_cast<const vec*>(src + a0);
            b = *reinterpret_cast<const vec*>(src + second(u, a0));
        };
        auto squares = [&](int u, float unit) LG_INLINE {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float x = (float)a.e[e] * unit, y = u < p.turn ? (float)b.e[e] * unit : 0.0f;
                sum += x * x;
                sum += y * y;
            }
            return sum;
        };
        float inv = 1.0f;
        bool down = false;
        const bool once = p.units <= LANES;  // (uniform)
        if (once && lane < p.units) load(lane);
        if (gain != nullptr) {
            auto total = [&](float unit) LG_INLINE {
                float sum = 0.0f;
                for (int u = lane; u < p.units; u += LANES) {
                    if (!once) load(u);
                    sum += squares(u, unit);
                }
                return head_lanes_sum<LANES>(sum);
            };
            const float sum = total(1.0f);
            inv = inv_rms(sum, (float)p.d, p.eps);
            down = !(sum < INFINITY);
            if (__builtin_expect(down, 0)) inv = inv_rms_down(total(kNormDown), (float)p.d, p.eps);
        }
        for (int u = lane; u < p.units; u += LANES) {
            if (!once) load(u);
            const int a0 = first(u), b0 = second(u, a0);
            float x[V], y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[e] = (float)a.e[e];
                y[e] = (float)b.e[e];
            }
            if (gain != nullptr) {
                if (__builtin_expect(down, 0)) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        x[e] *= kNormUnit;
                        y[e] *= kNormUnit;
                    }
                }
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[e] *= inv * gain[a0 + e];
                    y[e] *= inv * gain[b0 + e];
                }
            }
            vec one, two;
            if (u >= p.turn) {
#pragma unroll
                for (int e = 0; e < V; ++e) one.e[e] = (E)x[e];
                *reinterpret_cast<vec*>(dst + a0) = one;
                continue;
            }
            const int f = V * u;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                // interleaved: element 2e of the 2V behind one another pairs with 2e + 1
                const float p1 = INTERLEAVED ? (2 * e < V ? x[2 * e % V] : y[2 * e % V]) : x[e];
                const float p2 = INTERLEAVED ? (2 * e + 1 < V ? x[(2 * e + 1) % V] : y[(2 * e + 1) % V]) : y[e];
                const E n1 = (E)(p1 * c[f + e] - p2 * s[f + e]), n2 = (E)(p1 * s[f + e] + p2 * c[f + e]);
                if constexpr (INTERLEAVED) {
                    (2 * e < V ? one : two).e[2 * e % V] = n1;
                    (2 * e + 1 < V ? one : two).e[(2 * e + 1) % V] = n2;
                } else {
                    one.e[e] = n1;
                    two.e[e] = n2;
                }
            }
            *reinterpret_cast<vec*>(dst + a0) = one;
            *reinterpret_cast<vec*>(dst + b0) = two;
        }
    }
}

template <typename E, int V, bool INTERLEAVED>
static hipError_t norm_rope_by_lanes(const NormRopeParams& p, hipStream_t stream) {
    const unsigned grid = (unsigned)((p.tokens + p.tok - 1) / p.tok);
    auto go = [&](auto lanes) {
        norm_rope_packed_kernel<E, V, INTERLEAVED, decltype(lanes)::value><<<grid, kNormRopeThreads, 0, stream>>>(p);
    };
    if (p.units <= 4) go(ic<4>{});
    else if (p.units <= 8) go(ic<8>{});
    else if (p.units <= 16) go(ic<16>{});
    else if (p.units <= 32) go(ic<32>{});
    else go(ic<64>{});
    return hipGetLastError();
}

template <typename E, int V>
static hipError_t norm_rope_launch_v(const NormRopeParams& p, bool interleaved, hipStream_t stream) {
    return interleaved ? norm_rope_by_lanes<E, V, true>(p, stream) : norm_rope_by_lanes<E, V, false>(p, stream);
}

template <typename E>
static logismos_status_t norm_rope_launch(NormRopeParams p, bool interleaved, hipStream_t stream) {
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
    p.units = p.turn + rest / v;
    int tok = 4;
    while (tok > 1 && (tok * p.half > kNormRopeAngles || p.tokens < 1024 * tok)) tok /= 2;
    p.tok = tok;
    hipError_t rc = hipSuccess;
    if constexpr (sizeof(E) == 2)
        if (v == 8) rc = norm_rope_launch_v<E, 8>(p, interleaved, stream);
    if (v == 4) rc = norm_rope_launch_v<E, 4>(p, interleaved, stream);
    if (v == 2) rc = norm_rope_launch_v<E, 2>(p, interleaved, stream);
    if (v == 1) rc = norm_rope_launch_v<E, 1>(p, interleaved, stream);
    return static_cast<logismos_status_t>(rc);
}

static logismos_status_t norm_rope_packed(int elem_bytes, int type, NormRopeParams p, int rotary, int interleaved,
                                          logismos_stream_t stream) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    const int64_t strides[4] = {p.q_in_stride, p.k_in_stride, p.q_out_stride, p.k_out_stride};
    if (logismos_check_norm_rope_packed_shape(p.tokens, p.hq, p.hkv, p.d, rotary, p.axes, (int)p.position_stride,
                                              (int)strides[0], (int)strides[1], (int)strides[2], (int)strides[3],
                                              nullptr, 0) != 0)
        return bad;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.q_in) | reinterpret_cast<uintptr_t>(p.q_out) |
                         (p.hkv > 0 ? reinterpret_cast<uintptr_t>(p.k_in) | reinterpret_cast<uintptr_t>(p.k_out) : 0);
    if (!p.q_in || !p.q_out || (p.hkv > 0 && (!p.k_in || !p.k_out)) || at % (uintptr_t)elem_bytes != 0) return bad;
    if (rotary > 0 && (!p.positions || !p.inv_freq || (p.axes > 1 && !p.axis_of_pair))) return bad;
    if ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.q_gain) |
         reinterpret_cast<uintptr_t>(p.k_gain)) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(p.inv_freq) % 8 != 0)
        return bad;
    if (!isfinite(p.amplitude) || !((p.q_gain == nullptr && p.k_gain == nullptr) || (p.eps > 0.0f && isfinite(p.eps))))
        return bad;
    // (one address with two strides: rows would be read after others were written over them)
    if (p.tokens > 1 && ((p.q_in == p.q_out && p.q_in_stride != p.q_out_stride) ||
                         (p.hkv > 0 && p.k_in == p.k_out && p.k_in_stride != p.k_out_stride)))
        return bad;
    p.half = rotary / 2;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == 0) return norm_rope_launch<_Float16>(p, interleaved != 0, st);
    if (type == 1) return norm_rope_launch<__bf16>(p, interleaved != 0, st);
    return norm_rope_launch<float>(p, interleaved != 0, st);
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_norm_rope_packed_shape(int tokens, int num_q_heads, int num_kv_heads, int head_dim,
                                                        int rotary_dim, int num_axes, int position_stride,
                                                        int q_in_stride, int k_in_stride, int q_out_stride,
                                                        int k_out_stride, char* msg, size_t cap) {
    using lg::reject;
    if (rotary_dim != 0) {
        if (num_axes <= 0 || num_axes > 255)
            return reject(msg, cap, "num_axes must be between 1 and 255 (%d)", num_axes);
        if (num_axes > 1 && position_stride < tokens)
            return reject(msg, cap, "position_stride %d is smaller than the %d tokens of an axis", position_stride,
                          tokens);
    }
    // (everything else as rotary positions alone; no rotation at all is allowed here)
    return logismos_check_rope_packed_shape(tokens, num_q_heads, num_kv_heads, head_dim,
                                            rotary_dim == 0 ? 2 : rotary_dim, q_in_stride, k_in_stride, q_out_stride,
                                            k_out_stride, msg, cap);
}

#define LOGISMOS_NORM_ROPE_PACKED(name, bytes, type)                                                                  \
    logismos_status_t logismos_launch_norm_rope_packed_##name(                                                        \
        const void* q_in, const void* k_in, void* q_out, void* k_out, const int32_t* positions,                       \
        const uint8_t* axis_of_pair, const double* inv_freq, const float* q_gain, const float* k_gain, int tokens,    \
        int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim, int num_axes, int position_stride,           \
        int q_in_stride, int k_in_stride, int q_out_stride, int k_out_stride, float eps, float amplitude,             \
        int interleaved, logismos_stream_t stream) {                                                                  \
        lg::NormRopeParams p = {};                                                                                    \
        p.q_in = q_in;                                                                                                \
        p.k_in = k_in;                                                                                                \
        p.q_out = q_out;                                                                                              \
        p.k_out = k_out;                                                                                              \
        p.positions = positions;                                                                                      \
        p.axis_of_pair = axis_of_pair;                                                                                \
        p.inv_freq = inv_freq;                                                                                        \
        p.q_gain = q_gain;                                                                                            \
        p.k_gain = k_gain;                                                                                            \
        p.q_in_stride = q_in_stride;                                                                                  \
        p.k_in_stride = k_in_stride;                                                                                  \
        p.q_out_stride = q_out_stride;                                                                                \
        p.k_out_stride = k_out_stride;                                                                                \
        p.position_stride = position_stride;                                                                          \
        p.tokens = tokens;                                                                                            \
        p.hq = num_q_heads;                                                                                           \
        p.hkv = num_kv_heads;                                                                                         \
        p.d = head_dim;                                                                                               \
        p.axes = num_axes;                                                                                            \
        p.eps = eps;                                                                                                  \
        p.amplitude = amplitude;                                                                                      \
        return lg::norm_rope_packed(bytes, type, p, rotary_dim, interleaved, stream);                                 \
    }
LOGISMOS_NORM_ROPE_PACKED(fp16, 2, 0)
LOGISMOS_NORM_ROPE_PACKED(bf16, 2, 1)
LOGISMOS_NORM_ROPE_PACKED(f32, 4, 2)
#undef LOGISMOS_NORM_ROPE_PACKED

}  // extern "C"
