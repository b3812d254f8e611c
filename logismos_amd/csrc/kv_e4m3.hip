// K and V rows of a paged cache in 8 bits: quantised as they are written, and read back.
//
// A head row x of d elements is held as d e4m3 values (4 exponent and 3 mantissa bits, largest 448) and one power of two:
//
//   e = the smallest integer with max |x_i| <= 448 * 2^e, kept within [-64, 32]
//   c_i = e4m3(x_i * 2^-e), to nearest, ties to even;   x_i ~ c_i * 2^e
//
// With a power of two the product in front of the rounding and the one behind it are exact, so that an element is off by half a
// step of e4m3 and nothing else: at most 2^-4 of itself down to 2^-6 * 2^e, 2^-10 * 2^e below (a scale of max / 448 would use up to one bit
// more of the range of a type whose steps grow with the values, for two more roundings).  The exponents of neighbouring rows of a head lie
// side by side, so that the attention reads those of 16 keys at once.
//
// Bound by memory: an element is read and written once.  d / 8 lanes take a head row, 16 bytes each.  A workgroup takes the
// rows of up to 16 neighbouring tokens, so that the exponent bytes of a block are written within one compute unit.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"
#include "q4_common.hpp"

namespace lg {

constexpr int kE4m3Threads = 256;
constexpr int kE4m3Lowest = -64, kE4m3Highest = 32;  // exponents of a row

struct E4m3Params {
    const void* k_in;  // rows, or the pools when they are read
    const void* v_in;
    void* k_out;
    void* v_out;
    uint8_t* k_exp;
    uint8_t* v_exp;
    const int64_t* slots;
    int64_t k_stride, v_stride;  // elements, of the rows
    int64_t rows;                // of a pool
    int tokens, hkv, d, block_size;
    int tok;  // tokens per workgroup
};

// Largest of the LANES lanes of a head row (LANES a power of two up to 32).
template <int LANES>
__device__ __forceinline__ float row_lanes_max(float v) {
    if constexpr (LANES > 1) v = fmaxf(v, lane_xor_f32<1>(v));
    if constexpr (LANES > 2) v = fmaxf(v, lane_xor_f32<2>(v));
    if constexpr (LANES > 4) v = fmaxf(v, lane_xor_f32<4>(v));
    if constexpr (LANES > 8) v = fmaxf(v, lane_xor_f32<8>(v));
    if constexpr (LANES > 16) v = fmaxf(v, lane_xor_f32<16>(v));
    return v;
}

// The exponent of a row whose largest finite magnitude is `top` (0: the lowest).
__device__ __forceinline__ int e4m3_exponent(float top) {
    // (bf16 rows may hold subnormals: all of them get the lowest exponent, as everything below 448 * 2^-64 does)
    const unsigned u = __float_as_uint(top);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
    return e < kE4m3Lowest ? kE4m3Lowest : e > kE4m3Highest ? kE4m3Highest : e;
}

// (the type has no infinities: they become NaN)
__device__ __forceinline__ float e4m3_in_range(float x) {
    return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -448.0f, 448.0f) : NAN;
}

// Item i of a workgroup: (token, K or V, head), heads innermost.
struct E4m3Item {
    int64_t token;
    int head;
    bool is_v;
};
__device__ __forceinline__ E4m3Item e4m3_item(const E4m3Params& p, int t0, int i) {
    const int t = i / (2 * p.hkv), rest = i - t * 2 * p.hkv;
    return {t0 + t, rest >= p.hkv ? rest - p.hkv : rest, rest >= p.hkv};
}

template <typename E, int LANES>
__global__ __launch_bounds__(kE4m3Threads) void kv_write_e4m3_kernel(const E4m3Params p) {
    typedef E elems __attribute__((ext_vector_type(8)));
    constexpr int kGroups = kE4m3Threads / LANES, kAhead = 4;  // items that a group has in flight
    const int t0 = blockIdx.x * p.tok;
    const int n = (p.tokens - t0 < p.tok ? p.tokens - t0 : p.tok) * 2 * p.hkv;
    const int at = threadIdx.x % LANES;
    const bool mine = 8 * at < p.d;  // (a width that is no power of two leaves lanes over)
    for (int i0 = threadIdx.x / LANES; i0 < n; i0 += kAhead * kGroups) {
        elems x[kAhead];
        int64_t slot[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * kGroups;
            slot[a] = -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[a][j] = (E)0.0f;
            if (i >= n) continue;
            const E4m3Item it = e4m3_item(p, t0, i);
            slot[a] = p.slots[it.token];
            const E* src = static_cast<const E*>(it.is_v ? p.v_in : p.k_in) +
                           it.token * (it.is_v ? p.v_stride : p.k_stride) + (int64_t)it.head * p.d + 8 * at;
            if (mine) x[a] = *reinterpret_cast<const elems*>(src);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            float f[8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = (float)x[a][j];
                const float m = fabsf(f[j]);
                top = fmaxf(top, m < INFINITY ? m : 0.0f);  // (of the finite ones)
            }
            const int e = e4m3_exponent(row_lanes_max<LANES>(top));
            if (slot[a] < 0 || slot[a] >= p.rows) continue;
            const E4m3Item it = e4m3_item(p, t0, i0 + a * kGroups);
            const float scale = __int_as_float((127 - e) << 23);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = e4m3_in_range(f[j] * scale);
            uint2_t c;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                int word = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * w], f[4 * w + 1], 0, false);
                c[w] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * w + 2], f[4 * w + 3], word, true);
            }
            uint8_t* dst = static_cast<uint8_t*>(it.is_v ? p.v_out : p.k_out) +
                           (slot[a] * p.hkv + it.head) * p.d + 8 * at;
            if (mine) *reinterpret_cast<uint2_t*>(dst) = c;
            if (at == 0) {
                const int64_t block = (unsigned)slot[a] / (unsigned)p.block_size;
                const int64_t row = (unsigned)slot[a] % (unsigned)p.block_size;
                (it.is_v ? p.v_exp : p.k_exp)[(block * p.hkv + it.head) * p.block_size + row] = (uint8_t)(e + 127);
            }
        }
    }
}

template <typename E>
struct alignas(16) E4m3Out {
    E e[8];
};

template <typename E, int LANES>
__global__ __launch_bounds__(kE4m3Threads) void kv_gather_e4m3_kernel(const E4m3Params p) {
    constexpr int kGroups = kE4m3Threads / LANES, kAhead = 4;
    const int t0 = blockIdx.x * p.tok;
    const int n = (p.tokens - t0 < p.tok ? p.tokens - t0 : p.tok) * 2 * p.hkv;
    const int at = threadIdx.x % LANES;
    if (8 * at >= p.d) return;
    for (int i0 = threadIdx.x / LANES; i0 < n; i0 += kAhead * kGroups) {
        uint2_t c[kAhead];
        unsigned e[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * kGroups;
            c[a] = uint2_t{0, 0};
            e[a] = 127;
            if (i >= n) continue;
            const E4m3Item it = e4m3_item(p, t0, i);
            const int64_t slot = p.slots[it.token];
            if (slot < 0 || slot >= p.rows) continue;
            c[a] = *reinterpret_cast<const uint2_t*>(static_cast<const uint8_t*>(it.is_v ? p.v_in : p.k_in) +
                                                     (slot * p.hkv + it.head) * p.d + 8 * at);
            const int64_t block = (unsigned)slot / (unsigned)p.block_size;
            const int64_t row = (unsigned)slot % (unsigned)p.block_size;
            e[a] = (it.is_v ? p.v_exp : p.k_exp)[(block * p.hkv + it.head) * p.block_size + row];
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * kGroups;
            if (i >= n) continue;
            const E4m3Item it = e4m3_item(p, t0, i);
            const float scale = __int_as_float((int)(e[a] << 23));
            E4m3Out<E> y;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                typedef float float2_t __attribute__((ext_vector_type(2)));
                const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[a][w], false);
                const float2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[a][w], true);
                const float f[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = f[j] * scale;
                    if constexpr (sizeof(E) == 2 && !__is_same(E, __bf16)) {  // fp16 ends earlier than the cache
                        const float in = __builtin_amdgcn_fmed3f(v, -65504.0f, 65504.0f);
                        v = v == v ? in : v;
                    }
                    y.e[4 * w + j] = (E)v;
                }
            }
            E* dst = static_cast<E*>(it.is_v ? p.v_out : p.k_out) + it.token * (it.is_v ? p.v_stride : p.k_stride) +
                     (int64_t)it.head * p.d + 8 * at;
            *reinterpret_cast<E4m3Out<E>*>(dst) = y;
        }
    }
}

template <typename E, bool WRITE>
static hipError_t kv_e4m3_by_width(E4m3Params p, hipStream_t stream) {
    // up to 16 tokens to a workgroup, fewer where workgroups are what is missing
    int tok = 16;
    while (tok > 1 && p.tokens < 4 * tok * device_cu_count()) tok /= 2;
    p.tok = tok;
    const unsigned grid = (unsigned)((p.tokens + tok - 1) / tok);
    auto go = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        if constexpr (WRITE) kv_write_e4m3_kernel<E, L><<<grid, kE4m3Threads, 0, stream>>>(p);
        else kv_gather_e4m3_kernel<E, L><<<grid, kE4m3Threads, 0, stream>>>(p);
    };
    if (p.d <= 32) go(ic<4>{});
    else if (p.d <= 64) go(ic<8>{});
    else if (p.d <= 128) go(ic<16>{});
    else go(ic<32>{});
    return hipGetLastError();
}

static bool kv_e4m3_arguments(const E4m3Params& p) {
    if (!p.k_in || !p.v_in || !p.k_out || !p.v_out || !p.k_exp || !p.v_exp || !p.slots) return false;
    return (reinterpret_cast<uintptr_t>(p.k_in) | reinterpret_cast<uintptr_t>(p.v_in) |
            reinterpret_cast<uintptr_t>(p.k_out) | reinterpret_cast<uintptr_t>(p.v_out) |
            reinterpret_cast<uintptr_t>(p.k_exp) | reinterpret_cast<uintptr_t>(p.v_exp)) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(p.slots) % 8 == 0;
}

template <bool WRITE>
static logismos_status_t kv_e4m3(int type, const void* k_in, const void* v_in, void* k_out, void* v_out,
                                 const void* k_exp, const void* v_exp, const int64_t* slots, int tokens, int hkv,
                                 int d, int block_size, int num_blocks, int k_stride, int v_stride,
                                 logismos_stream_t stream) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (logismos_check_kv_e4m3_shape(tokens, hkv, d, block_size, num_blocks, k_stride, v_stride, nullptr, 0) != 0)
        return bad;
    if (tokens == 0) return 0;
    E4m3Params p = {};
    p.k_in = k_in;
    p.v_in = v_in;
    p.k_out = k_out;
    p.v_out = v_out;
    p.k_exp = static_cast<uint8_t*>(const_cast<void*>(k_exp));
    p.v_exp = static_cast<uint8_t*>(const_cast<void*>(v_exp));
    p.slots = slots;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.rows = (int64_t)num_blocks * block_size;
    p.tokens = tokens;
    p.hkv = hkv;
    p.d = d;
    p.block_size = block_size;
    if (!kv_e4m3_arguments(p)) return bad;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (type == 0) return static_cast<logismos_status_t>(kv_e4m3_by_width<_Float16, WRITE>(p, st));
    if constexpr (!WRITE)
        if (type == 2) return static_cast<logismos_status_t>(kv_e4m3_by_width<float, WRITE>(p, st));
    return static_cast<logismos_status_t>(kv_e4m3_by_width<__bf16, WRITE>(p, st));
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_kv_e4m3_shape(int total_tokens, int num_kv_heads, int head_dim, int block_size,
                                               int num_blocks, int k_stride, int v_stride, char* msg, size_t cap) {
    using lg::reject;
    if (total_tokens < 0 || total_tokens > lg::kPackedMaxRows)
        return reject(msg, cap, "total_tokens must be between 0 and %d (%d)", lg::kPackedMaxRows, total_tokens);
    if (num_kv_heads <= 0 || num_blocks <= 0)
        return reject(msg, cap, "num_kv_heads and num_blocks must be positive (%d, %d)", num_kv_heads, num_blocks);
    if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 256)
        return reject(msg, cap, "head_dim must be a multiple of 32 up to 256 (%d)", head_dim);
    if (block_size <= 0 || block_size % 16 != 0)
        return reject(msg, cap, "block_size must be a positive multiple of 16 (%d)", block_size);
    if ((int64_t)num_blocks * block_size > INT32_MAX)
        return reject(msg, cap, "num_blocks * block_size exceeds i32::MAX");
    const int64_t width = (int64_t)num_kv_heads * head_dim;
    if (width > (1 << 20)) return reject(msg, cap, "num_kv_heads * head_dim exceeds %d", 1 << 20);
    if (k_stride < width || v_stride < width)
        return reject(msg, cap, "a stride is smaller than its row (%d and %d of %lld)", k_stride, v_stride,
                      (long long)width);
    if ((k_stride | v_stride) % 8 != 0)
        return reject(msg, cap, "strides must be multiples of 8 (%d, %d)", k_stride, v_stride);
    return 0;
}

#define LOGISMOS_KV_WRITE_E4M3(name, type)                                                                             \
    logismos_status_t logismos_launch_kv_write_e4m3_##name(                                                            \
        const void* k_new, const void* v_new, void* k_pool, void* k_exp, void* v_pool, void* v_exp,                    \
        const int64_t* slot_mapping, int total_tokens, int num_kv_heads, int head_dim, int block_size, int num_blocks, \
        int k_stride, int v_stride, logismos_stream_t stream) {                                                        \
        return lg::kv_e4m3<true>(type, k_new, v_new, k_pool, v_pool, k_exp, v_exp, slot_mapping, total_tokens,         \
                                 num_kv_heads, head_dim, block_size, num_blocks, k_stride, v_stride, stream);          \
    }
LOGISMOS_KV_WRITE_E4M3(fp16, 0)
LOGISMOS_KV_WRITE_E4M3(bf16, 1)
#undef LOGISMOS_KV_WRITE_E4M3

#define LOGISMOS_KV_GATHER_E4M3(name, type)                                                                            \
    logismos_status_t logismos_launch_kv_gather_e4m3_##name(                                                           \
        const void* k_pool, const void* k_exp, const void* v_pool, const void* v_exp, const int64_t* slot_mapping,     \
        void* k_out, void* v_out, int total_tokens, int num_kv_heads, int head_dim, int block_size, int num_blocks,    \
        int k_stride, int v_stride, logismos_stream_t stream) {                                                        \
        return lg::kv_e4m3<false>(type, k_pool, v_pool, k_out, v_out, k_exp, v_exp, slot_mapping, total_tokens,        \
                                  num_kv_heads, head_dim, block_size, num_blocks, k_stride, v_stride, stream);         \
    }
LOGISMOS_KV_GATHER_E4M3(fp16, 0)
LOGISMOS_KV_GATHER_E4M3(bf16, 1)
LOGISMOS_KV_GATHER_E4M3(f32, 2)
#undef LOGISMOS_KV_GATHER_E4M3

}  // extern "C"
