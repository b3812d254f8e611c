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
// Bound by memory: an element is read and written once.  d / 8 lanes take a head row, 16 bytes each; its maximum is taken of the
// values' bits, and the conversions scale (two elements an instruction; written out in fp32, conversion, product, clamp and NaN, they
// were as long as the memory: 32768 rows of 8 heads of 128, 202 MB, 52 us, now 42, 4.8 TB/s; read back 47, a large copy 5.2).
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
__device__ __forceinline__ int row_lanes_max(int v) {
    if constexpr (LANES > 1) v = max(v, lane_xor_i32<1>(v));
    if constexpr (LANES > 2) v = max(v, lane_xor_i32<2>(v));
    if constexpr (LANES > 4) v = max(v, lane_xor_i32<4>(v));
    if constexpr (LANES > 8) v = max(v, lane_xor_i32<8>(v));
    if constexpr (LANES > 16) v = max(v, lane_xor_i32<16>(v));
    return v;
}

// The 16-bit types: magnitudes compare as their bits do.
struct E4m3F16 {
    static constexpr unsigned kInf = 0x7c00u;
    static __device__ __forceinline__ float value(unsigned bits) {
        return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
    }
    template <bool HI>
    static __device__ __forceinline__ unsigned pack(unsigned into, unsigned pair, float scale) {
        typedef short short2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(
                                                __builtin_bit_cast(short2_t, into), __builtin_bit_cast(half2_t, pair), scale, HI));
    }
};
struct E4m3Bf16 {
    static constexpr unsigned kInf = 0x7f80u;
    static __device__ __forceinline__ float value(unsigned bits) { return __uint_as_float(bits << 16); }
    template <bool HI>
    static __device__ __forceinline__ unsigned pack(unsigned into, unsigned pair, float scale) {
        typedef short short2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
                                                __builtin_bit_cast(short2_t, into), __builtin_bit_cast(bf16x2_t, pair), scale, HI));
    }
};

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

template <typename T, int LANES>
__global__ __launch_bounds__(kE4m3Threads) void kv_write_e4m3_kernel(const E4m3Params p) {
    constexpr int kGroups = kE4m3Threads / LANES, kAhead = 4;  // items that a group has in flight
    const int t0 = blockIdx.x * p.tok;
    const int n = (p.tokens - t0 < p.tok ? p.tokens - t0 : p.tok) * 2 * p.hkv;
    const int at = threadIdx.x % LANES;
    const bool mine = 8 * at < p.d;  // (a width that is no power of two leaves lanes over)
    for (int i0 = threadIdx.x / LANES; i0 < n; i0 += kAhead * kGroups) {
        uint4_t x[kAhead];
        int64_t slot[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * kGroups;
            slot[a] = -1;
            x[a] = uint4_t{0, 0, 0, 0};
            if (i >= n) continue;
            const E4m3Item it = e4m3_item(p, t0, i);
            slot[a] = p.slots[it.token];
            const unsigned short* src = static_cast<const unsigned short*>(it.is_v ? p.v_in : p.k_in) +
                                        it.token * (it.is_v ? p.v_stride : p.k_stride) + (int64_t)it.head * p.d + 8 * at;
            if (mine) x[a] = *reinterpret_cast<const uint4_t*>(src);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            unsigned most = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                most = max(most, max(x[a][w] & 0x7fffu, (x[a][w] >> 16) & 0x7fffu));
            most = (unsigned)row_lanes_max<LANES>((int)most);
            int e = e4m3_exponent(T::value(most));
            uint2_t c;
            if (__builtin_expect(most < T::kInf && !(T::value(most) > 448.0f * 4294967296.0f), 1)) {
                const float scale = __int_as_float((127 + e) << 23);
                c[0] = T::template pack<true>(T::template pack<false>(0u, x[a][0], scale), x[a][1], scale);
                c[1] = T::template pack<true>(T::template pack<false>(0u, x[a][2], scale), x[a][3], scale);
            } else {  // infinities, NaN, values beyond the cache's range
                unsigned finite = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const unsigned m = (x[a][w] >> (16 * y)) & 0x7fffu;
                        finite = max(finite, m < T::kInf ? m : 0u);
                    }
                e = e4m3_exponent(T::value((unsigned)row_lanes_max<LANES>((int)finite)));
                const float scale = __int_as_float((127 - e) << 23);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    float f[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        f[y] = e4m3_in_range(T::value((x[a][2 * w + (y >> 1)] >> (16 * (y & 1))) & 0xffffu) * scale);
                    const int word = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                    c[w] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], word, true);
                }
            }
            if (slot[a] < 0 || slot[a] >= p.rows) continue;
            const E4m3Item it = e4m3_item(p, t0, i0 + a * kGroups);
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

// Eight values times a power of two.
template <typename E>
__device__ __forceinline__ void e4m3_decode(uint2_t c, float scale, E (&y)[8]) {
    typedef E pair_t __attribute__((ext_vector_type(2)));
    static_for<2>([&](auto word) LG_INLINE {
        static_for<2>([&](auto half) LG_INLINE {
            constexpr int w = decltype(word)::value;
            constexpr bool kHi = decltype(half)::value != 0;
            pair_t v;
            if constexpr (__is_same(E, float)) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[w], scale, kHi);
            else if constexpr (__is_same(E, _Float16)) v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[w], scale, kHi);
            else v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[w], scale, kHi);
            y[4 * w + 2 * kHi] = v[0];
            y[4 * w + 2 * kHi + 1] = v[1];
        });
    });
}

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
            constexpr bool kF16 = __is_same(E, _Float16);
            if (!kF16 || __builtin_expect(e[a] <= 127 + 7, 1)) {  // (448 * 2^7 is within fp16)
                e4m3_decode(c[a], scale, y.e);
            } else {  // fp16 ends earlier than the cache
                float f[8];
                e4m3_decode(c[a], scale, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float in = __builtin_amdgcn_fmed3f(f[j], -65504.0f, 65504.0f);
                    y.e[j] = (E)(f[j] == f[j] ? in : f[j]);
                }
            }
            E* dst = static_cast<E*>(it.is_v ? p.v_out : p.k_out) + it.token * (it.is_v ? p.v_stride : p.k_stride) +
                     (int64_t)it.head * p.d + 8 * at;
            *reinterpret_cast<E4m3Out<E>*>(dst) = y;
        }
    }
}

template <typename E>
struct E4m3Rows {
    typedef E4m3F16 type;
};
template <>
struct E4m3Rows<__bf16> {
    typedef E4m3Bf16 type;
};

template <typename E, bool WRITE>
static hipError_t kv_e4m3_by_width(E4m3Params p, hipStream_t stream) {
    // as many tokens to a workgroup as keep all its lanes at work, fewer where workgroups are what is missing
    const int lanes = p.d <= 32 ? 4 : p.d <= 64 ? 8 : p.d <= 128 ? 16 : 32;
    int tok = 2 * kE4m3Threads / lanes / p.hkv;
    tok = tok < 1 ? 1 : tok > 64 ? 64 : tok;
    while (tok > 1 && p.tokens < 2 * (int64_t)tok * device_cu_count()) tok /= 2;
    p.tok = tok;
    const unsigned grid = (unsigned)((p.tokens + tok - 1) / tok);
    auto go = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        if constexpr (WRITE) kv_write_e4m3_kernel<typename E4m3Rows<E>::type, L><<<grid, kE4m3Threads, 0, stream>>>(p);
        else kv_gather_e4m3_kernel<E, L><<<grid, kE4m3Threads, 0, stream>>>(p);
    };
    switch (lanes) {
        case 4: go(ic<4>{}); break;
        case 8: go(ic<8>{}); break;
        case 16: go(ic<16>{}); break;
        default: go(ic<32>{});
    }
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
