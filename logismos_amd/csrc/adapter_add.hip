// Low-rank adapters of many requests beside a shared projection:
//
//   out[t][:] = base[t][:] + s_a * (x[t] . A_a^T) . B_a^T,   a = the adapter of the row's sequence
//
// Two launches.  The first takes a tile of one sequence's rows through A: v = x . A^T in fp32 into the workspace, in K parts
// (v is small; adding the parts up is the second launch's first step, in their order).  The second takes the
// same rows through B and adds the base.  Products on the matrix cores, the ranks as rows of the first product's
// result and the rows of x as its columns, the outputs as rows of the second's.
//
// v has to be an operand of the second product, so it is split into 16-bit terms: per row scaled by a power
// of two that brings its largest value into [1, 2) (exact, and undone in the fp32 result; fp16 could not hold the values
// as they are), then the rounded value and what the rounding left.  fp16: two terms, 22 bits; bf16: two terms,
// 16 bits, for outputs of 8, three, 24 bits, for fp32 outputs.
//
// Bound by memory: x, base and out once, A and B of the adapters in use.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"
#include "q4_common.hpp"

#include <math.h>

#include <type_traits>

namespace lg {

constexpr int kAdapterRows = 16;      // rows of a tile
constexpr int kAdapterMaxRank = 256;
constexpr int kAdapterMaxParts = 8;   // K parts of v

struct AdapterParams {
    const unsigned short* x;
    const unsigned short* a;  // [adapters][max_rank][k]
    const unsigned short* b;  // [adapters][n][max_rank]
    const int32_t* ranks;
    const float* scales;
    const int32_t* adapter_of_seq;
    const int32_t* cu;
    const void* base;
    void* out;
    float* v;  // [part][total][max_rank]
    int num_seqs, total, adapters, max_rank, n, k;
    int64_t x_stride, base_stride, out_stride;
    int parts, part_steps;  // K parts, steps of 32 columns of a part
};

// The rank that counts for sequence s; 0: no adapter.
__device__ __forceinline__ int adapter_rank(const AdapterParams& p, int s, int* adapter) {
    const int a = __builtin_amdgcn_readfirstlane(p.adapter_of_seq[s]);
    *adapter = a;
    if (a < 0 || a >= p.adapters) return 0;
    const int r = __builtin_amdgcn_readfirstlane(p.ranks[a]);
    return r < 0 ? 0 : r < p.max_rank ? r : p.max_rank;
}

// v[part][t][r] = sum over the part's columns of x[t][c] * A[r][c].  grid (tiles, K parts, 16 ranks each);
// the four waves share the part's steps and add up in LDS.
template <typename T>
__global__ __launch_bounds__(256) void adapter_down_kernel(const AdapterParams p) {
    __shared__ float sums[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = lane & 15, q = lane >> 4;
    const PackedTile t = packed_tile(p.cu, p.num_seqs, p.total, 1, kAdapterRows, blockIdx.x);
    const int r0 = t.tile * kAdapterRows;
    if (r0 >= t.rows) return;
    int adapter;
    const int rank = adapter_rank(p, t.seq, &adapter);
    const int rank0 = blockIdx.z * 16;
    if (rank0 >= rank) return;
    const int row = r0 + c < t.rows ? r0 + c : t.rows - 1;
    const unsigned short* x = p.x + (int64_t)(t.row0 + row) * p.x_stride;
    const int ar = rank0 + c < rank ? rank0 + c : rank - 1;
    const unsigned short* a = p.a + ((int64_t)adapter * p.max_rank + ar) * p.k;
    const int first = blockIdx.y * p.part_steps;
    const int all = (p.k + 31) / 32;
    const int last = first + p.part_steps < all ? first + p.part_steps : all;
    float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = first + wave; s < last; s += 4) {
        const int at = 32 * s + 8 * q;
        uint4_t xv = {0, 0, 0, 0}, av = {0, 0, 0, 0};
        if (at < p.k) {  // (k is a multiple of 8)
            xv = *reinterpret_cast<const uint4_t*>(x + at);
            av = *reinterpret_cast<const uint4_t*>(a + at);
        }
        acc = T::mfma16(av, xv, acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][lane * 4 + i] = acc[i];
    __syncthreads();
    // thread (row, rank): the value of lane (rank / 4, row), element rank % 4
    const int vr = threadIdx.x >> 4, rk = threadIdx.x & 15;
    if (r0 + vr < t.rows && rank0 + rk < p.max_rank) {
        const int i = ((rk >> 2) * 16 + vr) * 4 + (rk & 3);
        const float sum = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
        p.v[((int64_t)blockIdx.y * p.total + t.row0 + r0 + vr) * p.max_rank + rank0 + rk] = sum;
    }
}

// out = base + s (v . B^T): grid (tiles, 256 outputs each), a wave 64 of them.
template <typename T, bool F32, int TERMS>
__global__ __launch_bounds__(256) void adapter_up_kernel(const AdapterParams p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = lane & 15, q = lane >> 4;
    const PackedTile t = packed_tile(p.cu, p.num_seqs, p.total, 1, kAdapterRows, blockIdx.x);
    const int r0 = t.tile * kAdapterRows;
    if (r0 >= t.rows) return;
    int adapter;
    const int rank = adapter_rank(p, t.seq, &adapter);
    const int n0 = blockIdx.y * 256 + wave * 64;
    if (n0 >= p.n) return;
    if (rank == 0 && p.base == p.out) return;
    const bool live = r0 + c < t.rows;
    const int64_t row = t.row0 + (live ? r0 + c : t.rows - 1);
    // lane (c, q) holds row c's outputs n0 + 16 q .. + 15: element i of tile j is output 16 q + 4 j + i
    const int nl = n0 + 16 * q;
    float y[16];
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
        if (nl + e < p.n) {  // (n is a multiple of 8)
            if constexpr (F32) {
                const float4_t* src = reinterpret_cast<const float4_t*>(static_cast<const float*>(p.base) + row * p.base_stride + nl + e);
                const float4_t u0 = src[0], u1 = src[1];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[e + i] = u0[i];
                    y[e + 4 + i] = u1[i];
                }
            } else {
                const auto u = __builtin_bit_cast(typename T::vec8, *reinterpret_cast<const uint4_t*>(
                    static_cast<const unsigned short*>(p.base) + row * p.base_stride + nl + e));
#pragma unroll
                for (int i = 0; i < 8; ++i) y[e + i] = (float)u[i];
            }
        }
    }
    if (rank > 0) {
        const float* v = p.v + row * p.max_rank;
        const int64_t part = (int64_t)p.total * p.max_rank;
        auto value = [&](int r) LG_INLINE {  // (of 8 from r on, those behind the rank are 0)
            struct { float e[8]; } o;
#pragma unroll
            for (int i = 0; i < 8; ++i) o.e[i] = 0.0f;
            if (r < rank) {
                for (int s = 0; s < p.parts; ++s) {
                    const float4_t* src = reinterpret_cast<const float4_t*>(v + s * part + r);
                    const float4_t u0 = src[0], u1 = src[1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o.e[i] += u0[i];
                        o.e[4 + i] += u1[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) o.e[i] = r + i < rank ? o.e[i] : 0.0f;
            return o;
        };
        float top = 0.0f;
        for (int s = 0; s < rank; s += 32) {
            const auto u = value(s + 8 * q);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(u.e[i]));
        }
        top = fmaxf(top, lane_xor_f32<16>(top));
        top = fmaxf(top, lane_xor_f32<32>(top));
        // 2^-e of the largest value's exponent e, as far as fp32 has it
        const int ex = (int)(__float_as_uint(top) >> 23);
        const int down = ex < 1 ? 1 : ex > 253 ? 253 : ex;
        const float shrink = __uint_as_float((unsigned)(254 - down) << 23);
        const float grow = __uint_as_float((unsigned)down << 23);
        float4_t acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < rank; s += 32) {
            const int r = s + 8 * q;
            const auto u = value(r);
            uint4_t term[TERMS];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float a0 = u.e[i] * shrink, a1 = u.e[i + 1] * shrink;
#pragma unroll
                for (int k = 0; k < TERMS; ++k) {
                    const unsigned w = T::pack2(a0, a1);
                    term[k][i >> 1] = w;
                    typedef typename T::elem elem;
                    a0 -= (float)__builtin_bit_cast(elem, (unsigned short)(w & 0xffffu));
                    a1 -= (float)__builtin_bit_cast(elem, (unsigned short)(w >> 16));
                    a0 = a0 == a0 ? a0 : 0.0f;  // (an infinity is in its first term, with nothing left)
                    a1 = a1 == a1 ? a1 : 0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // row c of tile j
                const int nr = n0 + 16 * (c >> 2) + 4 * j + (c & 3);
                uint4_t bv = {0, 0, 0, 0};
                if (nr < p.n && r < rank) {
                    bv = *reinterpret_cast<const uint4_t*>(p.b + ((int64_t)adapter * p.n + nr) * p.max_rank + r);
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        bv[w] &= rank >= r + 2 * w + 2 ? ~0u : rank == r + 2 * w + 1 ? 0xffffu : 0u;
                }
#pragma unroll
                for (int k = 0; k < TERMS; ++k) acc[j] = T::mfma16(bv, term[k], acc[j]);
            }
        }
        const float scale = p.scales[adapter];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * j + i] = fmaf(acc[j][i] * grow, scale, y[4 * j + i]);
    }
    if (!live) return;
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
        if (nl + e < p.n) {
            if constexpr (F32) {
                float4_t* dst = reinterpret_cast<float4_t*>(static_cast<float*>(p.out) + row * p.out_stride + nl + e);
                dst[0] = float4_t{y[e], y[e + 1], y[e + 2], y[e + 3]};
                dst[1] = float4_t{y[e + 4], y[e + 5], y[e + 6], y[e + 7]};
            } else {
                uint4_t o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = T::pack2(y[e + 2 * i], y[e + 2 * i + 1]);
                *reinterpret_cast<uint4_t*>(static_cast<unsigned short*>(p.out) + row * p.out_stride + nl + e) = o;
            }
        }
    }
}

// K parts of the first product
static int adapter_parts(int k) {
    const int steps = (k + 31) / 32;
    int parts = steps / 16;
    return parts < 1 ? 1 : parts > kAdapterMaxParts ? kAdapterMaxParts : parts;
}

template <typename T>
static hipError_t adapter_launch(AdapterParams p, bool f32, hipStream_t stream) {
    const unsigned tiles = (unsigned)packed_tiles(p.total, p.num_seqs, 1, kAdapterRows);
    adapter_down_kernel<T><<<dim3(tiles, p.parts, (p.max_rank + 15) / 16), 256, 0, stream>>>(p);
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    const dim3 grid(tiles, (p.n + 255) / 256);
    if (!f32) adapter_up_kernel<T, false, 2><<<grid, 256, 0, stream>>>(p);
    else adapter_up_kernel<T, true, std::is_same<T, PackedF16>::value ? 2 : 3><<<grid, 256, 0, stream>>>(p);
    return hipGetLastError();
}

static logismos_status_t adapter_add(bool bf16, const void* x, const void* a, const void* b, const int32_t* ranks,
                                     const float* scales, const int32_t* adapter_of_seq, const int32_t* cu,
                                     const void* base, void* out, int f32, void* workspace, int num_seqs, int total,
                                     int adapters, int max_rank, int n, int k, int x_stride, int base_stride,
                                     int out_stride, logismos_stream_t stream) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (logismos_check_adapter_add_shape(num_seqs, total, adapters, max_rank, n, k, x_stride, base_stride, out_stride,
                                         nullptr, 0) != 0)
        return bad;
    if (!x || !a || !b || !ranks || !scales || !adapter_of_seq || !cu || !base || !out || !workspace) return bad;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
         reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(out) |
         reinterpret_cast<uintptr_t>(workspace)) % 16 != 0)
        return bad;
    if ((reinterpret_cast<uintptr_t>(ranks) | reinterpret_cast<uintptr_t>(scales) |
         reinterpret_cast<uintptr_t>(adapter_of_seq) | reinterpret_cast<uintptr_t>(cu)) % 4 != 0)
        return bad;
    if (base == out && base_stride != out_stride) return bad;
    AdapterParams p = {};
    p.x = static_cast<const unsigned short*>(x);
    p.a = static_cast<const unsigned short*>(a);
    p.b = static_cast<const unsigned short*>(b);
    p.ranks = ranks;
    p.scales = scales;
    p.adapter_of_seq = adapter_of_seq;
    p.cu = cu;
    p.base = base;
    p.out = out;
    p.v = static_cast<float*>(workspace);
    p.num_seqs = num_seqs;
    p.total = total;
    p.adapters = adapters;
    p.max_rank = max_rank;
    p.n = n;
    p.k = k;
    p.x_stride = x_stride;
    p.base_stride = base_stride;
    p.out_stride = out_stride;
    p.parts = adapter_parts(k);
    p.part_steps = ((k + 31) / 32 + p.parts - 1) / p.parts;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return static_cast<logismos_status_t>(bf16 ? adapter_launch<PackedBf16>(p, f32 != 0, st)
                                               : adapter_launch<PackedF16>(p, f32 != 0, st));
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_adapter_add_shape(int num_seqs, int total_tokens, int num_adapters, int max_rank,
                                                   int n, int k, int x_stride, int base_stride, int out_stride,
                                                   char* msg, size_t cap) {
    using lg::reject;
    if (num_seqs <= 0 || total_tokens <= 0 || num_adapters <= 0 || n <= 0 || k <= 0)
        return reject(msg, cap, "num_seqs, total_tokens, num_adapters, n and k must be positive (%d, %d, %d, %d, %d)",
                      num_seqs, total_tokens, num_adapters, n, k);
    if (max_rank <= 0 || max_rank % 8 != 0 || max_rank > lg::kAdapterMaxRank)
        return reject(msg, cap, "max_rank must be a multiple of 8 up to %d (%d)", lg::kAdapterMaxRank, max_rank);
    if (n % 8 != 0 || k % 8 != 0) return reject(msg, cap, "n and k must be multiples of 8 (%d, %d)", n, k);
    if (x_stride < k || base_stride < n || out_stride < n)
        return reject(msg, cap, "a stride is smaller than its row (%d of %d, %d and %d of %d)", x_stride, k, base_stride,
                      out_stride, n);
    if (x_stride % 8 != 0 || base_stride % 8 != 0 || out_stride % 8 != 0)
        return reject(msg, cap, "strides must be multiples of 8 (%d, %d, %d)", x_stride, base_stride, out_stride);
    if (n > 65535 * 256) return reject(msg, cap, "n must be at most %d (%d)", 65535 * 256, n);
    if ((int64_t)total_tokens + num_seqs > lg::kPackedMaxRows)
        return reject(msg, cap, "total_tokens + num_seqs exceeds %d", lg::kPackedMaxRows);
    return 0;
}

size_t logismos_adapter_add_workspace_bytes(int total_tokens, int max_rank) {
    if (total_tokens <= 0 || max_rank <= 0) return 0;
    return (size_t)lg::kAdapterMaxParts * (size_t)total_tokens * (size_t)max_rank * sizeof(float);
}

#define LOGISMOS_ADAPTER_ADD(name, bf16)                                                                              \
    logismos_status_t logismos_launch_adapter_add_##name(                                                             \
        const void* x, const void* a, const void* b, const int32_t* ranks, const float* scales,                       \
        const int32_t* adapter_of_seq, const int32_t* cu_seqlens, const void* base, void* out, int out_is_f32,        \
        void* workspace, int num_seqs, int total_tokens, int num_adapters, int max_rank, int n, int k, int x_stride,  \
        int base_stride, int out_stride, logismos_stream_t stream) {                                                  \
        return lg::adapter_add(bf16, x, a, b, ranks, scales, adapter_of_seq, cu_seqlens, base, out, out_is_f32,       \
                               workspace, num_seqs, total_tokens, num_adapters, max_rank, n, k, x_stride,             \
                               base_stride, out_stride, stream);                                                      \
    }
LOGISMOS_ADAPTER_ADD(fp16, false)
LOGISMOS_ADAPTER_ADD(bf16, true)
#undef LOGISMOS_ADAPTER_ADD

}  // extern "C"
