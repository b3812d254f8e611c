// Low-rank adapters of many requests beside a shared projection:
//
//   out[t][:] = base[t][:] + s_a * (x[t] . A_a^T) . B_a^T,   a = the adapter of the row's sequence
//
// Two launches.  The first takes a tile of one sequence's rows through A: v = x . A^T in fp32 into the workspace, in K parts
// (v is small; adding the parts up is the second launch's first step, in their order).  The second takes the
// same rows through B and adds the base.  Products on the matrix cores, the ranks as rows of the first product's
// result and the rows of x as its columns, the outputs as rows of the second's.
//
// s v has to be an operand of the second product, so it is split into 16-bit terms: per row scaled by a power
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

#include <algorithm>
#include <type_traits>

namespace lg {

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
    int n_slice, slices;    // outputs of a workgroup, a multiple of 256; how many of them
};

__device__ __forceinline__ int adapter_rank(const AdapterParams& p, int adapter) {
    if (adapter < 0 || adapter >= p.adapters) return 0;
    const int r = __builtin_amdgcn_readfirstlane(p.ranks[adapter]);
    return r < 0 ? 0 : r < p.max_rank ? r : p.max_rank;
}

// v[part][t][r] = sum over the part's columns of x[t][c] * A[r][c].  grid (tiles of 16 MT rows by K parts, 16 RT ranks
// each); the four waves share the part's steps of 32 columns and add up in LDS.
template <typename T, int MT, int RT>
__global__ __launch_bounds__(256, 2) void adapter_down_kernel(const AdapterParams p) {
    constexpr int kDeep = MT > 1 ? 4 : 8;  // steps asked for together, side by side: whole cache lines
    __shared__ float sums[4][MT * RT * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    const int part = (int)(blockIdx.x % (unsigned)p.parts);
    const PackedTile t = packed_tile<true>(p.cu, p.num_seqs, p.total, 1, 16 * MT, (int)(blockIdx.x / (unsigned)p.parts),
                                           p.adapter_of_seq);
    const int r0 = t.tile * 16 * MT;
    if (r0 >= t.rows || t.of < 0 || t.of >= p.adapters) return;
    const int rank0 = blockIdx.y * 16 * RT;
    // (ranks of the first tiles are not waited for: what lies behind the rank is left out when v is read)
    if (rank0 > 0 && rank0 >= adapter_rank(p, t.of)) return;
    const unsigned short* x[MT];
    const unsigned short* a[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = r0 + 16 * m + c < t.rows ? r0 + 16 * m + c : t.rows - 1;
        x[m] = p.x + (int64_t)(t.row0 + row) * p.x_stride;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = rank0 + 16 * i + c < p.max_rank ? rank0 + 16 * i + c : p.max_rank - 1;
        a[i] = p.a + ((int64_t)t.of * p.max_rank + r) * p.k;
    }
    const int all = (p.k + 31) / 32;
    const int first = part * p.part_steps + wave * kDeep;
    const int last = min((part + 1) * p.part_steps, all);
    float4_t acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[m][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // (whole: all steps are the wave's and inside the rows.  The others load the last columns instead of what is not there,
    // and take zeros: k is a multiple of 8)
    auto round = [&](auto whole_c, int s0) LG_INLINE {
        constexpr bool WHOLE = decltype(whole_c)::value != 0;
        uint4_t xv[kDeep][MT], av[kDeep][RT];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const int want = 32 * (s0 + d) + 8 * q;
            const int at = WHOLE || want < p.k ? want : p.k - 8;
#pragma unroll
            for (int m = 0; m < MT; ++m) xv[d][m] = *reinterpret_cast<const uint4_t*>(x[m] + at);
#pragma unroll
            for (int i = 0; i < RT; ++i) av[d][i] = *reinterpret_cast<const uint4_t*>(a[i] + at);
        }
        __builtin_amdgcn_sched_barrier(0);  // (all of them, then the products)
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if constexpr (!WHOLE) {
                const bool in = s0 + d < last && 32 * (s0 + d) + 8 * q < p.k;
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[d][m] = in ? xv[d][m] : uint4_t{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < RT; ++i) av[d][i] = in ? av[d][i] : uint4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < RT; ++i) acc[m][i] = T::mfma16(av[d][i], xv[d][m], acc[m][i]);
        }
    };
    int s0 = first;
    for (; s0 + kDeep <= last && 32 * (s0 + kDeep) <= p.k; s0 += 4 * kDeep) round(ic<1>{}, s0);
    if (s0 < last) round(ic<0>{}, s0);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < RT; ++i)
            *reinterpret_cast<float4_t*>(&sums[wave][((m * RT + i) * 64 + lane) * 4]) = acc[m][i];
    __syncthreads();
    // four ranks of a row per thread and turn: what lane (q, c) holds of tile (m, i)
    for (int e = threadIdx.x; e < MT * RT * 64; e += 256) {
        const int tile = e >> 6, m = tile / RT, i = tile - m * RT;
        const int row = r0 + 16 * m + (e & 15), rank = rank0 + 16 * i + 4 * ((e >> 4) & 3);
        float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const float4_t*>(&sums[w][e * 4]);
        if (row < t.rows && rank < p.max_rank)
            *reinterpret_cast<float4_t*>(p.v + ((int64_t)part * p.total + t.row0 + row) * p.max_rank + rank) = v;
    }
}

// out = base + (s v) . B^T.  grid: slices of the outputs (fastest: a slice of B then stays in the L2 of the XCDs that
// take it, for all rows of its adapter) by tiles of 16 MT rows; ranks in RS steps of 32.  The workgroup splits
// s v into terms once, in the order of the matrix operand, into LDS; a wave takes 64 outputs at a time, the four
// waves side by side.
template <typename T, bool F32, int TERMS, int MT, int RS>
__global__ __launch_bounds__(256, RS == 8 ? 1 : 2) void adapter_up_kernel(const AdapterParams p) {
    constexpr int kRows = 16 * MT, kChunks = 4 * RS;  // chunks of eight ranks
    __shared__ uint4_t operand[MT * RS * TERMS * 64];
    __shared__ float growth[kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    const int slice = (int)(blockIdx.x % (unsigned)p.slices);
    const PackedTile t = packed_tile<true>(p.cu, p.num_seqs, p.total, 1, kRows, (int)(blockIdx.x / (unsigned)p.slices),
                                           p.adapter_of_seq);
    const int r0 = t.tile * kRows;
    if (r0 >= t.rows) return;
    // What hangs on nothing but the tile is asked for in one go: rank and scale, the parts of v, the base.
    const bool named = t.of >= 0 && t.of < p.adapters;
    if (!named && p.base == p.out) return;
    const int raw_rank = p.ranks[named ? t.of : 0];
    const float scale = p.scales[named ? t.of : 0];
    const int left = t.rows - r0 < kRows ? t.rows - r0 : kRows;  // rows of this tile
    const int64_t row0 = t.row0 + r0;
    const int n_last = (slice + 1) * p.n_slice < p.n ? (slice + 1) * p.n_slice : p.n;
    int n0 = slice * p.n_slice + 64 * wave;
    // A wave's 64 outputs are four tiles of 16, ordered so that a lane (c, q) holds 16 bytes side by side of row c and
    // the four q of a row 64: fp32, element i of tile j is output 16 j + 4 q + i; 16 bits, 32 (j / 2) + 8 q + 4 (j % 2) + i.
    // What comes from memory is asked for ahead: the base by a step, B as soon as the step's products are done.
    constexpr int kBase = F32 ? 4 : 2, kSize = F32 ? 4 : 2;
    // (rows behind the tile's last, outputs behind the last and ranks behind the rank: others in their place, which count
    // for nothing -- a load under a condition of its own is a branch around it.  Offsets from the tile's first row and the
    // adapter's B have 32 bits.)
    uint4_t even[MT][kBase], odd[MT][kBase], bv[RS][4];
    const char* const base = static_cast<const char*>(p.base) + row0 * p.base_stride * kSize;
    char* const out = static_cast<char*>(p.out) + row0 * p.out_stride * kSize;
    const char* const b = reinterpret_cast<const char*>(p.b + (int64_t)(named ? t.of : 0) * p.n * p.max_rank);
    auto load_base = [&](uint4_t(&w)[MT][kBase], int at_n) LG_INLINE {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const unsigned row = (unsigned)min(16 * m + c, left - 1) * (unsigned)p.base_stride;
#pragma unroll
            for (int e = 0; e < kBase; ++e) {
                const unsigned n = (unsigned)min(at_n + (F32 ? 16 * e + 4 * q : 32 * e + 8 * q), p.n - 16 / kSize);
                w[m][e] = *reinterpret_cast<const uint4_t*>(base + (row + n) * (unsigned)kSize);
            }
        }
    };
    int rank = 0;
    auto load_b = [&](int at_n) LG_INLINE {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int want = at_n + (F32 ? 16 * j + c : 32 * (j >> 1) + 8 * (c >> 2) + 4 * (j & 1) + (c & 3));
            const unsigned row = (unsigned)min(want, p.n - 1) * (unsigned)p.max_rank;
#pragma unroll
            for (int s = 0; s < RS; ++s)
                bv[s][j] = *reinterpret_cast<const uint4_t*>(b + (row + (32 * s + 8 * q < rank ? 32 * s + 8 * q : 0)) * 2u);
        }
    };
    // Thread (row, chunk of eight ranks), the chunks of a row side by side; four parts of v at a time.
    struct Parts {
        float4_t w[4][2];
    };
    const int64_t part = (int64_t)p.total * p.max_rank;
    auto v_at = [&](int i) LG_INLINE {
        return p.v + (row0 + min(i / kChunks, left - 1)) * p.max_rank + min(8 * (i % kChunks), p.max_rank - 8);
    };
    auto load_v = [&](Parts& v, const float* at) LG_INLINE {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                v.w[s][e] = *reinterpret_cast<const float4_t*>(at + min(s, p.parts - 1) * part + 4 * e);
    };
    Parts v;
    load_v(v, v_at(threadIdx.x));
    load_base(even, min(n0, p.n - 1));
    if (named) rank = max(0, min(__builtin_amdgcn_readfirstlane(raw_rank), p.max_rank));
    if (rank == 0 && p.base == p.out) return;
    if (rank > 0) {
        load_b(n0);
        for (int i = threadIdx.x; i < kRows * kChunks; i += 256) {
            const int row = i / kChunks, chunk = i % kChunks, r = 8 * chunk;
            if (i >= 256) load_v(v, v_at(i));
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = 0.0f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (s < p.parts) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[e] += v.w[s][e >> 2][e & 3];
                }
            for (int s = 4; s < p.parts; ++s) {
                const float4_t* src = reinterpret_cast<const float4_t*>(v_at(i) + s * part);
                const float4_t u0 = src[0], u1 = src[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    u[e] += u0[e];
                    u[4 + e] += u1[e];
                }
            }
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                u[e] = row < left && r + e < rank ? u[e] * scale : 0.0f;
                top = fmaxf(top, fabsf(u[e]));
            }
#pragma unroll
            for (int m = 1; m < kChunks; m *= 2) top = fmaxf(top, shfl_xor_f32(top, m));
            // 2^-e of the largest value's exponent e, as far as fp32 has it
            const int ex = (int)(__float_as_uint(top) >> 23);
            const int down = ex < 1 ? 1 : ex > 253 ? 253 : ex;
            const float shrink = __uint_as_float((unsigned)(254 - down) << 23);
            if (chunk == 0) growth[row] = __uint_as_float((unsigned)down << 23);
            typedef typename T::elem elem;
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] *= shrink;
#pragma unroll
            for (int k = 0; k < TERMS; ++k) {
                uint4_t w;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    w[e >> 1] = T::pack2(u[e], u[e + 1]);
                    u[e] -= (float)__builtin_bit_cast(elem, (unsigned short)(w[e >> 1] & 0xffffu));
                    u[e + 1] -= (float)__builtin_bit_cast(elem, (unsigned short)(w[e >> 1] >> 16));
                    u[e] = u[e] == u[e] ? u[e] : 0.0f;  // (an infinity is in its first term, with nothing left)
                    u[e + 1] = u[e + 1] == u[e + 1] ? u[e + 1] : 0.0f;
                }
                operand[(((row >> 4) * RS + (chunk >> 2)) * TERMS + k) * 64 + (chunk & 3) * 16 + (row & 15)] = w;
            }
        }
        __syncthreads();
    }
    float grow[MT];
    uint4_t keep[RS];  // (the columns of B that count)
    // One step over the base `w`; WHOLE: of whole tiles, and the next one's B is asked for.
    auto compute = [&](auto adds_c, auto whole_c, uint4_t(&w)[MT][kBase], int at_n, int next_n) LG_INLINE {
        constexpr bool ADDS = decltype(adds_c)::value != 0, WHOLE = decltype(whole_c)::value != 0;
        float4_t acc[MT][4];
        if (ADDS) {
            asm volatile("" ::: "memory");  // (the terms are read again: kept over the steps they would not fit)
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) bv[s][j] &= keep[s];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < RS; ++s)
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
                        const uint4_t v = operand[((m * RS + s) * TERMS + k) * 64 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[m][j] = T::mfma16(bv[s][j], v, acc[m][j]);
                    }
            }
            if (WHOLE) {
                __builtin_amdgcn_sched_barrier(0);  // (into the registers that the products just read)
                load_b(next_n);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (!WHOLE && 16 * m + c >= left) continue;
            const unsigned row = (unsigned)(16 * m + c) * (unsigned)p.out_stride;
#pragma unroll
            for (int e = 0; e < kBase; ++e) {
                const int n = at_n + (F32 ? 16 * e + 4 * q : 32 * e + 8 * q);
                if (!WHOLE && n >= p.n) continue;
                uint4_t o = w[m][e];
                if constexpr (!ADDS) {
                } else if constexpr (F32) {
                    float4_t y = __builtin_bit_cast(float4_t, o);
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = fmaf(acc[m][e][i], grow[m], y[i]);
                    o = __builtin_bit_cast(uint4_t, y);
                } else {
                    const auto u = __builtin_bit_cast(typename T::vec8, o);
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        y[i] = fmaf(acc[m][2 * e + (i >> 2)][i & 3], grow[m], (float)u[i]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = T::pack2(y[2 * i], y[2 * i + 1]);
                }
                *reinterpret_cast<uint4_t*>(out + (row + (unsigned)n) * (unsigned)kSize) = o;
            }
        }
    };
    if (rank > 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) grow[m] = growth[16 * m + c];
#pragma unroll
        for (int s = 0; s < RS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 32 * s + 8 * q + 2 * i;
                keep[s][i] = rank >= r + 2 ? ~0u : rank == r + 1 ? 0xffffu : 0u;
            }
        if (left == kRows && n_last % 64 == 0) {
            // Straight-line code, two steps a turn: a condition around a load or a store would make every wait one for
            // everything in flight.  (The last step asks for itself again.)
            const int end = n0 < n_last ? n0 + (n_last - 1 - n0) / 256 * 256 : 0;
            while (n0 < n_last) {
                int next = min(n0 + 256, end);
                load_base(odd, next);
                compute(ic<1>{}, ic<1>{}, even, n0, next);
                n0 += 256;
                if (n0 >= n_last) break;
                next = min(n0 + 256, end);
                load_base(even, next);
                compute(ic<1>{}, ic<1>{}, odd, n0, next);
                n0 += 256;
            }
        } else {
            while (n0 < n_last) {
                compute(ic<1>{}, ic<0>{}, even, n0, 0);
                n0 += 256;
                if (n0 >= n_last) break;
                load_base(even, n0);
                load_b(n0);
            }
        }
    } else {
        while (n0 < n_last) {
            compute(ic<0>{}, ic<0>{}, even, n0, 0);
            n0 += 256;
            if (n0 < n_last) load_base(even, n0);
        }
    }
}

template <typename T, int MT, int RT>
static hipError_t adapter_down(AdapterParams p, hipStream_t stream) {
    const int64_t tiles = packed_tiles(p.total, p.num_seqs, 1, 16 * MT);
    const unsigned z = (unsigned)(p.max_rank + 16 * RT - 1) / (16 * RT);
    adapter_down_kernel<T, MT, RT><<<dim3((unsigned)(tiles * p.parts), z), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, bool F32, int MT, int RS>
static hipError_t adapter_up(AdapterParams p, hipStream_t stream) {
    constexpr int kTerms = F32 && std::is_same<T, PackedBf16>::value ? 3 : 2;
    const int64_t tiles = packed_tiles(p.total, p.num_seqs, 1, 16 * MT);
    // a workgroup takes 256 outputs, and more as long as there are eight workgroups per compute unit
    const int64_t steps = (p.n + 255) / 256;
    const int64_t per = std::max<int64_t>(1, std::min(steps, tiles * steps / (8 * device_cu_count())));
    p.n_slice = (int)per * 256;
    p.slices = (int)((steps + per - 1) / per);
    adapter_up_kernel<T, F32, kTerms, MT, RS><<<(unsigned)(tiles * p.slices), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, bool F32>
static hipError_t adapter_up_by_rank(const AdapterParams& p, bool long_seqs, hipStream_t stream) {
    constexpr int kLong = F32 ? 2 : 4;  // (what fits the registers twice: this step's and the next one's)
    if (p.max_rank <= 32) return long_seqs ? adapter_up<T, F32, kLong, 1>(p, stream) : adapter_up<T, F32, 1, 1>(p, stream);
    if (p.max_rank <= 64) return long_seqs ? adapter_up<T, F32, kLong, 2>(p, stream) : adapter_up<T, F32, 1, 2>(p, stream);
    if (p.max_rank <= 128) return !F32 && long_seqs ? adapter_up<T, F32, F32 ? 1 : 2, 4>(p, stream) : adapter_up<T, F32, 1, 4>(p, stream);
    return adapter_up<T, F32, 1, 8>(p, stream);
}

template <typename T>
static hipError_t adapter_launch(AdapterParams p, bool f32, hipStream_t stream) {
    const bool long_seqs = p.total >= 32 * (int64_t)p.num_seqs;
    const int steps = (p.k + 31) / 32, mt = long_seqs ? 4 : 1;
    const int rt = !long_seqs || p.max_rank <= 16 ? 1 : p.max_rank <= 32 ? 2 : 4;
    // K parts: two workgroups per compute unit, and steps for four waves
    const int64_t groups = packed_tiles(p.total, p.num_seqs, 1, 16 * mt) * ((p.max_rank + 16 * rt - 1) / (16 * rt));
    int parts = 1;  // (at most four for the loads of one round)
    while (parts < kAdapterMaxParts && groups * parts < 2 * device_cu_count() && steps >= 16 * parts) parts *= 2;
    p.parts = parts;
    p.part_steps = (steps + parts - 1) / parts;
    hipError_t rc;
    if (!long_seqs) rc = adapter_down<T, 1, 1>(p, stream);
    else if (rt == 1) rc = adapter_down<T, 4, 1>(p, stream);
    else if (rt == 2) rc = adapter_down<T, 4, 2>(p, stream);
    else rc = adapter_down<T, 4, 4>(p, stream);
    if (rc != hipSuccess) return rc;
    return f32 ? adapter_up_by_rank<T, true>(p, long_seqs, stream) : adapter_up_by_rank<T, false>(p, long_seqs, stream);
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
    if (n > (1 << 22) || k > (1 << 22)) return reject(msg, cap, "n and k must be at most %d (%d, %d)", 1 << 22, n, k);
    if (base_stride > (1 << 22) || out_stride > (1 << 22))
        return reject(msg, cap, "base and out strides must be at most %d (%d, %d)", 1 << 22, base_stride, out_stride);
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
