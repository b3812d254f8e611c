// Low-rank adapters of many requests beside a shared projection:
//
//   out[t][:] = base[t][:] + s_a * (x[t] . A_a^T) . B_a^T,   a = the adapter of the row's sequence
//
// Two launches (one for few rows).  The first takes a tile of one sequence's rows through A: v = x . A^T in fp32 into the
// workspace, in K parts (v is small; adding the parts up is the second launch's first step, in their order).  The second
// takes the same rows through B and adds the base.  Products on the matrix cores.
//
// s v has to be an operand of the second product, so it is split into 16-bit terms: per row scaled by a power
// of two that brings its largest value to where the type has most room (exact, and undone in the fp32 result; fp16 could not hold
// the values as they are), then the rounded value and what the rounding left.  Outputs of 16 bits: two terms,
// 22 bits for fp16's 11, 16 for bf16's 8; fp32 outputs: three, all 24 bits.
//
// Bound by memory: x, base and out once, A and B of the adapters in use.  16 prompts of 512 x 4096, rank 64, 24576 outputs in 16
// bits: 900 MB in 229 us, 3.9 TB/s (a large copy 5.2; the first launch 26 us, the second 203: its beginnings, and
// products and vector work that the memory time does not all cover; rank 32 192 us); 13 single rows and 5 chunks of 31 to 600, 8960 columns to 1536 in
// fp32: 54 MB in 22 us; 32 single rows on 8 adapters, 4096 to 6144: 10.5 us, a chain of dependent loads.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"
#include "q4_common.hpp"

#include <math.h>

#include <algorithm>

namespace lg {

constexpr int kAdapterMaxRank = 256;
constexpr int kAdapterMaxParts = 8;   // K parts of v, read four at a time
constexpr int kAdapterUnits = 256;    // compute units that K is dealt out to, at most

// K parts that `groups` workgroups of the first product are wanted in, two per compute unit.
inline int adapter_parts(int64_t groups, int units) {
    int parts = 1;
    while (parts < kAdapterMaxParts && groups * parts < 2 * units) parts *= 2;
    return parts;
}
// More than one part is made only while groups * parts / 2 < 2 * units, and a group is at most 64 rows by 64 ranks: rows * ranks * parts
// stay below this.
constexpr int64_t kAdapterPartElements = 4 * kAdapterUnits * 64 * 64;

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
    int n_slice, slices;    // outputs of a workgroup, whole steps of its waves; how many of them
};

__device__ __forceinline__ int adapter_rank(const AdapterParams& p, int adapter) {
    if (adapter < 0 || adapter >= p.adapters) return 0;
    const int r = __builtin_amdgcn_readfirstlane(p.ranks[adapter]);
    return r < 0 ? 0 : r < p.max_rank ? r : p.max_rank;
}

// A matrix operand (16 rows of 32 elements: lane (c, q) = row c, elements 8 q .. + 7) out of rows in memory.  Loaded as it
// is used, neighbouring lanes ask for different rows, and 16 bytes from each of 64 rows take four times as long as 64 bytes from
// each of 16 (measured in L2: 38 against 153 bytes per ns and compute unit, whatever the rows' distance).  So lane l loads
// chunk operand_chunk() of row l / 4, and the values change lanes through 1 KB of LDS that belongs to the wave; the
// chunks' order differs from row to row so that both ways touch every bank once.
__device__ __forceinline__ int operand_row() { return (threadIdx.x & 63) >> 2; }
__device__ __forceinline__ int operand_chunk() { return (threadIdx.x & 3) ^ ((threadIdx.x >> 4) & 3); }
__device__ __forceinline__ uint4_t operand_of(uint4_t loaded, uint4_t* scratch) {
    const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    scratch[lane] = loaded;
    __builtin_amdgcn_wave_barrier();
    const uint4_t v = scratch[4 * c + (q ^ (c >> 2))];
    __builtin_amdgcn_wave_barrier();
    return v;
}

// v[part][t][r] = sum over the part's columns of x[t][c] * A[r][c].  grid (tiles of 16 MT rows by K parts, 16 RT ranks
// each); the four waves share the part's steps of 32 columns and add up in LDS.
template <typename T, int MT, int RT>
__global__ __launch_bounds__(256, 2) void adapter_down_kernel(const AdapterParams p) {
    constexpr int kDeep = MT > 1 ? 4 : 8;  // steps asked for together, side by side: whole cache lines
    constexpr int kSlots = MT * RT > 4 ? MT * RT : 4;  // (1 KB each, on their way to the sums the operands' scratch)
    __shared__ __attribute__((aligned(16))) float sums[4][kSlots * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint4_t* const scratch = reinterpret_cast<uint4_t*>(sums[wave]);
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
    for (int m = 0; m < MT; ++m)
        x[m] = p.x + (int64_t)(t.row0 + min(r0 + 16 * m + operand_row(), t.rows - 1)) * p.x_stride;
#pragma unroll
    for (int i = 0; i < RT; ++i)
        a[i] = p.a + ((int64_t)t.of * p.max_rank + min(rank0 + 16 * i + operand_row(), p.max_rank - 1)) * p.k;
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
            const int want = 32 * (s0 + d) + 8 * operand_chunk();
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
                const bool in = s0 + d < last && 32 * (s0 + d) + 8 * operand_chunk() < p.k;
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[d][m] = in ? xv[d][m] : uint4_t{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < RT; ++i) av[d][i] = in ? av[d][i] : uint4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
                xv[d][m] = operand_of(xv[d][m], scratch + (d * (MT + RT) + m) % kSlots * 64);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const uint4_t av_of = operand_of(av[d][i], scratch + (d * (MT + RT) + MT + i) % kSlots * 64);
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][i] = T::mfma16(av_of, xv[d][m], acc[m][i]);
            }
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

// Where the terms' type has the row's largest value, as a power of two.  fp16 ends at 2^16 and loses bits below 2^-14: up there two terms
// are off by 2^-22 of every rank down to 2^-17 of the largest, three hold all of every rank down to 2^-15 of it, and what
// lies below is off by 2^-39 of the largest.  (With the largest at 1, by 2^-25 of
// it: a rank 2^-18 below it by 5.6 half steps of fp16, which show in every output whose B is small at the largest.)
//
// bf16 has the exponents of fp32, and so may B: with the largest below 2^-11, sums over 256 ranks of values up to 2^128 stay below that, so
// that what is finite in the result is finite on the way.
template <typename T>
constexpr int kAdapterTop = -12;
template <>
constexpr int kAdapterTop<PackedF16> = 14;

// Eight ranks u of a row (from rank r on), the chunks of a row in neighbouring lanes: times the adapter's scale, zero behind the
// rank and the rows, brought by a power of two to where the row's largest value lies in [2^kAdapterTop, twice that), split into terms of
// the operand's type, 64 words of four apart.  growth: what undoes the power of two.
template <typename T, int TERMS, int CHUNKS>
__device__ __forceinline__ void adapter_terms(float (&u)[8], bool live, int r, int rank, float scale, float* growth,
                                              uint4_t* operand) {
    typedef typename T::elem elem;
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        u[e] = live && r + e < rank ? u[e] * scale : 0.0f;
        top = fmaxf(top, fabsf(u[e]));
    }
#pragma unroll
    for (int m = 1; m < CHUNKS; m *= 2) top = fmaxf(top, shfl_xor_f32(top, m));
    const int ex = (int)(__float_as_uint(top) >> 23);  // (as far as fp32 has the power of two)
    constexpr int kTop = kAdapterTop<T>, kLow = std::max(1, 1 + kTop), kHigh = std::min(254, 253 + kTop);
    const int down = ex < kLow ? kLow : ex > kHigh ? kHigh : ex;
    const float shrink = __uint_as_float((unsigned)(254 + kTop - down) << 23);
    if (r == 0) *growth = __uint_as_float((unsigned)(down - kTop) << 23);
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
        operand[64 * k] = w;
    }
}

// Which of the eight columns of B from r on lie in front of the rank.
__device__ __forceinline__ uint4_t adapter_keep(int r, int rank) {
    uint4_t keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[i] = rank >= r + 2 * i + 2 ? ~0u : rank == r + 2 * i + 1 ? 0xffffu : 0u;
    return keep;
}

// Four outputs of a row: fp32 or two to a word.
template <bool F32>
struct Four {
    typedef uint2_t bits;
};
template <>
struct Four<true> {
    typedef uint4_t bits;
};
// The base's and the sums that belong to them, element e of the tiles.
template <typename T, bool F32>
__device__ __forceinline__ typename Four<F32>::bits adapter_sum(typename Four<F32>::bits base, const float4_t (&acc)[4], int e,
                                                                float grow) {
    if constexpr (F32) {
        float4_t y = __builtin_bit_cast(float4_t, base);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fmaf(acc[j][e], grow, y[j]);
        return __builtin_bit_cast(uint4_t, y);
    } else {
        typedef typename T::elem elem;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[j] = fmaf(acc[j][e], grow,
                        (float)__builtin_bit_cast(elem, (unsigned short)(j & 1 ? base[j >> 1] >> 16 : base[j >> 1] & 0xffffu)));
        return uint2_t{T::pack2(y[0], y[1]), T::pack2(y[2], y[3])};
    }
}

// out = base + (s v) . B^T.  grid: slices of the outputs (fastest: a slice of B then stays in the L2 of the XCDs that
// take it, for all rows of its adapter) by tiles of 16 MT GROUPS rows; ranks in RS steps of 32.  The workgroup splits
// s v into terms once, in the order of the matrix operand, into LDS.  A wave takes 16 MT rows by four tiles of 16 outputs at
// a time; GROUPS of the four waves lie one below the other (and read the same B), the others side by side.
//
// The rows are the rows of the product and the outputs its columns, output 4 c + j being column c of tile j: a lane then
// holds four outputs side by side of four rows, and the 16 lanes next to it those around them.
template <typename T, bool F32, int TERMS, int MT, int RS, int GROUPS>
__global__ __launch_bounds__(256, 2) void adapter_up_kernel(const AdapterParams p) {
    constexpr int kRows = 16 * MT * GROUPS, kChunks = 4 * RS;  // rows of a tile, chunks of eight ranks
    constexpr int kTiles = 4, kSize = F32 ? 4 : 2, kAcross = 16 * kTiles * (4 / GROUPS);
    typedef typename Four<F32>::bits four;
    __shared__ uint4_t operand[MT * GROUPS * RS * TERMS * 64];
    __shared__ __attribute__((aligned(16))) float growth[kRows];
    __shared__ uint4_t scratches[4][kTiles][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    const int group = wave % GROUPS;
    uint4_t(&scratch)[kTiles][64] = scratches[wave];
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
    const int my_row = 16 * MT * group + 4 * q;  // (16 m + e: the rows of this lane)
    const int n_last = (slice + 1) * p.n_slice < p.n ? (slice + 1) * p.n_slice : p.n;
    int n0 = slice * p.n_slice + 16 * kTiles * (wave / GROUPS);
    // (rows behind the tile's last, outputs behind the last and ranks behind the rank: others in their place, which count
    // for nothing -- a load under a condition of its own is a branch around it.  Offsets from the tile's first row and the
    // adapter's B have 32 bits.)
    // (B is asked for a step ahead, as soon as the products of the step before with these ranks are done; more than 64 ranks do not
    // fit and come 32 at a time)
    constexpr int kHeld = RS <= 2 ? RS : 1;
    four even[MT][4], odd[MT][4];
    uint4_t bv[kHeld][kTiles];
    const char* const base = static_cast<const char*>(p.base) + row0 * p.base_stride * kSize;
    char* const out = static_cast<char*>(p.out) + row0 * p.out_stride * kSize;
    const char* const b = reinterpret_cast<const char*>(p.b + (int64_t)(named ? t.of : 0) * p.n * p.max_rank);
    // (WHOLE: everything is there, and one offset per lane serves all rows)
    const unsigned base_lane = ((unsigned)my_row * (unsigned)p.base_stride + 4u * (unsigned)c) * (unsigned)kSize;
    auto load_base = [&](auto whole_c, four(&w)[MT][4], int at_n) LG_INLINE {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (decltype(whole_c)::value != 0) {
                    w[m][e] = *reinterpret_cast<const four*>(
                        base + ((int64_t)(16 * m + e) * p.base_stride + at_n) * kSize + base_lane);
                } else {
                    const unsigned row = (unsigned)min(my_row + 16 * m + e, left - 1);
                    const unsigned n = (unsigned)min(at_n + kTiles * c, p.n - kTiles);
                    w[m][e] = *reinterpret_cast<const four*>(base + (row * (unsigned)p.base_stride + n) * (unsigned)kSize);
                }
            }
    };
    int rank = 0;
    const unsigned b_lane = (unsigned)(kTiles * operand_row()) * (unsigned)p.max_rank * 2u;
    auto load_b = [&](auto whole_c, int at_n, int s) LG_INLINE {
        const int r = 32 * s + 8 * operand_chunk();
        const unsigned chunk = (unsigned)(r < rank ? r : 0) * 2u;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            if constexpr (decltype(whole_c)::value != 0) {
                bv[s % kHeld][j] = *reinterpret_cast<const uint4_t*>(b + (int64_t)(at_n + j) * p.max_rank * 2 + (b_lane + chunk));
            } else {
                const unsigned n = (unsigned)min(at_n + kTiles * operand_row() + j, p.n - 1);
                bv[s % kHeld][j] = *reinterpret_cast<const uint4_t*>(b + (n * (unsigned)p.max_rank * 2u + chunk));
            }
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
    auto load_v = [&](Parts& v, const float* at, int s0) LG_INLINE {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                v.w[s][e] = *reinterpret_cast<const float4_t*>(at + min(s0 + s, p.parts - 1) * part + 4 * e);
    };
    Parts v;
    load_v(v, v_at(threadIdx.x), 0);
    load_base(ic<0>{}, even, n0);
    if (named) rank = max(0, min(__builtin_amdgcn_readfirstlane(raw_rank), p.max_rank));
    if (rank == 0 && p.base == p.out) return;
    if (rank > 0) {
#pragma unroll
        for (int s = 0; s < kHeld; ++s) load_b(ic<0>{}, n0, s);
        for (int i = threadIdx.x; i < kRows * kChunks; i += 256) {
            const int row = i / kChunks, chunk = i % kChunks, r = 8 * chunk;
            if (i >= 256) load_v(v, v_at(i), 0);
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = 0.0f;
            auto add_v = [&](int s0) LG_INLINE {
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    if (s0 + s < p.parts) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) u[e] += v.w[s][e >> 2][e & 3];
                    }
            };
            add_v(0);
            if (p.parts > 4) {
                load_v(v, v_at(i), 4);
                add_v(4);
            }
            adapter_terms<T, TERMS, kChunks>(
                u, row < left, r, rank, scale, &growth[row],
                &operand[((row >> 4) * RS + (chunk >> 2)) * TERMS * 64 + (chunk & 3) * 16 + (row & 15)]);
        }
        __syncthreads();
    }
    uint4_t keep[RS];
    const unsigned out_lane = ((unsigned)my_row * (unsigned)p.out_stride + 4u * (unsigned)c) * (unsigned)kSize;
    // One step over the base `w`; WHOLE: of whole tiles, and the next one's B is asked for.
    auto compute = [&](auto adds_c, auto whole_c, four(&w)[MT][4], int at_n, int next_n) LG_INLINE {
        constexpr bool ADDS = decltype(adds_c)::value != 0, WHOLE = decltype(whole_c)::value != 0;
        float4_t acc[MT][kTiles];
        if (ADDS) {
            asm volatile("" ::: "memory");  // (terms and growth are read again: kept over the steps they cost a wave its place)
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                uint4_t(&w_b)[kTiles] = bv[s % kHeld];
                uint4_t term[MT][TERMS];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int k = 0; k < TERMS; ++k)
                        term[m][k] = operand[(((group * MT + m) * RS + s) * TERMS + k) * 64 + lane];
#pragma unroll
                for (int j = 0; j < kTiles; ++j) w_b[j] = operand_of(w_b[j] & keep[s], scratch[j]);
#pragma unroll
                for (int k = 0; k < TERMS; ++k)  // (the sums of a tile and row group as far apart as they can be)
#pragma unroll
                    for (int j = 0; j < kTiles; ++j)
#pragma unroll
                        for (int m = 0; m < MT; ++m) acc[m][j] = T::mfma16(term[m][k], w_b[j], acc[m][j]);
                if (s + kHeld < RS) load_b(whole_c, at_n, s + kHeld);
                else if (WHOLE) load_b(whole_c, next_n, (s + kHeld) % RS);
                __builtin_amdgcn_sched_barrier(0);  // (into the registers that the products just read)
            }
        }
        if (!WHOLE && at_n + kTiles * c >= p.n) return;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float4_t grow;
            if (ADDS) grow = *reinterpret_cast<const float4_t*>(&growth[my_row + 16 * m]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!WHOLE && my_row + 16 * m + e >= left) continue;
                four o = w[m][e];
                if constexpr (ADDS) o = adapter_sum<T, F32>(o, acc[m], e, grow[e]);
                *reinterpret_cast<four*>(out + ((int64_t)(16 * m + e) * p.out_stride + at_n) * kSize + out_lane) = o;
            }
        }
    };
    if (rank > 0) {
#pragma unroll
        for (int s = 0; s < RS; ++s) keep[s] = adapter_keep(32 * s + 8 * operand_chunk(), rank);
        if (left >= 16 * MT * (group + 1) && n_last % (16 * kTiles) == 0) {
            // Straight-line code, two steps a turn: a condition around a load or a store would make every wait one for
            // everything in flight.  (The last step asks for itself again.)
            const int end = n0 < n_last ? n0 + (n_last - 1 - n0) / kAcross * kAcross : 0;
            while (n0 < n_last) {
                int next = min(n0 + kAcross, end);
                load_base(ic<1>{}, odd, next);
                compute(ic<1>{}, ic<1>{}, even, n0, next);
                n0 += kAcross;
                if (n0 >= n_last) break;
                next = min(n0 + kAcross, end);
                load_base(ic<1>{}, even, next);
                compute(ic<1>{}, ic<1>{}, odd, n0, next);
                n0 += kAcross;
            }
        } else {
            while (n0 < n_last) {
                compute(ic<1>{}, ic<0>{}, even, n0, 0);
                n0 += kAcross;
                if (n0 >= n_last) break;
                load_base(ic<0>{}, even, n0);
#pragma unroll
                for (int s = 0; s < kHeld; ++s) load_b(ic<0>{}, n0, s);
            }
        }
    } else {
        while (n0 < n_last) {
            compute(ic<0>{}, ic<0>{}, even, n0, 0);
            n0 += kAcross;
            if (n0 < n_last) load_base(ic<0>{}, even, n0);
        }
    }
}

// Few rows: both products in one launch.  Every workgroup takes its tile of 16 rows through all of A by itself (sixteen waves
// share the steps of K) and then sixteen waves' outputs, tiles as in adapter_up_kernel: A is read once per 1024
// outputs, from L2, which for a handful of tiles costs less than a second launch.
template <typename T, bool F32, int TERMS, int RT>
__global__ __launch_bounds__(1024) void adapter_small_kernel(const AdapterParams p) {
    constexpr int kWaves = 16, kDeep = RT == 1 ? 8 : RT == 2 ? 4 : 2, RS = RT > 2 ? 2 : 1, kChunks = 4 * RS;
    constexpr int kTiles = 4, kSize = F32 ? 4 : 2, kAcross = 16 * kTiles * kWaves, kSlots = 4;
    typedef typename Four<F32>::bits four;
    static_assert(RT <= kSlots, "the sums fit the slots of 1 KB");
    __shared__ __attribute__((aligned(16))) float sums[kWaves][kSlots * 256];
    __shared__ uint4_t operand[RS * TERMS * 64];
    __shared__ __attribute__((aligned(16))) float growth[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    uint4_t* const scratch = reinterpret_cast<uint4_t*>(sums[wave]);
    const int slice = (int)(blockIdx.x % (unsigned)p.slices);
    const PackedTile t = packed_tile<true>(p.cu, p.num_seqs, p.total, 1, 16, (int)(blockIdx.x / (unsigned)p.slices),
                                           p.adapter_of_seq);
    const int r0 = t.tile * 16;
    if (r0 >= t.rows) return;
    const bool named = t.of >= 0 && t.of < p.adapters;
    if (!named && p.base == p.out) return;
    const int raw_rank = p.ranks[named ? t.of : 0];
    const float scale = p.scales[named ? t.of : 0];
    const int left = t.rows - r0 < 16 ? t.rows - r0 : 16;
    const int64_t row0 = t.row0 + r0;
    const int n0 = slice * kAcross + 16 * kTiles * wave, n = n0 + kTiles * c;
    int rank = 0;
    // (base and B: what lies behind the rank is masked where it is used)
    four base[4];
    uint4_t bv[RS][kTiles];
    const char* const base_rows = static_cast<const char*>(p.base) + (row0 * p.base_stride + min(n, p.n - kTiles)) * kSize;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        base[e] = *reinterpret_cast<const four*>(
            base_rows + (unsigned)min(4 * q + e, left - 1) * (unsigned)p.base_stride * (unsigned)kSize);
    const unsigned short* const b = p.b + (int64_t)(named ? t.of : 0) * p.n * p.max_rank;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int s = 0; s < RS; ++s)
            bv[s][j] = *reinterpret_cast<const uint4_t*>(b + (int64_t)min(n0 + kTiles * operand_row() + j, p.n - 1) * p.max_rank +
                                                         min(32 * s + 8 * operand_chunk(), p.max_rank - 8));
    if (named) {
        const unsigned short* const x = p.x + (row0 + min(operand_row(), left - 1)) * p.x_stride;
        const unsigned short* a[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
            a[i] = p.a + ((int64_t)t.of * p.max_rank + min(16 * i + operand_row(), p.max_rank - 1)) * p.k;
        const int last = (p.k + 31) / 32;
        float4_t acc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        // (columns behind the last: the last ones, taken as zeros)
        for (int s0 = wave * kDeep; s0 < last; s0 += kWaves * kDeep) {
            uint4_t xv[kDeep], av[kDeep][RT];
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                const int at = min(32 * (s0 + d) + 8 * operand_chunk(), p.k - 8);
                xv[d] = *reinterpret_cast<const uint4_t*>(x + at);
#pragma unroll
                for (int i = 0; i < RT; ++i) av[d][i] = *reinterpret_cast<const uint4_t*>(a[i] + at);
            }
            __builtin_amdgcn_sched_barrier(0);  // (all of them, then the products)
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                const bool in = 32 * (s0 + d) + 8 * operand_chunk() < p.k;
                const uint4_t xf = operand_of(in ? xv[d] : uint4_t{0, 0, 0, 0}, scratch + d * (1 + RT) % kSlots * 64);
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i] = T::mfma16(operand_of(in ? av[d][i] : uint4_t{0, 0, 0, 0},
                                                  scratch + (d * (1 + RT) + 1 + i) % kSlots * 64), xf, acc[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) *reinterpret_cast<float4_t*>(&sums[wave][(i * 64 + lane) * 4]) = acc[i];
        rank = max(0, min(__builtin_amdgcn_readfirstlane(raw_rank), p.max_rank));
    }
    if (rank == 0 && p.base == p.out) return;
    if (rank > 0) {
        __syncthreads();
        if (threadIdx.x < 16 * kChunks) {
            const int row = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks;
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = 0.0f;
            if (8 * chunk < 16 * RT) {
#pragma unroll
                for (int w = 0; w < kWaves; ++w)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float4_t v = *reinterpret_cast<const float4_t*>(
                            &sums[w][((chunk >> 1) * 64 + (2 * (chunk & 1) + g) * 16 + row) * 4]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) u[4 * g + e] += v[e];
                    }
            }
            adapter_terms<T, TERMS, kChunks>(u, row < left, 8 * chunk, rank, scale, &growth[row],
                                             &operand[(chunk >> 2) * TERMS * 64 + (chunk & 3) * 16 + row]);
        }
        __syncthreads();
    }
    float4_t acc[kTiles];
    float4_t grow = {0.0f, 0.0f, 0.0f, 0.0f};
    if (rank > 0) {
        grow = *reinterpret_cast<const float4_t*>(&growth[4 * q]);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            acc[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                const uint4_t f = operand_of(bv[s][j] & adapter_keep(32 * s + 8 * operand_chunk(), rank), scratch + j * 64);
#pragma unroll
                for (int k = 0; k < TERMS; ++k) acc[j] = T::mfma16(operand[(s * TERMS + k) * 64 + lane], f, acc[j]);
            }
        }
    }
    if (n >= p.n) return;
    char* const out_rows = static_cast<char*>(p.out) + (row0 * p.out_stride + n) * kSize;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (4 * q + e >= left) continue;
        const four o = rank > 0 ? adapter_sum<T, F32>(base[e], acc, e, grow[e]) : base[e];
        *reinterpret_cast<four*>(out_rows + (unsigned)(4 * q + e) * (unsigned)p.out_stride * (unsigned)kSize) = o;
    }
}

template <typename T, int MT, int RT>
static hipError_t adapter_down(AdapterParams p, hipStream_t stream) {
    const int64_t tiles = packed_tiles(p.total, p.num_seqs, 1, 16 * MT);
    const unsigned z = (unsigned)(p.max_rank + 16 * RT - 1) / (16 * RT);
    adapter_down_kernel<T, MT, RT><<<dim3((unsigned)(tiles * p.parts), z), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, bool F32, int MT, int RS, int GROUPS>
static hipError_t adapter_up(AdapterParams p, hipStream_t stream) {
    constexpr int kTerms = F32 ? 3 : 2;
    constexpr int kAcross = 64 * (4 / GROUPS);
    const int64_t tiles = packed_tiles(p.total, p.num_seqs, 1, 16 * MT * GROUPS);
    // A workgroup takes one step of outputs, and more as long as there are sixteen workgroups per compute unit: more of them spend
    // more on their beginnings, fewer stream worse (8192 rows x 24576 outputs, rank 64: 8 per unit 228 us, 16 215, 32 227).
    const int64_t steps = (p.n + kAcross - 1) / kAcross;
    const int64_t per = std::max<int64_t>(1, std::min(steps, tiles * steps / (16 * device_cu_count())));
    p.n_slice = (int)per * kAcross;
    p.slices = (int)((steps + per - 1) / per);
    adapter_up_kernel<T, F32, kTerms, MT, RS, GROUPS><<<(unsigned)(tiles * p.slices), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, bool F32>
static hipError_t adapter_up_by_rank(const AdapterParams& p, bool long_seqs, hipStream_t stream) {
    if (p.max_rank <= 32) return long_seqs ? adapter_up<T, F32, 2, 1, 2>(p, stream) : adapter_up<T, F32, 1, 1, 1>(p, stream);
    if (p.max_rank <= 64) return long_seqs ? adapter_up<T, F32, 2, 2, 2>(p, stream) : adapter_up<T, F32, 1, 2, 1>(p, stream);
    if (p.max_rank <= 128) return long_seqs ? adapter_up<T, F32, 1, 4, 2>(p, stream) : adapter_up<T, F32, 1, 4, 1>(p, stream);
    return adapter_up<T, F32, 1, 8, 1>(p, stream);
}

template <typename T, bool F32>
static hipError_t adapter_small(AdapterParams p, hipStream_t stream) {
    constexpr int kTerms = F32 ? 3 : 2;
    p.slices = (p.n + 1023) / 1024;
    const unsigned grid = (unsigned)(packed_tiles(p.total, p.num_seqs, 1, 16) * p.slices);
    if (p.max_rank <= 16) adapter_small_kernel<T, F32, kTerms, 1><<<grid, 1024, 0, stream>>>(p);
    else if (p.max_rank <= 32) adapter_small_kernel<T, F32, kTerms, 2><<<grid, 1024, 0, stream>>>(p);
    else adapter_small_kernel<T, F32, kTerms, 4><<<grid, 1024, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T>
static hipError_t adapter_launch(AdapterParams p, bool f32, hipStream_t stream) {
    // One launch where a workgroup reads little of A: in a graph it takes about as long as two (us, one row: rank 16 of 4096 to
    // 4096 7.8 / 6.9; 32 of 896 to 896 6.0 / 6.4; 32 of 4096 9.0 / 7.3), launched one by one a call costs the host 3.4 us less.
    if (p.max_rank <= 64 && (int64_t)p.max_rank * p.k <= 65536 &&
        packed_tiles(p.total, p.num_seqs, 1, 16) * ((p.n + 1023) / 1024) <= device_cu_count())
        return f32 ? adapter_small<T, true>(p, stream) : adapter_small<T, false>(p, stream);
    const bool long_seqs = p.total >= 32 * (int64_t)p.num_seqs;
    const int steps = (p.k + 31) / 32, mt = long_seqs ? 4 : 1;
    const int rt = !long_seqs || p.max_rank <= 16 ? 1 : p.max_rank <= 32 ? 2 : 4;
    // K parts: two workgroups per compute unit, and steps for four waves
    const int64_t groups = packed_tiles(p.total, p.num_seqs, 1, 16 * mt) * ((p.max_rank + 16 * rt - 1) / (16 * rt));
    int parts = adapter_parts(groups, std::min(device_cu_count(), kAdapterUnits));
    while (parts > 1 && steps < 8 * parts) parts /= 2;
    p.parts = parts;
    p.part_steps = (steps + parts - 1) / parts;
    // Whole rounds of the four waves where fewer parts are then enough (us before / then: 35 steps in rounds of 16, parts 8 to 6, 22.9 /
    // 22.0; 4 prompts of 512, 8960 to 1536, rank 16, 19.6 / 16.9; 32 single rows, 4864 to 896, 8.2 / 7.2; at worst, one of 200, 1536
    // to 8960, rank 128, 14.5 / 15.0)
    const int round = long_seqs ? 16 : 32, whole = (p.part_steps + round - 1) / round * round;
    if ((steps + whole - 1) / whole < parts) {
        p.part_steps = whole;
        p.parts = (steps + whole - 1) / whole;
    }
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
    // (never less for more tokens or a larger rank: a caller sizes it once, for the largest batch)
    const uint64_t rows = (uint64_t)total_tokens * (uint64_t)max_rank, most = lg::kAdapterMaxParts * rows;
    return (size_t)std::max(rows, std::min<uint64_t>(most, lg::kAdapterPartElements)) * sizeof(float);
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
