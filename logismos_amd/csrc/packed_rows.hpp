// What the operators over packed rows share (attention, rotary positions, adapters, cache rows): the 16-bit
// element types with their matrix instructions, and the way from a workgroup to the rows it takes.
#pragma once

#include "device_utils.hpp"

namespace lg {

typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

// Element types: vectors of eight (a matrix operand), two values packed into a word (rounded to
// nearest even, one v_cvt_pk each), the matrix instructions with their fp32 sums.
struct PackedF16 {
    typedef _Float16 elem;
    typedef half8_t vec8;
    static __device__ __forceinline__ unsigned pack2(float a, float b) {
        return __builtin_bit_cast(unsigned, half2_t{(_Float16)a, (_Float16)b});
    }
    static __device__ __forceinline__ float16_t mfma32(uint4_t a, uint4_t b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a),
                                                      __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4_t mfma16(uint4_t a, uint4_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                      __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
};
struct PackedBf16 {
    typedef __bf16 elem;
    typedef bf16x8_t vec8;
    static __device__ __forceinline__ unsigned pack2(float a, float b) {
        return __builtin_bit_cast(unsigned, bf16x2_t{(__bf16)a, (__bf16)b});
    }
    static __device__ __forceinline__ float16_t mfma32(uint4_t a, uint4_t b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4_t mfma16(uint4_t a, uint4_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};

constexpr int kPackedMaxRows = 1 << 23;  // rows and sequences of a launch

// Packed sequences in tiles of `tile` units (a row is `per_row` units).  Only the device knows the
// lengths, so a launch has packed_tiles() workgroups, the most that can be needed, and sequence s
// owns those from floor(cu[s] * per_row / tile) + s on: ceil(b - a) <= floor(b) - floor(a) + 1, so the
// ranges never overlap, and at most one workgroup per sequence finds nothing to do.
inline int64_t packed_tiles(int64_t rows, int num_seqs, int64_t per_row, int64_t tile) {
    return rows * per_row / tile + num_seqs;
}

struct PackedTile {
    int seq;
    int row0;  // first row of the sequence
    int rows;  // its rows (0 or less: nothing to do)
    int tile;  // which of its tiles
    int of;    // of_seq[seq], where given
};

// The sequence of workgroup `b` and its tile: candidates by the whole wave, 64 per round, and in the last round every lane
// holds what there is to know about one of them (nothing is loaded twice: few rows are all latency).
// Whatever the lengths hold, rows lie in [0, total).
template <bool OF = false>
__device__ __forceinline__ PackedTile packed_tile(const int32_t* __restrict__ cu, int num_seqs, int total,
                                                  int per_row, int tile, int b,
                                                  const int32_t* __restrict__ of_seq = nullptr) {
    const int lane = threadIdx.x & 63;
    auto start = [&](int at, int s) LG_INLINE {
        return (int)((unsigned)at * (unsigned)per_row / (unsigned)tile) + s;
    };
    int lo = 0, n = num_seqs;
    while (n > 63) {
        const int step = (n + 63) / 64;
        const int at = lane * step < n ? lane * step : 0;
        const bool in = lane * step < n && start(cu[lo + at], lo + at) <= b;
        const int count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
        const int skip = (count > 0 ? count - 1 : 0) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    const int mine = lo + (lane < n ? lane : n);
    const int edge = cu[mine];
    int of = 0;
    if constexpr (OF) of = of_seq[mine < num_seqs ? mine : num_seqs - 1];
    const bool in = lane < n && start(edge, mine) <= b;
    int last = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
    last = __builtin_amdgcn_readfirstlane(last > 0 ? last - 1 : 0);
    const int r0 = __builtin_amdgcn_readlane(edge, last), r1 = __builtin_amdgcn_readlane(edge, last + 1);
    PackedTile t;
    t.seq = lo + last;
    t.row0 = r0;
    t.rows = r0 >= 0 && r0 < total ? (r1 < total ? r1 : total) - r0 : 0;
    t.tile = b - start(r0, t.seq);
    if (t.tile < 0) t.rows = t.tile = 0;  // (rows in front of the first sequence)
    t.of = OF ? __builtin_amdgcn_readlane(of, last) : 0;
    return t;
}

// The same in the order of the sequences' lengths, longest first, for up to kPackedOrdered of them (every lane
// holds one): workgroups start in the order of their index, and long ones that start last are waited for by everybody.  The tiles
// of a sequence stay side by side, last ones first.  Every sequence has exactly the tiles that it needs.
constexpr int kPackedOrdered = 63;
__device__ __forceinline__ PackedTile packed_tile_ordered(const int32_t* __restrict__ cu, int num_seqs, int total,
                                                          int per_row, int tile, int b) {
    const int lane = threadIdx.x & 63;
    const int edge = cu[lane < num_seqs ? lane : num_seqs];
    const int next = __shfl_down(edge, 1);
    int rows = edge >= 0 && edge < total && lane < num_seqs ? (next < total ? next : total) - edge : 0;
    rows = rows > 0 ? rows : 0;
    const int tiles = (int)(((unsigned)rows * (unsigned)per_row + (unsigned)tile - 1) / (unsigned)tile);
    // (one key per lane, all different: longer first, then the earlier one; lanes behind the last have no rows and no tiles)
    const int key = rows * 64 + (63 - lane);
    int before = 0;  // tiles of the sequences in front of this lane's
    const int first = __builtin_amdgcn_readfirstlane(rows);
    if (__builtin_amdgcn_ballot_w64(lane < num_seqs && rows != first) == 0) {
        before = lane * tiles;
    } else {
        for (int j0 = 0; j0 < num_seqs; j0 += 8)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int other = __builtin_amdgcn_readlane(key, j0 + j);
                const int theirs =
                    (int)(((unsigned)(other >> 6) * (unsigned)per_row + (unsigned)tile - 1) / (unsigned)tile);
                before += other > key ? theirs : 0;
            }
    }
    const uint64_t mine = __builtin_amdgcn_ballot_w64(b >= before && b < before + tiles);
    PackedTile t = {0, 0, 0, 0, 0};
    if (mine == 0) return t;
    const int s = __builtin_ctzll(mine);
    t.seq = s;
    t.row0 = __builtin_amdgcn_readlane(edge, s);
    t.rows = __builtin_amdgcn_readlane(rows, s);
    t.tile = b - __builtin_amdgcn_readlane(before, s);
    return t;
}

// Normalises a wave's 32 columns and writes them, 16 at a time through its part of LDS (`stage`, 16 rows of D + 8): straight
// from the registers a store would put 16 bytes into each of 32 rows, from there it writes whole head rows.  `to` is where this
// lane's column goes, in elements from `out`, less than 2^31; cols the number of columns that are there.
template <typename T, int D>
__device__ __forceinline__ void attn_packed_write(unsigned short* out, unsigned to, int cols, unsigned short* stage,
                                                  const float16_t (&o)[D / 32], float l) {
    constexpr int kRow = D + 8, kLanes = D / 8;
    const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
    const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;  // (only keys that score -inf: zeros)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (16 * half >= cols) break;
        if ((col >> 4) == half) {
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *reinterpret_cast<uint2_t*>(stage + (col & 15) * kRow + 32 * dt + 8 * b + 4 * h) =
                        uint2_t{T::pack2(o[dt][4 * b] * inv, o[dt][4 * b + 1] * inv),
                                T::pack2(o[dt][4 * b + 2] * inv, o[dt][4 * b + 3] * inv)};
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = lane; i < 16 * kLanes; i += 64) {
            const int c = i / kLanes, piece = i % kLanes;
            const unsigned at = __shfl(to, 16 * half + c);
            const uint4_t v = *reinterpret_cast<const uint4_t*>(stage + c * kRow + 8 * piece);
            if (16 * half + c < cols) *reinterpret_cast<uint4_t*>(out + (at + 8u * piece)) = v;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

}  // namespace lg
