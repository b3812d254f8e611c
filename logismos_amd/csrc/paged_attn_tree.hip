// Attention of drafted tokens over a paged cache: the new rows of a sequence are the nodes of a tree (or several), their K and
// V already in the cache behind the context, and a row sees the whole context and those of the new tokens that its mask names.
//
//   out[t][h] = softmax_j(q[t][h] . k[j][h / g] * scale) . v[j][h / g],   j < prior, or bit j - prior of t's mask
//
// A column is a (token, head of the group) pair of one KV head; a unit is up to 32 WAVES columns of one sequence and KV head, a
// wave holds 32 of them, and every tile of 32 keys that a unit reads serves all its columns:
//
//   S^T[32 keys x 32 columns] = K . Q^T         v_mfma_f32_32x32x16
//   online softmax of a column, which lives in two lanes (fp32)
//   O^T[D x 32 columns] += V^T . P              v_mfma_f32_32x32x16, keys in the order that S^T leaves them in
//
// The tiles of all units, one behind the other, are dealt out to the workgroups in equal shares, whatever the contexts are; a
// unit that was cut is put together by a second, small launch from its parts (sums and the maxima they are relative to).
//
// e4m3 pools: a tile is decoded once, on its way into LDS: c * 2^(e - top) in 16 bits, top the largest exponent of the tile's
// rows, which goes into the scores of the tile (K) and into the exponents of its probabilities (V).  Elements below 2^-14 of the
// tile's largest row's step lose bits, to 2^-25 of it; bf16 queries take K as c * 2^e, which bf16 holds as it is.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"
#include "q4_common.hpp"

#include <math.h>

namespace lg {

constexpr int kTreeKeys = 32;       // keys of a tile
constexpr int kTreeWorkers = 512;   // workgroups that share the tiles, at most
constexpr int kTreeLeast = 8;       // tiles of a workgroup, at least
constexpr int kTreeMaskWords = 4;

struct TreeParams {
    const unsigned short* q;
    const uint8_t* k_pool;
    const uint8_t* v_pool;
    const uint8_t* k_exp;
    const uint8_t* v_exp;
    const int32_t* tables;
    const int32_t* cu;
    const int32_t* ctx;
    const uint32_t* mask;
    unsigned short* out;
    float* ws;
    int num_seqs, total, max_q, hkv, g, block_size, max_blocks, num_blocks, words;  // words: 32 bits each, of a row's mask
    int64_t q_stride, out_stride;
    float scale_log2e;
    int workers;
    int slot_waves;  // waves that a slot of the workspace has room for
};

// The sequences 64 at a time, one to a lane, with the tiles in front of them.
struct TreeChunk {
    int first;   // sequence of lane 0
    int row0, rows, ctx, prior, units, tiles;  // this lane's; tiles: of a unit
    unsigned before, behind;                   // tiles of all units in front of it, and with its own
    unsigned end;                              // ... with the last lane's
};

template <int COLS>
__device__ __forceinline__ TreeChunk tree_chunk(const TreeParams& p, int first, unsigned before) {
    const int lane = threadIdx.x & 63, s = first + lane;
    TreeChunk c;
    c.first = first;
    const bool in = s < p.num_seqs;
    const int r0 = p.cu[in ? s : p.num_seqs], r1 = p.cu[in ? s + 1 : p.num_seqs];
    const int context = in ? p.ctx[s] : 0;
    int rows = r0 >= 0 && r0 < p.total ? (r1 < p.total ? r1 : p.total) - r0 : 0;
    rows = rows < 0 || !in ? 0 : rows < p.max_q ? rows : p.max_q;
    c.row0 = r0;
    c.rows = rows;
    const int room = p.block_size * p.max_blocks;
    c.ctx = context < 0 ? 0 : context < room ? context : room;
    c.prior = c.ctx - rows;
    c.units = (rows * p.g + COLS - 1) / COLS * p.hkv;
    c.tiles = c.ctx > 0 ? (c.ctx + kTreeKeys - 1) / kTreeKeys : 1;
    unsigned sum = (unsigned)c.units * (unsigned)c.tiles;
    const unsigned mine = sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned other = __shfl_up(sum, d);
        sum += lane >= d ? other : 0u;
    }
    c.behind = before + sum;
    c.before = c.behind - mine;
    c.end = (unsigned)__builtin_amdgcn_readlane((int)c.behind, 63);
    return c;
}

// A unit and which of its tiles: everything the same in the whole wave.
struct TreeUnit {
    int seq, row0, rows, ctx, prior, head, group, tile, tiles;
};
__device__ __forceinline__ TreeUnit tree_unit(const TreeChunk& c, int hkv, unsigned pos) {
    const uint64_t behind = __builtin_amdgcn_ballot_w64(c.behind > pos);
    const int l = __builtin_ctzll(behind | (1ull << 63));
    auto of = [&](int v) LG_INLINE { return __builtin_amdgcn_readlane(v, l); };
    TreeUnit u;
    u.seq = c.first + l;
    u.row0 = of(c.row0);
    u.rows = of(c.rows);
    u.ctx = of(c.ctx);
    u.prior = of(c.prior);
    u.tiles = of(c.tiles);
    const unsigned rest = pos - (unsigned)of((int)c.before);
    const int unit = (int)(rest / (unsigned)u.tiles);
    u.tile = (int)(rest - (unsigned)unit * (unsigned)u.tiles);
    const int groups = of(c.units) / hkv;
    u.head = unit / groups;
    u.group = unit - u.head * groups;
    return u;
}

__device__ __forceinline__ unsigned tree_share(unsigned total, int workers) {
    const unsigned per = (total + workers - 1) / workers;
    return per > kTreeLeast ? per : kTreeLeast;
}

// Bytes of a wave's part of a slot: 32 columns of D sums, then maxima and denominators (a lane each, both lanes of a column).
constexpr int tree_wave_floats(int d) { return 32 * d + 128; }

// Probabilities are relative to a reference that follows the maximum lazily, as in attn_packed.hip: the largest lies between
// 2^kTreeHead and 2^(kTreeHead + kTreeLazy), so that those down to 2^-25 of a column's largest keep all bits of fp16.
constexpr float kTreeHead = 11.0f, kTreeLazy = 4.0f;

template <typename T, int D, int WAVES, bool E4M3>
__global__ __launch_bounds__(64 * WAVES) void paged_attn_tree_kernel(const TreeParams p) {
    constexpr int kCols = 32 * WAVES, kMovers = 32 * WAVES;  // threads that move K, and V
    constexpr int kSteps = D / 16, kTiles = D / 32;
    constexpr int kKRow = D + 8, kVRow = D / 32 % 2 ? D : D + 32;  // elements
    constexpr int kPer = kTreeKeys * D / 8 / kMovers;              // pieces of 8 elements that a thread moves per tile
    constexpr int kPiece = E4M3 ? 8 : 16;                          // their bytes
    constexpr int kRow = E4M3 ? D : 2 * D;                         // bytes of a head row
    constexpr int kTile = kTreeKeys * (kKRow + kVRow), kWayOut = WAVES * 16 * (D + 8);
    __shared__ __attribute__((aligned(16))) unsigned short lds[kTile > kWayOut ? kTile : kWayOut];
    __shared__ int tops[2];  // of the tile: exponents of K and V
    unsigned short* const ks = lds;
    unsigned short* const vs = lds + kTreeKeys * kKRow;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, col = lane & 31;
    const bool moves_v = wave >= WAVES / 2;
    const int s16 = lane & 15;
    const int v_lane = (4 * h + (s16 >> 2)) * kVRow + 16 * ((lane >> 4) & 1) + 4 * (s16 & 3);

    unsigned total = 0;
    for (int first = 0; first < p.num_seqs; first += 64) total = tree_chunk<kCols>(p, first, total).end;
    const unsigned per = tree_share(total, p.workers);
    unsigned pos = blockIdx.x * per;
    const unsigned end = total - pos < per ? total : pos + per;
    if (pos >= total) return;
    TreeChunk chunk = tree_chunk<kCols>(p, 0, 0);
    while (pos < end) {
        while (pos >= chunk.end) chunk = tree_chunk<kCols>(p, chunk.first + 64, chunk.end);
        const TreeUnit u = tree_unit(chunk, p.hkv, pos);
        const int tile0 = u.tile;
        const int tile1 = (unsigned)(u.tiles - tile0) < end - pos ? u.tiles : tile0 + (int)(end - pos);
        pos += (unsigned)(tile1 - tile0);

        const int cols = u.rows * p.g;
        const int c0 = u.group * kCols + wave * 32;
        const int gc = c0 + col < cols ? c0 + col : cols - 1;
        const int tok = gc / p.g, head = u.head * p.g + gc - tok * p.g;
        const bool active = c0 < cols;
        const uint32_t* const mask = p.mask + (int64_t)(u.row0 + tok) * p.words;

        uint4_t qb[kSteps];
        {
            const unsigned short* q = p.q + (int64_t)(u.row0 + tok) * p.q_stride + (int64_t)head * D + 8 * h;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) qb[j] = *reinterpret_cast<const uint4_t*>(q + 16 * j);
        }

        // ---- movement: the first half of the waves carries K, the second V
        const int32_t* const table = p.tables + (int64_t)u.seq * p.max_blocks;
        const uint8_t* const pool = moves_v ? p.v_pool : p.k_pool;
        const uint8_t* const exps = moves_v ? p.v_exp : p.k_exp;
        struct Regs {
            uint4_t x[kPer];
            int e;  // exponent of key lane % 32
        };
        auto key_of = [&](int i) LG_INLINE { return (tid % kMovers + kMovers * i) / (D / 8); };
        auto piece_of = [&](int i) LG_INLINE { return (tid % kMovers + kMovers * i) % (D / 8); };
        // The blocks of the two halves of a tile; bit 0 / 1 of `there`: the half has one.
        struct Blocks {
            int id[2], off[2], there;
        };
        auto blocks_of = [&](int tile) LG_INLINE {
            Blocks b;
            b.there = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = tile * kTreeKeys + 16 * i;
                const int at = key < u.ctx ? key / p.block_size : 0;
                const int id = key < u.ctx ? table[at] : -1;
                const bool ok = id >= 0 && id < p.num_blocks;
                b.id[i] = ok ? id : 0;
                b.off[i] = key < u.ctx ? key - at * p.block_size : 0;
                b.there |= ok ? 1 << i : 0;
            }
            return b;
        };
        auto gload = [&](const Blocks& b, int tile, Regs& r) LG_INLINE {
            const int left = u.ctx - tile * kTreeKeys;  // keys behind the last one: that one again
            int64_t row[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) row[i] = (int64_t)b.id[i] * p.block_size + b.off[i];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int key = key_of(i) < left ? key_of(i) : left - 1;
                const int64_t at = (key < 16 ? row[0] : row[1]) + (key & 15);
                const uint8_t* src = pool + (at * p.hkv + u.head) * kRow + kPiece * piece_of(i);
                if constexpr (E4M3) {
                    const uint2_t v = *reinterpret_cast<const uint2_t*>(src);
                    r.x[i][0] = v[0];
                    r.x[i][1] = v[1];
                } else {
                    r.x[i] = *reinterpret_cast<const uint4_t*>(src);
                }
            }
            if constexpr (E4M3) {
                const int key = col < left ? col : left - 1;
                const int half = key >> 4;
                const int64_t at = ((int64_t)(half ? b.id[1] : b.id[0]) * p.hkv + u.head) * p.block_size +
                                   (half ? b.off[1] : b.off[0]) + (key & 15);
                r.e = exps[at];
            }
        };
        auto lstore = [&](const Regs& r) LG_INLINE {
            unsigned short* at = moves_v ? vs : ks;
            const int row = moves_v ? kVRow : kKRow;
            int top = 127;
            constexpr bool kAsIs = __is_same(T, PackedBf16);  // K in bf16
            if constexpr (E4M3) {
                if (!kAsIs || moves_v) {
                    top = r.e;
                    top = max(top, lane_xor_i32<1>(top));
                    top = max(top, lane_xor_i32<2>(top));
                    top = max(top, lane_xor_i32<4>(top));
                    top = max(top, lane_xor_i32<8>(top));
                    top = max(top, lane_xor_i32<16>(top));
                }
                if (tid % kMovers == 0) tops[moves_v] = top - 127;
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                unsigned short* to = at + key_of(i) * row + 8 * piece_of(i);
                if constexpr (E4M3) {
                    const float scale = __int_as_float(max(__shfl(r.e, key_of(i)) - top + 127, 0) << 23);
                    uint4_t y;
                    if (kAsIs && !moves_v) {
                        y[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x[i][0], scale, false));
                        y[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x[i][0], scale, true));
                        y[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x[i][1], scale, false));
                        y[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x[i][1], scale, true));
                    } else {
                        y[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.x[i][0], scale, false));
                        y[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.x[i][0], scale, true));
                        y[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.x[i][1], scale, false));
                        y[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.x[i][1], scale, true));
                    }
                    *reinterpret_cast<uint4_t*>(to) = y;
                } else {
                    *reinterpret_cast<uint4_t*>(to) = r.x[i];
                }
            }
        };
        auto v_operand = [&](int kb, int dt) LG_INLINE {
            typedef short short4_t __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) short4_t lds_short4_t;
            const unsigned short* a = vs + v_lane + 16 * kb * kVRow + 32 * dt;
            const uint2_t lo = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)a));
            const uint2_t hi =
                __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(a + 8 * kVRow)));
            return uint4_t{lo[0], lo[1], hi[0], hi[1]};
        };
        auto k_operand = [&](int j) LG_INLINE {
            return *reinterpret_cast<const uint4_t*>(ks + col * kKRow + 16 * j + 8 * h);
        };

        float m = -INFINITY, l = 0.0f;
        float16_t o[kTiles];
#pragma unroll
        for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;

        Regs r;
        Blocks b = blocks_of(tile0);
        if (u.ctx > 0) gload(b, tile0, r);
        for (int tile = tile0; tile < tile1 && u.ctx > 0; ++tile) {
            const int key0 = tile * kTreeKeys, there = b.there;
            __syncthreads();
            lstore(r);
            __syncthreads();
            if (tile + 1 < tile1) {
                b = blocks_of(tile + 1);
                gload(b, tile + 1, r);
            }
            if (!active) continue;
            float scale = p.scale_log2e, v_top = 0.0f;
            if constexpr (E4M3) {
                scale = ldexpf(scale, tops[0]);
                v_top = (float)tops[1];
            }
            float16_t s;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) s = T::mfma32(k_operand(j), qb[j], s);
            // which of the tile's keys this column sees
            const bool masked = key0 + kTreeKeys > u.prior || there != 3;
            unsigned win = ~0u;
            if (masked) {
                const int j0 = key0 - u.prior;
                if (j0 > -32) {
                    auto word = [&](int i) LG_INLINE { return i < p.words ? mask[i] : 0u; };
                    if (j0 < 0) {
                        win = word(0) << -j0 | ((1u << -j0) - 1u);
                    } else {
                        const int i = j0 >> 5;
                        win = (unsigned)(((uint64_t)word(i + 1) << 32 | word(i)) >> (j0 & 31));
                    }
                }
                const int left = u.ctx - key0;
                if (left < 32) win &= (1u << left) - 1u;
                if ((there & 1) == 0) win &= 0xffff0000u;
                if ((there & 2) == 0) win &= 0x0000ffffu;
            }
            float x[16], tm = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[e] = s[e] * scale;
                if (masked) x[e] = (win >> (8 * (e >> 2) + 4 * h + (e & 3))) & 1u ? x[e] : -INFINITY;
                tm = fmaxf(tm, x[e]);
            }
            // (exponents of the tile's probabilities and of its rows of V together)
            tm = fmaxf(tm, lane_xor_f32<32>(tm)) + v_top - kTreeHead;
            const bool raise = tm > m + kTreeLazy;
            if (__builtin_amdgcn_ballot_w64(raise) != 0) {
                const float alpha = raise ? fast_exp2(m - tm) : 1.0f;
                m = raise ? tm : m;
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
            }
            const float ref = (m == -INFINITY ? 0.0f : m) - v_top;
            float sum = 0.0f;
            uint4_t pb[2];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                x[e] = fast_exp2(x[e] - ref);
                x[e + 1] = fast_exp2(x[e + 1] - ref);
                sum += x[e];
                sum += x[e + 1];
                pb[e >> 3][(e & 7) >> 1] = PackedF16::pack2(x[e], x[e + 1]);
            }
            l += E4M3 ? ldexpf(sum, -(int)v_top) : sum;
            uint4_t va[kSteps];
#pragma unroll
            for (int j = 0; j < kSteps; ++j) va[j] = v_operand(j / kTiles, j % kTiles);
            // A key that a column does not see has the probability 0 there, and 0 times an infinity or NaN of its V row is NaN: in
            // the new tokens' tiles such elements stay out of the product, and are added for the columns that see them.
            bool odd = false;
            if (masked) {
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const unsigned bad = ((va[j][w] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                        odd |= bad != 0;
                        va[j][w] &= ~((bad >> 15) * 0xffffu);
                    }
            }
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
                o[j % kTiles] = PackedF16::mfma32(va[j], pb[j / kTiles], o[j % kTiles]);
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0, 0)) {
                for (int key = 0; key < kTreeKeys; ++key) {
                    const int at = 4 * (key >> 3) + (key & 3);
                    float mine = x[0];
#pragma unroll
                    for (int e = 1; e < 16; ++e) mine = at == e ? x[e] : mine;
                    const float prob = __shfl(mine, col + 32 * ((key >> 2) & 1));
                    const bool seen = (win >> key) & 1u;
#pragma unroll
                    for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                        for (int q4 = 0; q4 < 4; ++q4) {
                            const half4_t v =
                                *reinterpret_cast<const half4_t*>(vs + key * kVRow + 32 * dt + 8 * q4 + 4 * h);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                o[dt][4 * q4 + i] += seen && !(fabsf((float)v[i]) < INFINITY) ? prob * (float)v[i] : 0.0f;
                        }
                }
            }
        }
        l += lane_xor_f32<32>(l);
        __syncthreads();  // (the next unit's tiles, and the columns on their way out, go where the last tile was)
        if (!active) continue;
        if (tile0 == 0 && tile1 == u.tiles) {
            const int tok0 = c0 / p.g;
            attn_packed_write<T, D>(p.out + (int64_t)(u.row0 + tok0) * p.out_stride,
                                    (unsigned)(tok - tok0) * (unsigned)p.out_stride + (unsigned)(head * D), cols - c0,
                                    lds + wave * 16 * (D + 8), o, l);
        } else {
            // a part: slot 1 of the workgroup holds the end of a unit, slot 0 everything else
            float* const slot = p.ws + ((int64_t)(2 * blockIdx.x + (tile1 == u.tiles ? 1 : 0)) * p.slot_waves + wave) *
                                           tree_wave_floats(D);
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    reinterpret_cast<float4_t*>(slot)[(4 * dt + q4) * 64 + lane] =
                        float4_t{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
            slot[32 * D + lane] = m;
            slot[32 * D + 64 + lane] = l;
        }
    }
}

// The parts of the units that were cut: a workgroup takes 32 columns and 32 elements of the heads, its waves every fourth part.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void paged_attn_tree_merge_kernel(const TreeParams p) {
    constexpr int kCols = 32 * WAVES, kTiles = D / 32;
    __shared__ float4_t theirs[3][4][64];
    __shared__ float ml[3][2][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int dt = blockIdx.x % kTiles;
    const int of_unit = blockIdx.x / kTiles % p.slot_waves;  // which 32 columns of a unit
    int unit = blockIdx.x / kTiles / p.slot_waves;           // of all units
    unsigned total = 0;
    for (int first = 0; first < p.num_seqs; first += 64) total = tree_chunk<kCols>(p, first, total).end;
    const unsigned per = tree_share(total, p.workers);
    // the sequence of the unit: units are counted as tiles are
    TreeChunk c = tree_chunk<kCols>(p, 0, 0);
    int seq_lane = 0;
    for (;;) {
        unsigned units = (unsigned)c.units;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const unsigned other = __shfl_up(units, d);
            units += lane >= d ? other : 0u;
        }
        const unsigned all = (unsigned)__builtin_amdgcn_readlane((int)units, 63);
        if ((unsigned)unit < all) {
            seq_lane = __builtin_ctzll(__builtin_amdgcn_ballot_w64(units > (unsigned)unit));
            unit -= __builtin_amdgcn_readlane((int)units, seq_lane) - __builtin_amdgcn_readlane(c.units, seq_lane);
            break;
        }
        unit -= (int)all;
        if (c.first + 64 >= p.num_seqs) return;
        c = tree_chunk<kCols>(p, c.first + 64, c.end);
    }
    const unsigned tiles = (unsigned)__builtin_amdgcn_readlane(c.tiles, seq_lane);
    const unsigned pos = (unsigned)__builtin_amdgcn_readlane((int)c.before, seq_lane) + (unsigned)unit * tiles;
    const int first = (int)(pos / per), last = (int)((pos + tiles - 1) / per);
    if (first == last) return;
    const TreeUnit u = tree_unit(c, p.hkv, pos);
    const int cols = u.rows * p.g, c0 = u.group * kCols + of_unit * 32;
    if (c0 >= cols) return;

    float m = -INFINITY, l = 0.0f;
    float4_t o[4];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) o[q4] = float4_t{0, 0, 0, 0};
    auto join = [&](float m2, float l2, const float4_t* o2) LG_INLINE {
        const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top;
        const float mine = fast_exp2(m - ref), its = fast_exp2(m2 - ref);
        m = top;
        l = l * mine + l2 * its;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[q4][e] = o[q4][e] * mine + o2[q4][e] * its;
    };
    for (int w = first + wave; w <= last; w += 4) {
        const float* slot =
            p.ws + ((int64_t)(2 * w + (w == last ? 1 : 0)) * p.slot_waves + of_unit) * tree_wave_floats(D);
        float4_t o2[4];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) o2[q4] = reinterpret_cast<const float4_t*>(slot)[(4 * dt + q4) * 64 + lane];
        join(slot[32 * D + lane], slot[32 * D + 64 + lane], o2);
    }
    if (wave > 0) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) theirs[wave - 1][q4][lane] = o[q4];
        ml[wave - 1][0][lane] = m;
        ml[wave - 1][1][lane] = l;
    }
    __syncthreads();
    if (wave > 0) return;
    for (int w = 0; w < 3; ++w) {
        float4_t o2[4];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) o2[q4] = theirs[w][q4][lane];
        join(ml[w][0][lane], ml[w][1][lane], o2);
    }
    const int h = lane >> 5, gc = c0 + (lane & 31);
    if (gc >= cols) return;
    const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
    const int tok = gc / p.g, head = u.head * p.g + gc - tok * p.g;
    unsigned short* out = p.out + (int64_t)(u.row0 + tok) * p.out_stride + (int64_t)head * D + 32 * dt + 4 * h;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<uint2_t*>(out + 8 * q4) =
            uint2_t{T::pack2(o[q4][0] * inv, o[q4][1] * inv), T::pack2(o[q4][2] * inv, o[q4][3] * inv)};
}

// Waves of a workgroup.
static int tree_waves(int) { return 4; }

static int tree_slot_waves(int max_q, int g, int waves) {
    const int64_t need = ((int64_t)max_q * g + 31) / 32;
    return need < waves ? (int)need : waves;
}

template <typename T, int D, bool E4M3>
static hipError_t tree_launch(TreeParams p, hipStream_t stream) {
    constexpr int WAVES = 4;
    p.slot_waves = tree_slot_waves(p.max_q, p.g, WAVES);
    const int64_t most = packed_tiles(p.total, p.num_seqs, p.g, 32 * WAVES) * p.hkv;  // units
    const int64_t room = (int64_t)p.block_size * p.max_blocks;
    const int64_t tiles = most * ((room + kTreeKeys - 1) / kTreeKeys);
    int64_t workers = 2 * device_cu_count();
    if (workers > kTreeWorkers) workers = kTreeWorkers;
    if (workers > (tiles + kTreeLeast - 1) / kTreeLeast) workers = (tiles + kTreeLeast - 1) / kTreeLeast;
    p.workers = (int)workers;
    paged_attn_tree_kernel<T, D, WAVES, E4M3><<<(unsigned)workers, 64 * WAVES, 0, stream>>>(p);
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess || workers == 1) return rc;
    paged_attn_tree_merge_kernel<T, D, WAVES><<<(unsigned)(most * p.slot_waves * (D / 32)), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, bool E4M3>
static hipError_t tree_by_width(const TreeParams& p, int d, hipStream_t stream) {
    switch (d) {
        case 32: return tree_launch<T, 32, E4M3>(p, stream);
        case 64: return tree_launch<T, 64, E4M3>(p, stream);
        case 96: return tree_launch<T, 96, E4M3>(p, stream);
        case 128: return tree_launch<T, 128, E4M3>(p, stream);
        case 160: return tree_launch<T, 160, E4M3>(p, stream);
        case 192: return tree_launch<T, 192, E4M3>(p, stream);
        case 224: return tree_launch<T, 224, E4M3>(p, stream);
        default: return tree_launch<T, 256, E4M3>(p, stream);
    }
}

static logismos_status_t tree_attention(bool e4m3, bool bf16, const TreeParams& p, int hq, int d, float scale,
                                        logismos_stream_t stream) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (logismos_check_paged_attn_tree_shape(p.num_seqs, p.total, p.max_q, hq, p.hkv, d, p.block_size, p.max_blocks,
                                             p.num_blocks, p.words / 2, (int)p.q_stride, (int)p.out_stride, nullptr,
                                             0) != 0)
        return bad;
    if (!p.q || !p.k_pool || !p.v_pool || !p.tables || !p.cu || !p.ctx || !p.mask || !p.out || !p.ws) return bad;
    if (e4m3 && (!p.k_exp || !p.v_exp)) return bad;
    if ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k_pool) |
         reinterpret_cast<uintptr_t>(p.v_pool) | reinterpret_cast<uintptr_t>(p.k_exp) |
         reinterpret_cast<uintptr_t>(p.v_exp) | reinterpret_cast<uintptr_t>(p.out) |
         reinterpret_cast<uintptr_t>(p.ws)) % 16 != 0 ||
        (reinterpret_cast<uintptr_t>(p.tables) | reinterpret_cast<uintptr_t>(p.cu) |
         reinterpret_cast<uintptr_t>(p.ctx)) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(p.mask) % 8 != 0)
        return bad;
    TreeParams q = p;
    q.g = hq / p.hkv;
    q.scale_log2e = scale * 1.4426950408889634f;
    if (!(scale > 0.0f) || !isfinite(q.scale_log2e)) return bad;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!e4m3) return static_cast<logismos_status_t>(tree_by_width<PackedF16, false>(q, d, st));
    return static_cast<logismos_status_t>(bf16 ? tree_by_width<PackedBf16, true>(q, d, st)
                                               : tree_by_width<PackedF16, true>(q, d, st));
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_paged_attn_tree_shape(int num_seqs, int total_tokens, int max_seqlen_q,
                                                       int num_q_heads, int num_kv_heads, int head_dim,
                                                       int block_size, int max_blocks_per_seq, int num_blocks,
                                                       int mask_words, int q_stride, int out_stride, char* msg,
                                                       size_t cap) {
    using lg::reject;
    if (num_seqs <= 0 || total_tokens <= 0 || max_seqlen_q <= 0)
        return reject(msg, cap, "num_seqs, total_tokens and max_seqlen_q must be positive (%d, %d, %d)", num_seqs,
                      total_tokens, max_seqlen_q);
    if (num_seqs > 65535 || total_tokens > 65535)
        return reject(msg, cap, "num_seqs and total_tokens must be <= 65535 (%d, %d)", num_seqs, total_tokens);
    if (max_seqlen_q > total_tokens)
        return reject(msg, cap, "max_seqlen_q %d exceeds total_tokens %d", max_seqlen_q, total_tokens);
    if (num_q_heads <= 0 || num_kv_heads <= 0)
        return reject(msg, cap, "num_q_heads and num_kv_heads must be positive (%d, %d)", num_q_heads, num_kv_heads);
    if (num_q_heads % num_kv_heads != 0)
        return reject(msg, cap, "num_q_heads %d is not a multiple of num_kv_heads %d", num_q_heads, num_kv_heads);
    if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 256)
        return reject(msg, cap, "head_dim must be a multiple of 32 up to 256 (%d)", head_dim);
    if (block_size <= 0 || block_size % 16 != 0)
        return reject(msg, cap, "block_size must be a positive multiple of 16 (%d)", block_size);
    if (max_blocks_per_seq <= 0 || num_blocks <= 0)
        return reject(msg, cap, "max_blocks_per_seq and num_blocks must be positive (%d, %d)", max_blocks_per_seq,
                      num_blocks);
    if ((int64_t)block_size * max_blocks_per_seq > INT32_MAX - 64 || (int64_t)block_size * num_blocks > INT32_MAX)
        return reject(msg, cap, "block_size * max_blocks_per_seq or block_size * num_blocks exceeds i32::MAX");
    if (mask_words <= 0 || mask_words > lg::kTreeMaskWords || max_seqlen_q > 64 * mask_words)
        return reject(msg, cap, "mask_words must be between 1 and %d, with a bit for each of max_seqlen_q tokens (%d, %d)",
                      lg::kTreeMaskWords, mask_words, max_seqlen_q);
    const int64_t width = (int64_t)num_q_heads * head_dim;
    if (width > (1 << 20)) return reject(msg, cap, "num_q_heads * head_dim exceeds %d", 1 << 20);
    if (q_stride < width || out_stride < width)
        return reject(msg, cap, "a stride is smaller than its row (%d and %d of %lld)", q_stride, out_stride,
                      (long long)width);
    if ((q_stride | out_stride) % 8 != 0)
        return reject(msg, cap, "strides must be multiples of 8 (%d, %d)", q_stride, out_stride);
    if (out_stride > (1 << 22)) return reject(msg, cap, "out_stride must be at most %d (%d)", 1 << 22, out_stride);
    // tiles of all units, and workgroups of the second launch
    const int64_t units = lg::packed_tiles(total_tokens, num_seqs, num_q_heads / num_kv_heads, 128) * num_kv_heads;
    const int64_t tiles = ((int64_t)block_size * max_blocks_per_seq + 31) / 32;
    if (units > (1 << 22) || tiles > INT32_MAX / units)
        return reject(msg, cap, "too many key tiles: %lld units of columns with up to %lld each", (long long)units,
                      (long long)tiles);
    return 0;
}

size_t logismos_paged_attn_tree_workspace_bytes(int total_tokens, int max_seqlen_q, int num_q_heads, int num_kv_heads,
                                                int head_dim) {
    if (total_tokens <= 0 || max_seqlen_q <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    if (max_seqlen_q > total_tokens || num_q_heads % num_kv_heads != 0 || head_dim > 256) return 0;
    const int g = num_q_heads / num_kv_heads;
    const int waves = lg::tree_slot_waves(max_seqlen_q, g, 4);
    return (size_t)2 * lg::kTreeWorkers * (size_t)waves * (size_t)lg::tree_wave_floats(head_dim) * sizeof(float);
}

#define LOGISMOS_TREE_PARAMS                                                                                           \
    lg::TreeParams p = {};                                                                                             \
    p.q = static_cast<const unsigned short*>(q);                                                                       \
    p.k_pool = static_cast<const uint8_t*>(k_pool);                                                                    \
    p.v_pool = static_cast<const uint8_t*>(v_pool);                                                                    \
    p.tables = block_tables;                                                                                           \
    p.cu = cu_seqlens_q;                                                                                               \
    p.ctx = context_lens;                                                                                              \
    p.mask = reinterpret_cast<const uint32_t*>(tree_mask);                                                             \
    p.out = static_cast<unsigned short*>(out);                                                                         \
    p.ws = static_cast<float*>(workspace);                                                                             \
    p.num_seqs = num_seqs;                                                                                             \
    p.total = total_tokens;                                                                                            \
    p.max_q = max_seqlen_q;                                                                                            \
    p.hkv = num_kv_heads;                                                                                              \
    p.block_size = block_size;                                                                                         \
    p.max_blocks = max_blocks_per_seq;                                                                                 \
    p.num_blocks = num_blocks;                                                                                         \
    p.words = mask_words > 0 && mask_words <= lg::kTreeMaskWords ? 2 * mask_words : 0;                                 \
    p.q_stride = q_stride;                                                                                             \
    p.out_stride = out_stride;

logismos_status_t logismos_launch_paged_attn_tree_fp16(
    const void* q, const void* k_pool, const void* v_pool, const int32_t* block_tables, const int32_t* cu_seqlens_q,
    const int32_t* context_lens, const uint64_t* tree_mask, void* out, void* workspace, int num_seqs, int total_tokens,
    int max_seqlen_q, int num_q_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq,
    int num_blocks, int mask_words, int q_stride, int out_stride, float scale, logismos_stream_t stream) {
    LOGISMOS_TREE_PARAMS
    return lg::tree_attention(false, false, p, num_q_heads, head_dim, scale, stream);
}

#define LOGISMOS_PAGED_ATTN_TREE_E4M3(name, bf16)                                                                      \
    logismos_status_t logismos_launch_paged_attn_tree_e4m3_##name(                                                     \
        const void* q, const void* k_pool, const void* k_exp, const void* v_pool, const void* v_exp,                   \
        const int32_t* block_tables, const int32_t* cu_seqlens_q, const int32_t* context_lens,                         \
        const uint64_t* tree_mask, void* out, void* workspace, int num_seqs, int total_tokens, int max_seqlen_q,       \
        int num_q_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq, int num_blocks,       \
        int mask_words, int q_stride, int out_stride, float scale, logismos_stream_t stream) {                         \
        LOGISMOS_TREE_PARAMS                                                                                           \
        p.k_exp = static_cast<const uint8_t*>(k_exp);                                                                  \
        p.v_exp = static_cast<const uint8_t*>(v_exp);                                                                  \
        return lg::tree_attention(true, bf16, p, num_q_heads, head_dim, scale, stream);                                \
    }
LOGISMOS_PAGED_ATTN_TREE_E4M3(fp16, false)
LOGISMOS_PAGED_ATTN_TREE_E4M3(bf16, true)
#undef LOGISMOS_PAGED_ATTN_TREE_E4M3
#undef LOGISMOS_TREE_PARAMS

logismos_status_t logismos_tree_mask(const int32_t* parents, int tokens, int mask_words, uint64_t* mask) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (tokens == 0 && mask_words > 0 && mask_words <= lg::kTreeMaskWords) return 0;
    if (!parents || !mask || tokens <= 0 || mask_words <= 0 || mask_words > lg::kTreeMaskWords ||
        tokens > 64 * mask_words)
        return bad;
    for (int i = 0; i < tokens; ++i)
        if (parents[i] < -1 || parents[i] >= i) return bad;
    for (int i = 0; i < tokens; ++i)
        for (int w = 0; w < mask_words; ++w) {
            const uint64_t above = parents[i] >= 0 ? mask[(size_t)parents[i] * mask_words + w] : 0;
            mask[(size_t)i * mask_words + w] = above | (i / 64 == w ? 1ull << (i % 64) : 0);
        }
    return 0;
}

}  // extern "C"
