// Attention of drafted tokens over a paged cache: the new rows of a sequence are the nodes of a tree (or several), their K and
// V already in the cache behind the context, and a row sees the whole context and those of the new tokens that its mask names.
//
//   out[t][h] = softmax_j(q[t][h] . k[j][h / g] * scale) . v[j][h / g],   j < prior, or bit j - prior of t's mask
//
// A column is a (token, head of the group) pair of one KV head; a unit is up to 32 COLW columns of one sequence and KV head, a
// wave holds 32 of them, and every tile of 32 keys that a unit reads serves all its columns:
//
//   S^T[32 keys x 32 columns] = K . Q^T         v_mfma_f32_32x32x16
//   online softmax of a column, which lives in two lanes (fp32)
//   O^T[D x 32 columns] += V^T . P              v_mfma_f32_32x32x16, keys in the order that S^T leaves them in
//
// The tiles of all units, one behind the other, are dealt out to the workgroups in equal shares, whatever the contexts are; a
// unit that was cut is put together by a second, small launch from its parts (sums and what they are relative to).  Where a table has room
// for few tiles, every unit has a workgroup and nothing is cut.
//
// Workgroups: eight waves side by side for more than 128 columns of heads of 64 and 128; four for 65 to 128, for any number of columns of other heads and
// always for heads wider than 128 (two parts of four where units of fp16 pools are few and long); two for 33 to 64 in two parts that take the tiles in turn,
// single waves in four parts for up to 32, so that narrow trees have several tiles in flight too (four side by side here as well for a middling
// number of tiles).  The rules and both sides are at tree_launch.  They go by the width of the block table, since only the device knows the contexts: short
// contexts in a wide table are dealt out and put together as long ones are (7 rows behind 300 15.2 us instead of 13.4, 16 behind 184 21.6 instead of 14.5).
//
// Schedule as in attn_packed.hip: step i issues S(i + 1) and O(i - 1) around the softmax of tile i; K goes into LDS two tiles
// ahead of its use and V one, asked for two steps before that.  Where the tiles lie (rows of the pools, for e4m3 the factors of
// every row) is worked out for 256 tiles at a time and kept in LDS: looked up step by step it was longer than the products.
//
// e4m3 pools: a tile is decoded once, on its way into LDS: c * 2^(e - top) in fp16, top the largest exponent of the tile's rows, which
// goes into the scores of the tile (K) and into the exponents of its probabilities (V).  Elements below 2^-21 of 2^top lose bits, to 2^-25 of it;
// bf16 queries take K as c * 2^e, which bf16 holds as it is.  Of a tile that not all columns see all of (drafted tokens, blocks that are not
// there) the rows go in as c, and their exponents into scores and probabilities key by key: otherwise a row that a column does not
// see would take bits from those that it does.  Such a tile takes 2 us more, two or three of them in a unit (32 users below 181 -> 190).
//
// Probabilities enter the second product as one fp16 term: results of fp16 rows are off by 2.6e-4 to 2.8e-4 of their size, of which
// rounding them is 2.1e-4 (bf16 rows 1.7e-3, all of it their rounding).  With a second term for what the rounding left it is 2.1e-4, but a
// context of 131072 took 142 instead of 119 us, 8 users over e4m3 76 instead of 63, trees of up to 64 columns up to 20 % more (registers).
//
// Bound by memory for narrow trees (one context of 131072, 32 / 8 heads of 128, fp16, 24 rows: 537 MB in 117 us, 4.6 TB/s, 107 of them
// the first launch), by the matrix cores and what surrounds their steps for wide ones: 32 contexts of 1000 to 8192, e4m3, 64 rows, 113 GFLOP in
// 191 us.  A step of eight waves over 32 keys takes 2300 clocks, of which its products are 1024 on each of the four matrix cores and the reads of
// K and V out of LDS (16 KB for each wave) as much; beginning a unit costs 6 us (its sequence, its places, its first tiles), and of a wide unit that is
// cut the parts are 135 KB each, written and read again: 28 us of the 191 under the profiler.  Heads of 128 and 96 take all 256 registers that two waves
// to a SIMD leave: 2 spilled in eight waves, 17 to 25 in four over e4m3 pools.
#pragma once

#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"
#include "q4_common.hpp"

#include <math.h>

namespace lg {

constexpr int kTreeKeys = 32;       // keys of a tile
constexpr int kTreeWorkers = 512;   // workgroups that share the tiles, at most
constexpr int kTreeLeast = 2;       // tiles of a workgroup, at least
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
    int whole;       // a workgroup has a unit, whole
    int by_unit;     // the second launch has a workgroup for every unit, not for every cut
    int slot_waves;  // waves that a slot of the workspace has room for
};

// The sequences 64 at a time, one to a lane, with the tiles in front of them.
struct TreeChunk {
    int first;   // sequence of lane 0
    int row0, rows, ctx, prior, units, tiles;  // this lane's; tiles: of a unit
    unsigned before, behind;                   // tiles of all units in front of it, and with its own
    unsigned end;                              // ... with the last lane's
};

// The launch's parameters read anew where they are needed: kept in scalar registers, those that the loop over the tiles has no use for
// would push out those that it has.
typedef const TreeParams __attribute__((address_space(4)))* TreeCold;
__device__ __forceinline__ TreeCold tree_cold() {
    auto at = (TreeCold)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return at;
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
    auto add = [&](auto ctrl, auto rows) LG_INLINE {
        v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    add(ic<0x111>{}, ic<0xf>{});  // from 1, 2, 4, 8 lanes below in a row of 16
    add(ic<0x112>{}, ic<0xf>{});
    add(ic<0x114>{}, ic<0xf>{});
    add(ic<0x118>{}, ic<0xf>{});
    add(ic<0x142>{}, ic<0xa>{});  // the first (third) row's total to the second (fourth)
    add(ic<0x143>{}, ic<0xc>{});  // that of the first two to the others
    return v;
}

template <int COLS>
__device__ __forceinline__ TreeChunk tree_chunk(int first, unsigned before) {
    const TreeCold c0 = tree_cold();
    const auto& p = *c0;
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
    const unsigned mine = (unsigned)c.units * (unsigned)c.tiles;
    c.behind = before + wave_scan(mine);
    c.before = c.behind - mine;
    c.end = (unsigned)__builtin_amdgcn_readlane((int)c.behind, 63);
    return c;
}

// A unit and which of its tiles: everything the same in the whole wave.
struct TreeUnit {
    int seq, row0, rows, ctx, prior, head, group, tile, tiles;
    unsigned at;  // the tile, counted over all units
};
__device__ __forceinline__ TreeUnit tree_unit(const TreeChunk& c, int hkv, unsigned pos) {
    const uint64_t behind = __builtin_amdgcn_ballot_w64(c.behind > pos);
    const int l = __builtin_ctzll(behind | (1ull << 63));
    auto of = [&](int v) LG_INLINE { return __builtin_amdgcn_readlane(v, l); };
    TreeUnit u;
    u.seq = c.first + l;
    u.at = pos;
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

// Where unit `unit` of all begins, counted in tiles (units are counted as tiles are), and its tiles; 0: there is no such unit.  Leaves
// the chunk that it is in.
template <int COLS>
__device__ __forceinline__ unsigned tree_unit_at(TreeChunk& c, int num_seqs, int unit, unsigned& pos) {
    for (;;) {
        const unsigned units = wave_scan((unsigned)c.units);
        const int all = __builtin_amdgcn_readlane((int)units, 63);
        if (unit < all) {
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(units > (unsigned)unit));
            unit -= __builtin_amdgcn_readlane((int)units, l) - __builtin_amdgcn_readlane(c.units, l);
            const unsigned tiles = (unsigned)__builtin_amdgcn_readlane(c.tiles, l);
            pos = (unsigned)__builtin_amdgcn_readlane((int)c.before, l) + (unsigned)unit * tiles;
            return tiles;
        }
        unit -= all;
        if (c.first + 64 >= num_seqs) return 0;
        c = tree_chunk<COLS>(c.first + 64, c.end);
    }
}

__device__ __forceinline__ unsigned tree_share(unsigned total, int workers) {
    const unsigned per = (total + workers - 1) / workers;
    return per > kTreeLeast ? per : kTreeLeast;
}

// Bytes of a wave's part of a slot: 32 columns of D sums, then maxima and denominators (a lane each, both lanes of a column).
constexpr int tree_wave_floats(int d) { return 32 * d + 128; }

// Probabilities are relative to a reference that follows the maximum lazily, as in attn_packed.hip: the largest lies between
// 2^kTreeHead and 2^(kTreeHead + kTreeLazy), so that those down to 2^-25 of a column's largest keep all bits of fp16.  It stands for the
// exponent of a probability and of the row of V that it goes with together, s * scale + v, and is kept as the score s and the exponent v:
// differences of scores are taken before the scale, and in one number the exponent would be rounded to steps of the score.
constexpr float kTreeHead = 11.0f, kTreeLazy = 4.0f;
struct TreeRef {
    float s, v;
};
// (s is NaN while a column has seen nothing above -inf)
__device__ __forceinline__ bool tree_none(TreeRef a) { return a.s != a.s; }
__device__ __forceinline__ float tree_above(TreeRef a, TreeRef b, float scale) {
    return tree_none(a) ? -INFINITY : tree_none(b) ? INFINITY : fmaf(a.s - b.s, scale, a.v - b.v);
}
__device__ __forceinline__ float tree_weight(TreeRef a, TreeRef top, float scale) { return fast_exp2(tree_above(a, top, scale)); }

// 8 elements as they lie in the pools.
template <bool E4M3>
struct TreePiece {
    typedef uint4_t type;
};
template <>
struct TreePiece<true> {
    typedef uint2_t type;
};

// A scaled score less the rounded product of the reference and the scale, in one rounding, is off by up to half a step of the reference, a
// factor of a tile's probabilities: up to here (in units of log 2) 2^-13, beyond it the difference of a column comes before the scale.
constexpr float kTreeFar = 4096.0f;

// Matrix operands of a product, and how many of them are read ahead of it (heads wider than 128 are short of registers).
constexpr int tree_steps(int d) { return d / 16; }
constexpr int tree_lead(int d) { return d > 128 ? 2 : tree_steps(d) < 3 ? tree_steps(d) : 3; }

// Elements of the rings of a part, and workgroups that a compute unit holds (by LDS, and two waves to a SIMD by registers).
constexpr int tree_rings(int d) { return 2 * kTreeKeys * (d + 8 + (d / 32 % 2 ? d : d + 32)); }
constexpr int tree_blocks(int d, int colw, int parts) {
    return colw * parts > 4 || d > 128 || (d > 64 && parts > 1) || 2 * parts * tree_rings(d) > 80 * 1024 ? 1 : 2;
}

// COLW waves side by side hold a unit's columns, PARTS groups of them take its tiles in turn.  One wave alone moves K and V of its
// tiles itself and waits for nobody; otherwise half of a part's waves move K and half V.
template <typename T, int D, int COLW, int PARTS, bool E4M3>
__global__ __launch_bounds__(64 * COLW * PARTS, tree_blocks(D, COLW, PARTS)) void paged_attn_tree_kernel(const TreeParams p) {
    constexpr bool kAlone = COLW == 1;
    constexpr int kCols = 32 * COLW, kMovers = kAlone ? 64 : 32 * COLW;  // threads that move K, and V
    constexpr int kSteps = tree_steps(D), kTiles = D / 32;
    constexpr int kKRow = D + 8, kVRow = D / 32 % 2 ? D : D + 32;  // elements
    constexpr int kKTile = kTreeKeys * kKRow, kVTile = kTreeKeys * kVRow;
    constexpr int kStride = kTreeKeys * PARTS;         // keys between two tiles of a part
    constexpr int kPer = kTreeKeys * D / 8 / kMovers;  // pieces of 8 elements that a thread moves per tile
    constexpr int kPiece = E4M3 ? 8 : 16;              // their bytes
    constexpr int kRow = E4M3 ? D : 2 * D;             // bytes of a head row
    constexpr int kRings = tree_rings(D);
    static_assert(kRings == 2 * kKTile + 2 * kVTile, "two tiles each");
    constexpr int kTab = E4M3 && PARTS * D > 256 ? 128 : 256;  // tiles whose places are in LDS at a time
    constexpr int kPlaces = kTab + 4 * PARTS;                  // ... with those that a step may ask for behind the last
    constexpr bool kWide = D > 128;  // (short of registers)
    // Steps between asking for a tile and storing it: two, one where a wave alone has no registers for more.
    constexpr int kDeep = (kAlone && !E4M3 && D > 64) || kWide ? 1 : 2;
    constexpr bool kAsIs = E4M3 && __is_same(T, PackedBf16);  // K in bf16, whose range is that of the cache
    constexpr bool kUnits = E4M3 && !kAsIs;                   // the scores of a tile have a unit of their own
    static_assert(kPer * kMovers * 8 == kTreeKeys * D, "whole pieces");
    constexpr int kJoin = PARTS > 1 ? COLW * PARTS * tree_wave_floats(D) * 2 : 0;  // where the parts' results meet
    __shared__ __attribute__((aligned(16))) unsigned short lds[PARTS * kRings > kJoin ? PARTS * kRings : kJoin];
    __shared__ __attribute__((aligned(16))) int rows_lds[2 * kPlaces];
    __shared__ __attribute__((aligned(16))) uint8_t exps_lds[E4M3 ? 64 * kPlaces : 16];
    __shared__ __attribute__((aligned(16))) unsigned short tops_lds[E4M3 ? 2 * kPlaces : 8];
    __shared__ int odd_parts[PARTS];
    const int wave_of_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave_of_all / COLW, wave = wave_of_all - part * COLW;
    const int tid = threadIdx.x - part * 64 * COLW, lane = tid & 63, h = lane >> 5, col = lane & 31;
    unsigned short* const ks = lds + part * kRings;
    unsigned short* const vs = ks + 2 * kKTile;
    const bool moves_k = kAlone || wave < COLW / 2, moves_v = kAlone || wave >= COLW / 2;
    const int mover = tid % kMovers;
    const int s16 = lane & 15;
    const int v_lane = (4 * h + (s16 >> 2)) * kVRow + 16 * ((lane >> 4) & 1) + 4 * (s16 & 3);
    auto together = [&] LG_INLINE {
        if constexpr (kAlone) __builtin_amdgcn_wave_barrier();
        else __syncthreads();
    };

    int first = 0;  // of the 64 sequences that the next unit is in, and the tiles in front of them
    unsigned before = 0;
    TreeChunk chunk = tree_chunk<kCols>(0, 0);
    unsigned pos, end;
    if (p.whole) {
        const unsigned tiles = tree_unit_at<kCols>(chunk, p.num_seqs, blockIdx.x, pos);
        if (tiles == 0) return;
        end = pos + tiles;
    } else {
        unsigned total = chunk.end;
        for (int f = 64; f < p.num_seqs; f += 64) total = tree_chunk<kCols>(f, total).end;
        const unsigned per = tree_share(total, p.workers);
        pos = blockIdx.x * per;
        if (pos >= total) return;
        end = total - pos < per ? total : pos + per;
    }
    for (bool again = false; pos < end; again = true) {
        if (again) chunk = tree_chunk<kCols>(first, before);
        while (pos >= chunk.end) {
            first += 64;
            if (first >= p.num_seqs) return;  // (lengths that overlap: their tiles may be more than 32 bits count)
            before = chunk.end;
            chunk = tree_chunk<kCols>(first, before);
        }
        const TreeUnit u = tree_unit(chunk, p.hkv, pos);
        const int tile0 = u.tile;
        const int tile1 = (unsigned)(u.tiles - tile0) < end - pos ? u.tiles : tile0 + (int)(end - pos);
        pos += (unsigned)(tile1 - tile0);

        const TreeCold unit_cold = tree_cold();
        const int g = unit_cold->g, cols = u.rows * g;
        const int c0 = u.group * kCols + wave * 32;
        const bool active = c0 < cols;
        // This lane's token and head (worked out anew where they are needed: registers are what the loop is short of).
        struct Column {
            int tok, head;
        };
        auto column = [&] LG_INLINE {
            int c = c0 + col;
            asm volatile("" : "+v"(c));
            c = c < cols ? c : cols - 1;
            const int tok = c / g;
            return Column{tok, u.head * g + c - tok * g};
        };

        uint4_t qb[kSteps];
        {
            const Column c = column();
            const unsigned short* q =
                unit_cold->q + (int64_t)(u.row0 + c.tok) * unit_cold->q_stride + (int64_t)c.head * D + 8 * h;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) qb[j] = *reinterpret_cast<const uint4_t*>(q + 16 * j);
        }

        // ---- where the tiles lie: for kTab of them at a time in LDS, worked out by all threads together
        struct Place {
            int row[2];  // of the pools, at which the halves begin; -1: there is none, or the table's entry names no block
        };
        auto is_there = [](const Place& w) LG_INLINE { return (w.row[0] & w.row[1]) >= 0; };  // one half at least
        // A tile that all columns see, all of it.
        auto is_whole = [&](const Place& w, int key0) LG_INLINE {
            return (w.row[0] | w.row[1]) >= 0 && key0 + kTreeKeys <= u.prior;
        };
        // A key's entry of the table (-1: none) and row in its block; the entry's row of the pools, -1: it names no block.
        struct Entry {
            int block, off;
        };
        auto entry_of = [&](int key) LG_INLINE {
            const TreeCold t = tree_cold();
            const int entry = key / t->block_size;
            Entry e = {-1, key - entry * t->block_size};
            if (key < u.ctx) e.block = t->tables[(int64_t)u.seq * t->max_blocks + entry];
            if (e.block >= t->num_blocks) e.block = -1;
            return e;
        };
        auto row_of = [&](const Entry& e) LG_INLINE { return e.block < 0 ? -1 : e.block * p.block_size + e.off; };
        // First the rows, then (they are loaded while the first tiles are on their way) the exponents.
        constexpr int kThreads = 64 * COLW * PARTS, kRounds = (2 * kPlaces + kThreads - 1) / kThreads;
        auto half_key = [&](int i, int from, int count) LG_INLINE { return i < 2 * count ? from * kTreeKeys + 16 * i : u.ctx; };
        auto fill = [&](int from, int count, int halves, Entry (&entry)[kRounds]) LG_INLINE {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int i = threadIdx.x + r * kThreads;
                if (i < halves) {
                    entry[r] = entry_of(half_key(i, from, count));
                    rows_lds[i] = row_of(entry[r]);
                }
            }
        };
        auto fill_exps = [&](int from, int count, int halves, const Entry (&entry)[kRounds]) LG_INLINE {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int i = threadIdx.x + r * kThreads;
                if (i < halves) {
                    // the exponents of the 16 rows of K and of V (of those that there are), and the largest of each
                    const TreeCold t = tree_cold();
                    const Entry& at = entry[r];
                    const int64_t first = at.block < 0 ? 0 : ((int64_t)at.block * t->hkv + u.head) * t->block_size + at.off;
                    const int left = at.block < 0 ? 0 : u.ctx - half_key(i, from, count);
                    unsigned top[2];
                    uint4_t both[2];
                    both[0] = *reinterpret_cast<const uint4_t*>(t->k_exp + first);
                    both[1] = *reinterpret_cast<const uint4_t*>(t->v_exp + first);
                    const bool other_there = lane_xor_i32<1>(at.block) >= 0;
                    const bool whole = at.block >= 0 && other_there && half_key(i & ~1, from, count) + kTreeKeys <= u.prior;
#pragma unroll
                    for (int kind = 0; kind < 2; ++kind) {
                        uint4_t e = both[kind];
                        unsigned most = 0;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int bytes = left - 4 * w;
                            e[w] = bytes >= 4 ? e[w] : bytes > 0 ? e[w] & ((1u << (8 * bytes)) - 1u) : 0u;
                            most = max(max(most, e[w] >> 24), max(e[w] & 0xffu, max((e[w] >> 8) & 0xffu, (e[w] >> 16) & 0xffu)));
                        }
                        // (kept as what the rows are to be multiplied by, relative to the tile's largest; where not all columns see the same
                        // rows, as they come)
                        const unsigned other = (unsigned)lane_xor_i32<1>((int)most);
                        top[kind] = whole ? most : 127u;
                        const int top_of_tile = !whole || (kAsIs && kind == 0) ? 127 : (int)max(most, other);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            unsigned r4 = 0;
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                r4 |= (unsigned)max((int)((e[w] >> (8 * y)) & 0xffu) - top_of_tile + 127, 0) << (8 * y);
                            e[w] = r4;
                        }
                        *reinterpret_cast<uint4_t*>(exps_lds + (i >> 1) * 64 + 32 * kind + 16 * (i & 1)) = e;
                    }
                    tops_lds[i] = (unsigned short)(top[0] | top[1] << 8);
                }
            }
        };
        // Tile i of this part in the table: as it comes, in vector registers, and for the whole wave.
        auto place = [&](int i) LG_INLINE {
            return *reinterpret_cast<const uint2_t*>(rows_lds + 2 * (i * PARTS + part));
        };
        auto uniform = [](uint2_t v) LG_INLINE {
            return Place{{__builtin_amdgcn_readfirstlane((int)v[0]), __builtin_amdgcn_readfirstlane((int)v[1])}};
        };
        // The largest exponents of a tile's rows of K and V (0: every row is taken by its own).
        struct Tops {
            int k, v;
        };
        auto top_bytes = [&](int i) LG_INLINE { return *reinterpret_cast<const unsigned*>(tops_lds + 2 * (i * PARTS + part)); };
        auto tops_of = [&](unsigned bytes) LG_INLINE {
            const unsigned both = __builtin_amdgcn_readfirstlane(bytes);
            Tops t;
            t.k = max((int)(both & 0xffu), (int)((both >> 16) & 0xffu)) - 127;
            t.v = max((int)((both >> 8) & 0xffu), (int)(both >> 24)) - 127;
            if (kAsIs) t.k = 0;
            return t;
        };

        typedef typename TreePiece<E4M3>::type piece_t;
        struct Regs {
            piece_t k[kAlone ? kPer : 1], v[kPer];  // (of several waves: v holds whichever a wave moves)
        };
        // Piece i of a mover: of key key_of(i).  Where a round of the movers' pieces is whole keys, it lies kRound keys behind piece
        // i - 1 and one offset serves all; within a wave they are then of the same half of the tile.
        constexpr bool kEven = kMovers % (D / 8) == 0;
        constexpr int kRound = kMovers / (D / 8);
        auto key_of = [&](int i) LG_INLINE {
            return kEven ? mover / (D / 8) + kRound * i : (mover + kMovers * i) / (D / 8);
        };
        auto piece_of = [&](int i) LG_INLINE { return (mover + (kEven ? 0 : kMovers * i)) % (D / 8); };
        const unsigned row_bytes = (unsigned)p.hkv * kRow;
        const int wave_key = __builtin_amdgcn_readfirstlane(mover / (D / 8)) & ~15;  // (kEven: of which 16 keys piece 0 is)
        unsigned piece_at[kEven ? 1 : kPer];
#pragma unroll
        for (int i = 0; i < (kEven ? 1 : kPer); ++i)
            piece_at[i] = ((unsigned)key_of(i) & 15u) * row_bytes + (unsigned)(kPiece * piece_of(i));
        // (a half that is not there: the first rows of the pool; rows behind the last key lie in its block)
        auto load = [&](const uint8_t* pool, const Place& w, piece_t* x) LG_INLINE {
            const uint8_t* const half0 = pool + (int64_t)max(w.row[0], 0) * row_bytes + u.head * kRow;
            const uint8_t* const half1 = pool + (int64_t)max(w.row[1], 0) * row_bytes + u.head * kRow;
            // (a scalar base and 32-bit offsets: otherwise the compiler keeps 64-bit sums of everything that does not change)
            unsigned at0 = piece_at[0];
            asm volatile("" : "+v"(at0));
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if constexpr (kEven) {
                    const uint8_t* from = (wave_key + kRound * i < 16 ? half0 : half1) + (unsigned)(kRound * i % 16) * row_bytes;
                    x[i] = *reinterpret_cast<const piece_t*>(from + at0);
                } else {
                    x[i] = *reinterpret_cast<const piece_t*>((key_of(i) < 16 ? half0 : half1) + piece_at[i]);
                }
            }
        };
        // A piece of 8 as the kernel wants it: e4m3 rows times 2^(e - top) in 16 bits, those of a tile that is not whole as they are.
        auto decoded = [&](const piece_t& x, int e, bool as_bf16) LG_INLINE {
            if constexpr (!E4M3) return x;
            else {
            const float scale = __int_as_float(e << 23);
            uint4_t y;
            if (as_bf16) {
                y[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[0], scale, false));
                y[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[0], scale, true));
                y[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[1], scale, false));
                y[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[1], scale, true));
            } else {
                y[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[0], scale, false));
                y[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[0], scale, true));
                y[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[1], scale, false));
                y[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[1], scale, true));
            }
            return y;
            }
        };
        auto exps_at = [&](int i, int kind) LG_INLINE { return exps_lds + (i * PARTS + part) * 64 + 32 * kind; };
        // (a row's byte without a branch around its read: 1 where the tile is not whole)
        struct Byte {
            int keep, set;
        };
        auto byte_if = [](bool by_row) LG_INLINE { return by_row ? Byte{0xff, 0} : Byte{0, 127}; };
        auto store_k = [&](int buf, const piece_t* x, const uint8_t* e, const Place& w, int key0) LG_INLINE {
            unsigned short* const to = ks + buf * kKTile;
            const Byte which = byte_if(kAsIs || is_whole(w, key0));
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int row = E4M3 ? (e[key_of(i)] & which.keep) | which.set : 0;
                *reinterpret_cast<uint4_t*>(to + key_of(i) * kKRow + 8 * piece_of(i)) = decoded(x[i], row, kAsIs);
            }
        };
        // A key that a column does not see has the probability 0 there, and 0 times an infinity or NaN of its V row is NaN: in
        // tiles that are not seen whole such elements go in as 0, and are added at the end for the columns that see them, from the part's
        // first tile on in which there is one (of keys that somebody may see: what lies behind the last one costs nothing).
        auto store_v = [&](int buf, const piece_t* x, const uint8_t* e, const Place& w, int key0) LG_INLINE {
            unsigned short* const to = vs + buf * kVTile;
            if (__builtin_expect(is_whole(w, key0), 1)) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const int row = E4M3 ? e[key_of(i)] : 0;
                    *reinterpret_cast<uint4_t*>(to + key_of(i) * kVRow + 8 * piece_of(i)) = decoded(x[i], row, false);
                }
                return;
            }
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                uint4_t y = decoded(x[i], 127, false);
                const int key = key_of(i);
                const bool there = key0 + key < u.ctx && (key < 16 ? w.row[0] : w.row[1]) >= 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned bad = ((y[j] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                    odd |= there && bad != 0;
                    y[j] = !is_there(w) ? 0u : y[j] & ~((bad >> 15) * 0xffffu);
                }
                *reinterpret_cast<uint4_t*>(to + key * kVRow + 8 * piece_of(i)) = y;
            }
            // (several waves of a part, if more than one finds such an element first: in the same tile)
            if (__builtin_amdgcn_ballot_w64(odd) != 0 && lane == 0 && odd_parts[part] < 0) odd_parts[part] = key0 / kTreeKeys;
        };
        auto v_operand = [&](int buf, int kb, int dt) LG_INLINE {
            typedef short short4_t __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) short4_t lds_short4_t;
            const unsigned short* a = vs + buf * kVTile + v_lane + 16 * kb * kVRow + 32 * dt;
            const uint2_t lo = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)a));
            const uint2_t hi =
                __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(a + 8 * kVRow)));
            return uint4_t{lo[0], lo[1], hi[0], hi[1]};
        };
        auto k_operand = [&](int buf, int j) LG_INLINE {
            return *reinterpret_cast<const uint4_t*>(ks + buf * kKTile + col * kKRow + 16 * j + 8 * h);
        };
        // Which keys of a tile this column sees.
        auto window = [&](const Place& w, int key0) LG_INLINE {
            unsigned win = ~0u;
            const int j0 = key0 - u.prior;
            if (j0 > -32) {
                const TreeCold t = tree_cold();
                const int words = t->words;
                const uint32_t* const mask = t->mask + (int64_t)(u.row0 + column().tok) * words;
                auto word = [&](int i) LG_INLINE { return i < words ? mask[i] : 0u; };
                if (j0 < 0) {
                    win = word(0) << -j0 | ((1u << -j0) - 1u);
                } else {
                    const int i = j0 >> 5;
                    win = (unsigned)(((uint64_t)word(i + 1) << 32 | word(i)) >> (j0 & 31));
                }
            }
            const int left = u.ctx - key0;
            if (left < 32) win &= left > 0 ? (1u << left) - 1u : 0u;
            if (w.row[0] < 0) win &= 0xffff0000u;
            if (w.row[1] < 0) win &= 0x0000ffffu;
            return win;
        };

        TreeRef m;  // what the probabilities and sums of a column are relative to
        float l;
        float16_t o[kTiles];
        uint4_t p_prev[2];
        float16_t s_even, s_odd;  // scores of a tile by its parity

        // A tile that not all columns see all of, in front of its step: leaves in s_cur what the exponents of the probabilities are above the
        // reference, and for e4m3 rows the sum without those of V; returns what raising the reference takes off the exponents so far.
        // The exponents of e4m3 rows (at `exps`) go into the scores and into those of the probabilities key by key, so that a column has
        // to do with the keys alone that it sees: its reference is the largest sum of the two.
        auto apart = [&](float16_t& s_cur, const Place& w, int key0, const uint8_t* exps, float& sum) LG_INLINE {
            const float scale = p.scale_log2e;
            const unsigned win = window(w, key0) >> (4 * h);
            unsigned ek[4], ev[4];
            if constexpr (E4M3) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    ek[b] = *reinterpret_cast<const unsigned*>(exps + 8 * b + 4 * h);
                    ev[b] = *reinterpret_cast<const unsigned*>(exps + 32 + 8 * b + 4 * h);
                }
            }
            auto byte = [](const unsigned (&x)[4], int e) LG_INLINE { return (x[e >> 2] >> (8 * (e & 3))) & 0xffu; };
            float tm = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = kUnits ? ldexpf(s_cur[e], (int)byte(ek, e) - 127) : s_cur[e];
                const unsigned sees = (unsigned)((int)(win << (31 - (8 * (e >> 2) + (e & 3)))) >> 31);  // all bits, or none
                s_cur[e] = __uint_as_float((__float_as_uint(x) & sees) | (0xff800000u & ~sees));
                tm = fmaxf(tm, s_cur[e]);
            }
            tm = fmaxf(tm, lane_xor_f32<32>(tm));
            const float base = tm == -INFINITY ? 0.0f : tm;
            float most = -INFINITY;  // (e4m3: the exponents as their bytes)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s_cur[e] = E4M3 ? fmaf(s_cur[e] - base, scale, (float)byte(ev, e)) : (s_cur[e] - base) * scale;
                most = fmaxf(most, s_cur[e]);
            }
            most = E4M3 ? fmaxf(most, lane_xor_f32<32>(most)) - 127.0f : tm == -INFINITY ? tm : 0.0f;
            const bool none = tree_none(m);
            const float rel = fmaf(base - m.s, scale, most - m.v);
            // (a little before the step would do it)
            const bool up = none ? tm > -INFINITY : rel > kTreeLazy - 0.0625f;
            m.s = up ? tm : m.s;
            if (E4M3) m.v = up ? most : m.v;
            // (nothing to see: from anywhere, since the difference times the scale may be beyond fp32)
            const float off = (up ? -most : tm == -INFINITY ? 0.0f : fmaf(base - m.s, scale, -m.v)) - (E4M3 ? 127.0f : 0.0f);
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s_cur[e] += off;
                if (E4M3) sum += fast_exp2(s_cur[e] - (float)byte(ev, e) + (127.0f + kTreeHead));
            }
            return up ? (none ? -INFINITY : -rel) : 0.0f;
        };

        // Tile i with S(i) in s_cur (of parity H), K(i + 1) in K buffer 1 - H and V(i - 1) in V buffer 1 - H; leaves S(i + 1) and P(i).
        auto step = [&](auto h_c, const Place& w, int key0, const Tops& top, const uint8_t* exps) LG_INLINE {
            constexpr int H = decltype(h_c)::value;
            float16_t &s_cur = H ? s_odd : s_even, &s_nxt = H ? s_even : s_odd;
            const bool whole = is_whole(w, key0);
            // The tile's scores in its own unit, the reference in it and the exponents of V above that of the reference; what raising the reference
            // takes off the exponents so far.
            float scale = kUnits ? fminf(ldexpf(p.scale_log2e, top.k), 3e38f) : p.scale_log2e;
            float ref = kUnits ? ldexpf(m.s, -top.k) : m.s, v_above = E4M3 ? (float)top.v - m.v : 0.0f, drop = 0.0f;
            float sum_apart = 0.0f;
            if (__builtin_expect(!whole, 0)) {
                drop = apart(s_cur, w, key0, exps, sum_apart);
                scale = 1.0f;
                ref = v_above = 0.0f;
            }
            // The products in pairs of S and O, so that none waits for the one before it, operands kLead pairs ahead, and between any two of
            // them a share of the softmax: its maximum first, then the probabilities.
            constexpr int kLead = tree_lead(D), kSlots = 2 * kSteps, kFirst = kSlots * 3 / 16 > 2 ? kSlots * 3 / 16 : 2;
            static_assert(kLead <= kSteps, "no operand behind the last");
            uint4_t ka[kSteps], va[kSteps];
#pragma unroll
            for (int e = 0; e < 16; ++e) s_nxt[e] = 0.0f;
            float tm = -INFINITY, off = 0.0f, sum = 0.0f, even = 0.0f;
            uint4_t pb[2];
            auto read = [&](int j) LG_INLINE {
                ka[j] = k_operand(1 - H, j);
                va[j] = v_operand(1 - H, j / kTiles, j % kTiles);
            };
            auto share = [&](auto slot_c) LG_INLINE {
                constexpr int kSlot = decltype(slot_c)::value;
                if constexpr (kSlot == 0) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) tm = fmaxf(tm, s_cur[e]);
                }
                if constexpr (kSlot == kFirst - 1) {
                    tm = fmaxf(tm, lane_xor_f32<32>(tm));
                    const float rel = fmaf(tm - ref, scale, v_above);
                    off = fmaf(-ref, scale, kTreeHead + v_above);
                    const bool rare = !(rel <= kTreeLazy) | !(fabsf(ref * scale) < kTreeFar);  // (nothing seen so far: NaN)
                    if (__builtin_expect(__builtin_amdgcn_ballot_w64(rare) != 0, 0)) {
                        const bool none = tree_none(m), up = none ? tm > -INFINITY : rel > kTreeLazy;
                        drop = up ? (none ? -INFINITY : -rel) : drop;
                        m.s = up ? (kUnits ? ldexpf(tm, top.k) : tm) : m.s;
                        if (E4M3) m.v = up ? (float)top.v : m.v;
                        ref = up ? tm : none ? 0.0f : ref;
                        v_above = up ? 0.0f : v_above;
                        const bool far = !(fabsf(ref * scale) < kTreeFar);
                        const float by = far ? ref : 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) s_cur[e] -= by;
                        off = fmaf(far ? 0.0f : -ref, scale, kTreeHead + v_above);
                    }
                }
                static_for<16>([&](auto e_c) LG_INLINE {
                    constexpr int e = decltype(e_c)::value;
                    if constexpr (kFirst + e * (kSlots - kFirst) / 16 == kSlot) {
                        const float prob = fast_exp2(fmaf(s_cur[e], scale, off));
                        sum += prob;
                        if constexpr (e % 2 == 0) even = prob;
                        else pb[e >> 3][(e & 7) >> 1] = PackedF16::pack2(even, prob);
                    }
                });
            };
#pragma unroll
            for (int j = 0; j < kLead; ++j) read(j);
            static_for<kSteps>([&](auto step_c) LG_INLINE {
                constexpr int j = decltype(step_c)::value;
                if constexpr (j + kLead < kSteps) read(j + kLead);
                s_nxt = T::mfma32(ka[j], qb[j], s_nxt);
                share(ic<2 * j>{});
                __builtin_amdgcn_sched_barrier(0);
                o[j % kTiles] = PackedF16::mfma32(va[j], p_prev[j / kTiles], o[j % kTiles]);
                share(ic<2 * j + 1>{});
                __builtin_amdgcn_sched_barrier(0);
            });
            // (F belongs to this step: its results are used by the next one only, and would sink there)
            asm volatile("" : "+v"(pb[0]), "+v"(pb[1]), "+v"(sum));
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(drop != 0.0f) != 0, 0)) {  // O(i - 1) was relative to the old one
                const float alpha = fast_exp2(drop);
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
            }
            l += !E4M3 ? sum : whole ? ldexpf(sum, -top.v) : sum_apart;
            p_prev[0] = pb[0];
            p_prev[1] = pb[1];
        };

        // The tiles of the part.
        auto walk_tiles = [&] LG_INLINE {
            for (int from = tile0; from < tile1; from += kTab) {
                const int count = min(tile1 - from, kTab), steps = (count + PARTS - 1) / PARTS;
                if (from != tile0) __syncthreads();  // (the last waves are done with the table)
                const int halves = 2 * (steps + 4) * PARTS;
                Entry entry[kRounds];
                fill(from, count, halves, entry);
                __syncthreads();
                int key0 = (from + part) * kTreeKeys;  // of tile i
                p_prev[0] = p_prev[1] = uint4_t{0, 0, 0, 0};
                Place w0 = uniform(place(0)), w1 = uniform(place(1)), w2 = uniform(place(2)), w3 = w2;
                uint2_t ahead = place(1 + kDeep);
                unsigned tops_ahead = 0;
                Regs ra, rb;
                Tops t0 = {0, 0}, t1 = {0, 0}, t2 = {0, 0};
                auto kregs = [](Regs& r) LG_INLINE { return kAlone ? r.k : r.v; };
                // K out of `lead` and V out of `behind`; of several waves each its own kind
                auto ask = [&](const Place& lead, const Place& behind, Regs& r) LG_INLINE {
                    if constexpr (kAlone) {
                        load(p.k_pool, lead, r.k);
                        load(p.v_pool, behind, r.v);
                    } else {
                        const Place w = {{moves_v ? behind.row[0] : lead.row[0], moves_v ? behind.row[1] : lead.row[1]}};
                        load(moves_v ? p.v_pool : p.k_pool, w, r.v);
                    }
                };
                {
                    piece_t x0[kPer];
                    load(p.k_pool, w0, x0);
                    load(p.k_pool, w1, kregs(rb));
                    if constexpr (kDeep == 2) ask(w2, w0, ra);
                    if constexpr (E4M3) {
                        fill_exps(from, count, halves, entry);
                        __syncthreads();
                        t0 = tops_of(top_bytes(0));
                        t1 = tops_of(top_bytes(1));
                        tops_ahead = top_bytes(2);
                    }
                    if (moves_k) {
                        store_k(0, x0, exps_at(0, 0), w0, key0);
                        store_k(1, kregs(rb), exps_at(1, 0), w1, key0 + kStride);
                    }
                }
                // V buffer 1 plays V(-1) in the first step, whose P is 0: finite values
                for (int i = tid; i < kVTile / 2; i += 64 * COLW) reinterpret_cast<unsigned*>(vs + kVTile)[i] = 0u;
                together();
#pragma unroll
                for (int e = 0; e < 16; ++e) s_even[e] = 0.0f;
#pragma unroll
                for (int j = 0; j < kSteps; ++j) s_even = T::mfma32(k_operand(0, j), qb[j], s_even);
                together();  // (the first step ends with a store into the buffer just read)
                // step i, H its parity: what a later step needs is asked for in front of it and goes to LDS behind it
                auto one = [&](auto h_c, int i, Regs& now, Regs& next) LG_INLINE {
                    constexpr int H = decltype(h_c)::value;
                    Place& lead = kDeep == 2 ? w3 : w2;
                    lead = uniform(ahead);
                    ahead = place(i + 2 + kDeep);
                    ask(lead, kDeep == 2 ? w1 : w0, next);
                    if constexpr (E4M3) {
                        t2 = tops_of(tops_ahead);
                        tops_ahead = top_bytes(i + 3);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (COLW >= 4 && D >= 96) __builtin_amdgcn_s_setprio(1);
                    if (active) step(h_c, w0, key0, t0, exps_at(i, 0));
                    if constexpr (COLW >= 4 && D >= 96) __builtin_amdgcn_s_setprio(0);
                    __builtin_amdgcn_sched_barrier(0);
                    Regs& then = kDeep == 2 ? now : next;
                    // (waited for here, whichever of the two follows: not known to have arrived, they would be waited for with the next ones)
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        if constexpr (kAlone) asm volatile("" : "+v"(then.k[j]));
                        asm volatile("" : "+v"(then.v[j]));
                    }
                    if (moves_k) store_k(H, kregs(then), exps_at(i + 2, 0), w2, key0 + 2 * kStride);  // K(i + 2)
                    if (moves_v) store_v(H, then.v, exps_at(i, 1), w0, key0);  // V(i)
                    t0 = t1;
                    t1 = t2;
                    w0 = w1;
                    w1 = w2;
                    w2 = w3;
                    key0 += kStride;
                    together();
                };
                int i = 0;
                for (; i + 1 < steps; i += 2) {
                    one(ic<0>{}, i, ra, rb);
                    one(ic<1>{}, i + 1, rb, ra);
                }
                if (i < steps) one(ic<0>{}, i, ra, rb);
                const int buf = (steps - 1) & 1;
                if (active) {
#pragma unroll
                    for (int j = 0; j < kSteps; ++j)
                        o[j % kTiles] = PackedF16::mfma32(v_operand(buf, j / kTiles, j % kTiles), p_prev[j / kTiles], o[j % kTiles]);
                }
            }
        };

        if (wave_of_all == 0 && lane < PARTS) odd_parts[lane] = -1;
        __syncthreads();
        m = TreeRef{NAN, 0.0f};
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
        if (u.ctx > 0) walk_tiles();
        __syncthreads();
        const int odd0 = __builtin_amdgcn_readfirstlane(odd_parts[part]);
        if (__builtin_expect(odd0 >= 0, 0)) {
            for (int tile = odd0; tile < tile1 && active; ++tile) {
                const int key0 = tile * kTreeKeys;
                const Place w = {{__builtin_amdgcn_readfirstlane(row_of(entry_of(key0))),
                                  __builtin_amdgcn_readfirstlane(row_of(entry_of(key0 + 16)))}};
                // (each part for its own tiles: the parts are added up)
                if ((tile - tile0) % kTab % PARTS != part || !is_there(w) || is_whole(w, key0)) continue;
                const unsigned win = window(w, key0);
                for (int key = 0; key < kTreeKeys; ++key) {
                    const bool sees = (win >> key) & 1u;
                    if (__builtin_amdgcn_ballot_w64(sees) == 0) continue;  // (nobody: perhaps it is not there)
                    const uint8_t* row =
                        p.v_pool + ((int64_t)(key < 16 ? w.row[0] : w.row[1]) + (key & 15)) * row_bytes + u.head * kRow;
#pragma unroll
                    for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int at = 32 * dt + 8 * (e >> 2) + 4 * h + (e & 3);
                            float v;
                            if constexpr (E4M3) v = (row[at] & 0x7f) == 0x7f ? NAN : 0.0f;
                            else v = (float)reinterpret_cast<const _Float16*>(row)[at];
                            o[dt][e] += sees && !(fabsf(v) < INFINITY) ? v : 0.0f;
                        }
                }
            }
        }
        l += lane_xor_f32<32>(l);
        __syncthreads();  // (the next unit's tiles, and the columns on their way out, go where the last tiles were)
        const bool all = tile0 == 0 && tile1 == u.tiles;
        // a part of a unit: slot 1 of the workgroup holds the end of one, slot 0 everything else
        const TreeCold t = tree_cold();
        float* const slot = t->ws + ((int64_t)(2 * blockIdx.x + (tile1 == u.tiles ? 1 : 0)) * t->slot_waves + wave) *
                                        tree_wave_floats(D);
        if constexpr (PARTS == 1) {
            if (!active) continue;
            if (all) {
                const int tok0 = c0 / g;
                const Column c = column();
                static_assert(COLW * 16 * (D + 8) <= kRings, "the columns on their way out fit");
                attn_packed_write<T, D>(t->out + (int64_t)(u.row0 + tok0) * t->out_stride,
                                        (unsigned)(c.tok - tok0) * (unsigned)t->out_stride + (unsigned)(c.head * D), cols - c0,
                                        lds + wave * 16 * (D + 8), o, l);
            } else {
#pragma unroll
                for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4)
                        reinterpret_cast<float4_t*>(slot)[(4 * dt + q4) * 64 + lane] =
                            float4_t{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
                slot[32 * D + lane] = h ? m.v : m.s;
                slot[32 * D + 64 + lane] = l;
            }
        } else {
            // the parts through LDS; of a wave's 32 columns each part then joins every PARTS-th 32 elements
            float* const mine = reinterpret_cast<float*>(lds) + (wave * PARTS + part) * tree_wave_floats(D);
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    reinterpret_cast<float4_t*>(mine)[(4 * dt + q4) * 64 + lane] =
                        float4_t{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
            mine[32 * D + lane] = h ? m.v : m.s;
            mine[32 * D + 64 + lane] = l;
            __syncthreads();
            if (active) {
                const float* const parts = reinterpret_cast<const float*>(lds) + wave * PARTS * tree_wave_floats(D);
                TreeRef refs[PARTS], top = {NAN, 0.0f};
                float weight[PARTS], sum = 0.0f;
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    refs[q] = {parts[q * tree_wave_floats(D) + 32 * D + col], parts[q * tree_wave_floats(D) + 32 * D + 32 + col]};
                    if (tree_above(refs[q], top, t->scale_log2e) > 0.0f) top = refs[q];
                }
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    weight[q] = tree_weight(refs[q], top, t->scale_log2e);
                    sum += parts[q * tree_wave_floats(D) + 32 * D + 64 + lane] * weight[q];
                }
                const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
                const Column c = column();
                unsigned short* const out =
                    t->out + (int64_t)(u.row0 + c.tok) * t->out_stride + (int64_t)c.head * D + 4 * h;
                for (int dt = part; dt < kTiles; dt += PARTS)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        float4_t v = {0, 0, 0, 0};
#pragma unroll
                        for (int q = 0; q < PARTS; ++q) {
                            const float4_t w = reinterpret_cast<const float4_t*>(parts + q * tree_wave_floats(D))[(4 * dt + q4) * 64 + lane];
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] += w[e] * weight[q];
                        }
                        if (!all) reinterpret_cast<float4_t*>(slot)[(4 * dt + q4) * 64 + lane] = v;
                        else if (c0 + col < cols)
                            *reinterpret_cast<uint2_t*>(out + 32 * dt + 8 * q4) =
                                uint2_t{T::pack2(v[0] * inv, v[1] * inv), T::pack2(v[2] * inv, v[3] * inv)};
                    }
                if (!all && part == 0) {
                    slot[32 * D + lane] = h ? top.v : top.s;
                    slot[32 * D + 64 + lane] = sum;
                }
            }
            __syncthreads();
        }
    }
}

// The units that were cut: a workgroup takes the first cut of one (or the unit), 32 of its columns and 8 Q elements of the heads, its
// waves every fourth part of the unit, a few of them in flight.
// (E4M3 keeps the instances of two source files apart.)
template <typename T, int D, int COLW, int Q, bool E4M3>
__global__ __launch_bounds__(256) void paged_attn_tree_merge_kernel(const TreeParams p) {
    constexpr int kCols = 32 * COLW, kPieces = D / 8 / Q, kAhead = 16 / Q;
    __shared__ float4_t theirs[3][Q][64];
    __shared__ float ml[3][3][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int piece = blockIdx.x % kPieces;
    const int of_unit = blockIdx.x / kPieces % p.slot_waves;     // which 32 columns of a unit
    const int cut = (int)(blockIdx.x / kPieces) / p.slot_waves;  // behind the tiles of this workgroup, or the unit
    TreeChunk c = tree_chunk<kCols>(0, 0);
    unsigned total = c.end;
    for (int first = 64; first < p.num_seqs; first += 64) total = tree_chunk<kCols>(first, total).end;
    const unsigned per = tree_share(total, p.workers);
    TreeUnit u;
    if (p.by_unit) {
        unsigned pos;
        if (tree_unit_at<kCols>(c, p.num_seqs, cut, pos) == 0) return;
        u = tree_unit(c, p.hkv, pos);
    } else {
        const unsigned pos = (unsigned)(cut + 1) * per;
        if (pos >= total) return;
        while (pos >= c.end) {
            if (c.first + 64 >= p.num_seqs) return;
            c = tree_chunk<kCols>(c.first + 64, c.end);
        }
        u = tree_unit(c, p.hkv, pos);
        if (u.tile == 0) return;
    }
    const unsigned begin = u.at - (unsigned)u.tile;
    const int first = (int)(begin / per), last = (int)((begin + (unsigned)u.tiles - 1) / per);
    const int cols = u.rows * p.g, c0 = u.group * kCols + of_unit * 32;
    if (first == last || (!p.by_unit && first != cut) || c0 >= cols) return;

    TreeRef m = {NAN, 0.0f};
    float l = 0.0f;
    float4_t o[Q];
#pragma unroll
    for (int q4 = 0; q4 < Q; ++q4) o[q4] = float4_t{0, 0, 0, 0};
    auto join = [&](TreeRef m2, float l2, const float4_t* o2) LG_INLINE {
        const float above = tree_above(m2, m, p.scale_log2e);
        const bool up = above > 0.0f;
        const float other = fast_exp2(-fabsf(above)), mine = up ? other : 1.0f, its = up ? 1.0f : other;
        m = {up ? m2.s : m.s, up ? m2.v : m.v};
        l = l * mine + l2 * its;
#pragma unroll
        for (int q4 = 0; q4 < Q; ++q4)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[q4][e] = o[q4][e] * mine + o2[q4][e] * its;
    };
    for (int w0 = first + wave; w0 <= last; w0 += 4 * kAhead) {
        float4_t o2[kAhead][Q];
        TreeRef m2[kAhead];
        float l2[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int w = w0 + 4 * a <= last ? w0 + 4 * a : w0;
            const float* slot =
                p.ws + ((int64_t)(2 * w + (w == last ? 1 : 0)) * p.slot_waves + of_unit) * tree_wave_floats(D);
            m2[a] = {slot[32 * D + (lane & 31)], slot[32 * D + 32 + (lane & 31)]};
            l2[a] = slot[32 * D + 64 + lane];
#pragma unroll
            for (int q4 = 0; q4 < Q; ++q4) o2[a][q4] = reinterpret_cast<const float4_t*>(slot)[(Q * piece + q4) * 64 + lane];
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (w0 + 4 * a <= last) join(m2[a], l2[a], o2[a]);
    }
    if (wave > 0) {
#pragma unroll
        for (int q4 = 0; q4 < Q; ++q4) theirs[wave - 1][q4][lane] = o[q4];
        ml[wave - 1][0][lane] = m.s;
        ml[wave - 1][1][lane] = m.v;
        ml[wave - 1][2][lane] = l;
    }
    __syncthreads();
    if (wave > 0) return;
    for (int w = 0; w < 3; ++w) {
        float4_t o2[Q];
#pragma unroll
        for (int q4 = 0; q4 < Q; ++q4) o2[q4] = theirs[w][q4][lane];
        join({ml[w][0][lane], ml[w][1][lane]}, ml[w][2][lane], o2);
    }
    const int h = lane >> 5, gc = c0 + (lane & 31);
    if (gc >= cols) return;
    const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
    const int tok = gc / p.g, head = u.head * p.g + gc - tok * p.g;
    unsigned short* out = p.out + (int64_t)(u.row0 + tok) * p.out_stride + (int64_t)head * D + 8 * Q * piece + 4 * h;
#pragma unroll
    for (int q4 = 0; q4 < Q; ++q4)
        *reinterpret_cast<uint2_t*>(out + 8 * q4) =
            uint2_t{T::pack2(o[q4][0] * inv, o[q4][1] * inv), T::pack2(o[q4][2] * inv, o[q4][3] * inv)};
}

inline int tree_slot_waves(int max_q, int g, int waves) {
    const int64_t need = ((int64_t)max_q * g + 31) / 32;
    return need < waves ? (int)need : waves;
}

template <typename T, int D, int COLW, int PARTS, bool E4M3>
static hipError_t tree_launch_as(TreeParams p, hipStream_t stream) {
    p.slot_waves = tree_slot_waves(p.max_q, p.g, COLW);
    const int64_t most = packed_tiles(p.total, p.num_seqs, p.g, 32 * COLW) * p.hkv;  // units
    const int64_t room = (int64_t)p.block_size * p.max_blocks;
    const int64_t tiles = most * ((room + kTreeKeys - 1) / kTreeKeys);
    // Few tiles to a unit: a workgroup for every unit, whole, and no second launch.  us, cut / whole, 12 / 2 heads of 128, 7 rows behind 300:
    // 15.2 / 13.4; 32 / 8, 16 rows behind 184: 21.6 / 14.5; four times 40 behind 210: 19.3 / 16.5; but heads of 256, 8 rows behind 242 eight times: 15.0 / 18.6.
    p.whole = (room + kTreeKeys - 1) / kTreeKeys <= (D > 128 ? 4 : 8) * PARTS;
    if (p.whole) {
        paged_attn_tree_kernel<T, D, COLW, PARTS, E4M3><<<(unsigned)most, 64 * COLW * PARTS, 0, stream>>>(p);
        return hipGetLastError();
    }
    int64_t workers = tree_blocks(D, COLW, PARTS) * device_cu_count();
    if (workers > kTreeWorkers * 4 / (COLW > 4 ? COLW : 4)) workers = kTreeWorkers * 4 / (COLW > 4 ? COLW : 4);
    if (workers > (tiles + kTreeLeast - 1) / kTreeLeast) workers = (tiles + kTreeLeast - 1) / kTreeLeast;
    p.workers = (int)workers;
    p.by_unit = most < workers;
    paged_attn_tree_kernel<T, D, COLW, PARTS, E4M3><<<(unsigned)workers, 64 * COLW * PARTS, 0, stream>>>(p);
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess || workers == 1) return rc;
    // (32 elements of the heads to a workgroup where there are enough of them, 8 otherwise)
    const int64_t groups = (p.by_unit ? most : workers - 1) * p.slot_waves;
    if (groups * (D / 32) >= device_cu_count() / 2)
        paged_attn_tree_merge_kernel<T, D, COLW, 4, E4M3><<<(unsigned)(groups * (D / 32)), 256, 0, stream>>>(p);
    else
        paged_attn_tree_merge_kernel<T, D, COLW, 1, E4M3><<<(unsigned)(groups * (D / 8)), 256, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T, int D, bool E4M3>
static hipError_t tree_launch(const TreeParams& p, hipStream_t stream) {
    const int64_t cols = (int64_t)p.max_q * p.g;  // of the longest tree
    if constexpr (D <= 128) {
        const int64_t units = packed_tiles(p.total, p.num_seqs, p.g, 128) * p.hkv;
        const int64_t tiles = ((int64_t)p.block_size * p.max_blocks + kTreeKeys - 1) / kTreeKeys;
        // Up to 64 columns: the waves that have none take tiles of their own, which pays where workgroups have few tiles or many, not
        // between, where joining the parts costs more.  us, parts / four waves side by side, heads of 128, by 32-key tiles of all units, e4m3 and
        // fp16: up to 32 columns 1000 21.7 / 28.2 and 20.4 / 26.0, 1024 18.3 / 20.2 and 17.2 / 18.2, 4000 32.5 / 29.3 and 30.3 / 26.1, 4750 33.1 / 28.2
        // and 30.5 / 25.9, 9954 40.0 / 35.6 and 37.3 / 34.0, 16384 42.9 / 44.2 and 53.3 / 55.3, 19000 52.0 / 48.8 and 53.6 / 54.2 (but 256 18.5 / 16.1 and
        // 17.0 / 14.2); up to 64 columns 1000 24.3 / 30.8 and 23.1 / 29.8, 1280 21.4 / 24.1 and 19.8 / 22.7, 5500 35.1 / 32.4 and 31.6 / 28.7, 11466 46.5 / 42.1
        // and 40.2 / 39.4, 16384 57.3 / 52.1 and 55.5 / 59.4.
        const bool between = units * tiles >= 4 * kTreeWorkers && units * tiles < 24 * kTreeWorkers;
        if (cols <= 32 && (!between || tiles <= 32)) return tree_launch_as<T, D, 1, 4, E4M3>(p, stream);
        if (cols <= 64 && (!between || tiles <= 16)) return tree_launch_as<T, D, 2, 2, E4M3>(p, stream);
        // Few units of many tiles over fp16 pools: eight waves of two parts, one workgroup to a compute unit, leave half as many parts of units to be
        // put together as two workgroups of four waves do.  us, four / eight waves, 32 / 8 heads of 128, 28 rows: one context of 131072 124.8 / 119.0,
        // of 65536 66.8 / 62.9, four of 40000, 24 rows, 148.6 / 140.8; heads of 96 98.3 / 99.0, 52.6 / 51.5, 115.9 / 110.3; but of 64 72.5 / 71.2,
        // 43.5 / 43.4, 82.3 / 85.0, and e4m3, whose step is short of registers in eight waves, 109.6 / 106.6, 61.2 / 61.8, 118.3 / 127.9.
        if constexpr (!E4M3 && D >= 96)
            if (cols > 64 && cols <= 128 && units <= 64 && units * tiles >= 16 * kTreeWorkers)
                return tree_launch_as<T, D, 4, 2, E4M3>(p, stream);
    }
    // More than 128 columns of heads of 64 and 128: eight waves, which read a tile once where two workgroups of four read it twice.  us, four / eight
    // waves, e4m3 and fp16: 32 contexts of 1000 to 8192, 256 columns of heads of 128, 217 / 200 and 225 / 203; of 4096, 448 columns of heads of 64,
    // 76.3 / 75.8 and 72.6 / 67.7; 64 contexts of 1000, 168 columns of them, 35.3 / 31.8 and 31.7 / 28.7; 210 columns 45.0 / 44.5 and 40.5 / 39.9.  It loses where
    // the last eight waves have few columns, which the rule does not look at: 280 columns 65.6 / 75.6 and 57.7 / 66.9, 336 65.9 / 75.9 and 59.5 / 67.0.
    if constexpr (D == 64 || D == 128)
        if (cols > 128) return tree_launch_as<T, D, 8, 1, E4M3>(p, stream);
    return tree_launch_as<T, D, 4, 1, E4M3>(p, stream);
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

// The launches of each source file.
hipError_t tree_launch_fp16(const TreeParams& p, int d, hipStream_t stream);
hipError_t tree_launch_e4m3_fp16(const TreeParams& p, int d, hipStream_t stream);
hipError_t tree_launch_e4m3_bf16(const TreeParams& p, int d, hipStream_t stream);

}  // namespace lg
