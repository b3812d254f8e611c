// Attention of whole packed sequences: q, k and v are rows of the same tokens, sequences one behind the
// other (cu_seqlens), causal or over the whole sequence, G = num_q_heads / num_kv_heads query heads per KV head.
//
// A column is a (token, head of the group) pair of one KV head, in that order over the sequence.  A wave owns 32 columns,
// their queries in registers; a workgroup's waves share the key tiles in LDS.  Per tile of 32 keys:
//
//   S^T[32 keys x 32 columns] = K . Q^T         v_mfma_f32_32x32x16
//   online softmax of a column, which lives in two lanes (fp32)
//   O^T[D x 32 columns] += V^T . P              v_mfma_f32_32x32x16
//
// The result layout of S^T is the operand layout of P when the keys of a step of 16 are taken in the order
// 4h + i, 8 + 4h + i (h: half of the wave, i < 4); V comes out of its row-major tile in that order through the
// transposing LDS read.  P goes in rounded to the rows' type: every term is off by at most half a step of that type
// relative to itself, as every output is by its own rounding (fp16: terms below 2^-25 of the largest by more, see ApRange).
// The errors against 64 bits are a quarter to a third above those of unrounded probabilities; a second term, as the decode rows of the paged
// form have it, would be half as many products again.
//
// Schedule: the stages of a tile -- S(t) and O(t) on the matrix cores, F(t), the softmax, on the vector units -- run
// one behind the other in a wave: step t issues S(t + 1) and O(t - 1) around F(t), so that the products of a step
// do not depend on its vector work and the two can be interleaved instruction by instruction.  K is stored into LDS two
// tiles ahead of its use and V one step, each by half of the waves; the rings are two deep.  Rows of K lie 2 D + 16 bytes
// apart and those of V an odd multiple of 64: the operand reads of 16 (32) lanes then touch every bank once.
//
// Few long sequences: HALVES == 2, twice the waves, of which the second part takes every other key tile; its sums join the
// first part's, each relative to its own maximum, through LDS.
//
// Bound by the matrix cores at heads of 128 and long sequences (one prompt of 16384 tokens, 32 / 8 heads: 1950 to 2150 us by card, 1020 to
// 1130 TFLOP/s, a large matrix product of the library 1130; the first few calls on a card that has rested take 2270); by the vector units at
// heads of 64 (per step 76 vector instructions, 16 of them exponentials, to 8 products; nothing but those takes 520 clocks a step, this
// 770, of which a barrier and a store into LDS for every 32 keys are a part: 4 prompts of 8192, 14 / 2 heads, 580 us, 830 TFLOP/s).
//
// The step is that of the paged prefill kernel (paged_attn.hip) with width and type as parameters: a change to one concerns the other.
#include "device_utils.hpp"
#include "launch_common.hpp"
#include "packed_rows.hpp"
#include "q4_common.hpp"

#include <math.h>

namespace lg {

struct AttnPackedParams {
    const unsigned short* q;
    const unsigned short* k;
    const unsigned short* v;
    const int32_t* cu;
    unsigned short* out;
    int num_seqs, total, hkv, g;
    int64_t q_stride, k_stride, v_stride, out_stride;
    float scale_log2e;
    int causal;
    int ordered;  // longest sequences first
};

constexpr int kApKeys = 32;

// What the exponentials are taken relative to is a reference that follows the maximum lazily: it is raised when a tile
// exceeds it by more than 2^kLazy, so that rescaling the sums is rare.  The largest probability of a column then lies between
// 2^kHead and 2^(kHead + kLazy); numerator and denominator carry the same factor.
//
// fp16 ends at 2^16 and loses bits below 2^-14, so its probabilities start as high as they can: those down to 2^-25 of a column's largest
// keep all bits, smaller ones are off by up to 2^-36 of it.  (With the largest at 1, 16384 keys at 2^-21.5 of one whose row of V is
// zero were off by 6 %, and below 2^-25 they vanished.)
//
// bf16 has the exponents of fp32, and V may hold anything up to 2^128: probabilities of at most 2^-24 add up to less than that over
// the 2^23 keys that there can be, so that finite values have a finite mean.  Those below 2^-94 of a column's largest vanish.
template <typename T>
struct ApRange;
template <>
struct ApRange<PackedF16> {
    static constexpr float kHead = 11.0f, kLazy = 4.0f;
};
template <>
struct ApRange<PackedBf16> {
    static constexpr float kHead = -32.0f, kLazy = 8.0f;
};

// The reference for a maximum.  (Not fused: the constant is then part of the instruction, and needs no register.)
template <typename T>
__device__ __forceinline__ float attn_packed_reference(float top, float scale_log2e) {
    float scaled = top * scale_log2e;
    asm("" : "+v"(scaled));
    return scaled - ApRange<T>::kHead;
}

// Probabilities of the 16 keys that a lane holds of its column (keys first + 8 (e / 4) + e % 4), the running maximum (of the
// scores as they are: their differences are taken before the scale) and sum; returns what the sums so far are to be
// multiplied by.
template <typename T>
__device__ __forceinline__ float attn_packed_softmax(float16_t sc, int first, int vis, float scale_log2e, float& m,
                                                     float& l, uint4_t (&pb)[2]) {
    float tm = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        sc[e] = first + 8 * (e >> 2) + (e & 3) < vis ? sc[e] : -INFINITY;
        tm = fmaxf(tm, sc[e]);
    }
    tm = fmaxf(tm, lane_xor_f32<32>(tm));
    const float m_new = fmaxf(m, tm);
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = fast_exp2((m - ref) * scale_log2e);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        const float p0 = fast_exp2(fmaf(sc[e] - ref, scale_log2e, ApRange<T>::kHead));
        const float p1 = fast_exp2(fmaf(sc[e + 1] - ref, scale_log2e, ApRange<T>::kHead));
        l += p0 + p1;
        pb[e >> 3][(e & 7) >> 1] = T::pack2(p0, p1);
    }
    return alpha;
}

// Of a V operand of 16 keys (lane: keys 4 h .. + 3 and 8 + 4 h .. + 3 of them) the first ones, the others zero: `keys` counts
// from key 4 h of the tile of 32.
__device__ __forceinline__ uint4_t attn_packed_first_keys(uint4_t v, int kb, int keys) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int at = 16 * kb + 2 * w + (w > 1 ? 4 : 0);
        v[w] &= keys >= at + 2 ? ~0u : keys == at + 1 ? 0xffffu : 0u;
    }
    return v;
}

// A scaled score less the rounded product of the maximum and the scale, in one rounding: off by up to half a step of the
// maximum, the same for all keys of a column.  Up to here that is at most 1 in the exponent and falls out of the result.
constexpr float kApExact = 16777216.0f;
// The reference of a column that has seen nothing above -inf yet: finite, so that such a key weighs 0 without a test, and so far
// down that whoever still has it in the end goes the plain way.
constexpr float kApNone = -3e38f;

template <typename T, int D, int WAVES, int HALVES>
__global__ __launch_bounds__(64 * WAVES * HALVES) void attn_packed_kernel(const AttnPackedParams p) {
    constexpr int kCols = 32 * WAVES, kMovers = 32 * WAVES;  // threads that move K, and V
    constexpr int kSteps = D / 16, kTiles = D / 32;  // operands of K (and of V) per key tile; output tiles
    constexpr int kKRow = D + 8, kVRow = D / 32 % 2 ? D : D + 32;  // elements
    constexpr int kKTile = kApKeys * kKRow, kVTile = kApKeys * kVRow;
    constexpr int kPer = kApKeys * D / 8 / kMovers;      // 16-byte pieces that a thread moves per tile
    constexpr int kRings = 2 * kKTile + 2 * kVTile;
    __shared__ __attribute__((aligned(16))) unsigned short lds[HALVES * kRings];
    __shared__ unsigned odd_waves[WAVES * HALVES];
    const int wave_of_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = HALVES == 1 ? 0 : wave_of_all / WAVES;  // (takes the key tiles HALVES t + part)
    const int wave = wave_of_all - part * WAVES, tid = threadIdx.x - part * 64 * WAVES, lane = tid & 63;
    unsigned short* const ks = lds + part * kRings;
    unsigned short* const vs = ks + 2 * kKTile;
    const int h = lane >> 5, col = lane & 31;
    const int kvh = (int)(blockIdx.x % (unsigned)p.hkv);
    const int at = (int)(blockIdx.x / (unsigned)p.hkv);
    const PackedTile t = p.ordered != 0 ? packed_tile_ordered(p.cu, p.num_seqs, p.total, p.g, kCols, at)
                                                      : packed_tile(p.cu, p.num_seqs, p.total, p.g, kCols, at);
    const int cols = t.rows * p.g;
    const int groups = (cols + kCols - 1) / kCols;
    const int group = groups - 1 - t.tile;  // (the last columns see the most keys: they start first)
    if (t.rows <= 0 || group < 0) return;
    const int c0 = group * kCols + wave * 32;
    const int gc = c0 + col;
    const bool live = gc < cols;
    const int tok = (live ? gc : cols - 1) / p.g, head = kvh * p.g + (live ? gc : cols - 1) % p.g;
    const int vis = p.causal ? tok + 1 : t.rows;  // keys of this lane's column
    const int last = (group + 1) * kCols < cols ? (group + 1) * kCols - 1 : cols - 1;
    const int visible = p.causal ? last / p.g + 1 : t.rows;  // ... of the workgroup's last
    const int all_see = p.causal ? group * kCols / p.g + 1 : t.rows;  // ... of the workgroup's first
    const int first_vis = p.causal ? (c0 < cols ? c0 : cols - 1) / p.g + 1 : t.rows;  // ... of the wave's first
    const int last_vis = p.causal ? (c0 + 31 < cols ? c0 + 31 : cols - 1) / p.g + 1 : t.rows;

    uint4_t qb[kSteps];
    {
        const unsigned short* q = p.q + (int64_t)(t.row0 + tok) * p.q_stride + (int64_t)head * D + 8 * h;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) qb[j] = *reinterpret_cast<const uint4_t*>(q + 16 * j);
    }

    // ---- movement: the first half of a part's waves carries K, the second V, a thread kPer pieces of 16 bytes of a tile
    const bool moves_v = wave >= WAVES / 2;
    const int64_t stride = moves_v ? p.v_stride : p.k_stride;
    const unsigned short* const src = (moves_v ? p.v : p.k) + (int64_t)t.row0 * stride + (int64_t)kvh * D;
    struct Regs {
        uint4_t x[kPer];
    };
    auto key_of = [&](int u) LG_INLINE { return (tid % kMovers + kMovers * u) / (D / 8); };
    auto piece_of = [&](int u) LG_INLINE { return (tid % kMovers + kMovers * u) % (D / 8); };
    // Byte offsets in a whole tile; the rest of the address is the same for the whole wave. Where a mover's pieces are
    // whole keys apart (heads of 32, 64, 128, 256) one offset serves all of them.
    constexpr bool kEven = kMovers % (D / 8) == 0;
    constexpr int kOffsets = kEven ? 1 : kPer;
    unsigned whole_at[kOffsets];
#pragma unroll
    for (int u = 0; u < kOffsets; ++u)
        whole_at[u] = ((unsigned)key_of(u) * (unsigned)stride + 8u * (unsigned)piece_of(u)) * 2u;
    auto gload = [&](int tile, Regs& r) LG_INLINE {
        // (past the last visible key that key again: its probability is 0 for everybody who sees less)
        const int key0 = min((HALVES * tile + part) * kApKeys, visible - 1);
        const char* at = reinterpret_cast<const char*>(src + (int64_t)key0 * stride);
        if (key0 + kApKeys <= visible) {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const char* piece = kEven ? at + (int64_t)stride * (u * (kMovers / (D / 8)) * 2) : at;
                r.x[u] = *reinterpret_cast<const uint4_t*>(piece + whole_at[kEven ? 0 : u]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const unsigned k = (unsigned)min(key_of(u), visible - 1 - key0);
                r.x[u] = *reinterpret_cast<const uint4_t*>(at + (k * (unsigned)stride + 8u * (unsigned)piece_of(u)) * 2u);
            }
        }
    };
    auto lstore = [&](int buf, const Regs& r) LG_INLINE {
        unsigned short* at = moves_v ? vs + buf * kVTile : ks + buf * kKTile;
        const int row = moves_v ? kVRow : kKRow;
#pragma unroll
        for (int u = 0; u < kPer; ++u) *reinterpret_cast<uint4_t*>(at + key_of(u) * row + 8 * piece_of(u)) = r.x[u];
    };
    const int s16 = lane & 15;
    const int v_lane = (4 * h + (s16 >> 2)) * kVRow + 16 * ((lane >> 4) & 1) + 4 * (s16 & 3);
    auto v_operand = [&](int buf, int kb, int dt) LG_INLINE {
        typedef short short4_t __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) short4_t lds_short4_t;
        const unsigned short* a = vs + buf * kVTile + v_lane + 16 * kb * kVRow + 32 * dt;
        const uint2_t lo = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)a));
        const uint2_t hi = __builtin_bit_cast(
            uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(a + 8 * kVRow)));
        return uint4_t{lo[0], lo[1], hi[0], hi[1]};
    };
    auto k_operand = [&](int buf, int j) LG_INLINE {
        return *reinterpret_cast<const uint4_t*>(ks + buf * kKTile + col * kKRow + 16 * j + 8 * h);
    };

    float m = kApNone, l = 0.0f;
    float16_t o[kTiles];
#pragma unroll
    for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    uint4_t p_prev[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    float16_t s_cur;

    // Tile `tile` with S(tile) in s_cur, K(tile + 1) in K buffer 1 - H and V(tile - 1) in V buffer 1 - H; leaves
    // S(tile + 1) and P(tile).  MASKED: a column of the workgroup ends in the tile or in front of it.
    auto step = [&](auto masked_c, auto h_c, int tile) LG_INLINE {
        constexpr bool MASKED = decltype(masked_c)::value != 0;
        constexpr int H = decltype(h_c)::value;
        uint4_t ka[kSteps], va[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            ka[j] = k_operand(1 - H, j);
            va[j] = v_operand(1 - H, j / kTiles, j % kTiles);
        }
        const int key0 = (HALVES * tile + part) * kApKeys;
        float sc[16];
        float tm = -INFINITY;
        if (!MASKED || key0 + kApKeys <= first_vis) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[e] = s_cur[e];
                tm = fmaxf(tm, sc[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[e] = key0 + 8 * (e >> 2) + 4 * h + (e & 3) < vis ? s_cur[e] : -INFINITY;
                tm = fmaxf(tm, sc[e]);
            }
        }
        tm = attn_packed_reference<T>(fmaxf(tm, lane_xor_f32<32>(tm)), p.scale_log2e);
        const bool raise = tm > m + ApRange<T>::kLazy;
        const float m_before = m;
        m = raise ? tm : m;
        float16_t s_nxt;
#pragma unroll
        for (int e = 0; e < 16; ++e) s_nxt[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            s_nxt = T::mfma32(ka[j], qb[j], s_nxt);
            o[j % kTiles] = T::mfma32(va[j], p_prev[j / kTiles], o[j % kTiles]);
        }
        float sum = 0.0f;
        uint4_t pb[2];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float p0 = fast_exp2(fmaf(sc[e], p.scale_log2e, -m));
            const float p1 = fast_exp2(fmaf(sc[e + 1], p.scale_log2e, -m));
            sum += p0;
            sum += p1;
            pb[e >> 3][(e & 7) >> 1] = T::pack2(p0, p1);
        }
        if constexpr (!MASKED) {
            // half of the operand reads (64 wide five sixths: 1 to 2.5 % less, 128 wide 2 % more), then the products, each followed by a read (into registers freed before) and
            // its share of the vector work (128 wide, four instructions and not five: one prompt of 16384 2054 -> 2003 us, one of
            // 8192 at 12 / 2 heads 235 -> 220; 64 wide, ten and not nine: one of 2048 at 14 / 2 heads 27.5 -> 26.4)
            constexpr int kReads = 3 * kSteps, kFirst = (D > 64 ? 12 : 20) * kSteps / 8, kShare = (D < 128 ? 80 : 72) / (2 * kSteps);
            __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
            for (int g = 0; g < 2 * kSteps; ++g) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (g < kReads - kFirst) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, kShare, 0);
            }
        }
        // (F belongs to this step: its results are used by the next one only, and would sink there)
        asm volatile("" : "+v"(pb[0]), "+v"(pb[1]), "+v"(sum));
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(raise) != 0, 0)) {  // O(tile - 1) was relative to the old one
            const float alpha = raise ? fast_exp2(m_before - m) : 1.0f;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        }
        l += sum;
        s_cur = s_nxt;
        p_prev[0] = pb[0];
        p_prev[1] = pb[1];
    };

    const int tiles = (visible + HALVES * kApKeys - 1) / (HALVES * kApKeys);  // of a part (past the last key: nobody sees it)
    Regs ra, rb;
    {
        // V buffer 1 plays V(-1) in the first step, whose P is 0: finite values
        for (int i = tid; i < kVTile / 2; i += 64 * WAVES) reinterpret_cast<unsigned*>(vs + kVTile)[i] = 0u;
        gload(0, ra);
        if (!moves_v) {
            gload(1, rb);
            lstore(0, ra);
            lstore(1, rb);
            gload(2, ra);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) s_cur[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) s_cur = T::mfma32(k_operand(0, j), qb[j], s_cur);
        __syncthreads();  // (the first step ends with a store into the buffer just read)
        const int ahead = moves_v ? 1 : 3;  // K(tile + 3), V(tile + 1)
        // step `tile`, H its parity: what the step after the next needs is asked for in front of it and goes to LDS behind it
        auto one = [&](auto masked_c, auto h_c, int tile, Regs& now, Regs& next) LG_INLINE {
            gload(tile + ahead, next);
            __builtin_amdgcn_sched_barrier(0);
            // (a wave in the middle of a step goes before one that moves tiles.  us with / without, 32 / 8 heads of 128: one of 4096 155 /
            // 161, six of 1500 140 / 143; 96 wide 19.2 / 20.0; but 64 wide, three waves to a SIMD, 16 heads, 8 of 1000 42.9 / 37.9)
            if constexpr (D >= 96) __builtin_amdgcn_s_setprio(1);
            step(masked_c, h_c, tile);
            if constexpr (D >= 96) __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            lstore(decltype(h_c)::value, now);  // K(tile + 2), V(tile)
            __syncthreads();
        };
        const int plain = min(tiles, all_see / (HALVES * kApKeys)) & ~1;
        int tile = 0;
        for (; tile < plain; tile += 2) {
            one(ic<0>{}, ic<0>{}, tile, ra, rb);
            one(ic<0>{}, ic<1>{}, tile + 1, rb, ra);
        }
        while (tile < tiles) {
            one(ic<1>{}, ic<0>{}, tile, ra, rb);
            if (++tile >= tiles) break;
            one(ic<1>{}, ic<1>{}, tile, rb, ra);
            ++tile;
        }
        const int buf = (tiles - 1) & 1;
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
            o[j % kTiles] = T::mfma32(v_operand(buf, j / kTiles, j % kTiles), p_prev[j / kTiles], o[j % kTiles]);
    }
    // A key that a column does not see has the probability 0 there, and 0 times an infinity or NaN of its V row is a NaN.
    // If the results are not all finite, or a maximum is too large for the fused difference, the keys are gone through again,
    // plainly, and in the tiles in which columns of the wave end with a pass of its own for every number of keys that one of them
    // sees.  (Workgroup by workgroup; a call all of whose workgroups do takes 1.8 times as long for short documents, 2.5 at heads of 64
    // and for one of 16384 at heads of 128, 3.9 where key tiles are dealt out to two parts at heads of 128, whose second walk spills.)
    float unit = 1.0f;  // of m, in powers of two
    {
        float odds[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // NaN if a result is not finite
#pragma unroll
        for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) odds[e & 3] = fmaf(o[dt][e], 0.0f, odds[e & 3]);
        const float odd = (odds[0] + odds[1]) + (odds[2] + odds[3]);
        // (a column that sees keys, none of them above -inf times the scale, may hold scores that are finite before it)
        const bool far = fabsf(m) > kApExact && vis > kApKeys * part;
        const bool any = __builtin_amdgcn_ballot_w64(odd != odd || far) != 0;
        if (lane == 0) odd_waves[wave_of_all] = any;
        __syncthreads();
        unsigned all = 0;
#pragma unroll
        for (int w = 0; w < WAVES * HALVES; ++w) all |= odd_waves[w];
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(all) != 0, 0)) {
            unit = p.scale_log2e;
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
            for (int tile = 0; tile < tiles; ++tile) {
                const int key0 = (HALVES * tile + part) * kApKeys;
                __syncthreads();
                gload(tile, ra);
                lstore(0, ra);
                __syncthreads();
                float16_t sc;
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
                for (int j = 0; j < kSteps; ++j) sc = T::mfma32(k_operand(0, j), qb[j], sc);
                uint4_t pb[2];
                const float alpha = attn_packed_softmax<T>(sc, key0 + 4 * h, vis, p.scale_log2e, m, l, pb);
#pragma unroll
                for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
                if (key0 + kApKeys <= first_vis) {
#pragma unroll
                    for (int j = 0; j < kSteps; ++j)
                        o[j % kTiles] = T::mfma32(v_operand(0, j / kTiles, j % kTiles), pb[j / kTiles], o[j % kTiles]);
                } else {
                    for (int seen = first_vis; seen <= last_vis; ++seen) {
#pragma unroll
                        for (int dt = 0; dt < kTiles; ++dt) {
                            float16_t acc = o[dt];
#pragma unroll
                            for (int kb = 0; kb < 2; ++kb)
                                acc = T::mfma32(attn_packed_first_keys(v_operand(0, kb, dt), kb, seen - key0 - 4 * h),
                                                pb[kb], acc);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[dt][e] = vis == seen ? acc[e] : o[dt][e];
                        }
                    }
                }
            }
            __syncthreads();
        }
    }
    l += lane_xor_f32<32>(l);
    unsigned short* stage = lds + wave * 16 * kKRow;
    if constexpr (HALVES == 2) {
        // the second part's results through LDS, each wave's own 128 D bytes, then its maxima and sums
        static_assert(WAVES * (128 * D + 512) <= 2 * HALVES * kRings, "the second part's results fit");
        float4_t* const theirs = reinterpret_cast<float4_t*>(lds) + wave * 8 * D;
        float* const ml = reinterpret_cast<float*>(reinterpret_cast<float4_t*>(lds) + WAVES * 8 * D) + wave * 128;
        if (part == 1) {
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    theirs[(4 * dt + b) * 64 + lane] =
                        float4_t{o[dt][4 * b], o[dt][4 * b + 1], o[dt][4 * b + 2], o[dt][4 * b + 3]};
            ml[lane] = m;
            ml[64 + lane] = l;
        }
        __syncthreads();
        if (part == 1) return;
        const float other = ml[lane];
        const float top = fmaxf(m, other), ref = top == -INFINITY ? 0.0f : top;
        const float mine = fast_exp2((m - ref) * unit), its = fast_exp2((other - ref) * unit);
        l = l * mine + ml[64 + lane] * its;
#pragma unroll
        for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4_t w = theirs[(4 * dt + b) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[dt][4 * b + e] = o[dt][4 * b + e] * mine + w[e] * its;
            }
        stage = reinterpret_cast<unsigned short*>(theirs);
        __builtin_amdgcn_wave_barrier();
    }
    if (c0 >= cols) return;
    static_assert(WAVES * 16 * kKRow <= kRings && 32 * kKRow <= 128 * D, "the columns on their way out fit");
    const int tok0 = c0 / p.g;  // of the wave's first column
    attn_packed_write<T, D>(p.out + (int64_t)(t.row0 + tok0) * p.out_stride,
                            (unsigned)(tok - tok0) * (unsigned)p.out_stride + (unsigned)(head * D), cols - c0,
                            stage, o, l);
}

template <typename T, int D, int WAVES, int HALVES = 1>
static hipError_t attn_packed_launch(const AttnPackedParams& p, hipStream_t stream) {
    const int64_t tiles = packed_tiles(p.total, p.num_seqs, p.g, 32 * WAVES);
    attn_packed_kernel<T, D, WAVES, HALVES><<<(unsigned)(tiles * p.hkv), 64 * WAVES * HALVES, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T>
static hipError_t attn_packed_by_width(const AttnPackedParams& p, int d, hipStream_t stream) {
    // 256 columns to a workgroup (eight waves, K and V moved half as often) where the sequences are long and there are
    // many of them; otherwise 128, of which a compute unit holds two or three that fill each other's waits.  us, 8 / 4 waves, 128
    // wide, 32 / 8 heads: one of 16384 1968 / 2079, one of 4096 138 / 145, 8 of 2048 317 / 317, but 16 of 1500 383 / 362, 16 of
    // 512 72 / 70; 12 / 2: one of 16384 794 / 819, one of 8192 227 / 226.  64 wide: 4 x 8192, 14 / 2, 586 / 582; one of 2048 41 / 31.
    const bool wide = d == 128 && p.total >= 2048 * (int64_t)p.num_seqs &&
                      packed_tiles(p.total, p.num_seqs, p.g, 256) * p.hkv >= 2 * device_cu_count();
    // Key tiles dealt out to two parts of a workgroup, joined at its end, where workgroups are few and keys many: the steps of a
    // workgroup alone on its compute unit are latency (1000 clocks of the 770 that a step takes of three side by side), twice the
    // waves hide it, but have a join, and no room for a second workgroup beside them.  us, one part / two, 64 wide, 14 / 2 heads:
    // one of 512 11.8 / 11.2, of 2048 33.1 / 27.2, of 4096 64.0 / 54.5, two of 2048 40.2 / 33.6, but one of 256 8.4 / 8.8, four
    // of 1024 22.6 / 26.7 and one of 6000 97 / 104; 128 wide, 12 / 2: one of 4096 90 / 70, but 32 / 8, one of 512 15.7 / 16.2; 32 wide,
    // 24 / 4: one of 512 10.0 / 9.4, of 2048 28.0 / 23.7, but one of 256 7.1 / 7.3, four of 600 13.5 / 14.3; 96 wide, 16 / 16: one of 768
    // 18.0 / 16.6, of 4096 83 / 73, but one of 256 10.0 / 10.5, four of 800 23.8 / 30.3; at worst, 8 / 2, four of 2048 53.0 / 54.1.
    const int64_t groups = (int64_t)p.total * p.g / 128 * p.hkv;
    const bool split =
        (groups <= device_cu_count() && p.total >= (d > 64 ? 8 * d : 512) * (int64_t)p.num_seqs) ||
        (groups <= 2 * device_cu_count() && p.total >= 2048 * (int64_t)p.num_seqs);
    switch (d) {
        case 32: return split ? attn_packed_launch<T, 32, 4, 2>(p, stream) : attn_packed_launch<T, 32, 4>(p, stream);
        case 64: return split ? attn_packed_launch<T, 64, 4, 2>(p, stream) : attn_packed_launch<T, 64, 4>(p, stream);
        case 96: return split ? attn_packed_launch<T, 96, 4, 2>(p, stream) : attn_packed_launch<T, 96, 4>(p, stream);
        case 128:
            return wide    ? attn_packed_launch<T, 128, 8>(p, stream)
                   : split ? attn_packed_launch<T, 128, 4, 2>(p, stream)
                           : attn_packed_launch<T, 128, 4>(p, stream);
        case 160: return attn_packed_launch<T, 160, 4>(p, stream);
        case 192: return attn_packed_launch<T, 192, 4>(p, stream);
        case 224: return attn_packed_launch<T, 224, 4>(p, stream);
        default: return attn_packed_launch<T, 256, 4>(p, stream);
    }
}

static logismos_status_t attn_packed(bool bf16, const void* q, const void* k, const void* v, const int32_t* cu,
                                     void* out, int num_seqs, int total, int hq, int hkv, int d, int q_stride,
                                     int k_stride, int v_stride, int out_stride, float scale, int causal,
                                     logismos_stream_t stream) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (logismos_check_attn_packed_shape(num_seqs, total, hq, hkv, d, q_stride, k_stride, v_stride, out_stride,
                                         nullptr, 0) != 0)
        return bad;
    const float scale_log2e = scale * 1.4426950408889634f;
    if (!q || !k || !v || !cu || !out || !(scale > 0.0f) || !isfinite(scale_log2e)) return bad;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
         reinterpret_cast<uintptr_t>(out)) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(cu) % 4 != 0)
        return bad;
    AttnPackedParams p = {};
    p.q = static_cast<const unsigned short*>(q);
    p.k = static_cast<const unsigned short*>(k);
    p.v = static_cast<const unsigned short*>(v);
    p.cu = cu;
    p.out = static_cast<unsigned short*>(out);
    p.num_seqs = num_seqs;
    p.total = total;
    p.hkv = hkv;
    p.g = hq / hkv;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.out_stride = out_stride;
    p.scale_log2e = scale_log2e;
    p.causal = causal != 0;
    // (putting them in order takes every workgroup about 1 us: 8 prompts of 100 to 4096 tokens 93 -> 85 us, 8 of 1000 43 -> 40,
    // but 16 of 512 76 -> 79)
    p.ordered = num_seqs > 1 && num_seqs <= kPackedOrdered && total > 512 * (int64_t)num_seqs;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return static_cast<logismos_status_t>(bf16 ? attn_packed_by_width<PackedBf16>(p, d, st)
                                               : attn_packed_by_width<PackedF16>(p, d, st));
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_attn_packed_shape(int num_seqs, int total_tokens, int num_q_heads, int num_kv_heads,
                                                   int head_dim, int q_stride, int k_stride, int v_stride,
                                                   int out_stride, char* msg, size_t cap) {
    using lg::reject;
    if (num_seqs <= 0 || total_tokens <= 0) return reject(msg, cap, "num_seqs and total_tokens must be positive (%d, %d)", num_seqs, total_tokens);
    if (num_q_heads <= 0 || num_kv_heads <= 0)
        return reject(msg, cap, "num_q_heads and num_kv_heads must be positive (%d, %d)", num_q_heads, num_kv_heads);
    if (num_q_heads % num_kv_heads != 0)
        return reject(msg, cap, "num_q_heads %d is not a multiple of num_kv_heads %d", num_q_heads, num_kv_heads);
    if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 256)
        return reject(msg, cap, "head_dim must be a multiple of 32 up to 256 (%d)", head_dim);
    if ((int64_t)total_tokens + num_seqs > lg::kPackedMaxRows)
        return reject(msg, cap, "total_tokens + num_seqs exceeds %d", lg::kPackedMaxRows);
    if ((int64_t)total_tokens * num_q_heads / 128 + (int64_t)num_seqs * num_kv_heads > (1 << 22))
        return reject(msg, cap, "total_tokens * num_q_heads / 128 + num_seqs * num_kv_heads exceeds %d", 1 << 22);
    const int64_t qw = (int64_t)num_q_heads * head_dim, kw = (int64_t)num_kv_heads * head_dim;
    if (q_stride < qw || out_stride < qw || k_stride < kw || v_stride < kw)
        return reject(msg, cap, "a stride is smaller than its row (%d and %d of %lld, %d and %d of %lld)", q_stride,
                      out_stride, (long long)qw, k_stride, v_stride, (long long)kw);
    if ((q_stride | k_stride | v_stride | out_stride) % 8 != 0)
        return reject(msg, cap, "strides must be multiples of 8 (%d, %d, %d, %d)", q_stride, k_stride, v_stride,
                      out_stride);
    if (k_stride > (1 << 22) || v_stride > (1 << 22) || out_stride > (1 << 22))
        return reject(msg, cap, "k, v and out strides must be at most %d (%d, %d, %d)", 1 << 22, k_stride, v_stride,
                      out_stride);
    return 0;
}

#define LOGISMOS_ATTN_PACKED(name, bf16)                                                                              \
    logismos_status_t logismos_launch_attn_packed_##name(                                                             \
        const void* q, const void* k, const void* v, const int32_t* cu_seqlens, void* out, int num_seqs,              \
        int total_tokens, int num_q_heads, int num_kv_heads, int head_dim, int q_stride, int k_stride, int v_stride,  \
        int out_stride, float scale, int causal, logismos_stream_t stream) {                                          \
        return lg::attn_packed(bf16, q, k, v, cu_seqlens, out, num_seqs, total_tokens, num_q_heads, num_kv_heads,     \
                               head_dim, q_stride, k_stride, v_stride, out_stride, scale, causal, stream);            \
    }
LOGISMOS_ATTN_PACKED(fp16, false)
LOGISMOS_ATTN_PACKED(bf16, true)
#undef LOGISMOS_ATTN_PACKED

}  // extern "C"
