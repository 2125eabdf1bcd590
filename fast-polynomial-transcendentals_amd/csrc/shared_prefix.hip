// shared_prefix.hip -- attention of a batch whose sequences share one prefix,
// for gfx950: the new tokens of every sequence attend to the prefix's keys,
// held once for all, and to the keys of their own suffix cache.
//
//   out[b, t] = softmax(s) V over prefix keys 0 .. P - 1 and suffix keys
//   0 .. lens[b] - T + t of sequence b (the last T of which are the new tokens'
//   own), s = q.k scale, or cap tanh(q.k scale / cap)
//
// For one KV head the rows that meet the prefix are all B T g rows of the batch
// (g query heads to a KV head), so the prefix is one product over many rows,
// read once per row tile; each sequence's suffix has T g rows of its own.  Both
// are cut along the keys into enough parts to fill the chip, each part leaves its
// rows' O, maximum and sum in FP32 in a workspace, and a second launch joins the
// parts of a row: O = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
//
// A part is a block of four waves, two blocks to a CU (three at head_dim 64):
//  * up to 32 rows ("narrow"): every wave has all rows and a quarter of the
//    keys, in tiles of 32 keys that it alone moves to its LDS; K of
//    the next tile flies while the scores are turned into probabilities, V of the
//    next while the next scores are made, and no wave waits for another;
//  * more ("wide"): each wave has 32 of 128 rows and all waves share 64-key tiles,
//    K two and V one staged ahead (three and two at head_dim 64); with up to 64 rows
//    two waves share a row and halve each tile's keys.
// Products are S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16, so a lane
// keeps one row (query) and a row's reductions stay in two lanes
// (flash_attn.hpp).
//
// What bounds it: up to about 128 rows a KV head the bytes of K and V, beyond
// that the matrix cores and the exponentials beside them.  Measured (BF16, 32 / 8
// heads, both launches): 2 sequences behind 131072 keys, heads of 64, 57 us, 4.7 TB/s (5.4
// in the first launch); 64 behind 32768 with caches of up to 2048 keys, heads of 128, 95 us
// (403 MB, 35 GFLOP); 16 x 100 tokens behind 8192 247 us, 900 TFLOP/s; 8 sequences
// behind 1024, caches of 256, 11 us.
//
// The host does not know the caches' lengths: parts, workspace and launch go by what
// they are allocated for, and a part without keys still writes its rows.  64 sequences
// with 500 to 2000 keys behind 4096: 71 us in caches of 2048, 90 in 8192, 176 in 32768
// (behind 32768 keys 96, 131, 541); views of the longest length keep it at 69 and 96.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "row_state.hpp"
#include "spline_ops_hip.h"

namespace pt {

constexpr int kWideRows = 128, kNarrowRows = 32;
constexpr int kLeastKeys = 128;   // of a part: a tile for each wave of a narrow block
// Of a part of a cache with few rows: 64 caches of 1 to 2048 keys take 57 us in parts
// of up to 768, 64 in one, 64 to 73 in parts of 256 to 512 (a block costs 5 us
// beside its keys).
constexpr int kMostOwnKeys = 768;
constexpr int kBlockKeys = 128;

struct PrefixParams {
    const uint16_t* q;
    const uint16_t *pk, *pv, *sk, *sv;
    const int32_t* lens;
    float* part_o;  // [parts][rows][HD]
    float2* part_ml;  // [parts][rows]
    void* out;
    float* lse;
    AttnStrides qs, pks, pvs, sks, svs;  // prefix: b unused
    int64_t rows;     // B T Hq
    int64_t mrows;    // B T g: rows of a KV head
    int hq, hkv, group, tokens, batch;
    int prefix, suffix;
    int parts_p, parts_s;      // along the keys
    int chunk;                 // prefix keys per part, a multiple of 64
    int tiles_p, tiles_s;      // row tiles of a KV head; of a sequence and KV head
    int groups_p;              // hkv * parts_p
    int64_t blocks_p;
    int narrow_p, narrow_s, wide_strides;
    int once;                  // K and V do not stay in the caches
    float scale, cap;
};

template <bool BF>
__device__ __forceinline__ f32x16_t mfma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
}

// Values that are no finite numbers: bit 15 of each half of the result.
template <bool BF>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & (BF ? 0x7f807f80u : 0x7c007c00u)) + (BF ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
// A BF16 fragment with the largest finite value in the place of what is not finite
// in V, and zeros elsewhere.
typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
template <bool BF>
__device__ __forceinline__ bf16x8_t where_not_finite(bf16x8_t f) {
    constexpr uint16_t kInf = BF ? 0x7f80 : 0x7c00;
    u16x8_t u = __builtin_bit_cast(u16x8_t, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = (u[e] & kInf) == kInf ? (uint16_t)0x7f7f : (uint16_t)0;
    return __builtin_bit_cast(bf16x8_t, u);
}

// N loads of a wave, STEP rows apart, from row0 on, to their rows of a tile (the
// first is tile_row).  Whole tiles take one decision for all loads; a tile with
// rows past `last`, or rows too far apart for a lane's offset, one for each.
template <int HD, int N, int STEP, bool ONCE>
__device__ __forceinline__ void stage_rows(const RowLoader<HD>& loader, uint32_t tile, int tile_row, const uint16_t* base,
                                           int64_t stride, int row0, int last) {
    constexpr int kLoadRows = RowLoader<HD>::kLoadRows;
    if (row0 + STEP * (N - 1) + kLoadRows - 1 <= last && !loader.wide) {  // wave-uniform
        const uint16_t* rows = base + row0 * stride;
        const uint32_t lane = (uint32_t)loader.lr * (uint32_t)(int)stride * 2;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = tile_row + STEP * j;
            const uint32_t offset = lane + (uint32_t)((loader.lc ^ row_swizzle<HD>((r & 7) + loader.lr)) * 16);
            if constexpr (ONCE) load_to_lds_once(tile + lds_row<HD>(r), rows, offset);
            else load_to_lds(tile + lds_row<HD>(r), rows, offset);
            rows += STEP * stride;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = tile_row + STEP * j;
            loader.template load<ONCE>(tile + lds_row<HD>(r), r & 7, base, stride, row0 + STEP * j, last);
        }
    }
}

template <int HD>
struct PrefixShape {
    static constexpr int kNarrowKeys = 32;  // one accumulator
    static constexpr int kNarrowTileB = lds_row<HD>(kNarrowKeys);
    static constexpr int kWideTileB = lds_row<HD>(kAttnBlockK);
    static constexpr int kWideRing = HD == 64 ? 3 : 2;
    static constexpr int kRegionB = 32 * HD * 4;  // 32 FP32 rows of O
    static constexpr int kNarrowB = 2 * kNarrowTileB > kRegionB ? 2 * kNarrowTileB : kRegionB;  // per wave
    static constexpr int kWideB = 2 * kWideRing * kWideTileB;
    static constexpr int kLds = 4 * kNarrowB > kWideB ? 4 * kNarrowB : kWideB;
    static_assert(4 * kRegionB <= kLds, "O leaves through LDS");
};

// The keys of part s of a cache, for rows r0 .. r0 + nrows - 1 of a sequence; seen:
// keys that its token 0 sees (token t: t more).
struct SuffixPart {
    int seen, k0, kend;

    __device__ __forceinline__ SuffixPart(const PrefixParams& p, int b, int s, int r0, int nrows) {
        int len = p.lens[b];
        len = len < 0 ? 0 : len < p.suffix ? len : p.suffix;  // held to the cache
        seen = len - p.tokens + 1;
        const int last_token = (r0 + nrows - 1) / p.group;
        const int visible = seen + last_token > 0 ? seen + last_token : 0;  // keys that any row sees
        const int each = ((visible + p.parts_s - 1) / p.parts_s + 63) & ~63;
        k0 = s * each;
        kend = k0 + each < visible ? k0 + each : visible;
    }
};

// Blocks to a CU: two at head_dim 128 (220 registers), three at 64 (168), where
// the D4 softcap needs 172.
template <int MODE, int HD, bool BF>
__global__ void __launch_bounds__(256) __attribute__((
    amdgpu_waves_per_eu(HD == 64 && MODE != kAttnSoftcapD4 ? 3 : 2))) shared_prefix_kernel(PrefixParams p) {
    using F = PrefixShape<HD>;
    constexpr int kC = HD / 16, kD = HD / 32;
    __shared__ __align__(1024) unsigned char smem[F::kLds];
    __shared__ float2 sml[4][32];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int h = lane >> 5, c32 = lane & 31;

    // ---- which rows and keys
    int kvh, part, nrows;           // nrows: of this block
    int64_t m0;                     // the block's first row among its KV head's
    const uint16_t *kp, *vp;
    int64_t kstride, vstride;
    int k0, kend;                   // keys of the block
    int seen = 0;                   // suffix keys that the sequence's token 0 sees (token t: t more)
    const bool own = (int64_t)blockIdx.x >= p.blocks_p;
    if (!own) {
        // neighbours in a row of eight blocks go to eight XCDs: the row tiles of
        // one part and KV head follow each other on one XCD, whose L2 holds its keys
        const uint32_t idx = blockIdx.x, xcd = idx & 7, slot = idx >> 3;
        const uint32_t g = slot / (uint32_t)p.tiles_p * 8 + xcd, tile = slot % (uint32_t)p.tiles_p;
        if (g >= (uint32_t)p.groups_p) return;
        part = (int)(g / (uint32_t)p.hkv);
        kvh = (int)(g % (uint32_t)p.hkv);
        m0 = (int64_t)tile * kWideRows;
        const int64_t left = p.mrows - m0;
        nrows = left < kWideRows ? (int)left : kWideRows;
        kp = p.pk + kvh * p.pks.h;
        vp = p.pv + kvh * p.pvs.h;
        kstride = p.pks.s;
        vstride = p.pvs.s;
        k0 = part * p.chunk;
        kend = k0 + p.chunk < p.prefix ? k0 + p.chunk : p.prefix;
    } else {
        uint32_t rest = (uint32_t)((int64_t)blockIdx.x - p.blocks_p);
        const uint32_t tile = rest % (uint32_t)p.tiles_s;
        rest /= (uint32_t)p.tiles_s;
        kvh = (int)(rest % (uint32_t)p.hkv);
        rest /= (uint32_t)p.hkv;
        const int s = (int)(rest % (uint32_t)p.parts_s), b = (int)(rest / (uint32_t)p.parts_s);
        part = p.parts_p + s;
        const int per = p.tokens * p.group, r0 = (int)tile * kWideRows;
        m0 = (int64_t)b * per + r0;
        nrows = per - r0 < kWideRows ? per - r0 : kWideRows;
        kp = p.sk + b * p.sks.b + kvh * p.sks.h;
        vp = p.sv + b * p.svs.b + kvh * p.svs.h;
        kstride = p.sks.s;
        vstride = p.svs.s;
        const SuffixPart keys(p, b, s, r0, nrows);
        seen = keys.seen;
        k0 = keys.k0;
        kend = keys.kend;
    }
    // the waves that share a row's keys among them: narrow four, half two, else one
    const bool narrow = own ? p.narrow_s : p.narrow_p, half = !narrow && nrows <= 64;
    const int rbase = narrow ? 0 : half ? (wave & 1) * 32 : wave * 32;  // the wave's rows in the block
    const bool rin = rbase + c32 < nrows;                                // this lane has a row

    // ---- staging; the first tiles fly while the rows are found
    const RowLoader<HD> loader(lane, p.wide_strides);
    constexpr int kLoadRows = RowLoader<HD>::kLoadRows;
    const int all = kend > k0 ? kend - k0 : 0;
    // narrow: wave w moves tiles w, w + 4, .. to its own place
    constexpr int kNarrowKeys = F::kNarrowKeys, kNarrowLoads = kNarrowKeys / kLoadRows;
    constexpr int NK = kAttnBlockK, kWideLoads = NK / kLoadRows / 4, kRing = F::kWideRing;
    const int tiles = narrow ? (all + kNarrowKeys - 1) / kNarrowKeys : (all + NK - 1) / NK;
    const uint32_t own_k = lds0 + (uint32_t)(wave * F::kNarrowB), own_v = own_k + F::kNarrowTileB;
    auto load_own = [&](uint32_t lds, const uint16_t* base, int64_t stride, int i) __attribute__((always_inline)) {
        const int row0 = k0 + i * kNarrowKeys;
        if (p.once) stage_rows<HD, kNarrowLoads, kLoadRows, true>(loader, lds, 0, base, stride, row0, kend - 1);
        else stage_rows<HD, kNarrowLoads, kLoadRows, false>(loader, lds, 0, base, stride, row0, kend - 1);
    };
    // wide: the block's rings, K a tile further ahead than V
    constexpr uint32_t kV = kRing * F::kWideTileB;
    auto stage_k = [&](int i) __attribute__((always_inline)) {
        const int r = kLoadRows * wave;
        if (i < tiles)
            stage_rows<HD, kWideLoads, 4 * kLoadRows, false>(loader, lds0 + (uint32_t)(i % kRing * F::kWideTileB), r, kp,
                                                             kstride, k0 + i * NK + r, kend - 1);
    };
    auto stage_v = [&](int i) __attribute__((always_inline)) {
        const int r = kLoadRows * wave;
        if (i < tiles)
            stage_rows<HD, kWideLoads, 4 * kLoadRows, false>(loader, lds0 + kV + (uint32_t)(i % kRing * F::kWideTileB), r,
                                                             vp, vstride, k0 + i * NK + r, kend - 1);
    };
    if (narrow) {
        if (wave < tiles) {
            load_own(own_k, kp, kstride, wave);
            load_own(own_v, vp, vstride, wave);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) {
            stage_k(i);
            if (i > 0) stage_v(i - 1);
        }
    }

    // row m of a KV head is (b, t, head in the group); fewer than 2^31 of them
    const uint32_t mrow = (uint32_t)m0 + (uint32_t)(rin ? rbase + c32 : 0);
    const uint32_t bt = mrow / (uint32_t)p.group;
    const uint32_t b = bt / (uint32_t)p.tokens;
    const int t = (int)(bt - b * (uint32_t)p.tokens);
    const uint16_t* qrow =
        p.q + b * p.qs.b + t * p.qs.s + (kvh * p.group + (int)(mrow - bt * (uint32_t)p.group)) * p.qs.h;
    // the last key that the lane's row sees (a lane without a row computes one
    // that is not stored, and asks for no mask)
    int klast = own && rin ? seen + t - 1 : kend - 1;
    klast = klast < kend - 1 ? klast : kend - 1;

    RowState<HD> st;
    bf16x8_t qf[kC];  // Q^T fragments: columns 16c + 8h .. of row c32
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        qf[c] = (bf16x8_t){};
        if (rin) qf[c] = *reinterpret_cast<const bf16x8_t*>(qrow + 16 * c + 8 * h);
    }
    const TileReader<HD> reader(lane);
    ScoreConsts consts;
    consts.sl = attn_is_plain_softmax(MODE) ? p.scale * kLog2e : kLog2e;
    if constexpr (!attn_is_plain_softmax(MODE)) {
        // in VGPRs (faster operands) where there is room
        auto hold = [](float x) __attribute__((always_inline)) { return HD == 128 ? vgpr(x) : x; };
        consts.scale = hold(p.scale);
        consts.cap = hold(p.cap);
        consts.inv_cap = hold(1.0f / p.cap);
        if constexpr (MODE == kAttnSoftcapD4)
#pragma unroll
            for (int i = 1; i <= SoftcapConsts::T::P.deg; ++i) consts.tanh[i] = hold(bf16_value(SoftcapConsts::T::P.c[i]));
    }

    // S^T of the NT 32-key accumulators at kt0, fragments read six ahead
    auto scores = [&](auto& s, const unsigned char* kt0) __attribute__((always_inline)) {
        constexpr int NT = sizeof(s) / sizeof(f32x16_t), kN = NT * kC;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) s[kt] = (f32x16_t){};
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
            for (int kt = 0; kt < NT; ++kt)
                s[kt] = mfma<BF>(reader.row_frag(kt0 + lds_row<HD>(kt * 32), c), qf[c], s[kt]);
        constexpr int kAhead = kN < 6 ? kN : 6;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int g = 0; g < kN - kAhead; ++g) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // O^T += V^T P^T, three fragments (two reads each) ahead.  One rounding of P
    // costs as much as the result's own (their sum is 1.4 times it).  Narrow blocks
    // wait for memory, so they add the product with what it left (exact).  Wide ones round once,
    // as the attention forward does; the same there took 341 us against 247 with
    // 16 x 100 tokens behind 8192 keys, 72 against 59 with 64 decoding behind 32768, 77
    // against 60 with 128 behind 16384, 101 against 98 with caches of 2048 besides.
    auto accumulate = [&](auto exact, const auto& s, const unsigned char* vt0) __attribute__((always_inline)) {
        constexpr bool EXACT = decltype(exact)::value;
        constexpr int NT = sizeof(s) / sizeof(f32x16_t), kN = 2 * NT * kD;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < 2 * NT; ++g) {
            const bf16x8_t pf = prob_frag<BF>(s[g >> 1], g & 1);
            bf16x8_t rest;
            if constexpr (EXACT) rest = prob_rest<BF>(s[g >> 1], g & 1, pf);
#pragma unroll
            for (int dt = 0; dt < kD; ++dt) {
                const bf16x8_t v = reader.col_frag(vt0 + lds_row<HD>(16 * g), dt);
                st.o[dt] = mfma<BF>(v, pf, st.o[dt]);
                if constexpr (EXACT) st.o[dt] = mfma<BF>(v, rest, st.o[dt]);
            }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int g = 0; g < kN - 3; ++g) {
            __builtin_amdgcn_sched_group_barrier(0x008, EXACT ? 2 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, EXACT ? 6 : 3, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // The same for a tile with keys that some of the rows do not see: 0 * Inf is NaN,
    // so what is not finite in V is taken out, and the rows that see its key (diag as
    // in score_state) get an infinity, as four times the largest BF16 value.  It marks
    // the element: the join looks up what it has to be.
    auto accumulate_seen = [&](auto exact, const auto& s, const unsigned char* vt0, int diag)
                               __attribute__((always_inline)) {
        constexpr bool EXACT = decltype(exact)::value;
        constexpr int NT = sizeof(s) / sizeof(f32x16_t);
        uint32_t bad = 0;
#pragma unroll
        for (int g = 0; g < 2 * NT; ++g) {
            __builtin_amdgcn_sched_barrier(0);  // here and below: few registers at a time
            const bf16x8_t pf = prob_frag<BF>(s[g >> 1], g & 1);
            bf16x8_t rest;
            if constexpr (EXACT) rest = prob_rest<BF>(s[g >> 1], g & 1, pf);
#pragma unroll
            for (int dt = 0; dt < kD; ++dt) {
                u32x4_t v = __builtin_bit_cast(u32x4_t, reader.col_frag(vt0 + lds_row<HD>(16 * g), dt));
                const u32x4_t t = {not_finite<BF>(v.x), not_finite<BF>(v.y), not_finite<BF>(v.z), not_finite<BF>(v.w)};
                bad |= t.x | t.y | t.z | t.w;
                v &= ~((t << 1) - (t >> 15));
                st.o[dt] = mfma<BF>(__builtin_bit_cast(bf16x8_t, v), pf, st.o[dt]);
                if constexpr (EXACT) st.o[dt] = mfma<BF>(__builtin_bit_cast(bf16x8_t, v), rest, st.o[dt]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!__any(bad != 0)) return;
        asm("" : "+v"(diag));  // no comparison with it is made ahead of the branch
#pragma unroll
        for (int g = 0; g < 2 * NT; ++g) {
            bf16x8_t seen;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                seen[e] = (__bf16)(diag + 16 * g + 8 * (e >> 2) + (e & 3) > 0 ? 0.0f : 4.0f);
#pragma unroll
            for (int dt = 0; dt < kD; ++dt) {
                __builtin_amdgcn_sched_barrier(0);
                st.o[dt] = mfma<true>(where_not_finite<BF>(reader.col_frag(vt0 + lds_row<HD>(16 * g), dt)), seen, st.o[dt]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const bool some_see = own && p.tokens > 1;
    // the first and the last key that bound what the wave's rows see: tiles that
    // end ahead of the first need no mask, tiles behind the last no arithmetic
    int kfull = kend - 1, kmost = kend - 1;
    if (some_see) {
        kfull = kmost = klast;
#pragma unroll
        for (int step = 1; step < 32; step *= 2) {
            const int x = __shfl_xor(kfull, step), y = __shfl_xor(kmost, step);
            kfull = x < kfull ? x : kfull;
            kmost = y > kmost ? y : kmost;
        }
        kfull = __builtin_amdgcn_readfirstlane(kfull);
        kmost = __builtin_amdgcn_readfirstlane(kmost);
    }

    if (narrow) {
        constexpr int NT = kNarrowKeys / 32;
        const unsigned char* kt0 = smem + wave * F::kNarrowB;
        const unsigned char* vt0 = kt0 + F::kNarrowTileB;
        f32x16_t s[NT];
        auto tile = [&](auto masked, int i) __attribute__((always_inline)) {
            wait_loads<kNarrowLoads>();  // K(i) has landed; V(i) may fly
            scores(s, kt0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K(i) is read: its place is free
            const bool more = i + 4 < tiles;
            if (more) load_own(own_k, kp, kstride, i + 4);
            const int diag = k0 + i * kNarrowKeys + 4 * h - klast;
            const float mul = score_state<MODE, HD, BF, NT, decltype(masked)::value>(s, st, consts, diag);
            score_exps<HD, NT>(s, st, mul);
            if (more) wait_loads<kNarrowLoads>();  // V(i) has landed; K(i + 4) may fly
            else wait_loads<0>();
            if constexpr (decltype(masked)::value) accumulate_seen(std::integral_constant<bool, true>{}, s, vt0, diag);
            else accumulate(std::integral_constant<bool, true>{}, s, vt0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) load_own(own_v, vp, vstride, i + 4);
        };
        const int full = (kfull + 1 - k0) / kNarrowKeys;  // tiles without a masked key (negative: none)
        int i = wave;
        for (; i < tiles && i < full; i += 4) tile(std::integral_constant<bool, false>{}, i);
        for (; i < tiles; i += 4) tile(std::integral_constant<bool, true>{}, i);
    } else {
        // sync(i), i = 0 .. tiles: K(i) and V(i - 1) are whole, and every wave is
        // done with K(i - 1) and V(i - 2), whose places the next loads take.  The
        // loads of the sync before may still fly where the rings hold three tiles.
        auto sync = [&](int i) __attribute__((always_inline)) {
            if (kRing > 2 && i + 1 < tiles) wait_loads<2 * kWideLoads * (kRing - 2)>();
            else wait_loads<0>();
            block_barrier();
            stage_k(i + kRing - 1);
            stage_v(i + kRing - 2);
        };
        // the wave's keys of a tile: all 64, or with half of the rows 32 of them
        auto run = [&](auto nt_c, int off) __attribute__((always_inline)) {
            constexpr int NT = decltype(nt_c)::value;
            constexpr int kFirst = 1;  // K chunks whose products go with the maximum
            // tiles without a masked key, and with one that a row sees; a wave
            // without rows only stages
            const int x = kfull + 1 - k0 - off - 32 * NT, y = kmost - k0 - off;
            const int whole = x < 0 ? 0 : x / NK + 1, most = y < 0 || rbase >= nrows ? 0 : y / NK + 1;
            const int last = most < tiles ? most : tiles;
            const unsigned char* ks = smem + lds_row<HD>(off);
            auto k_tile = [&](int i) __attribute__((always_inline)) { return ks + i % kRing * F::kWideTileB; };
            // S of tile i + 1 between the maximum and the exponentials of tile i, so
            // that the matrix cores work while scores become probabilities.  At
            // head_dim 64, which has 168 registers for it, it spills.  16 x 100
            // tokens behind 8192 keys 253 us against 271, 256 sequences behind 8192
            // 69 against 76, memory-bound cases alike; 512 tokens of one sequence
            // 95 against 92.
            auto step = [&](f32x16_t (&cur)[NT], f32x16_t (&nxt)[NT], int i) __attribute__((always_inline)) {
                sync(i + 1);
                const unsigned char *kt0 = k_tile(i + 1), *vt0 = k_tile(i) + kV;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int kt = 0; kt < NT; ++kt) nxt[kt] = (f32x16_t){};
#pragma unroll
                for (int c = 0; c < kFirst; ++c)
#pragma unroll
                    for (int kt = 0; kt < NT; ++kt)
                        nxt[kt] = mfma<BF>(reader.row_frag(kt0 + lds_row<HD>(kt * 32), c), qf[c], nxt[kt]);
                const float mul = score_state<MODE, HD, BF, NT, false>(cur, st, consts, 0);
#pragma unroll
                for (int c = kFirst; c < kC; ++c)
#pragma unroll
                    for (int kt = 0; kt < NT; ++kt)
                        nxt[kt] = mfma<BF>(reader.row_frag(kt0 + lds_row<HD>(kt * 32), c), qf[c], nxt[kt]);
                score_exps<HD, NT>(cur, st, mul);
#pragma unroll
                for (int g = 0; g < 2 * NT; ++g) {
                    const bf16x8_t pf = prob_frag<BF>(cur[g >> 1], g & 1);
#pragma unroll
                    for (int dt = 0; dt < kD; ++dt)
                        st.o[dt] = mfma<BF>(reader.col_frag(vt0 + lds_row<HD>(16 * g), dt), pf, st.o[dt]);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            // one thing after the other
            auto finish = [&](auto masked, f32x16_t (&s)[NT], int i) __attribute__((always_inline)) {
                sync(i + 1);
                const int diag = k0 + i * NK + off + 4 * h - klast;
                const float mul = score_state<MODE, HD, BF, NT, decltype(masked)::value>(s, st, consts, diag);
                score_exps<HD, NT>(s, st, mul);
                if constexpr (decltype(masked)::value)
                    accumulate_seen(std::integral_constant<bool, false>{}, s, k_tile(i) + kV, diag);
                else accumulate(std::integral_constant<bool, false>{}, s, k_tile(i) + kV);
                if (i + 1 < last) scores(s, k_tile(i + 1));
            };
            int synced = 0;  // syncs met
            if (last > 0) {
                f32x16_t s[NT];
                sync(0);
                scores(s, k_tile(0));
                int i = 0;
                if constexpr (HD == 128) {
                    f32x16_t s2[NT];
                    for (; i + 2 < last && i + 1 < whole; i += 2) {
                        step(s, s2, i);
                        step(s2, s, i + 1);
                    }
                }
                for (; i < last && i < whole; ++i) finish(std::integral_constant<bool, false>{}, s, i);
                for (; i < last; ++i) finish(std::integral_constant<bool, true>{}, s, i);
                synced = last + 1;
            }
            if (tiles > 0)
                for (int i = synced; i <= tiles; ++i) sync(i);
        };
        if (half) run(std::integral_constant<int, 1>{}, (wave >> 1) * 32);
        else run(std::integral_constant<int, 2>{}, 0);
    }

    // ---- the rows to the workspace, whole rows through LDS
    __syncthreads();  // every wave has read its tiles
    unsigned char* region = smem + wave * F::kRegionB;
    spill_rows<HD>(region, st, h, c32);
    const float l = half_sum(st.l);
    if (h == 0) sml[wave][c32] = make_float2(st.m, l);
    __syncthreads();
    const int64_t prow = (int64_t)part * p.rows + (int64_t)kvh * p.mrows + m0;
    float* po = p.part_o + prow * HD;
    constexpr int kChunks = HD / 4;
    for (int i = tid; i < nrows * kChunks; i += 256) {
        const int row = i / kChunks, chunk = i % kChunks;
        // the row's share of each wave that has it
        const int first = narrow ? 0 : row >> 5, step = narrow ? 1 : 2, shares = narrow ? 4 : half ? 2 : 1, r = row & 31;
        float2 ml = sml[first][r];
        f32x4_t o = *reinterpret_cast<const f32x4_t*>(smem + first * F::kRegionB + o_chunk<HD>(r, chunk));
        if (shares > 1) {
            const float own_max = ml.x;
            for (int w = 1; w < shares; ++w) ml.x = __builtin_fmaxf(ml.x, sml[first + w * step][r].x);
            const float a = __builtin_amdgcn_exp2f(own_max - ml.x);
            o *= a;
            ml.y *= a;
            for (int w = 1; w < shares; ++w) {
                const float2 x = sml[first + w * step][r];
                const float a2 = __builtin_amdgcn_exp2f(x.x - ml.x);
                o += *reinterpret_cast<const f32x4_t*>(smem + (first + w * step) * F::kRegionB + o_chunk<HD>(r, chunk)) * a2;
                ml.y = __builtin_fmaf(x.y, a2, ml.y);
            }
        }
        *reinterpret_cast<f32x4_t*>(po + (int64_t)row * HD + chunk * 4) = o;
        if (chunk == 0) p.part_ml[prow + row] = ml;
    }
}

typedef int16_t i16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// Elements 4 chunk .. of a row whose sum is a number while they are not: each
// infinity and NaN that the row sees in V, from the parts that hold one (Inf for
// infinities of one sign, NaN otherwise).  What the parts' products made of them depends on
// rounding: an infinity times the zero that a probability was rounded to, or times
// what that rounding left, is a NaN or has the other sign.  An element that sees none
// (its finite values overflowed) keeps what it has.  Each row looks for itself: an infinity in
// the prefix takes 0.34 ms with 64 sequences behind 32768 keys, 6 ms with 16 x 100 tokens
// behind 8192; finite values pay a comparison.
template <int HD, bool BF>
__device__ __forceinline__ void look_up_values(const PrefixParams& p, int64_t row, int chunk, f32x4_t& o) {
    const int kvh = (int)(row / p.mrows), per = p.tokens * p.group;
    const int64_t mrow = row - kvh * p.mrows;
    const int b = (int)(mrow / per), r = (int)(mrow - (int64_t)b * per), t = r / p.group;
    const int r0 = r & ~(kWideRows - 1), nrows = per - r0 < kWideRows ? per - r0 : kWideRows;
    // the largest halves as signed numbers, which positive ones are ordered as, and as
    // unsigned ones, negative
    i16x2_t top[2] = {};
    u16x2_t low[2] = {};
    for (int i = 0; i < p.parts_p + p.parts_s; ++i) {
        const f32x4_t x =
            *reinterpret_cast<const f32x4_t*>(p.part_o + ((int64_t)i * p.rows + row) * HD + chunk * 4) * 0.0f;
        if (x[0] + x[1] + x[2] + x[3] == 0.0f) continue;
        int k, kend;
        const uint16_t* v;
        int64_t stride;
        if (i < p.parts_p) {
            k = i * p.chunk;
            kend = k + p.chunk < p.prefix ? k + p.chunk : p.prefix;
            v = p.pv + kvh * p.pvs.h;
            stride = p.pvs.s;
        } else {
            const SuffixPart keys(p, b, i - p.parts_p, r0, nrows);
            k = keys.k0;
            kend = keys.kend < keys.seen + t ? keys.kend : keys.seen + t;
            v = p.sv + b * p.svs.b + kvh * p.svs.h;
            stride = p.svs.s;
        }
        for (; k < kend; k += 6) {  // six loads in flight; the last key again past the end
            uint2 w[6];
#pragma unroll
            for (int u = 0; u < 6; ++u)
                w[u] = *reinterpret_cast<const uint2*>(v + (k + u < kend ? k + u : kend - 1) * stride + chunk * 4);
#pragma unroll
            for (int u = 0; u < 6; ++u) {
                top[0] = __builtin_elementwise_max(top[0], __builtin_bit_cast(i16x2_t, w[u].x));
                top[1] = __builtin_elementwise_max(top[1], __builtin_bit_cast(i16x2_t, w[u].y));
                low[0] = __builtin_elementwise_max(low[0], __builtin_bit_cast(u16x2_t, w[u].x));
                low[1] = __builtin_elementwise_max(low[1], __builtin_bit_cast(u16x2_t, w[u].y));
            }
        }
    }
    constexpr int kInf = BF ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int plus = (int)top[e >> 1][e & 1] - kInf, minus = (int)low[e >> 1][e & 1] - (kInf | 0x8000);
        if (plus > 0 || minus > 0 || (plus == 0 && minus == 0)) o[e] = __builtin_nanf("");
        else if (plus == 0 || minus == 0) o[e] = plus == 0 ? __builtin_inff() : -__builtin_inff();
    }
}

// Joins the parts of each row.  HD / 4 lanes hold a row, and G groups of them
// take the parts in turn, four loads in flight each, so that few rows with many
// parts do not wait for one load after the other.
template <int HD, bool BF, int G>
__global__ void __launch_bounds__(256) shared_prefix_join_kernel(PrefixParams p) {
    constexpr int kChunks = HD / 4, kRows = 256 / (kChunks * G);
    const int chunk = threadIdx.x % kChunks, g = threadIdx.x / kChunks % G, r = threadIdx.x / (kChunks * G);
    const int64_t row = (int64_t)blockIdx.x * kRows + r;
    const int parts = p.parts_p + p.parts_s;
    float m = kEmptyMax, l = 0.0f;
    f32x4_t o = (f32x4_t){};
    auto add = [&](float m2, float l2, f32x4_t o2) {
        const float top = __builtin_fmaxf(m, m2);
        const float a = __builtin_amdgcn_exp2f(m - top), a2 = __builtin_amdgcn_exp2f(m2 - top);
        l = __builtin_fmaf(l, a, l2 * a2);
        o = o * a + o2 * a2;
        m = top;
    };
    if (row < p.rows) {
        for (int i = g; i < parts; i += 4 * G) {
            float2 ml[4];
            f32x4_t part[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool in = i + u * G < parts;
                const int64_t at = (int64_t)(in ? i + u * G : i) * p.rows + row;
                ml[u] = p.part_ml[at];
                part[u] = *reinterpret_cast<const f32x4_t*>(p.part_o + at * HD + chunk * 4);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * G < parts) add(ml[u].x, ml[u].y, part[u]);
        }
    }
    if constexpr (G > 1) {
        __shared__ f32x4_t so[256];
        __shared__ float2 sml[256 / kChunks];
        so[threadIdx.x] = o;
        if (chunk == 0) sml[threadIdx.x / kChunks] = make_float2(m, l);
        __syncthreads();
        if (g != 0) return;
#pragma unroll
        for (int u = 1; u < G; ++u) {
            const float2 ml = sml[r * G + u];
            add(ml.x, ml.y, so[threadIdx.x + u * kChunks]);
        }
    }
    if (row >= p.rows) return;
    const f32x4_t zero = o * 0.0f;  // NaN where not finite; a sum that is none makes the row NaN
    if (zero[0] + zero[1] + zero[2] + zero[3] != 0.0f && l - l == 0.0f) look_up_values<HD, BF>(p, row, chunk, o);
    // a row that sees no key is zero
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t kvh = row / p.mrows, mrow = row - kvh * p.mrows, bt = mrow / p.group;
    const int64_t head = kvh * p.group + (mrow - bt * p.group);
    uint2 w;
    if constexpr (BF) {
        w = make_uint2(pack_bf(o[0] * inv, o[1] * inv), pack_bf(o[2] * inv, o[3] * inv));
    } else {
        w = make_uint2(as_u32((h2_t){(_Float16)(o[0] * inv), (_Float16)(o[1] * inv)}),
                       as_u32((h2_t){(_Float16)(o[2] * inv), (_Float16)(o[3] * inv)}));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (bt * p.hq + head) * HD + chunk * 4) = w;
    if (chunk == 0 && p.lse != nullptr) {
        const int64_t b = bt / p.tokens, t = bt - b * p.tokens;
        p.lse[(b * p.hq + head) * p.tokens + t] =
            l == 0.0f ? -__builtin_inff() : (m + __builtin_log2f(l)) * kLn2;
    }
}

// ---- host side -----------------------------------------------------------------

namespace {

constexpr int64_t kMaxBlocks = 0xffffffffll / 256;  // a grid counts its threads in 32 bits

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the work is cut: sets the parts, tiles and blocks.  False: too large.
bool plan(const spline_hip_shared_prefix* a, PrefixParams& p, int64_t& blocks) {
    const int64_t group = a->q_heads / a->kv_heads, per = a->tokens * group;
    if (a->batch > 0x7fffffff / per || a->batch * per > 0x7fffffff / a->kv_heads) return false;
    p.batch = (int)a->batch;
    p.tokens = (int)a->tokens;
    p.hq = (int)a->q_heads;
    p.hkv = (int)a->kv_heads;
    p.group = (int)group;
    p.prefix = (int)a->prefix;
    p.suffix = (int)a->suffix;
    p.mrows = a->batch * per;
    p.rows = p.mrows * p.hkv;
    p.narrow_p = p.mrows <= kNarrowRows;
    p.narrow_s = per <= kNarrowRows;
    p.tiles_p = (int)ceil_div(p.mrows, kWideRows);
    p.tiles_s = (int)ceil_div(per, kWideRows);
    // one round of blocks, two to a CU, if the caches are half full; a narrow block
    // counts kBlockKeys more than its keys.  64 sequences behind 8192 keys, caches of 256:
    // 29.5 us with 128 of them, 31.6 with none, 27.5 with 256; heads of 64: 20.5, 23.4,
    // 22.6; 33 sequences, ungrouped heads of 64: 21.1, 22.5, 22.7.  32 behind 65536,
    // caches of 3000, heads of 64: 57.8 counting each of a cache's blocks, 64.5 one.
    const int64_t slots = 2 * (int64_t)device_shape().cus;
    const int64_t own_blocks = p.narrow_s ? ceil_div(a->suffix, kMostOwnKeys) : 0;
    const int64_t per_cache = (a->suffix + 1) / 2 + kBlockKeys * own_blocks;
    const int64_t keys = p.hkv * (p.tiles_p * a->prefix + a->batch * p.tiles_s * per_cache);
    int64_t each = ceil_div(keys, slots);
    each = each < kLeastKeys ? kLeastKeys : each;
    auto parts_of = [&](int64_t n) { return n <= each ? 1 : n / each; };
    p.parts_p = p.parts_s = 0;
    p.chunk = 64;
    if (p.prefix > 0) {
        p.chunk = (int)(ceil_div(ceil_div(p.prefix, parts_of(p.prefix)), 64) * 64);
        p.parts_p = (int)ceil_div(p.prefix, p.chunk);
    }
    if (p.suffix > 0) {
        // caches differ in length: blocks with few rows take short enough parts to
        // even that out
        const int64_t parts = parts_of(p.suffix), least = own_blocks > 1 ? own_blocks : 1;
        p.parts_s = (int)(parts > least ? parts : least);
    }
    p.once = 4.0 * a->head_dim * p.hkv * ((double)a->prefix + (double)a->batch * a->suffix) >= kMallBytes;
    p.groups_p = p.hkv * p.parts_p;
    p.blocks_p = ceil_div(p.groups_p, 8) * 8 * p.tiles_p;
    const int64_t blocks_s = a->batch * p.parts_s * p.hkv * p.tiles_s;
    blocks = p.blocks_p + blocks_s;
    return blocks <= kMaxBlocks && p.rows <= kMaxBlocks;
}

bool sizes_ok(const spline_hip_shared_prefix* a) {
    const int64_t limit = 1 << 30;  // keys and tokens: those of a part's end stay within 32 bits
    return a && a->batch >= 0 && a->tokens >= 0 && a->q_heads > 0 && a->kv_heads > 0 && a->q_heads % a->kv_heads == 0 &&
           a->q_heads <= 65536 && (a->head_dim == 64 || a->head_dim == 128) && a->prefix >= 0 && a->prefix <= limit &&
           a->suffix >= 0 && a->suffix <= limit && a->tokens <= limit / 65536;
}

template <int MODE, int HD, bool BF>
void go(const PrefixParams& p, int64_t blocks, hipStream_t st) {
    if (blocks > 0)
        hipLaunchKernelGGL((shared_prefix_kernel<MODE, HD, BF>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    if (p.parts_p + p.parts_s > 4)
        hipLaunchKernelGGL((shared_prefix_join_kernel<HD, BF, 8>), dim3((unsigned)ceil_div(p.rows, 128 / HD)), dim3(256),
                           0, st, p);
    else
        hipLaunchKernelGGL((shared_prefix_join_kernel<HD, BF, 1>), dim3((unsigned)ceil_div(p.rows, 1024 / HD)), dim3(256),
                           0, st, p);
}

template <bool BF>
int run(const spline_hip_shared_prefix* a, void* stream) {
    if (!sizes_ok(a) || !(a->scale > 0.0f && a->scale <= __FLT_MAX__)) return hipErrorInvalidValue;
    if (a->mode != kAttnSoftmaxNative && a->mode != kAttnSoftcapNative && !(BF && a->mode == kAttnSoftcapD4))
        return hipErrorInvalidValue;
    if (a->mode != kAttnSoftmaxNative && !(a->cap > 0.0f && a->cap <= __FLT_MAX__)) return hipErrorInvalidValue;
    if (a->batch == 0 || a->tokens == 0) return hipSuccess;
    PrefixParams p{};
    int64_t blocks = 0;
    if (!plan(a, p, blocks)) return hipErrorInvalidValue;
    auto rows_ok = [](const void* x, const int64_t* s, int n) {
        bool ok = x != nullptr && aligned16(x);
        for (int i = 0; i < n; ++i) ok = ok && s[i] >= 0 && s[i] % 8 == 0;
        return ok;
    };
    if (!rows_ok(a->q, a->q_strides, 3) || !a->out || !aligned16(a->out) || ((uintptr_t)a->lse & 3) != 0)
        return hipErrorInvalidValue;
    if (a->prefix > 0 && (!rows_ok(a->prefix_k, a->prefix_k_strides, 2) || !rows_ok(a->prefix_v, a->prefix_v_strides, 2)))
        return hipErrorInvalidValue;
    if (a->suffix > 0 && (!rows_ok(a->suffix_k, a->suffix_k_strides, 3) || !rows_ok(a->suffix_v, a->suffix_v_strides, 3) ||
                          !a->suffix_lens || ((uintptr_t)a->suffix_lens & 3) != 0))
        return hipErrorInvalidValue;
    const int64_t parts = p.parts_p + p.parts_s;
    if (parts > 0 && (!a->workspace || !aligned16(a->workspace))) return hipErrorInvalidValue;
    p.q = static_cast<const uint16_t*>(a->q);
    p.pk = static_cast<const uint16_t*>(a->prefix_k);
    p.pv = static_cast<const uint16_t*>(a->prefix_v);
    p.sk = static_cast<const uint16_t*>(a->suffix_k);
    p.sv = static_cast<const uint16_t*>(a->suffix_v);
    p.lens = a->suffix_lens;
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + parts * p.rows * a->head_dim);
    p.out = a->out;
    p.lse = a->lse;
    p.qs = {a->q_strides[0], a->q_strides[2], a->q_strides[1]};
    p.pks = {0, a->prefix_k_strides[1], a->prefix_k_strides[0]};
    p.pvs = {0, a->prefix_v_strides[1], a->prefix_v_strides[0]};
    p.sks = {a->suffix_k_strides[0], a->suffix_k_strides[2], a->suffix_k_strides[1]};
    p.svs = {a->suffix_v_strides[0], a->suffix_v_strides[2], a->suffix_v_strides[1]};
    // staging adds up to 7 rows to a wave's address as a 32-bit byte offset
    for (const AttnStrides* s : {&p.pks, &p.pvs, &p.sks, &p.svs}) p.wide_strides |= s->s > (int64_t(1) << 27);
    p.scale = a->scale;
    p.cap = a->cap;
    const hipStream_t st = hs(stream);
    auto head = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        a->head_dim == 128 ? go<MODE, 128, BF>(p, blocks, st) : go<MODE, 64, BF>(p, blocks, st);
    };
    if (a->mode == kAttnSoftmaxNative) head(std::integral_constant<int, kAttnSoftmaxNative>{});
    else if (a->mode == kAttnSoftcapNative) head(std::integral_constant<int, kAttnSoftcapNative>{});
    else if constexpr (BF) head(std::integral_constant<int, kAttnSoftcapD4>{});
    return hipGetLastError();
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" int64_t spline_hip_shared_prefix_workspace_bytes(const spline_hip_shared_prefix* a) {
    if (!sizes_ok(a)) return -1;
    if (a->batch == 0 || a->tokens == 0) return 0;
    PrefixParams p{};
    int64_t blocks = 0;
    if (!plan(a, p, blocks)) return -1;
    return (int64_t)(p.parts_p + p.parts_s) * p.rows * (a->head_dim + 2) * 4;
}
extern "C" int launch_shared_prefix_attention_bf16(const spline_hip_shared_prefix* args, void* stream) {
    return run<true>(args, stream);
}
extern "C" int launch_shared_prefix_attention_fp16(const spline_hip_shared_prefix* args, void* stream) {
    return run<false>(args, stream);
}
