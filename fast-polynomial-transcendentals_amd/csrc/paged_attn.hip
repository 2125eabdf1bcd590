// paged_attn.hip -- attention of new tokens over a cache in pages of 4-bit numbers
// (fp4.hpp), for gfx950.
//
//   out[b, t] = softmax(s) V over keys 0 .. lens[b] - T + t of sequence b,
//   s = q.k scale, or cap tanh(q.k scale / cap)
//
// The T g rows of a sequence and KV head (g query heads to a KV head) are cut into
// tiles of 16, 32, 64 or 128; a tile, its keys and a KV head are a unit.  The keys of
// all units, laid end to end in steps, are divided evenly among a fixed number of
// blocks, whatever the lengths are: a block takes its stretch of this line, which
// may begin inside a unit and reach over several.  A unit within one block leaves
// as its result; the pieces of one that is cut leave O, maximum and sum in FP32,
// two pieces a block at most, and a second launch joins them:
// O = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  So neither time nor workspace goes
// by what the table could hold.
//
// Up to 32 rows ("narrow"): of a step's 128 keys each of a block's four waves has 32, and
// none waits for another.  Products are S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32, a lane keeping one row (query).  K needs no LDS: the sum over the head
// dimension may take its elements in any order, so a lane loads 16 bytes of a key, 32 elements
// of one block, and turns each word into a fragment of K (v_cvt_scalef32_pk_bf16_fp4,
// exact); Q's fragments follow that order.  V has to be turned by keys: BF16 rows in the
// wave's own LDS, read back transposed (ds_read_b64_tr_b16).  One token's rows have a form
// of their own where it pays (below), and so have more than 32 rows.
//
// What bounds it: with few rows the bytes of K and V (17 a block of 32 elements), whose loads
// alone take 91 us where 64 sequences of up to 16384 keys (571 MB) take 103 to 109, 6.2 TB/s a
// further key and 15 us a call; from about 64 rows a KV head on the matrix cores and the
// exponentials and conversions beside them: 4 x 512 tokens over 17408 keys 784 us, 734 TFLOP/s (half as
// many products again are those of P's second terms), over up to 8700 keys each 222 us, 655 TFLOP/s, where
// first keys and results of 512 units count.  FP16 queries, of two terms as well, take 1.2 times as long.
// Two sequences of up to 131072 keys take 37 us, 8 of up to 1200 12 us, most of it latency: lengths,
// table, codes and the join one behind the other.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "fp4.hpp"
#include "row_state.hpp"

namespace pt {

// Keys of a block's step
constexpr int kNarrowStep = 128;  // each wave 32 of them
constexpr int kWaveKeys = 32;
constexpr int kDecodeStep = 256;  // each wave 64
constexpr int kWideStep = 64;
// A block's stretch is so long that the longest unit is cut into at most this many pieces, one more for each
// 32 of its steps, and one where it begins inside a stretch: the blocks that join a unit have not more to do
// than those that make its pieces.  One KV head, 131072 keys: with 8 heads of 64 21 us, 41 with a piece a
// block; 4 heads of 128 26 and 57; 8 of 128 beside 15 sequences of 100 keys 29, 66 where the pieces of all
// units are counted together, so that the short ones leave theirs to the long one.
constexpr int kPieces = 64;
// A unit's first keys and its result cost as much as so many steps more: 4 x 512 tokens
// over up to 8700 keys 311 us counting none, 280 with one, 254 with two, 231 with four, 238 with
// eight; 64 decoding sequences 136, 131 with one or two, 135 with four.
constexpr int unit_steps(int step) { return step == kWideStep ? 4 : 2; }

struct PagedParams {
    const uint16_t* q;
    Fp4Pages c;
    AttnStrides qs;
    float* part_o;    // [2 blocks][ROWS][HD]
    float2* part_ml;  // [2 blocks][ROWS]
    int4* cut;        // [blocks] the unit that leaves a block unfinished: batch, KV head and (from bit 16
                      // on) the block's number on the line, pieces (0: no such unit), first row
    void* out;
    float* lse;
    int hq, group, tokens, rows, tiles, capacity;
    int places;  // batch * tiles
    float scale, cap;
};

__device__ __forceinline__ f32x4_t mfma16(bf16x8_t a, bf16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Has the compiler wait for a fragment's load here: where it is first used inside a loop,
// the wait there would be for every load issued since, in every turn.
__device__ __forceinline__ void loaded(bf16x8_t& f) { asm volatile("" : "+v"(f)); }

// Over the lanes of a row (l ^ 16 and l ^ 32): the largest of N scores, NaN if one is
// (v_maximum3_f32: no instructions that quiet its operands), and a sum.
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <int N>
__device__ __forceinline__ float row_max(const float (&y)[N]) {
    float x = maximum(maximum(y[0], y[1]), y[2]);
#pragma unroll
    for (int e = 3; e + 1 < N; e += 2) x = maximum(maximum(x, y[e]), y[e + 1]);
    x = maximum(x, y[N - 1]);
    const auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
    x = maximum(as_f32(r[0]), as_f32(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
    return maximum(as_f32(t[0]), as_f32(t[1]));
}
__device__ __forceinline__ float row_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
    return half_sum(as_f32(r[0]) + as_f32(r[1]));
}

// ---- the line of all units ------------------------------------------------------

// A row tile of a sequence.
template <int ROWS, int STEP>
struct Place {
    int b;
    int r0, nrows;  // rows of the sequence
    int seen;       // keys that token 0 sees (token t: t more), not held to the table
    int visible;    // keys that the tile's last row sees

    __device__ __forceinline__ Place(const PagedParams& p, int place) {
        b = place / p.tiles;
        r0 = (place - b * p.tiles) * ROWS;
        nrows = p.rows - r0 < ROWS ? p.rows - r0 : ROWS;
        seen = p.c.len(b) - p.tokens + 1;
        visible = keys_of(p, (r0 + nrows - 1) / p.group);
    }
    // Keys that a token sees.
    __device__ __forceinline__ int keys_of(const PagedParams& p, int token) const {
        const int64_t n = (int64_t)seen + token;
        return n < 0 ? 0 : n < p.capacity ? (int)n : p.capacity;
    }
    // One at least: a tile without keys leaves zeros.
    __device__ __forceinline__ int steps() const { return visible <= STEP ? 1 : (visible + STEP - 1) / STEP; }
    // On the line.
    __device__ __forceinline__ int length() const { return steps() + unit_steps(STEP); }
};

// A block's stretch of the line: x to x1 of all steps (fewer than 2^31), from `in` of a
// place and KV head on.  The first `longer` blocks have each + 1 steps, the others each.
template <int ROWS, int STEP>
struct Stretch {
    using At = Place<ROWS, STEP>;
    static constexpr int kUnit = unit_steps(STEP);
    int block, each, longer, x, x1, place, kvh, in;

    // False: none (and the block's cut says so).  SHARED: neighbours on the line, which read
    // the same keys, are on one XCD, whose L2 holds them.
    template <bool SHARED>
    __device__ __forceinline__ bool find(const PagedParams& p) {
        __shared__ int sums[4], most[4], start[2];
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int per = (p.places + 255) / 256;
        const int64_t first = (int64_t)tid * per;
        const int from = first < p.places ? (int)first : p.places, to = p.places - from < per ? p.places : from + per;
        int mine = 0, plane = 0, ahead = 0;  // steps of the thread's places, of a KV head, ahead
        int top = 0;                         // the thread's longest place
        for (int i = from; i < to; ++i) {
            const int n = At(p, i).length();
            mine += n;
            top = n > top ? n : top;
        }
        int inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(inc, d);
            inc += lane >= d ? y : 0;
            const int z = __shfl_xor(top, d);
            top = z > top ? z : top;
        }
        if (lane == 63) {
            sums[wave] = inc;
            most[wave] = top;
        }
        __syncthreads();
        int longest = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ahead += w < wave ? sums[w] : 0;
            plane += sums[w];
            longest = most[w] > longest ? most[w] : longest;
        }
        ahead += inc - mine;
        const int all = plane * p.c.hkv;
        const int pieces = kPieces + longest / 32, least = (longest + pieces - 1) / pieces;  // steps of a stretch
        int blocks = all / least;
        blocks = blocks < (int)gridDim.x ? blocks : (int)gridDim.x;
        const int id = (int)blockIdx.x, share = (blocks + 7) / 8;
        block = SHARED ? id % 8 * share + id / 8 : id;
        if (block >= blocks || (SHARED && id / 8 >= share)) {
            if (tid == 0) p.cut[id] = make_int4(0, 0, 0, 0);
            return false;
        }
        each = all / blocks;
        longer = all - each * blocks;
        x = block * each + (block < longer ? block : longer);
        x1 = x + each + (block < longer ? 1 : 0);
        kvh = x / plane;
        const int at = x - kvh * plane;
        if (at >= ahead && at < ahead + mine)
            for (int i = from; i < to; ++i) {
                const int n = At(p, i).length();
                if (at < ahead + n) {
                    start[0] = i;
                    start[1] = at - ahead;
                    break;
                }
                ahead += n;
            }
        __syncthreads();
        place = start[0];
        in = start[1];
        return true;
    }
    // The block's steps of the unit that it is at: the first, and behind the last.
    __device__ __forceinline__ int first() const { return in > kUnit ? in - kUnit : 0; }
    __device__ __forceinline__ int last(int steps) const {
        const int end = in + (x1 - x) - kUnit;
        return end < 0 ? 0 : end < steps ? end : steps;
    }
    // Goes on behind a unit.  What the block leaves unfinished is its cut.
    __device__ __forceinline__ void advance(const PagedParams& p, const At& at) {
        const int steps = at.steps(), end = x - in + steps + kUnit;  // of the unit
        if (threadIdx.x == 0 && end >= x1) {
            int4 cut = make_int4(0, 0, 0, 0);
            if (first() == 0 && last(steps) > 0 && last(steps) < steps) {
                // the block with the unit's last step
                const int to = end - 1, many = longer * (each + 1);
                const int stop = to < many ? to / (each + 1) : longer + (to - many) / each;
                cut = make_int4(at.b, block << 16 | kvh, stop - block + 1, at.r0);
            }
            p.cut[blockIdx.x] = cut;
        }
        x = end;
        in = 0;
        if (++place == p.places) {
            place = 0;
            ++kvh;
        }
    }
};

// ---- scores -----------------------------------------------------------------------

// The capped scores of a softcap mode (softmax_exponents for any even number).
template <int MODE, int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], const ScoreConsts& k) {
    if constexpr (MODE == kAttnSoftcapD4) {
#pragma unroll
        for (int r = 0; r < N; r += 2) {
            const uint32_t u = pack_bf(rbf(x[r] * k.scale) * k.inv_cap, rbf(x[r + 1] * k.scale) * k.inv_cap);
            float t0, t1;
            SoftcapConsts::T::eval2(u, k.tanh, t0, t1);
            x[r] = rbf(t0 * k.cap);
            x[r + 1] = rbf(t1 * k.cap);
        }
    } else if constexpr (MODE == kAttnSoftcapNative) {
#pragma unroll
        for (int r = 0; r < N; ++r) x[r] = k.cap * native_lane<kTanh, kFwd>(x[r] * k.scale * k.inv_cap);
    }
}

__device__ __forceinline__ bf16x8_t row_probs(const float (&s)[8]) {
    bf16x8_t f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (__bf16)s[e];
    return f;
}
// What that rounding left, as a second operand.
__device__ __forceinline__ bf16x8_t row_rests(const float (&s)[8], bf16x8_t hi) {
    bf16x8_t f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (__bf16)(s[e] - (float)hi[e]);
    return f;
}

// Eight FP16 numbers as the sum of two BF16 ones, which is exact.
__device__ __forceinline__ void split_fp16(bf16x8_t bits, bf16x8_t& hi, bf16x8_t& lo) {
    const f16x8_t x = __builtin_bit_cast(f16x8_t, bits);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = (float)x[e];
        hi[e] = (__bf16)v;
        const float left = v - (float)hi[e];
        lo[e] = (__bf16)(left - left == 0.0f ? left : 0.0f);  // none of an infinity
    }
}

// FP32 rows of O in LDS, 16 bytes between them: 16 rows' chunks fall on different columns.
template <int HD>
__device__ __forceinline__ constexpr uint32_t o_at(int row, int chunk) {
    return (uint32_t)(row * (HD * 4 + 16) + chunk * 16);
}

// Elements 4 chunk .. of a row of a place, divided by their sum, to the result.
template <int HD, bool BF>
__device__ __forceinline__ void write_row(const PagedParams& p, int b, int row, int kvh, int chunk, f32x4_t o,
                                          float2 ml) {
    const float inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;  // a row that sees no key is zero
    const int t = row / p.group, head = kvh * p.group + (row - t * p.group);
    const int64_t bt = (int64_t)b * p.tokens + t;
    uint2 w;
    if constexpr (BF) {
        w = make_uint2(pack_bf(o[0] * inv, o[1] * inv), pack_bf(o[2] * inv, o[3] * inv));
    } else {
        w = make_uint2(as_u32((h2_t){(_Float16)(o[0] * inv), (_Float16)(o[1] * inv)}),
                       as_u32((h2_t){(_Float16)(o[2] * inv), (_Float16)(o[3] * inv)}));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (bt * p.hq + head) * HD + chunk * 4) = w;
    if (chunk == 0 && p.lse != nullptr)
        p.lse[((int64_t)b * p.hq + head) * p.tokens + t] =
            ml.y == 0.0f ? -__builtin_inff() : (ml.x + __builtin_log2f(ml.y)) * kLn2;
}

// ---- a wave's tile of 32 keys -------------------------------------------------------

// A wave's rows of V in BF16, 32 bytes between them and 16 more between groups of eight.
// A transposing read takes 256 bytes at once, eight rows by 32 bytes, which fall on
// different columns; a write 128 bytes, 16 of eight lanes: lanes 0..7 have the rows 0..3
// and 8..11 (v_key), and those do.
template <int HD>
__device__ __forceinline__ constexpr uint32_t v_at(int row, int chunk) {
    return (uint32_t)(row * (HD * 2 + 32) + (row >> 3) * 16 + chunk * 16);
}

// The key of 16 whose values a lane holds.
__device__ __forceinline__ int v_key(int c16) { return (c16 & 3) | (c16 & 4) << 1 | (c16 & 8) >> 1; }

// Where a lane's codes of 16 keys lie: HD / 4 elements of a key (row) from quarter HD / 4
// on, and the word with their block's byte.
template <int HD>
struct LaneCodes {
    uint32_t code, word, shift;

    __device__ __forceinline__ LaneCodes(const Fp4Pages& c, int row, int quarter) {
        code = (uint32_t)(row * (HD / 2) + quarter * (HD / 8));
        const uint32_t byte = (uint32_t)(c.page_size * (HD / 2) + row * (HD / kFp4Block) + quarter * (HD / 4) / kFp4Block);
        word = byte & ~3u;
        shift = (byte & 3) * 8;
    }
};

// The codes of 16 keys that a lane holds.  The byte is loaded in its word: what the
// compiler makes of a byte that goes round a loop waits for it too early.
template <int HD>
struct Codes {
    uint32_t w[HD / 32];
    uint32_t word;

    __device__ __forceinline__ uint32_t byte(const LaneCodes<HD>& lane) const {
        return __builtin_amdgcn_ubfe(word, lane.shift, 8);
    }

    template <bool ONCE>
    __device__ __forceinline__ void load(const uint8_t* head, uint32_t code, uint32_t at) {
        typedef typename std::conditional<HD == 128, u32x4_t, u32x2_t>::type Words;
        const Words* src = reinterpret_cast<const Words*>(head + code);
        const Words a = ONCE ? __builtin_nontemporal_load(src) : *src;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) w[i] = a[i];
        const uint32_t* bytes = reinterpret_cast<const uint32_t*>(head + at);
        word = ONCE ? __builtin_nontemporal_load(bytes) : *bytes;
    }
    // Of page 0 where there is none (its keys are masked, its values cleared): a branch would
    // have every wait for a load wait for all of them.
    // ONCE: a block's keys are its own, and pass the caches: 32 sequences of up to 8191 keys, 32 / 8 heads of
    // 128, 46 us, 51 through them.  Rows of a fork read the pages that they share once each, which
    // the caches would serve in part: 64 prompts of up to 2000 keys with four samples each 92 us, 82 through
    // them, of up to 8191 297 and 284.  A call does not know what its tables share.
    template <bool ONCE>
    __device__ __forceinline__ void load(const Fp4Pages& c, int page, int row, int kv, int h, const LaneCodes<HD>& lane) {
        load<ONCE>(c.head(page < 0 ? 0 : page, kv, h), (uint32_t)row * (HD / 2) + lane.code,
                   (uint32_t)row * (HD / kFp4Block) + lane.word);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) w[i] = 0;
        word = 0;
    }
};

// The rows that a lane's query has seen so far.
template <int HD>
struct PagedState {
    f32x4_t o[HD / 16];  // O^T: o[dt][r] = element 16 dt + 4 (lane / 16) + r of row lane % 16
    float m, l;          // log2 units; l of this lane's quarter of the keys

    __device__ __forceinline__ PagedState() : m(kEmptyMax), l(0.0f) {
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) o[dt] = (f32x4_t){};
    }
};

// Up to 32 rows: NR tiles of 16, which share a wave's fragments of K and V.
template <int MODE, int HD, int NR, bool BF>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NR == 1 ? (HD == 64 ? 4 : 3) : 2))) paged_narrow_kernel(PagedParams p) {
    constexpr int ROWS = 16 * NR, kC = HD / 32, kD = HD / 16;
    constexpr int kVTile = v_at<HD>(kWaveKeys, 0), kSpill = o_at<HD>(16, 0);
    constexpr int kRegion = kVTile > kSpill ? kVTile : kSpill;
    __shared__ __align__(1024) unsigned char smem[4 * kRegion];
    __shared__ float2 sml[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c16 = lane & 15, quarter = lane >> 4;
    Stretch<ROWS, kNarrowStep> line;
    if (!line.template find<false>(p)) return;

    ScoreConsts consts;
    consts.sl = attn_is_plain_softmax(MODE) ? p.scale * kLog2e : kLog2e;
    consts.scale = p.scale;
    consts.cap = p.cap;
    consts.inv_cap = 1.0f / p.cap;
    if constexpr (MODE == kAttnSoftcapD4)
#pragma unroll
        for (int i = 1; i <= SoftcapConsts::T::P.deg; ++i) consts.tanh[i] = bf16_value(SoftcapConsts::T::P.c[i]);

    unsigned char* vt = smem + wave * kRegion;
    while (line.x < line.x1) {
        const Place<ROWS, kNarrowStep> at(p, line.place);
        const int steps = at.steps(), step0 = line.first(), n = line.last(steps) - step0, kvh = line.kvh;
        if (n == 0) {
            line.advance(p, at);
            break;
        }
        // ---- Q^T fragments: elements (HD / 4) quarter + 8 c .. of row c16
        bf16x8_t qf[NR][kC], ql[BF ? 1 : NR][kC];
        int klast[NR];  // the last key that the lane's row sees
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const int row = nr * 16 + c16;
            const bool rin = row < at.nrows;
            const int t = (at.r0 + (rin ? row : 0)) / p.group;
            klast[nr] = (rin ? at.keys_of(p, t) : at.visible) - 1;
            const uint16_t* src = p.q + at.b * p.qs.b + t * p.qs.s +
                                  (kvh * p.group + (at.r0 + (rin ? row : 0) - t * p.group)) * p.qs.h + quarter * (HD / 4);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                bf16x8_t f = {};
                if (rin) f = *reinterpret_cast<const bf16x8_t*>(src + 8 * c);
                if constexpr (!BF) split_fp16(f, qf[nr][c], ql[nr][c]);
                else qf[nr][c] = f;
            }
        }
        PagedState<HD> st[NR];
        const int kfull = at.keys_of(p, at.r0 / p.group) - 1;  // every row sees the keys up to it

        // ---- the wave's tiles of 32 keys, one a step.  Lane 2 i + g knows where group g
        // of step i lies, 32 steps at a time.  Codes of the next tile fly from where this
        // one's are used on.
        int my_page = -1, my_row = 0;
        auto look_up = [&](int i0) __attribute__((always_inline)) {
            const int key = (step0 + i0 + (lane >> 1)) * kNarrowStep + wave * kWaveKeys + (lane & 1) * 16;
            const int entry = key / p.c.page_size;
            my_page = i0 + (lane >> 1) < n && key < at.visible ? p.c.page_of(at.b, entry) : -1;
            my_row = key - entry * p.c.page_size;
        };
        const LaneCodes<HD> k_lane(p.c, c16, quarter), v_lane(p.c, v_key(c16), quarter);
        const int vkey = v_key(c16);
        unsigned char* const v_write = vt + v_at<HD>(vkey, quarter * kC);
        auto load = [&](Codes<HD>& codes, int kv, int i, int g) __attribute__((always_inline)) {
            const int l = 2 * (i & 31) + g;
            codes.template load<true>(p.c, __builtin_amdgcn_readlane(my_page, l), __builtin_amdgcn_readlane(my_row, l), kv, kvh,
                                      kv ? v_lane : k_lane);
        };
        const unsigned char* const v_read = vt + v_at<HD>(4 * quarter + (c16 >> 2), (c16 & 3) >> 1) + (c16 & 1) * 8;
        // columns 16 dt + c16 of rows 4 quarter .. + 3 and 16 + 4 quarter .. + 3
        auto value_frag = [&](int dt) __attribute__((always_inline)) {
            const uint16_t* src = reinterpret_cast<const uint16_t*>(v_read + dt * 32);
            const u32x2_t lo = __builtin_bit_cast(u32x2_t, lds_read_tr16(src));
            const u32x2_t hi = __builtin_bit_cast(u32x2_t, lds_read_tr16(src + v_at<HD>(16, 0) / 2));
            return __builtin_bit_cast(bf16x8_t, (u32x4_t){lo.x, lo.y, hi.x, hi.y});
        };
        Codes<HD> k[2], v[2];
        const int tiles = p.c.pages > 0 ? n : 0;
        if (tiles > 0) {
            look_up(0);
#pragma unroll
            for (int g = 0; g < 2; ++g) load(k[g], 0, 0, g);
#pragma unroll
            for (int g = 0; g < 2; ++g) load(v[g], 1, 0, g);
        }
        if constexpr (BF)
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int c = 0; c < kC; ++c) loaded(qf[nr][c]);
        for (int i = 0; i < tiles; ++i) {
            const int key0 = (step0 + i) * kNarrowStep + wave * kWaveKeys;
            const bool hole[2] = {__builtin_amdgcn_readlane(my_page, 2 * (i & 31)) < 0,
                                  __builtin_amdgcn_readlane(my_page, 2 * (i & 31) + 1) < 0};
            const bool masked = key0 + kWaveKeys - 1 > kfull || hole[0] || hole[1];
            if ((i & 31) == 31) look_up(i + 1);  // no page behind the last tile
            f32x4_t s[2][NR];
            const float scale[2] = {fp4_scale(k[0].byte(k_lane)), fp4_scale(k[1].byte(k_lane))};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) s[0][nr] = s[1][nr] = (f32x4_t){};
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const bf16x8_t kf = fp4_to_bf16(k[g].w[c], scale[g]);
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        s[g][nr] = mfma16(kf, qf[nr][c], s[g][nr]);
                        if constexpr (!BF) s[g][nr] = mfma16(kf, ql[nr][c], s[g][nr]);
                    }
                }
#pragma unroll
            for (int g = 0; g < 2; ++g) load(k[g], 0, i + 1, g);
            // V to LDS; in a tile with keys that some row does not see, blocks that are no
            // numbers as zeros (0 * NaN is NaN)
            bool bad[2] = {false, false};
            if (masked)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    bad[g] = v[g].byte(v_lane) > (uint32_t)kFp4Most && !hole[g];
                    if (bad[g] || hole[g]) v[g].clear();
                }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float scale = fp4_scale(v[g].byte(v_lane));
#pragma unroll
                for (int c = 0; c < kC; ++c)
                    *reinterpret_cast<bf16x8_t*>(v_write + v_at<HD>(16 * g, c)) = fp4_to_bf16(v[g].w[c], scale);
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) load(v[g], 1, i + 1, g);
            __builtin_amdgcn_sched_barrier(0);
            // probabilities of keys 4 quarter + r of the first group, then of the second
            bf16x8_t pf[NR], pr[NR];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = s[e >> 2][nr][e & 3];
                cap_scores<MODE>(y, consts);
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (hole[e >> 2] || key0 + 16 * (e >> 2) + 4 * quarter + (e & 3) > klast[nr]) y[e] = -__builtin_inff();
                }
                const float mx = row_max(y) * consts.sl;
                const bool move = mx - st[nr].m > 8.0f;  // the lanes of a row decide alike
                if (__any(move)) {
                    const float m = move ? mx : st[nr].m;
                    const float alpha = __builtin_amdgcn_exp2f(st[nr].m - m);
                    st[nr].m = m;
                    st[nr].l *= alpha;
#pragma unroll
                    for (int dt = 0; dt < kD; ++dt) st[nr].o[dt] *= alpha;
                }
                float mul = consts.sl;
                const bool far = __builtin_fabsf(st[nr].m) >= kFarMax;
                if (__any(far)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = far ? y[e] * mul : y[e];
                    mul = far ? 1.0f : mul;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[e], mul, -st[nr].m));
                st[nr].l += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
                pf[nr] = row_probs(y);
                pr[nr] = row_rests(y, pf[nr]);
            }
            // O^T += V^T P^T, fragments of V three ahead
            __builtin_amdgcn_sched_barrier(0);
            bf16x8_t vf[kD];
#pragma unroll
            for (int dt = 0; dt < kD && dt < 3; ++dt) vf[dt] = value_frag(dt);
#pragma unroll
            for (int dt = 0; dt < kD; ++dt) {
                if (dt + 3 < kD) vf[dt + 3] = value_frag(dt + 3);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    st[nr].o[dt] = mfma16(vf[dt], pf[nr], st[nr].o[dt]);
                    st[nr].o[dt] = mfma16(vf[dt], pr[nr], st[nr].o[dt]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // what is NaN in V reaches the rows that see it
#pragma unroll
            for (int g = 0; g < 2; ++g)
                for (uint64_t m = __ballot(bad[g]); m != 0; m &= m - 1) {
                    const int l = __builtin_ctzll(m), key = key0 + 16 * g + v_key(l & 15), part = l >> 4;  // of the head, in four
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                        for (int dt = 0; dt < kD; ++dt)
                            if (key <= klast[nr] && dt / (kD / 4) == part)
#pragma unroll
                                for (int r = 0; r < 4; ++r) st[nr].o[dt][r] = __builtin_nanf("");
                }
        }

        // ---- the waves' shares of each row
        const bool begins = step0 == 0, ends = step0 + n == steps;
        const int slot = 2 * line.block + (begins ? 1 : 0);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            if (nr * 16 >= at.nrows) break;
            __syncthreads();  // the region is free
            unsigned char* region = smem + wave * kRegion;
#pragma unroll
            for (int dt = 0; dt < kD; ++dt)
                *reinterpret_cast<f32x4_t*>(region + o_at<HD>(c16, 4 * dt + quarter)) = st[nr].o[dt];
            const float l = row_sum(st[nr].l);
            if (quarter == 0) sml[wave][c16] = make_float2(st[nr].m, l);
            __syncthreads();
            constexpr int kChunks = HD / 4;
            for (int i = tid; i < 16 * kChunks; i += 256) {
                const int row = i / kChunks, chunk = i % kChunks;
                if (nr * 16 + row >= at.nrows) continue;
                float2 ml = make_float2(kEmptyMax, 0.0f);
#pragma unroll
                for (int w = 0; w < 4; ++w) ml.x = __builtin_fmaxf(ml.x, sml[w][row].x);
                f32x4_t o = {};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float2 y = sml[w][row];
                    const float a = __builtin_amdgcn_exp2f(y.x - ml.x);
                    o += *reinterpret_cast<const f32x4_t*>(smem + w * kRegion + o_at<HD>(row, chunk)) * a;
                    ml.y = __builtin_fmaf(y.y, a, ml.y);
                }
                if (begins && ends) {
                    write_row<HD, BF>(p, at.b, at.r0 + nr * 16 + row, kvh, chunk, o, ml);
                } else {
                    *reinterpret_cast<f32x4_t*>(p.part_o + (int64_t)(slot * ROWS + nr * 16 + row) * HD + chunk * 4) = o;
                    if (chunk == 0) p.part_ml[slot * ROWS + nr * 16 + row] = ml;
                }
            }
        }
        __syncthreads();
        line.advance(p, at);
    }
}

// ---- one new token -------------------------------------------------------------------
//
// The same for the up to 8 rows of a single token, all of which see the same keys.  A
// wave has 64 keys of a step, in groups of 16, and its 16 columns hold the rows NC =
// 2 or 4 times, 16 / NC columns each.  All columns of a group's scores are alike, so
// column class c takes those of group c: the maximum, the exponentials and a softcap run
// over NC groups at once.  In P the other groups' rows of a column are zero, so that a
// column keeps a softmax over its class's keys, and the classes of a row are joined as the
// waves are.
template <int MODE, int HD, int NC, bool BF>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 || BF ? 3 : 2))) paged_decode_kernel(PagedParams p) {
    constexpr int ROWS = 16, W = 16 / NC, kA = 4 / NC;  // rows' columns; accumulators of scores
    constexpr int kC = HD / 32, kD = HD / 16;
    constexpr int kVTile = v_at<HD>(32, 0), kSpill = o_at<HD>(16, 0);
    constexpr int kRegion = kVTile > kSpill ? kVTile : kSpill;
    __shared__ __align__(1024) unsigned char smem[4 * kRegion];
    __shared__ float2 sml[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c16 = lane & 15, quarter = lane >> 4, cls = c16 / W;
    Stretch<ROWS, kDecodeStep> line;
    if (!line.template find<false>(p)) return;

    ScoreConsts consts;
    consts.sl = attn_is_plain_softmax(MODE) ? p.scale * kLog2e : kLog2e;
    consts.scale = p.scale;
    consts.cap = p.cap;
    consts.inv_cap = 1.0f / p.cap;
    if constexpr (MODE == kAttnSoftcapD4)
#pragma unroll
        for (int i = 1; i <= SoftcapConsts::T::P.deg; ++i) consts.tanh[i] = bf16_value(SoftcapConsts::T::P.c[i]);

    unsigned char* const vt = smem + wave * kRegion;
    const int vkey = v_key(c16);
    unsigned char* const v_write = vt + v_at<HD>(vkey, quarter * kC);
    const unsigned char* const v_read = vt + v_at<HD>(4 * quarter + (c16 >> 2), (c16 & 3) >> 1) + (c16 & 1) * 8;
    auto value_frag = [&](int dt) __attribute__((always_inline)) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(v_read + dt * 32);
        const u32x2_t lo = __builtin_bit_cast(u32x2_t, lds_read_tr16(src));
        const u32x2_t hi = __builtin_bit_cast(u32x2_t, lds_read_tr16(src + v_at<HD>(16, 0) / 2));
        return __builtin_bit_cast(bf16x8_t, (u32x4_t){lo.x, lo.y, hi.x, hi.y});
    };
    const LaneCodes<HD> k_lane(p.c, c16, quarter), v_lane(p.c, v_key(c16), quarter);

    while (line.x < line.x1) {
        const Place<ROWS, kDecodeStep> at(p, line.place);
        const int steps = at.steps(), step0 = line.first(), n = line.last(steps) - step0, kvh = line.kvh;
        if (n == 0) {
            line.advance(p, at);
            break;
        }
        // ---- Q^T fragments, the rows in every class
        bf16x8_t qf[kC], ql[BF ? 1 : kC];
        {
            const int row = c16 % W;
            const uint16_t* src = p.q + at.b * p.qs.b + (kvh * p.group + (row < p.group ? row : 0)) * p.qs.h + quarter * (HD / 4);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                bf16x8_t f = {};
                if (row < p.group) f = *reinterpret_cast<const bf16x8_t*>(src + 8 * c);
                if constexpr (!BF) split_fp16(f, qf[c], ql[c]);
                else qf[c] = f;
            }
        }
        // ---- pages: lane 4 i + g knows where group g of step i lies, 16 steps at a time
        int my_page = -1, my_row = 0;
        auto look_up = [&](int i0) __attribute__((always_inline)) {
            const int key = (step0 + i0 + (lane >> 2)) * kDecodeStep + wave * 64 + (lane & 3) * 16;
            const int entry = key / p.c.page_size;
            my_page = i0 + (lane >> 2) < n && key < at.visible ? p.c.page_of(at.b, entry) : -1;
            my_row = key - entry * p.c.page_size;
        };
        Codes<HD> k[4], v[4];
        auto load = [&](Codes<HD>& codes, int kv, int i, int g) __attribute__((always_inline)) {
            const int l = 4 * (i & 15) + g;
            codes.template load<true>(p.c, __builtin_amdgcn_readlane(my_page, l), __builtin_amdgcn_readlane(my_row, l), kv, kvh,
                                      kv ? v_lane : k_lane);
        };
        const int tiles = p.c.pages > 0 ? n : 0;
        if (tiles > 0) {
            look_up(0);
#pragma unroll
            for (int g = 0; g < 4; ++g) load(k[g], 0, 0, g);
#pragma unroll
            for (int g = 0; g < 4; ++g) load(v[g], 1, 0, g);
        }
        if constexpr (BF)
#pragma unroll
            for (int c = 0; c < kC; ++c) loaded(qf[c]);
        PagedState<HD> st;
        for (int i = 0; i < tiles; ++i) {
            const int key0 = (step0 + i) * kDecodeStep + wave * 64;
            const uint32_t holes = (uint32_t)(__ballot(my_page < 0) >> (4 * (i & 15))) & 15;
            const bool masked = key0 + 63 >= at.visible || holes != 0;
            if ((i & 15) == 15) look_up(i + 1);  // no page behind the last tile
            f32x4_t s[4];
            float scale[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                s[g] = (f32x4_t){};
                scale[g] = fp4_scale(k[g].byte(k_lane));
            }
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const bf16x8_t kf = fp4_to_bf16(k[g].w[c], scale[g]);
                    s[g] = mfma16(kf, qf[c], s[g]);
                    if constexpr (!BF) s[g] = mfma16(kf, ql[c], s[g]);
                }
#pragma unroll
            for (int g = 0; g < 4; ++g) load(k[g], 0, i + 1, g);
            // scores of the column's groups: keys 16 (NC a + cls) + 4 quarter + r
            float y[4 * kA];
#pragma unroll
            for (int a = 0; a < kA; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = s[NC * a][r];
#pragma unroll
                    for (int c = 1; c < NC; ++c) x = cls == c ? s[NC * a + c][r] : x;
                    y[4 * a + r] = x;
                }
            cap_scores<MODE>(y, consts);
            if (masked) {
#pragma unroll
                for (int g = 0; g < 4; ++g)  // what is not seen may be no number
                    if ((holes >> g & 1) || key0 + 16 * g + vkey >= at.visible) v[g].clear();
#pragma unroll
                for (int a = 0; a < kA; ++a)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int g = NC * a + cls;
                        if ((holes >> g & 1) || key0 + 16 * g + 4 * quarter + r >= at.visible) y[4 * a + r] = -__builtin_inff();
                    }
            }
            const float mx = row_max(y) * consts.sl;
            const bool move = mx - st.m > 8.0f;  // the lanes of a column decide alike
            if (__any(move)) {
                const float m = move ? mx : st.m;
                const float alpha = __builtin_amdgcn_exp2f(st.m - m);
                st.m = m;
                st.l *= alpha;
#pragma unroll
                for (int dt = 0; dt < kD; ++dt) st.o[dt] *= alpha;
            }
            float mul = consts.sl;
            const bool far = __builtin_fabsf(st.m) >= kFarMax;
            if (__any(far)) {
#pragma unroll
                for (int e = 0; e < 4 * kA; ++e) y[e] = far ? y[e] * mul : y[e];
                mul = far ? 1.0f : mul;
            }
            uint32_t hi[2 * kA], lo[2 * kA];  // pairs of probabilities in two BF16 terms
#pragma unroll
            for (int e = 0; e < 4 * kA; e += 2) {
                const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(y[e], mul, -st.m));
                const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(y[e + 1], mul, -st.m));
                st.l += a + b;
                const bf16x2_t h = {(__bf16)a, (__bf16)b};
                const bf16x2_t rest = {(__bf16)(a - (float)h.x), (__bf16)(b - (float)h.y)};
                hi[e / 2] = __builtin_bit_cast(uint32_t, h);
                lo[e / 2] = __builtin_bit_cast(uint32_t, rest);
            }
            // O^T += V^T P^T, 32 keys at a time
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int a = 2 * t / NC, c0 = 2 * t % NC;  // the classes of its groups: c0 and c0 + 1
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float sv = fp4_scale(v[2 * t + g].byte(v_lane));
#pragma unroll
                    for (int c = 0; c < kC; ++c)
                        *reinterpret_cast<bf16x8_t*>(v_write + v_at<HD>(16 * g, c)) = fp4_to_bf16(v[2 * t + g].w[c], sv);
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) load(v[2 * t + g], 1, i + 1, 2 * t + g);
                auto frag = [&](const uint32_t (&w)[2 * kA]) __attribute__((always_inline)) {
                    const bool x = cls == c0, z = cls == c0 + 1;
                    return __builtin_bit_cast(bf16x8_t, (u32x4_t){x ? w[2 * a] : 0, x ? w[2 * a + 1] : 0, z ? w[2 * a] : 0,
                                                                  z ? w[2 * a + 1] : 0});
                };
                const bf16x8_t pf = frag(hi), pr = frag(lo);
                __builtin_amdgcn_sched_barrier(0);
                bf16x8_t vf[kD];
#pragma unroll
                for (int dt = 0; dt < 3; ++dt) vf[dt] = value_frag(dt);
#pragma unroll
                for (int dt = 0; dt < kD; ++dt) {
                    if (dt + 3 < kD) vf[dt + 3] = value_frag(dt + 3);
                    st.o[dt] = mfma16(vf[dt], pf, st.o[dt]);
                    st.o[dt] = mfma16(vf[dt], pr, st.o[dt]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }

        // ---- the shares of each row: four waves' classes
        const bool begins = step0 == 0, ends = step0 + n == steps;
        const int slot = 2 * line.block + (begins ? 1 : 0);
        __syncthreads();  // the region is free
#pragma unroll
        for (int dt = 0; dt < kD; ++dt) *reinterpret_cast<f32x4_t*>(vt + o_at<HD>(c16, 4 * dt + quarter)) = st.o[dt];
        const float l = row_sum(st.l);
        if (quarter == 0) sml[wave][c16] = make_float2(st.m, l);
        __syncthreads();
        constexpr int kChunks = HD / 4;
        for (int i = tid; i < at.nrows * kChunks; i += 256) {
            const int row = i / kChunks, chunk = i % kChunks;
            float2 ml = make_float2(kEmptyMax, 0.0f);
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int c = 0; c < NC; ++c) ml.x = __builtin_fmaxf(ml.x, sml[w][W * c + row].x);
            f32x4_t o = {};
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float2 x = sml[w][W * c + row];
                    const float a = __builtin_amdgcn_exp2f(x.x - ml.x);
                    o += *reinterpret_cast<const f32x4_t*>(smem + w * kRegion + o_at<HD>(W * c + row, chunk)) * a;
                    ml.y = __builtin_fmaf(x.y, a, ml.y);
                }
            if (begins && ends) {
                write_row<HD, BF>(p, at.b, row, kvh, chunk, o, ml);
            } else {
                *reinterpret_cast<f32x4_t*>(p.part_o + (int64_t)(slot * ROWS + row) * HD + chunk * 4) = o;
                if (chunk == 0) p.part_ml[slot * ROWS + row] = ml;
            }
        }
        __syncthreads();
        line.advance(p, at);
    }
}

// ---- many rows ----------------------------------------------------------------------
//
// A block has 128 rows, each wave 32 of them (or 64 rows, two waves sharing a row
// and halving each tile's keys), on v_mfma_f32_32x32x16 (row_state.hpp).  All waves share
// tiles of 64 keys, which they turn into BF16 rows in LDS, each wave 16 keys, a tile
// ahead; the codes of the tile behind that are in flight meanwhile.
//
// P enters P V in two BF16 terms, as in the kernels of fewer rows: a token's result is as exact,
// whether it is decoded alone, verified among a few or part of a prompt.  One term, off by
// 2^-8, is as large an error as the result's own rounding (root mean square 0.0023 instead of 0.0017)
// and saves its products: 32 x 5 tokens over up to 4100 keys take 30 us with it, 33 with two,
// 4 x 512 over up to 8700 keys 178 and 227, over 17408 588 and 781.

// Rows of K are read 16 rows at a time, 16 bytes of each, rows of V transposed, four rows by
// 64 bytes: 16 bytes lie between rows of K, 64 between those of V and 16 more between
// groups of four, so that the 256 bytes of a read fall on different columns, and the 128 of a
// write: 16 of eight rows of K, or of two rows of V in each group of four.
template <int MODE, int HD, int ROWS, bool BF>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) paged_wide_kernel(PagedParams p) {
    constexpr int kC = HD / 16, kD = HD / 32, kW = HD / 32;      // kW: words of codes of a lane
    constexpr int NT = ROWS == 128 ? 2 : 1;                      // 32-key accumulators of a wave
    constexpr uint32_t kRowK = HD * 2 + 16, kRowV = HD * 2 + 64;
    constexpr uint32_t kTileK = kWideStep * kRowK, kTileV = kWideStep * kRowV + kWideStep / 4 * 16;
    constexpr uint32_t kSlot = kTileK + kTileV, kRegion = 32 * (HD * 4 + 16);
    constexpr uint32_t kLds = 2 * kSlot > 4 * kRegion ? 2 * kSlot : 4 * kRegion;
    __shared__ __align__(1024) unsigned char smem[kLds];
    __shared__ float2 sml[4][32];
    __shared__ uint8_t marks[2][kWideStep];  // blocks of V that are NaN, where some row does not see all keys
    __shared__ int marked[2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int h = lane >> 5, c32 = lane & 31, c16 = lane & 15, quarter = lane >> 4;
    Stretch<ROWS, kWideStep> line;
    if (!line.template find<true>(p)) return;

    ScoreConsts consts;
    consts.sl = vgpr(attn_is_plain_softmax(MODE) ? p.scale * kLog2e : kLog2e);
    consts.scale = p.scale;
    consts.cap = p.cap;
    consts.inv_cap = 1.0f / p.cap;
    if constexpr (MODE == kAttnSoftcapD4)
#pragma unroll
        for (int i = 1; i <= SoftcapConsts::T::P.deg; ++i) consts.tanh[i] = bf16_value(SoftcapConsts::T::P.c[i]);

    const int rbase = ROWS == 128 ? wave * 32 : (wave & 1) * 32;  // the wave's rows in the block
    const int koff = ROWS == 128 ? 0 : (wave >> 1) * 32;          // and keys in a tile
    while (line.x < line.x1) {
        const Place<ROWS, kWideStep> at(p, line.place);
        const int steps = at.steps(), step0 = line.first(), n = line.last(steps) - step0, kvh = line.kvh;
        if (n == 0) {
            line.advance(p, at);
            break;
        }

        // ---- staging: the wave's 16 keys of a tile.  Lane 4 i + g knows the page of group g
        // of step i, 16 steps at a time.
        int my_page = -1, my_row = 0;
        uint32_t ahead_holes = 0;  // of the tile whose codes are in flight
        Codes<HD> ck, cv;
        // the wave's keys, lanes 0..7 with values of keys whose rows' writes do not meet
        const int vkey = (c16 & 1) | (c16 & 8) >> 2 | (c16 & 6) << 1;
        const LaneCodes<HD> k_lane(p.c, c16, quarter), v_lane(p.c, vkey, quarter);
        const int key16 = wave * 16 + c16, val16 = wave * 16 + vkey;
        auto fetch = [&](int i) __attribute__((always_inline)) {
            if ((i & 15) == 0) {
                const int key = (step0 + i + (lane >> 2)) * kWideStep + (lane & 3) * 16;
                const int entry = key / p.c.page_size;
                my_page = i + (lane >> 2) < n && key < at.visible ? p.c.page_of(at.b, entry) : -1;
                my_row = key - entry * p.c.page_size;
            }
            ahead_holes = (uint32_t)(__ballot(my_page < 0) >> (4 * (i & 15))) & 15;
            const int l = 4 * (i & 15) + wave;
            const int page = __builtin_amdgcn_readlane(my_page, l), row = __builtin_amdgcn_readlane(my_row, l);
            ck.template load<false>(p.c, page, row, 0, kvh, k_lane);
            cv.template load<false>(p.c, page, row, 1, kvh, v_lane);
        };
        const int kfull = at.keys_of(p, at.r0 / p.group) - 1;  // every row sees the keys up to it
        // the tile in flight to slot i % 2
        auto stage = [&](int i) __attribute__((always_inline)) {
            unsigned char* slot = smem + (i & 1) * kSlot;
            const bool masked = (step0 + i + 1) * kWideStep - 1 > kfull || ahead_holes != 0;
            if (masked) {  // blocks of V that are NaN are zeros (0 * NaN is NaN), and marked
                const bool hole = ahead_holes >> wave & 1, bad = cv.byte(v_lane) > (uint32_t)kFp4Most && !hole;
                const uint64_t any = __ballot(bad);
                if (bad || hole) cv.clear();
                if (any != 0) {
                    if (quarter == 0) {
                        uint32_t m = 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q) m |= (uint32_t)(any >> (16 * q + c16) & 1) << (q * kD / 4);
                        marks[i & 1][val16] = (uint8_t)m;
                    }
                    if (lane == 0) marked[i & 1] = 1;
                } else if (quarter == 0) marks[i & 1][val16] = 0;
            }
            const float sk = fp4_scale(ck.byte(k_lane)), sv = fp4_scale(cv.byte(v_lane));
            unsigned char* k = slot + key16 * kRowK + quarter * kW * 16;
            unsigned char* v = slot + kTileK + val16 * kRowV + (val16 >> 2) * 16 + quarter * kW * 16;
#pragma unroll
            for (int c = 0; c < kW; ++c) *reinterpret_cast<bf16x8_t*>(k + c * 16) = fp4_to_bf16(ck.w[c], sk);
#pragma unroll
            for (int c = 0; c < kW; ++c) *reinterpret_cast<bf16x8_t*>(v + c * 16) = fp4_to_bf16(cv.w[c], sv);
        };
        const int tiles = p.c.pages > 0 ? n : 0;
        if (tiles > 0) fetch(0);

        // ---- Q^T fragments: columns 16 c + 8 h .. of row c32
        const int row = rbase + c32;
        const bool rin = row < at.nrows;
        const int t = (at.r0 + (rin ? row : 0)) / p.group;
        const int klast = (rin ? at.keys_of(p, t) : at.visible) - 1;  // the last key that the lane's row sees
        const uint16_t* src = p.q + at.b * p.qs.b + t * p.qs.s + (kvh * p.group + (at.r0 + (rin ? row : 0) - t * p.group)) * p.qs.h;
        bf16x8_t qf[kC], ql[BF ? 1 : kC];
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            bf16x8_t f = {};
            if (rin) f = *reinterpret_cast<const bf16x8_t*>(src + 16 * c + 8 * h);
            if constexpr (!BF) split_fp16(f, qf[c], ql[c]);
            else qf[c] = f;
        }
        RowState<HD> st;
        __syncthreads();  // the tiles and marks of the unit before are read
        if (tid < 2) marked[tid] = 0;
        __syncthreads();
        uint32_t holes = ahead_holes;
        if (tiles > 0) stage(0);
        if (tiles > 1) fetch(1);
        __syncthreads();
        if constexpr (BF)
#pragma unroll
            for (int c = 0; c < kC; ++c) loaded(qf[c]);
        for (int i = 0; i < tiles; ++i) {
            const unsigned char* ks = smem + (i & 1) * kSlot + (koff + c32) * kRowK + h * 16;
            // transposing reads: row 4 h + (l % 16) / 4, columns 16 ((l / 16) % 2) + 4 (l % 4)
            const int tr = koff + 4 * h + (c16 >> 2);
            const unsigned char* vs = smem + (i & 1) * kSlot + kTileK + tr * kRowV + (tr >> 2) * 16 + (quarter & 1) * 32 + (lane & 3) * 8;
            const int key0 = (step0 + i) * kWideStep;
            const bool masked = key0 + kWideStep - 1 > kfull || holes != 0;
            constexpr int kTerms = BF ? 1 : 2;  // products a fragment of K
            f32x16_t s[NT];
            // fragments of K are read six ahead of their products
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kt = 0; kt < NT; ++kt) s[kt] = (f32x16_t){};
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int kt = 0; kt < NT; ++kt) {
                    const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(ks + kt * 32 * kRowK + c * 32);
                    s[kt] = mfma32(kf, qf[c], s[kt]);
                    if constexpr (!BF) s[kt] = mfma32(kf, ql[c], s[kt]);
                }
            constexpr int kReads = NT * kC, kAhead = kReads < 6 ? kReads : 6;
            __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
            for (int g = 0; g < kReads - kAhead; ++g) {
                __builtin_amdgcn_sched_group_barrier(0x008, kTerms, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, kAhead * kTerms, 0);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            if constexpr (!attn_is_plain_softmax(MODE)) {
#pragma unroll
                for (int kt = 0; kt < NT; ++kt) {
                    float x[16];
                    softmax_exponents<MODE>(s[kt], consts, x);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kt][r] = x[r];
                }
            }
            if (masked) {  // keys of accumulator kt: 32 kt + 8 (r / 4) + 4 h + r % 4
                const int diag = key0 + koff + 4 * h - klast;
#pragma unroll
                for (int kt = 0; kt < NT; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (diag + kt * 32 + 8 * (r >> 2) + (r & 3) > 0 || (holes >> (koff / 16 + 2 * kt + (r >> 3)) & 1))
                            s[kt][r] = -__builtin_inff();
            }
            const float mul = score_state<kAttnSoftmaxNative, HD, true, NT, false>(s, st, consts, 0);
            score_exps<HD, NT>(s, st, mul);
            // the compiler's order of reads and products: fragments of V three ahead take 788 us where it takes
            // 781 (4 x 512 tokens over 17408 keys)
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int g = 0; g < 2 * NT; ++g) {
                const bf16x8_t pf = prob_frag<true>(s[g >> 1], g & 1);
                const bf16x8_t rest = prob_rest<true>(s[g >> 1], g & 1, pf);
#pragma unroll
                for (int dt = 0; dt < kD; ++dt) {
                    const uint16_t* vp = reinterpret_cast<const uint16_t*>(vs + g * (16 * kRowV + 64) + dt * 64);
                    const u32x2_t lo = __builtin_bit_cast(u32x2_t, lds_read_tr16(vp));
                    const u32x2_t hi = __builtin_bit_cast(u32x2_t, lds_read_tr16(vp + (8 * kRowV + 32) / 2));
                    const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, (u32x4_t){lo.x, lo.y, hi.x, hi.y});
                    st.o[dt] = mfma32(vf, pf, st.o[dt]);
                    st.o[dt] = mfma32(vf, rest, st.o[dt]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            if (masked && marked[i & 1] != 0)
                for (int key = koff; key < koff + 32 * NT; ++key) {
                    const uint32_t m = marks[i & 1][key];
#pragma unroll
                    for (int dt = 0; dt < kD; ++dt)
                        if ((m >> dt & 1) && key0 + key <= klast)
#pragma unroll
                            for (int r = 0; r < 16; ++r) st.o[dt][r] = __builtin_nanf("");
                }
            if (i + 1 < tiles) {
                holes = ahead_holes;
                stage(i + 1);
                if (i + 2 < tiles) fetch(i + 2);
            }
            __syncthreads();
        }

        // ---- the rows: whole ones through LDS
        unsigned char* region = smem + wave * kRegion;
#pragma unroll
        for (int dt = 0; dt < kD; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4_t*>(region + o_at<HD>(c32, dt * 8 + 2 * g + h)) =
                    (f32x4_t){st.o[dt][4 * g], st.o[dt][4 * g + 1], st.o[dt][4 * g + 2], st.o[dt][4 * g + 3]};
        const float l = half_sum(st.l);
        if (h == 0) sml[wave][c32] = make_float2(st.m, l);
        __syncthreads();
        const bool begins = step0 == 0, ends = step0 + n == steps;
        const int slot = 2 * line.block + (begins ? 1 : 0);
        constexpr int kChunks = HD / 4;
        for (int i = tid; i < at.nrows * kChunks; i += 256) {
            const int orow = i / kChunks, chunk = i % kChunks, w = orow >> 5, r = orow & 31;
            float2 ml = sml[w][r];
            f32x4_t o = *reinterpret_cast<const f32x4_t*>(smem + w * kRegion + o_at<HD>(r, chunk));
            if constexpr (ROWS == 64) {
                const float2 y = sml[w + 2][r];
                const float top = __builtin_fmaxf(ml.x, y.x);
                const float a = __builtin_amdgcn_exp2f(ml.x - top), a2 = __builtin_amdgcn_exp2f(y.x - top);
                o = o * a + *reinterpret_cast<const f32x4_t*>(smem + (w + 2) * kRegion + o_at<HD>(r, chunk)) * a2;
                ml = make_float2(top, __builtin_fmaf(ml.y, a, y.y * a2));
            }
            if (begins && ends) {
                write_row<HD, BF>(p, at.b, at.r0 + orow, kvh, chunk, o, ml);
            } else {
                *reinterpret_cast<f32x4_t*>(p.part_o + (int64_t)(slot * ROWS + orow) * HD + chunk * 4) = o;
                if (chunk == 0) p.part_ml[slot * ROWS + orow] = ml;
            }
        }
        line.advance(p, at);
    }
}

// Joins the pieces of the unit of a block's cut.  HD / 4 lanes
// hold a row, and the groups of them beyond the rows take the pieces in turn.
template <int HD, int ROWS, bool BF>
__global__ void __launch_bounds__(512) paged_join_kernel(PagedParams p) {
    constexpr int kChunks = HD / 4, kSlots = 512 / kChunks;  // row slots
    const int4 cut = p.cut[blockIdx.x];
    const int pieces = cut.z, block = cut.y >> 16, kvh = cut.y & 0xffff;
    if (pieces == 0) return;
    const int nrows = p.rows - cut.w < ROWS ? p.rows - cut.w : ROWS;
    int span = 1;  // a power of two that holds the block's share of the rows
    while (span * (int)gridDim.y < nrows && span < kSlots) span *= 2;
    const int shares = kSlots / span;
    const int chunk = threadIdx.x % kChunks, s = threadIdx.x / kChunks, share = s / span;
    __shared__ f32x4_t so[512];
    __shared__ float2 sml[kSlots];
    const int first = s % span + (int)blockIdx.y * span;
    for (int row = first; row < nrows; row += kSlots * (int)gridDim.y) {  // more than once where all slots have a row
        float m = kEmptyMax, l = 0.0f;
        f32x4_t o = (f32x4_t){};
        auto add = [&](float m2, float l2, f32x4_t o2) {
            const float top = __builtin_fmaxf(m, m2);
            const float a = __builtin_amdgcn_exp2f(m - top), a2 = __builtin_amdgcn_exp2f(m2 - top);
            l = __builtin_fmaf(l, a, l2 * a2);
            o = o * a + o2 * a2;
            m = top;
        };
        for (int i = share; i < pieces; i += 4 * shares) {
            float2 ml[4];
            f32x4_t part[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = i + u * shares < pieces ? i + u * shares : i;
                const int slot = 2 * (block + j) + (j == 0 ? 1 : 0);
                ml[u] = p.part_ml[slot * ROWS + row];
                part[u] = *reinterpret_cast<const f32x4_t*>(p.part_o + (int64_t)(slot * ROWS + row) * HD + chunk * 4);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * shares < pieces) add(ml[u].x, ml[u].y, part[u]);
        }
        if (shares > 1) {
            so[threadIdx.x] = o;
            if (chunk == 0) sml[s] = make_float2(m, l);
        }
        if (shares == 1) write_row<HD, BF>(p, cut.x, cut.w + row, kvh, chunk, o, make_float2(m, l));
    }
    if (shares == 1) return;
    __syncthreads();
    if (share != 0 || first >= nrows) return;
    const int row = first;
    float top = kEmptyMax, l = 0.0f;
    for (int u = 0; u < shares; ++u) top = __builtin_fmaxf(top, sml[s + u * span].x);
    f32x4_t o = (f32x4_t){};
    for (int u = 0; u < shares; ++u) {
        const float2 ml = sml[s + u * span];
        const float a = __builtin_amdgcn_exp2f(ml.x - top);
        o += so[threadIdx.x + u * span * kChunks] * a;
        l = __builtin_fmaf(ml.y, a, l);
    }
    write_row<HD, BF>(p, cut.x, cut.w + row, kvh, chunk, o, make_float2(top, l));
}

// ---- host side -----------------------------------------------------------------

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct PagedPlan {
    int rows;        // of a tile
    int classes;     // of columns, for one token
    int64_t blocks;  // a fixed number: the device divides the keys among them
    int64_t bytes;   // of the workspace
};

// Where columns of several groups pay: 32 sequences of 8192 keys, heads of 64, 16 ungrouped
// ones 64 us against 75, with a softcap 63 against 89, 32 / 8 heads 39 and 40, with a softcap 40
// and 48.  Heads of 128, 32 / 8: 57 against 54, with a softcap 58 against 63; FP16 queries, whose second
// terms take the registers of a third block, 74 against 58 and 77 against 66.
constexpr bool has_classes(int mode, int head_dim, bool bf) {
    return head_dim == 64 || (bf && mode != kAttnSoftmaxNative);
}

bool plan(const spline_hip_fp4_cache* c, const spline_hip_fp4_attention* a, bool bf, PagedPlan& p) {
    if (!a || !fp4_sizes_ok(c, a->tokens) || a->q_heads <= 0 || a->q_heads > 65536 || a->q_heads % c->kv_heads != 0)
        return false;
    const int64_t rows = a->tokens * (a->q_heads / c->kv_heads);
    if (rows > 1 << 30) return false;  // of a sequence, in 32 bits
    p.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.classes = 1;
    if (a->tokens == 1 && rows <= 8 && has_classes(a->mode, (int)c->head_dim, bf)) p.classes = rows > 4 ? 2 : 4;
    p.blocks = ceil_div(device_shape().cus * (rows > 16 ? 2 : 3), 8) * 8;  // whole rows of XCDs
    const int64_t tiles = ceil_div(rows, p.rows);
    // places, and the steps of the line, are counted in 32 bits
    if (c->batch > 0x7fffffff / (tiles ? tiles : 1)) return false;
    const int step = p.classes > 1 ? kDecodeStep : p.rows <= 32 ? kNarrowStep : kWideStep;
    const int64_t steps = ceil_div(c->entries * c->page_size, step) + 1 + unit_steps(step);
    if (c->batch * tiles > 0x7fffffff / (steps * c->kv_heads)) return false;
    p.bytes = p.blocks * (16 + 2 * p.rows * (c->head_dim + 2) * 4);
    return true;
}

// Blocks that join a unit: with two for up to 32 rows two sequences of up to 131072 keys, 48 pieces
// a unit, take 37.2 us instead of 39.3 (four 37.1), calls with fewer pieces the same to 1 %.
template <int ROWS>
dim3 join_grid(const PagedParams& p, int64_t blocks) {
    return dim3((unsigned)blocks, ROWS > 32 ? 4 : p.rows > 1 ? 2 : 1);
}
template <int MODE, int HD, int ROWS, bool BF>
void go(const PagedParams& p, int64_t blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks);
    if constexpr (ROWS <= 32) hipLaunchKernelGGL((paged_narrow_kernel<MODE, HD, ROWS / 16, BF>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_wide_kernel<MODE, HD, ROWS, BF>), grid, dim3(256), 0, st, p);
    hipLaunchKernelGGL((paged_join_kernel<HD, ROWS, BF>), join_grid<ROWS>(p, blocks), dim3(512), 0, st, p);
}
template <int MODE, int HD, int NC, bool BF>
void decode(const PagedParams& p, int64_t blocks, hipStream_t st) {
    const dim3 grid((unsigned)blocks);
    hipLaunchKernelGGL((paged_decode_kernel<MODE, HD, NC, BF>), grid, dim3(256), 0, st, p);
    hipLaunchKernelGGL((paged_join_kernel<HD, 16, BF>), join_grid<16>(p, blocks), dim3(512), 0, st, p);
}
template <int MODE, int HD, bool BF>
void go(const PagedParams& p, const PagedPlan& plan, hipStream_t st) {
    if constexpr (has_classes(MODE, HD, BF)) {
        if (plan.classes == 4) return decode<MODE, HD, 4, BF>(p, plan.blocks, st);
        if (plan.classes == 2) return decode<MODE, HD, 2, BF>(p, plan.blocks, st);
    }
    if (plan.rows == 16) go<MODE, HD, 16, BF>(p, plan.blocks, st);
    else if (plan.rows == 32) go<MODE, HD, 32, BF>(p, plan.blocks, st);
    else if (plan.rows == 64) go<MODE, HD, 64, BF>(p, plan.blocks, st);
    else go<MODE, HD, 128, BF>(p, plan.blocks, st);
}

template <bool BF>
int run(const spline_hip_fp4_cache* c, const spline_hip_fp4_attention* a, void* stream) {
    PagedPlan plan_{};
    if (!plan(c, a, BF, plan_) || !(a->scale > 0.0f && a->scale <= __FLT_MAX__)) return hipErrorInvalidValue;
    if (a->mode != kAttnSoftmaxNative && a->mode != kAttnSoftcapNative && !(BF && a->mode == kAttnSoftcapD4))
        return hipErrorInvalidValue;
    if (a->mode != kAttnSoftmaxNative && !(a->cap > 0.0f && a->cap <= __FLT_MAX__)) return hipErrorInvalidValue;
    if (c->batch == 0 || a->tokens == 0) return hipSuccess;
    bool ok = fp4_pointers_ok(c) && a->q && aligned16(a->q) && a->out && aligned16(a->out) &&
              ((uintptr_t)a->lse & 3) == 0 && a->workspace && aligned16(a->workspace);
    for (int i = 0; i < 3; ++i) ok = ok && a->q_strides[i] >= 0 && a->q_strides[i] % 8 == 0;
    if (!ok) return hipErrorInvalidValue;
    PagedParams p{};
    p.q = static_cast<const uint16_t*>(a->q);
    p.c = fp4_pages(c);
    p.qs = {a->q_strides[0], a->q_strides[2], a->q_strides[1]};
    const int64_t rows = plan_.blocks * 2 * plan_.rows;
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * c->head_dim);
    p.cut = reinterpret_cast<int4*>(p.part_ml + rows);
    p.out = a->out;
    p.lse = a->lse;
    p.hq = (int)a->q_heads;
    p.group = (int)(a->q_heads / c->kv_heads);
    p.tokens = (int)a->tokens;
    p.rows = p.tokens * p.group;
    p.tiles = (int)ceil_div(p.rows, plan_.rows);
    p.capacity = p.c.entries * p.c.page_size;
    p.places = (int)c->batch * p.tiles;
    p.scale = a->scale;
    p.cap = a->cap;
    const hipStream_t st = hs(stream);
    auto shape = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        if (c->head_dim == 128) go<MODE, 128, BF>(p, plan_, st);
        else go<MODE, 64, BF>(p, plan_, st);
    };
    if (a->mode == kAttnSoftmaxNative) shape(std::integral_constant<int, kAttnSoftmaxNative>{});
    else if (a->mode == kAttnSoftcapNative) shape(std::integral_constant<int, kAttnSoftcapNative>{});
    else if constexpr (BF) shape(std::integral_constant<int, kAttnSoftcapD4>{});
    return hipGetLastError();
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" int64_t spline_hip_paged_fp4_workspace_bytes(const spline_hip_fp4_cache* cache,
                                                        const spline_hip_fp4_attention* args) {
    PagedPlan p{};
    PagedPlan q{};  // the types' plans differ; the larger one
    if (!plan(cache, args, true, p) || !plan(cache, args, false, q)) return -1;
    return cache->batch == 0 || args->tokens == 0 ? 0 : p.bytes > q.bytes ? p.bytes : q.bytes;
}
extern "C" int launch_paged_fp4_attention_fp16(const spline_hip_fp4_cache* cache, const spline_hip_fp4_attention* args,
                                               void* stream) {
    return run<false>(cache, args, stream);
}
extern "C" int launch_paged_fp4_attention_bf16(const spline_hip_fp4_cache* cache, const spline_hip_fp4_attention* args,
                                               void* stream) {
    return run<true>(cache, args, stream);
}
