// qk_rope.hip -- what a query or key head passes between its projection and
// the attention, in one pass over memory for gfx950: the RMS norm of the head
// with its weight, then the rotary rotation by positions that the caller gives,
// on one axis or on several (time, height, width); and the gradients of both.
//
//   n = x r,  r = 1 / sqrt(mean(x^2) + eps),  u = n w
//   (y_a, y_b) = (u_a cos t - u_b sin t, u_a sin t + u_b cos t)
//   backward:  g = R(-t) dy,  dw = sum g n,  dx = r (w g - n mean(w g n))
//
// x [B, S, H, D] -> y [B, H, S, D], 16-bit, any strides over a contiguous head
// dimension; a frequency's pair is (2i, 2i + 1) or (i, i + R/2) of the R rotated
// elements, and elements from R on are only normalised.  The phase of position
// p is p * increment in Q0.32 turns, exact modulo a turn for every position.
//
// A row is spread over L lanes (a power of two) that own two vectors of V
// elements each, so both elements of every pair lie in one lane and the mean
// takes log2 L lane exchanges.  A thread evaluates its V sines and cosines once
// for a token and applies them to the heads of a group, whose loads it issues
// ahead of all arithmetic.  Lanes of neighbouring rows are neighbouring tokens.
//
// The gradient of w sums over every row: a block keeps its sums in registers
// over all its tokens, adds its rows through LDS and stores one partial row;
// a second launch adds the partial rows.  Every order of addition is fixed.
//
// What bounds it: memory, 4 bytes an element forward and 6 backward.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "ops.hpp"
#include "spline_ops_hip.h"

namespace pt {

// sin and cos of a Q0.32 phase, FP32: the nearest quarter turn is taken off in
// integers, t = the rest in units of 1/8 turn, |t| <= 1, and sin(pi/4 t) = t S(t^2),
// cos(pi/4 t) = C(t^2) with the interpolants at Chebyshev nodes (in t^2) of
// S and of (C - 1) / t^2.  Largest error 8.5e-8 and 6.1e-8, over 2^21 phases.
__device__ __forceinline__ void phase_sincos(uint32_t phase, float& c, float& s) {
    const uint32_t q = (phase + 0x20000000u) >> 30;
    const float t = (float)(int32_t)(phase - (q << 30)) * 0x1p-29f;
    const float t2 = t * t;
    float sp = __builtin_fmaf(-3.595429e-05f, t2, 0.0024900069f);
    sp = __builtin_fmaf(sp, t2, -0.080745436f);
    sp = __builtin_fmaf(sp, t2, 0.7853982f);
    sp *= t;
    float cp = __builtin_fmaf(3.5419528e-06f, t2, -0.0003259614f);
    cp = __builtin_fmaf(cp, t2, 0.015854338f);
    cp = __builtin_fmaf(cp, t2, -0.30842513f);
    cp = __builtin_fmaf(cp, t2, 1.0f);
    const bool swap = q & 1u;
    s = as_f32(as_u32(swap ? cp : sp) ^ ((q & 2u) << 30));
    c = as_f32(as_u32(swap ? sp : cp) ^ (((q + 1u) & 2u) << 30));
}

// x combined with the lane `STEP` of a group away, in every lane of the group.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + as_f32((uint32_t)__builtin_amdgcn_mov_dpp((int)as_u32(x), CTRL, 0xf, 0xf, true));
}
// The sum over an aligned group of 2^log lanes; all 64 lanes take part.
__device__ __forceinline__ float group_sum(float x, int log) {
    if (log > 0) x = dpp_add<0xB1>(x);   // quad_perm 1 0 3 2
    if (log > 1) x = dpp_add<0x4E>(x);   // quad_perm 2 3 0 1
    if (log > 2) x = dpp_add<0x141>(x);  // row_half_mirror
    if (log > 3) x = dpp_add<0x140>(x);  // row_mirror
    if (log > 4) {
        const auto r = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
        x = as_f32(r[0]) + as_f32(r[1]);
    }
    if (log > 5) {
        const auto r = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
        x = as_f32(r[0]) + as_f32(r[1]);
    }
    return x;
}

template <bool BF>
__device__ __forceinline__ void widen(uint32_t w, float& lo, float& hi) {
    if constexpr (BF) {
        lo = bf_lo(w);
        hi = bf_hi(w);
    } else {
        const h2_t h = as_h2(w);
        lo = (float)h.x;
        hi = (float)h.y;
    }
}
template <bool BF>
__device__ __forceinline__ uint32_t narrow(float lo, float hi) {
    if constexpr (BF) return pack_bf(lo, hi);
    else return as_u32((h2_t){(_Float16)lo, (_Float16)hi});
}

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// V elements, V / 2 words.
template <int V>
struct Words {
    uint32_t w[V / 2];
};
template <int V>
__device__ __forceinline__ Words<V> load_words(const uint16_t* p) {
    Words<V> o;
    if constexpr (V == 8) {
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(p);
        o.w[0] = v.x; o.w[1] = v.y; o.w[2] = v.z; o.w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        o.w[0] = v.x; o.w[1] = v.y;
    }
    return o;
}
template <int V, bool NT>
__device__ __forceinline__ void store_words(uint16_t* p, const Words<V>& o) {
    if constexpr (V == 8) {
        const u32x4_t v = {o.w[0], o.w[1], o.w[2], o.w[3]};
        if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(p));
        else *reinterpret_cast<u32x4_t*>(p) = v;
    } else {
        const u32x2_t v = {o.w[0], o.w[1]};
        if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x2_t*>(p));
        else *reinterpret_cast<u32x2_t*>(p) = v;
    }
}

struct Strides {
    int64_t b, s, h;
};

// The queries or the keys.
struct QkSide {
    const uint16_t* x;
    uint16_t* y;
    const uint16_t* dy;  // backward: the gradient at the output; y then receives the input's
    const void* w;       // [D], or null
    float* dw;           // backward: [blocks, D] partial sums, or null
    Strides xs, ys, dys;
    int heads, splits;   // parts that the heads are cut into
    int blocks;          // backward: blocks of this side
};

struct QkParams {
    QkSide q, k;
    const uint32_t* inc;
    const uint32_t* pos;    // low words of the positions, or null: 0 .. S - 1
    Strides poss;           // axis (in h), batch and sequence, in words
    const int32_t* axes;    // axis of each frequency, or null: one axis
    int axis_count;
    uint32_t tokens, seq;
    int head_dim, rotary;
    int lanes, log_lanes;   // lanes that own vectors, and log2 of the lanes of a row
    float eps, inv_d;
    bool w32, neg, nt;      // FP32 weights; the inverse rotation; non-temporal stores
};

// Where a lane's two vectors lie in a row and what they turn by.
template <int V, bool INTER>
struct LanePart {
    int e[2];
    bool rot[2];

    __device__ __forceinline__ LanePart(const QkParams& p, int l) {
        if constexpr (INTER) {
            e[0] = V * l;
            e[1] = (p.head_dim >> 1) + V * l;
            rot[0] = e[0] < p.rotary;
            rot[1] = e[1] < p.rotary;
        } else {
            const int half = p.rotary / (2 * V);
            rot[0] = rot[1] = l < half;
            e[0] = l < half ? V * l : p.rotary + 2 * V * (l - half);
            e[1] = l < half ? (p.rotary >> 1) + V * l : e[0] + V;
        }
    }
    // Pair j < V of the lane: elements first(j), second(j) of its 2 V.
    __device__ __forceinline__ static constexpr int first(int j) { return INTER ? 2 * j : j; }
    __device__ __forceinline__ static constexpr int second(int j) { return INTER ? 2 * j + 1 : V + j; }

    __device__ __forceinline__ void angles(const QkParams& p, uint32_t b, uint32_t s, float (&cs)[V],
                                           float (&sn)[V]) const {
        const uint32_t* pos = p.pos == nullptr ? nullptr : p.pos + b * p.poss.b + s * p.poss.s;
        const uint32_t one = pos == nullptr ? s : p.axes == nullptr ? *pos : 0u;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            cs[j] = 1.0f;
            sn[j] = 0.0f;
            if (rot[INTER && j >= V / 2]) {
                const int f = INTER ? (j < V / 2 ? (e[0] >> 1) + j : (e[1] >> 1) + j - V / 2) : e[0] + j;
                uint32_t at = one;
                if (p.axes != nullptr) {
                    const int a = p.axes[f];  // held to the axes that there are
                    at = pos[(a < 0 ? 0 : a < p.axis_count ? a : p.axis_count - 1) * p.poss.h];
                }
                const uint32_t phase = at * p.inc[f];
                phase_sincos(p.neg ? 0u - phase : phase, cs[j], sn[j]);
            }
        }
    }

    template <bool BF>
    __device__ __forceinline__ void weights(const QkParams& p, const void* w, float (&out)[2 * V]) const {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (w == nullptr) {
#pragma unroll
                for (int i = 0; i < V; ++i) out[c * V + i] = 1.0f;
            } else if (p.w32) {
#pragma unroll
                for (int i = 0; i < V; ++i) out[c * V + i] = static_cast<const float*>(w)[e[c] + i];
            } else {
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const uint16_t* t = static_cast<const uint16_t*>(w) + e[c] + i;
                    widen<BF>((uint32_t)t[0] | (uint32_t)t[1] << 16, out[c * V + i], out[c * V + i + 1]);
                }
            }
        }
    }
};

template <bool BF, int V>
__device__ __forceinline__ void widen_row(const Words<V> (&raw)[2], float (&f)[2 * V]) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        widen<BF>(raw[0].w[i / 2], f[i], f[i + 1]);
        widen<BF>(raw[1].w[i / 2], f[V + i], f[V + i + 1]);
    }
}
template <bool BF, int V, bool NT>
__device__ __forceinline__ void store_row(uint16_t* row, const int (&e)[2], const float (&f)[2 * V]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        Words<V> o;
#pragma unroll
        for (int i = 0; i < V; i += 2) o.w[i / 2] = narrow<BF>(f[c * V + i], f[c * V + i + 1]);
        store_words<V, NT>(row + e[c], o);
    }
}

template <int V>
__device__ __forceinline__ float sum_squares(const float (&f)[2 * V]) {
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) t[i & 3] = __builtin_fmaf(f[i], f[i], t[i & 3]);
    return (t[0] + t[1]) + (t[2] + t[3]);
}

// The heads of the queries and of the keys are cut into splits, and a block takes
// one split of a chunk of tokens (blockIdx.x runs over the splits first), so the
// blocks that run together share whole rows of memory, and a thread evaluates its
// angles once for all heads of its split.  Loads of the next HPT heads are in
// flight behind the arithmetic of these.  With the norm, w is folded into the
// rotation, y_a = r (x_a (w_a cos) - x_b (w_b sin)), which leaves r for the end.
template <bool BF, int V, bool INTER, bool NORM, bool NT, int HPT>
__global__ void __launch_bounds__(kBlock, 4) qk_rope_kernel(QkParams p) {
    using Part = LanePart<V, INTER>;
    const int l = threadIdx.x & ((1 << p.log_lanes) - 1);
    const bool own = l < p.lanes;
    const Part part(p, l);
    const uint32_t splits = p.q.splits + p.k.splits;
    const uint32_t chunk0 = blockIdx.x / splits;
    int split = (int)(blockIdx.x - chunk0 * splits);
    const bool is_k = split >= p.q.splits;
    split -= is_k ? p.q.splits : 0;
    const int heads = is_k ? p.k.heads : p.q.heads, parts = is_k ? p.k.splits : p.q.splits;
    const int h_begin = heads * split / parts, h_end = heads * (split + 1) / parts;
    const Strides xs = is_k ? p.k.xs : p.q.xs, ys = is_k ? p.k.ys : p.q.ys;
    const int64_t rows = kBlock >> p.log_lanes, stride = gridDim.x / splits * rows;
    for (int64_t t0 = chunk0 * rows; t0 < p.tokens; t0 += stride) {
        const int64_t token = t0 + (threadIdx.x >> p.log_lanes);
        const bool in = own && token < p.tokens;
        const uint32_t b = (uint32_t)token / p.seq, s = (uint32_t)token - b * p.seq;
        const uint16_t* x = (is_k ? p.k.x : p.q.x) + b * xs.b + s * xs.s;
        uint16_t* y = (is_k ? p.k.y : p.q.y) + b * ys.b + s * ys.s;
        auto load = [&](int h, Words<V> (&raw)[HPT][2]) {
#pragma unroll
            for (int u = 0; u < HPT; ++u)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    raw[u][c] = Words<V>{};
                    if (in && h + u < h_end) raw[u][c] = load_words<V>(x + (h + u) * xs.h + part.e[c]);
                }
        };
        Words<V> raw[2][HPT][2];
        load(h_begin, raw[0]);
        // y_a = ca x_a - sb x_b, y_b = sa x_a + cb x_b
        float ca[V] = {}, sa[V] = {}, cb[V], sb[V];
        if (in) part.angles(p, b, s, ca, sa);
        if constexpr (NORM) {
            float w[2 * V] = {};
            if (own) part.template weights<BF>(p, is_k ? p.k.w : p.q.w, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                cb[j] = ca[j] * w[Part::second(j)];
                sb[j] = sa[j] * w[Part::second(j)];
                ca[j] *= w[Part::first(j)];
                sa[j] *= w[Part::first(j)];
            }
        }
        auto turn = [&](int h, const Words<V> (&now)[HPT][2]) {
#pragma unroll
            for (int u = 0; u < HPT; ++u) {
                if (h + u >= h_end) break;  // the same for every thread of the block
                float f[2 * V];
                widen_row<BF, V>(now[u], f);
                float r = 1.0f;
                if constexpr (NORM)
                    r = __builtin_amdgcn_rsqf(
                        __builtin_fmaf(group_sum(sum_squares<V>(f), p.log_lanes), p.inv_d, p.eps));
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float a = f[Part::first(j)], d = f[Part::second(j)];
                    const float ya = __builtin_fmaf(a, ca[j], -(d * (NORM ? sb[j] : sa[j])));
                    const float yb = __builtin_fmaf(a, sa[j], d * (NORM ? cb[j] : ca[j]));
                    f[Part::first(j)] = NORM ? ya * r : ya;
                    f[Part::second(j)] = NORM ? yb * r : yb;
                }
                if (in) store_row<BF, V, NT>(y + (h + u) * ys.h, part.e, f);
            }
        };
        for (int h = h_begin; h < h_end; h += 2 * HPT) {
            if (h + HPT < h_end) load(h + HPT, raw[1]);
            turn(h, raw[0]);
            if (h + HPT >= h_end) break;
            if (h + 2 * HPT < h_end) load(h + 2 * HPT, raw[0]);
            turn(h + HPT, raw[1]);
        }
    }
}

// Grid q.blocks + k.blocks; a block takes items (a split of the side's heads of a
// chunk of tokens) blocks apart, and a thread evaluates its angles once an item.
// Three waves a SIMD (168 registers), two where FP16's conversions need more.
template <bool BF, int V, bool INTER, bool NT, int HPT>
__global__ void __launch_bounds__(kBlock, !BF && V == 8 ? 2 : 3) qk_rope_bwd_kernel(QkParams p) {
    using Part = LanePart<V, INTER>;
    const bool is_k = (int)blockIdx.x >= p.q.blocks;
    const uint16_t* x = is_k ? p.k.x : p.q.x;
    const uint16_t* dy = is_k ? p.k.dy : p.q.dy;
    uint16_t* dx = is_k ? p.k.y : p.q.y;
    float* dw = is_k ? p.k.dw : p.q.dw;
    const Strides xs = is_k ? p.k.xs : p.q.xs, ys = is_k ? p.k.ys : p.q.ys, dys = is_k ? p.k.dys : p.q.dys;
    const int heads = is_k ? p.k.heads : p.q.heads;
    const uint32_t blocks = is_k ? p.k.blocks : p.q.blocks, splits = is_k ? p.k.splits : p.q.splits;
    const uint32_t block = (uint32_t)((int)blockIdx.x - (is_k ? p.q.blocks : 0));
    const int l = threadIdx.x & ((1 << p.log_lanes) - 1), row = threadIdx.x >> p.log_lanes;
    const int rows = kBlock >> p.log_lanes;
    const bool own = l < p.lanes;
    const Part part(p, l);
    float w[2 * V] = {}, acc[2 * V] = {};
    if (own) part.template weights<BF>(p, is_k ? p.k.w : p.q.w, w);

    // item = chunk * splits + split, stepped without a division
    const int64_t chunks = ((int64_t)p.tokens + rows - 1) / rows;
    const uint32_t chunk_step = blocks / splits, split_step = blocks - chunk_step * splits;
    int64_t chunk = block / splits;
    uint32_t split = block - (uint32_t)chunk * splits;
    while (chunk < chunks) {
        const int64_t token = chunk * rows + row;
        const bool in = own && token < p.tokens;
        const uint32_t b = (uint32_t)token / p.seq, s = (uint32_t)token - b * p.seq;
        const int h_begin = heads * (int)split / (int)splits, h1 = heads * ((int)split + 1) / (int)splits;
        const uint16_t* xtoken = x + b * xs.b + s * xs.s;
        const uint16_t* dytoken = dy + b * dys.b + s * dys.s;
        uint16_t* dxtoken = dx + b * ys.b + s * ys.s;
        float cs[V] = {}, sn[V] = {};
        for (int h0 = h_begin; h0 < h1; h0 += HPT) {
            Words<V> rx[HPT][2], rdy[HPT][2];
#pragma unroll
            for (int u = 0; u < HPT; ++u)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    rx[u][c] = rdy[u][c] = Words<V>{};
                    if (in && h0 + u < h1) {
                        rx[u][c] = load_words<V>(xtoken + (h0 + u) * xs.h + part.e[c]);
                        rdy[u][c] = load_words<V>(dytoken + (h0 + u) * dys.h + part.e[c]);
                    }
                }
            if (in && h0 == h_begin) part.angles(p, b, s, cs, sn);
#pragma unroll
            for (int u = 0; u < HPT; ++u) {
                if (h0 + u >= h1) break;  // the same for every thread of the block
                float n[2 * V], g[2 * V];
                widen_row<BF, V>(rx[u], n);
                widen_row<BF, V>(rdy[u], g);
                const float r = __builtin_amdgcn_rsqf(
                    __builtin_fmaf(group_sum(sum_squares<V>(n), p.log_lanes), p.inv_d, p.eps));
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float a = g[Part::first(j)], d = g[Part::second(j)];
                    g[Part::first(j)] = __builtin_fmaf(a, cs[j], d * sn[j]);
                    g[Part::second(j)] = __builtin_fmaf(d, cs[j], -(a * sn[j]));
                }
                float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    n[i] *= r;
                    if (in) acc[i] = __builtin_fmaf(g[i], n[i], acc[i]);
                    g[i] *= w[i];
                    t[i & 3] = __builtin_fmaf(g[i], n[i], t[i & 3]);
                }
                const float mean = group_sum((t[0] + t[1]) + (t[2] + t[3]), p.log_lanes) * p.inv_d;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) g[i] = r * __builtin_fmaf(n[i], -mean, g[i]);
                if (in) store_row<BF, V, NT>(dxtoken + (h0 + u) * ys.h, part.e, g);
            }
        }
        chunk += chunk_step;
        split += split_step;
        if (split >= splits) {
            split -= splits;
            ++chunk;
        }
    }
    if (dw == nullptr) return;  // the same for every thread of the block

    // acc of every row to LDS, then one thread a column adds the rows
    __shared__ float sums[kBlock * 2 * V];
    if (own) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) sums[row * p.head_dim + part.e[c] + i] = acc[c * V + i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.head_dim; e += kBlock) {
        float t = 0.0f;
        for (int i = 0; i < rows; ++i) t += sums[i * p.head_dim + e];
        dw[(int64_t)block * p.head_dim + e] = t;
    }
}

struct DwSide {
    const float* part;
    void* out;
    int rows;
};

// Adds the partial rows: 16 columns a block, 64 rows at a time.
template <bool BF>
__global__ void __launch_bounds__(1024) qk_dw_kernel(DwSide q, DwSide k, int head_dim, bool w32) {
    const DwSide s = blockIdx.y ? k : q;
    if (s.part == nullptr) return;
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
    float t = 0.0f;
    if (e < head_dim) {
#pragma unroll 8
        for (int r = r0; r < s.rows; r += 64) t += s.part[(int64_t)r * head_dim + e];
    }
    __shared__ float sums[64][17];
    sums[r0][c] = t;
    __syncthreads();
    if (r0 != 0 || e >= head_dim) return;
    float total = 0.0f;
#pragma unroll 16
    for (int r = 0; r < 64; ++r) total += sums[r][c];
    if (w32) static_cast<float*>(s.out)[e] = total;
    else static_cast<uint16_t*>(s.out)[e] = (uint16_t)narrow<BF>(total, 0.0f);
}

// ---- host side -----------------------------------------------------------------

namespace {

bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// Elements that every row of the operand lets a vector hold: 8, 4 or 0.
int vector_of(const void* p, const Strides& s) {
    const int64_t all = s.b | s.s | s.h;
    return aligned_to(p, 16) && all % 8 == 0 ? 8 : aligned_to(p, 8) && all % 4 == 0 ? 4 : 0;
}

Strides strides_of(const int64_t (&s)[3]) { return Strides{s[0], s[1], s[2]}; }

constexpr int64_t kMaxHeads = 1 << 16;

// Checks the arguments and lays them out; V receives the vector width, 0 where
// there is nothing to do.
int make_params(const spline_hip_qk_rope* a, bool norm, bool backward, QkParams& p, int& V) {
    if (a == nullptr || a->batch < 0 || a->sequence_length < 0 || a->q_heads < 0 || a->k_heads < 0)
        return hipErrorInvalidValue;
    const int64_t d = a->head_dim, r = a->rotary_dim;
    if (d <= 0 || d > 256 || d % 8 != 0 || r < 0 || r > d || r % 8 != 0) return hipErrorInvalidValue;
    if (a->q_heads > kMaxHeads || a->k_heads > kMaxHeads) return hipErrorInvalidValue;
    V = 0;
    if (a->batch == 0 || a->sequence_length == 0 || a->q_heads + a->k_heads == 0) return hipSuccess;
    if (a->batch > 0x7fffffff / a->sequence_length) return hipErrorInvalidValue;
    if (r > 0 && (!a->phase_increments || !aligned_to(a->phase_increments, 4))) return hipErrorInvalidValue;
    if (a->position_bytes != 4 && a->position_bytes != 8) return hipErrorInvalidValue;
    if (a->positions && !aligned_to(a->positions, a->position_bytes)) return hipErrorInvalidValue;
    if (a->frequency_axes && (!a->positions || a->axes < 1 || !aligned_to(a->frequency_axes, 4)))
        return hipErrorInvalidValue;
    const int wa = a->weight_f32 ? 4 : 2;
    if (!aligned_to(a->q_weight, wa) || !aligned_to(a->k_weight, wa)) return hipErrorInvalidValue;

    p = QkParams{};
    V = d % 16 == 0 && r % 16 == 0 ? 8 : 4;
    auto side = [&](QkSide& s, int64_t heads, const void* x, void* y, const void* w, const void* dy,
                    const int64_t (&xs)[3], const int64_t (&ys)[3], const int64_t (&dys)[3]) {
        s.heads = (int)heads;
        if (heads == 0) return true;
        if ((!x && (norm || !backward)) || !y || (backward && !dy)) return false;
        s.x = static_cast<const uint16_t*>(x);
        s.y = static_cast<uint16_t*>(y);
        s.dy = static_cast<const uint16_t*>(dy);
        s.w = norm ? w : nullptr;
        s.xs = strides_of(xs);
        s.ys = strides_of(ys);
        s.dys = strides_of(dys);
        int v = vector_of(y, s.ys);
        if (norm || !backward) v = vector_of(x, s.xs) < v ? vector_of(x, s.xs) : v;
        if (backward) v = vector_of(dy, s.dys) < v ? vector_of(dy, s.dys) : v;
        V = v < V ? v : V;
        return v != 0;
    };
    if (!side(p.q, a->q_heads, a->q, a->q_out, a->q_weight, a->dq_out, a->q_strides, a->q_out_strides,
              a->dq_out_strides) ||
        !side(p.k, a->k_heads, a->k, a->k_out, a->k_weight, a->dk_out, a->k_strides, a->k_out_strides,
              a->dk_out_strides))
        return hipErrorInvalidValue;
    p.inc = static_cast<const uint32_t*>(a->phase_increments);
    // a position's low word holds it modulo the 2^32 that its phase wraps at
    const int64_t words = a->position_bytes / 4;
    p.pos = static_cast<const uint32_t*>(a->positions);
    p.poss = Strides{a->position_strides[1] * words, a->position_strides[2] * words, a->position_strides[0] * words};
    p.axes = a->frequency_axes;
    p.axis_count = a->axes > 0x7fffffff ? 0x7fffffff : (int)a->axes;
    p.tokens = (uint32_t)(a->batch * a->sequence_length);
    p.seq = (uint32_t)a->sequence_length;
    p.head_dim = (int)d;
    p.rotary = (int)r;
    p.lanes = (int)d / (2 * V);
    while ((1 << p.log_lanes) < p.lanes) ++p.log_lanes;
    p.eps = a->eps;
    p.inv_d = 1.0f / (float)d;
    p.w32 = a->weight_f32 != 0;
    // Non-temporal stores from half of the elementwise kernels' threshold on for
    // the forward: alone 22.5 us against 27.5 with 59 MiB of results, 24.7
    // against 25.9 with 44, and neutral with the attention behind it, which reads them
    // (40 to 59 MiB: within 1 %).  The backward keeps the threshold (63 MiB:
    // 55 us with them, 53 without).
    p.nt = (a->q_heads + a->k_heads) * (int64_t)p.tokens * d * 2 >= (backward ? kNtStoreBytes : kNtStoreBytes / 2);
    return hipSuccess;
}

// Cuts the heads of both sides: 8 heads to a split, fewer where the items would
// not make two blocks a CU.  4 x 4096 tokens, 32 + 8 heads of 128, forward /
// backward by heads to a split: 5 64.6 / 111 us, 8 66 / 101, 16 69 / 114, all 76 / -;
// 6001 tokens forward: 2 37.9, 6 31.5, 8 to 11 29.7 (each with cached stores).
void cut_heads(QkParams& p, int64_t chunks) {
    const int64_t want = (2 * device_shape().cus + chunks - 1) / chunks, heads = p.q.heads + p.k.heads;
    auto splits = [&](int n) {
        const int64_t even = (want * n + heads - 1) / heads, full = (n + 8 - 1) / 8;
        return (int)(even > n ? n : even < full ? full : even);
    };
    p.q.splits = splits(p.q.heads);
    p.k.splits = splits(p.k.heads);
}

template <bool BF, int V, bool INTER, bool NORM>
void run_forward(QkParams& p, hipStream_t stream) {
    const int64_t rows = kBlock >> p.log_lanes, chunks = (p.tokens + rows - 1) / rows;
    cut_heads(p, chunks);
    const int64_t splits = p.q.splits + p.k.splits;
    const int64_t most = 0xffffffffll / kBlock / splits;  // a grid counts its threads in 32 bits
    const int64_t grid = (chunks < most ? chunks : most) * splits;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kBlock), 0, stream, p); };
    p.nt ? go(qk_rope_kernel<BF, V, INTER, NORM, true, 2>) : go(qk_rope_kernel<BF, V, INTER, NORM, false, 2>);
}

template <bool BF, bool NORM>
int forward(QkParams& p, int V, bool inter, hipStream_t stream) {
    if (V == 0) return hipSuccess;
    if (V == 8) inter ? run_forward<BF, 8, true, NORM>(p, stream) : run_forward<BF, 8, false, NORM>(p, stream);
    else inter ? run_forward<BF, 4, true, NORM>(p, stream) : run_forward<BF, 4, false, NORM>(p, stream);
    return hipGetLastError();
}

// Blocks of both sides, which bounds the partial rows (1024: 119 us at the size
// above, where items make 2.5 rounds of them).
constexpr int kBwdBlocks = 2048;

template <bool BF>
int backward(const spline_hip_qk_rope* a, QkParams& p, int V, hipStream_t stream) {
    if (V == 0) return hipSuccess;
    const int64_t rows = kBlock >> p.log_lanes, chunks = (p.tokens + rows - 1) / rows;
    cut_heads(p, chunks);
    const int64_t items = chunks * (p.q.splits + p.k.splits);
    const int64_t each = (items + kBwdBlocks - 1) / kBwdBlocks;  // per block
    p.q.blocks = (int)((chunks * p.q.splits + each - 1) / each);
    p.k.blocks = (int)((chunks * p.k.splits + each - 1) / each);
    float* ws = a->dw_workspace;
    if (p.q.w) p.q.dw = ws, ws += (int64_t)p.q.blocks * p.head_dim;
    if (p.k.w) p.k.dw = ws;
    if ((p.q.w && (!a->dq_weight || !a->dw_workspace)) || (p.k.w && (!a->dk_weight || !a->dw_workspace)))
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)(p.q.blocks + p.k.blocks));
    const bool inter = a->interleaved != 0;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, p); };
    auto pick = [&](auto nt) {
        constexpr bool NT = decltype(nt)::value;
        if (V == 8) inter ? go(qk_rope_bwd_kernel<BF, 8, true, NT, 2>) : go(qk_rope_bwd_kernel<BF, 8, false, NT, 2>);
        else inter ? go(qk_rope_bwd_kernel<BF, 4, true, NT, 2>) : go(qk_rope_bwd_kernel<BF, 4, false, NT, 2>);
    };
    p.nt ? pick(std::integral_constant<bool, true>{}) : pick(std::integral_constant<bool, false>{});
    int rc = hipGetLastError();
    if (rc != hipSuccess || (!p.q.w && !p.k.w)) return rc;
    hipLaunchKernelGGL((qk_dw_kernel<BF>), dim3((p.head_dim + 15) / 16, 2), dim3(1024), 0, stream,
                       DwSide{p.q.dw, a->dq_weight, p.q.blocks}, DwSide{p.k.dw, a->dk_weight, p.k.blocks},
                       p.head_dim, p.w32);
    return hipGetLastError();
}

template <bool BF>
int norm_forward(const spline_hip_qk_rope* a, void* stream) {
    QkParams p;
    int V;
    const int rc = make_params(a, true, false, p, V);
    return rc != hipSuccess ? rc : forward<BF, true>(p, V, a->interleaved != 0, hs(stream));
}
template <bool BF>
int norm_backward(const spline_hip_qk_rope* a, void* stream) {
    QkParams p;
    int V;
    const int rc = make_params(a, true, true, p, V);
    return rc != hipSuccess ? rc : backward<BF>(a, p, V, hs(stream));
}
template <bool BF>
int rotate(const spline_hip_qk_rope* a, int inverse, void* stream) {
    QkParams p;
    int V;
    const int rc = make_params(a, false, false, p, V);
    p.neg = inverse != 0;
    return rc != hipSuccess ? rc : forward<BF, false>(p, V, a->interleaved != 0, hs(stream));
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" int launch_qk_norm_rope_bf16(const spline_hip_qk_rope* args, void* stream) {
    return norm_forward<true>(args, stream);
}
extern "C" int launch_qk_norm_rope_fp16(const spline_hip_qk_rope* args, void* stream) {
    return norm_forward<false>(args, stream);
}
extern "C" int64_t spline_hip_qk_norm_rope_bwd_bytes(int64_t head_dim) {
    return head_dim > 0 ? (int64_t)(kBwdBlocks + 2) * head_dim * 4 : 0;
}
extern "C" int launch_qk_norm_rope_bwd_bf16(const spline_hip_qk_rope* args, void* stream) {
    return norm_backward<true>(args, stream);
}
extern "C" int launch_qk_norm_rope_bwd_fp16(const spline_hip_qk_rope* args, void* stream) {
    return norm_backward<false>(args, stream);
}
extern "C" int launch_rope_axes_bf16(const spline_hip_qk_rope* args, int inverse, void* stream) {
    return rotate<true>(args, inverse, stream);
}
extern "C" int launch_rope_axes_fp16(const spline_hip_qk_rope* args, int inverse, void* stream) {
    return rotate<false>(args, inverse, stream);
}
