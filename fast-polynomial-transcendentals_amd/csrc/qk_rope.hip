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
// A lane owns one vector of V elements of a row, so that a wave's accesses are
// whole rows of neighbouring tokens (halves of rows: a copy of rows of 64, 80 or 96
// elements takes a quarter longer).  The other elements of its pairs lie in the same
// vector, or in the lane half a rotated row away, which sends them (ds_bpermute).
// With the norm a row takes a power of two of lanes, for the mean's exchanges,
// else as many as it fills.  A thread evaluates its sines and cosines once for a
// token and applies them to the heads of its split.
//
// The gradient of w sums over every row: a block keeps its sums in registers
// over all its tokens, adds its rows through LDS and stores one partial row;
// a second launch adds the partial rows.  Every order of addition is fixed.
//
// What bounds it: memory, 4 bytes an element forward and 6 backward.  Measured at
// 4 x 4096 tokens, 32 + 8 heads of 128 in BF16, each by itself over inputs in turn:
// forward 62.7 to 64.2 us, 5.3 TB/s, backward 97.7 to 99.0 us for both launches, 5.1 TB/s (a
// copy of as much: 6.6 TB/s).  Behind the forward, which leaves part of x in the MALL, the
// backward kernel takes 84 to 89 us and the sum of the partial rows 4 to 5, so that
// one pass of both takes 153.  The rotation alone by three axes, 2 x 8190 tokens: 61.4 us,
// 5.5 TB/s.  Few tokens take a launch, 4 us.  Rows of 80 elements with 40 rotated, by halves,
// take 4-element vectors and 20 of 32 lanes: 11.8 us forward for 3003 tokens of 32
// heads in FP16, where a copy takes 4.7, and 19.2 backward.
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
    int lanes, log_lanes;   // lanes that own vectors; log2 of the lanes between rows (with the norm)
    int wave_rows, rows;    // rows of a wave, of a block
    float eps, inv_d;
    bool w32, neg, nt;      // FP32 weights; the inverse rotation; non-temporal stores
};

// Where a lane's vector lies in a row, and what it turns by: y_i = c_i x_i + s_i x_i',
// i' the other element of i's pair.
template <int V, bool INTER>
struct LanePart {
    int e, pe;    // first element, and that of the lane with the other halves of the pairs
    int partner;  // its lane in the wave, times 4
    bool rot, first;

    __device__ __forceinline__ LanePart(const QkParams& p, int l, int lane) {
        const int half = p.rotary >> 1;
        e = V * l;
        rot = e < p.rotary;
        first = e < half;
        pe = INTER || !rot ? e : first ? e + half : e - half;
        partner = 4 * (lane + (pe - e) / V);
    }

    __device__ __forceinline__ void angles(const QkParams& p, uint32_t b, uint32_t s, float (&cs)[V],
                                           float (&sn)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            cs[i] = 1.0f;
            sn[i] = 0.0f;
        }
        if (!rot) return;
        const uint32_t* pos = p.pos == nullptr ? nullptr : p.pos + b * p.poss.b + s * p.poss.s;
        const uint32_t one = pos == nullptr ? s : p.axes == nullptr ? *pos : 0u;
        // V / 2 angles a lane: of halves, the lane with the other half evaluates the rest
        const int f0 = INTER ? e >> 1 : first ? e : pe + V / 2;
        float c[V / 2], t[V / 2];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            uint32_t at = one;
            if (p.axes != nullptr) {
                const int a = p.axes[f0 + j];  // held to the axes that there are
                at = pos[(a < 0 ? 0 : a < p.axis_count ? a : p.axis_count - 1) * p.poss.h];
            }
            const uint32_t phase = at * p.inc[f0 + j];
            phase_sincos(p.neg ? 0u - phase : phase, c[j], t[j]);
        }
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            if constexpr (INTER) {
                cs[2 * j] = cs[2 * j + 1] = c[j];
                sn[2 * j] = -t[j];
                sn[2 * j + 1] = t[j];
            } else {
                // both lanes of a pair are here or neither is
                const float c2 = as_f32((uint32_t)__builtin_amdgcn_ds_bpermute(partner, (int)as_u32(c[j])));
                const float t2 = as_f32((uint32_t)__builtin_amdgcn_ds_bpermute(partner, (int)as_u32(t[j])));
                cs[j] = first ? c[j] : c2;
                cs[V / 2 + j] = first ? c2 : c[j];
                sn[j] = first ? -t[j] : t2;
                sn[V / 2 + j] = first ? -t2 : t[j];
            }
        }
    }

    // w[start ..], ones without a weight.
    template <bool BF>
    __device__ __forceinline__ void weights(const QkParams& p, const void* w, int start, float (&out)[V]) const {
        if (w == nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = 1.0f;
        } else if (p.w32) {
            const float* t = static_cast<const float*>(w) + start;
            if (((uintptr_t)w & 15) == 0) {
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(t + i);
                    out[i] = v.x, out[i + 1] = v.y, out[i + 2] = v.z, out[i + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) out[i] = t[i];
            }
        } else {
            const uint16_t* t = static_cast<const uint16_t*>(w) + start;
            Words<V> o;
            if (((uintptr_t)w & 15) == 0) {
                o = load_words<V>(t);
            } else {  // a view of other weights
#pragma unroll
                for (int i = 0; i < V / 2; ++i) o.w[i] = (uint32_t)t[2 * i] | (uint32_t)t[2 * i + 1] << 16;
            }
#pragma unroll
            for (int i = 0; i < V; i += 2) widen<BF>(o.w[i / 2], out[i], out[i + 1]);
        }
    }

    // The other elements of the pairs; zeros where nothing turns (an infinity
    // there stays where it is).  All lanes take part.
    template <bool BF>
    __device__ __forceinline__ void others(const QkParams& p, const Words<V>& raw, const float (&f)[V],
                                           float (&out)[V]) const {
        if constexpr (INTER) {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = f[i ^ 1];
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i)
                widen<BF>((uint32_t)__builtin_amdgcn_ds_bpermute(partner, (int)raw.w[i]), out[2 * i], out[2 * i + 1]);
        }
        if (p.rotary < p.head_dim) {  // the same for every thread
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = rot ? out[i] : 0.0f;
        }
    }
};

template <bool BF, int V>
__device__ __forceinline__ void widen_row(const Words<V>& raw, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 2) widen<BF>(raw.w[i / 2], f[i], f[i + 1]);
}
template <bool BF, int V, bool NT>
__device__ __forceinline__ void store_row(uint16_t* at, const float (&f)[V]) {
    Words<V> o;
#pragma unroll
    for (int i = 0; i < V; i += 2) o.w[i / 2] = narrow<BF>(f[i], f[i + 1]);
    store_words<V, NT>(at, o);
}

template <int V>
__device__ __forceinline__ float sum_squares(const float (&f)[V]) {
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < V; ++i) t[i & 3] = __builtin_fmaf(f[i], f[i], t[i & 3]);
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
    const int lane = threadIdx.x & 63;
    const int wrow = NORM ? lane >> p.log_lanes : lane / (uint32_t)p.lanes;
    const int l = NORM ? lane & ((1 << p.log_lanes) - 1) : lane - wrow * p.lanes;
    const bool own = NORM ? l < p.lanes : wrow < p.wave_rows;
    const int row = (int)(threadIdx.x >> 6) * p.wave_rows + wrow;
    const Part part(p, own ? l : 0, own ? lane : 0);
    const uint32_t splits = p.q.splits + p.k.splits;
    const uint32_t chunk0 = blockIdx.x / splits;
    int split = (int)(blockIdx.x - chunk0 * splits);
    const bool is_k = split >= p.q.splits;
    split -= is_k ? p.q.splits : 0;
    const int heads = is_k ? p.k.heads : p.q.heads, parts = is_k ? p.k.splits : p.q.splits;
    const int h_begin = heads * split / parts, h_end = heads * (split + 1) / parts;
    const Strides xs = is_k ? p.k.xs : p.q.xs, ys = is_k ? p.k.ys : p.q.ys;
    const int64_t stride = gridDim.x / splits * (int64_t)p.rows;
    for (int64_t t0 = chunk0 * (int64_t)p.rows; t0 < p.tokens; t0 += stride) {
        const int64_t token = t0 + row;
        const bool in = own && token < p.tokens;
        const uint32_t b = (uint32_t)token / p.seq, s = (uint32_t)token - b * p.seq;
        const uint16_t* x = (is_k ? p.k.x : p.q.x) + b * xs.b + s * xs.s + part.e;
        uint16_t* y = (is_k ? p.k.y : p.q.y) + b * ys.b + s * ys.s + part.e;
        auto load = [&](int h, Words<V> (&raw)[HPT]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < HPT; ++u) {
                raw[u] = Words<V>{};
                if (in && h + u < h_end) raw[u] = load_words<V>(x + (h + u) * xs.h);
            }
        };
        Words<V> raw[2][HPT];
        load(h_begin, raw[0]);
        float cs[V] = {}, sn[V] = {};
        if (in) part.angles(p, b, s, cs, sn);
        if constexpr (NORM) {
            const void* w = is_k ? p.k.w : p.q.w;
            float mine[V] = {}, other[V] = {};
            if (own) part.template weights<BF>(p, w, part.e, mine);
            if (!INTER && own) part.template weights<BF>(p, w, part.pe, other);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                cs[i] *= mine[i];
                // nothing is added where nothing turns: a weight there may be infinite
                sn[i] = part.rot ? sn[i] * (INTER ? mine[i ^ 1] : other[i]) : 0.0f;
            }
        }
        auto turn = [&](int h, const Words<V> (&now)[HPT]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < HPT; ++u) {
                if (h + u >= h_end) break;  // the same for every thread of the block
                float f[V], o[V];
                widen_row<BF, V>(now[u], f);
                part.template others<BF>(p, now[u], f, o);
                float r = 1.0f;
                if constexpr (NORM)
                    r = __builtin_amdgcn_rsqf(
                        __builtin_fmaf(group_sum(sum_squares<V>(f), p.log_lanes), p.inv_d, p.eps));
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float t = __builtin_fmaf(cs[i], f[i], sn[i] * o[i]);
                    f[i] = NORM ? t * r : t;
                }
                if (in) store_row<BF, V, NT>(y + (h + u) * ys.h, f);
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
template <bool BF, int V, bool INTER, bool NT, int HPT>
__global__ void __launch_bounds__(kBlock, 4) qk_rope_bwd_kernel(QkParams p) {
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
    const int lane = threadIdx.x & 63, l = lane & ((1 << p.log_lanes) - 1), rows = p.rows;
    const int row = (int)(threadIdx.x >> 6) * p.wave_rows + (lane >> p.log_lanes);
    const bool own = l < p.lanes;
    const Part part(p, own ? l : 0, own ? lane : 0);
    float w[V] = {}, acc[V] = {};
    if (own) part.template weights<BF>(p, is_k ? p.k.w : p.q.w, part.e, w);

    // item = chunk * splits + split, stepped without a division
    const int64_t chunks = ((int64_t)p.tokens + rows - 1) / rows;
    const uint32_t chunk_step = blocks / splits, split_step = blocks - chunk_step * splits;
    int64_t chunk = block / splits;
    uint32_t split = block - (uint32_t)chunk * splits;
    while (chunk < chunks) {
        const int64_t token = chunk * rows + row;
        const bool in = own && token < p.tokens;
        const uint32_t b = (uint32_t)token / p.seq, s = (uint32_t)token - b * p.seq;
        const int h_begin = heads * (int)split / (int)splits, h_end = heads * ((int)split + 1) / (int)splits;
        const uint16_t* xtoken = x + b * xs.b + s * xs.s + part.e;
        const uint16_t* dytoken = dy + b * dys.b + s * dys.s + part.e;
        uint16_t* dxtoken = dx + b * ys.b + s * ys.s + part.e;
        float cs[V] = {}, sn[V] = {};
        for (int h = h_begin; h < h_end; h += HPT) {
            Words<V> rx[HPT], rdy[HPT];
#pragma unroll
            for (int u = 0; u < HPT; ++u) {
                rx[u] = rdy[u] = Words<V>{};
                if (in && h + u < h_end) {
                    rx[u] = load_words<V>(xtoken + (h + u) * xs.h);
                    rdy[u] = load_words<V>(dytoken + (h + u) * dys.h);
                }
            }
            if (in && h == h_begin) part.angles(p, b, s, cs, sn);
#pragma unroll
            for (int u = 0; u < HPT; ++u) {
                if (h + u >= h_end) break;  // the same for every thread of the block
                float n[V], g[V], o[V];
                widen_row<BF, V>(rx[u], n);
                widen_row<BF, V>(rdy[u], g);
                part.template others<BF>(p, rdy[u], g, o);
                const float r = __builtin_amdgcn_rsqf(
                    __builtin_fmaf(group_sum(sum_squares<V>(n), p.log_lanes), p.inv_d, p.eps));
                float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    g[i] = __builtin_fmaf(cs[i], g[i], -(sn[i] * o[i]));  // the rotation by -t
                    n[i] *= r;
                    if (in) acc[i] = __builtin_fmaf(g[i], n[i], acc[i]);
                    g[i] *= w[i];
                    t[i & 3] = __builtin_fmaf(g[i], n[i], t[i & 3]);
                }
                const float mean = group_sum((t[0] + t[1]) + (t[2] + t[3]), p.log_lanes) * p.inv_d;
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = r * __builtin_fmaf(n[i], -mean, g[i]);
                if (in) store_row<BF, V, NT>(dxtoken + (h + u) * ys.h, g);
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
    __shared__ float sums[kBlock * V];
    if (own) {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[row * p.head_dim + part.e + i] = acc[i];
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
    if (s.out == nullptr) return;
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
    p = QkParams{};
    if (a->batch == 0 || a->sequence_length == 0 || a->q_heads + a->k_heads == 0) return hipSuccess;
    if (a->batch > 0x7fffffff / a->sequence_length) return hipErrorInvalidValue;
    if (r > 0 && (!a->phase_increments || !aligned_to(a->phase_increments, 4))) return hipErrorInvalidValue;
    if (a->position_bytes != 4 && a->position_bytes != 8) return hipErrorInvalidValue;
    if (a->positions && !aligned_to(a->positions, a->position_bytes)) return hipErrorInvalidValue;
    if (a->frequency_axes && (!a->positions || a->axes < 1 || !aligned_to(a->frequency_axes, 4)))
        return hipErrorInvalidValue;
    const int wa = a->weight_f32 ? 4 : 2;
    if (!aligned_to(a->q_weight, wa) || !aligned_to(a->k_weight, wa)) return hipErrorInvalidValue;

    V = a->interleaved || r % 16 == 0 ? 8 : 4;  // a vector holds pairs, or one half of its pairs
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
    p.lanes = (int)d / V;
    while ((1 << p.log_lanes) < p.lanes) ++p.log_lanes;
    p.wave_rows = norm ? 64 >> p.log_lanes : 64 / p.lanes;
    p.rows = kBlock / 64 * p.wave_rows;
    p.eps = a->eps;
    p.inv_d = 1.0f / (float)d;
    p.w32 = a->weight_f32 != 0;
    // Non-temporal stores from half of the elementwise kernels' threshold on:
    // forward 22.3 us against 28.6 with 59 MiB of results, 19.4 against 21.9 with 44,
    // and neutral with the attention behind it, which reads them (40 to 59 MiB:
    // within 1 %); backward 46.1 against 48.3 with 62 MiB, 36.4 against 40.8 with 44.
    p.nt = (a->q_heads + a->k_heads) * (int64_t)p.tokens * d * 2 >= kNtStoreBytes / 2;
    return hipSuccess;
}

// Cuts the heads of both sides: `each` heads to a split, 8 forward and 12 backward,
// fewer where the items would not make two blocks a CU.  Forward / backward by heads
// to a split, us: 4 x 4096 tokens, 32 + 8 heads of 128: 4 64.4 / 104, 8 64.7 / 103,
// 12 63.0 / 98, 16 64.4 / 108; 2 x 4096 tokens, heads of 96: 4 30.7 / 51.6,
// 8 24.6 / 51.9, 12 23.4 / 47.6, 16 25.1 / 47.5; 6001 tokens forward: 4 27.7, 8 22.1,
// 12 23.4, 16 26.0.  1000 tokens, forward / backward at 2, 4 and 8 blocks a CU:
// 7.7 / 14.8, 9.8 / 17.3, 12.3 / 18.9; 300 tokens 5.6 / 11.3, 5.5 / 9.9, 5.5 / 9.9.
void cut_heads(QkParams& p, int64_t chunks, int each) {
    const int64_t want = (2 * device_shape().cus + chunks - 1) / chunks, heads = p.q.heads + p.k.heads;
    auto splits = [&](int n) {
        const int64_t even = (want * n + heads - 1) / heads, full = (n + each - 1) / each;
        return (int)(even > n ? n : even < full ? full : even);
    };
    p.q.splits = splits(p.q.heads);
    p.k.splits = splits(p.k.heads);
}

template <bool BF, int V, bool INTER, bool NORM>
void run_forward(QkParams& p, hipStream_t stream) {
    const int64_t chunks = (p.tokens + (int64_t)p.rows - 1) / p.rows;
    cut_heads(p, chunks, 8);
    const int64_t splits = p.q.splits + p.k.splits;
    const int64_t most = 0xffffffffll / kBlock / splits;  // a grid counts its threads in 32 bits
    const int64_t grid = (chunks < most ? chunks : most) * splits;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kBlock), 0, stream, p); };
    p.nt ? go(qk_rope_kernel<BF, V, INTER, NORM, true, 4>) : go(qk_rope_kernel<BF, V, INTER, NORM, false, 4>);
}

template <bool BF, bool NORM>
int forward(QkParams& p, int V, bool inter, hipStream_t stream) {
    if (V == 0) return hipSuccess;
    if (V == 8) inter ? run_forward<BF, 8, true, NORM>(p, stream) : run_forward<BF, 8, false, NORM>(p, stream);
    else inter ? run_forward<BF, 4, true, NORM>(p, stream) : run_forward<BF, 4, false, NORM>(p, stream);
    return hipGetLastError();
}

// Blocks of both sides, which bounds the partial rows.  1024 instead: 98.8 us against
// 97.7 at the first size above, 21.5 against 19.4 with 3003 tokens of 16 + 16 heads of 80.
constexpr int kBwdBlocks = 2048;

template <bool BF>
int backward(const spline_hip_qk_rope* a, QkParams& p, int V, hipStream_t stream) {
    // a side without rows has no partial rows either: its weight's gradient is zero
    const bool qw = a->q_weight != nullptr, kw = a->k_weight != nullptr;
    if ((qw && (!a->dq_weight || !a->dw_workspace)) || (kw && (!a->dk_weight || !a->dw_workspace)))
        return hipErrorInvalidValue;
    auto add_rows = [&]() -> int {
        if (!qw && !kw) return hipSuccess;
        hipLaunchKernelGGL((qk_dw_kernel<BF>), dim3((unsigned)(a->head_dim + 15) / 16, 2), dim3(1024), 0, stream,
                           DwSide{p.q.dw, qw ? a->dq_weight : nullptr, p.q.dw ? p.q.blocks : 0},
                           DwSide{p.k.dw, kw ? a->dk_weight : nullptr, p.k.dw ? p.k.blocks : 0}, (int)a->head_dim,
                           a->weight_f32 != 0);
        return hipGetLastError();
    };
    if (V == 0) return add_rows();
    const int64_t chunks = (p.tokens + (int64_t)p.rows - 1) / p.rows;
    cut_heads(p, chunks, 12);
    const int64_t items = chunks * (p.q.splits + p.k.splits);
    const int64_t each = (items + kBwdBlocks - 1) / kBwdBlocks;  // per block
    p.q.blocks = (int)((chunks * p.q.splits + each - 1) / each);
    p.k.blocks = (int)((chunks * p.k.splits + each - 1) / each);
    float* ws = a->dw_workspace;
    if (p.q.w) p.q.dw = ws, ws += (int64_t)p.q.blocks * p.head_dim;
    if (p.k.w) p.k.dw = ws;
    const dim3 grid((unsigned)(p.q.blocks + p.k.blocks));
    const bool inter = a->interleaved != 0;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, p); };
    auto pick = [&](auto nt) {
        constexpr bool NT = decltype(nt)::value;
        if (V == 8) inter ? go(qk_rope_bwd_kernel<BF, 8, true, NT, 2>) : go(qk_rope_bwd_kernel<BF, 8, false, NT, 2>);
        else inter ? go(qk_rope_bwd_kernel<BF, 4, true, NT, 2>) : go(qk_rope_bwd_kernel<BF, 4, false, NT, 2>);
    };
    p.nt ? pick(std::integral_constant<bool, true>{}) : pick(std::integral_constant<bool, false>{});
    const int rc = hipGetLastError();
    return rc != hipSuccess ? rc : add_rows();
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
