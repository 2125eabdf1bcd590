// paged_cache.hip -- storing into, reading from and rearranging the pages of a
// serving cache, for gfx950.
//
// Store and load: the last T keys and values of each sequence to and from E2M1 codes
// (fp4.hpp).  A thread has 8 elements, four threads a block of 32: its largest value
// lies in [7/2, 7) times the power of two that they choose, 2^(floor(log2 max) - 2),
// twice that if the largest is past 7/4 of its own power, so that no value loses more
// than half a step when 6 is the greatest number (a choice of [4, 8) cuts up to a
// fourth off).  v_cvt_scalef32_pk_fp4 rounds to nearest, ties to the even code.
// Both are bound by the 16-bit side's bytes.
#include <hip/hip_runtime.h>

#include "fp4.hpp"

namespace pt {

// n / d for n below 2^31: the high half of n m, shifted, with m = 2^(31 + s) / d rounded up
// and 2^s >= d, which is off by less than 1 / d.
struct Divisor {
    uint32_t d, m, s;

    Divisor() = default;
    explicit Divisor(uint32_t d_) : d(d_), s(0) {
        while ((uint64_t(1) << s) < d) ++s;
        m = (uint32_t)((uint64_t(1) << (31 + s)) / d + 1);
    }
    __device__ __forceinline__ uint32_t divide(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> (s - 1); }
};

struct Fp4Rows {
    const uint16_t *k, *v;
    AttnStrides ks, vs;
    uint32_t threads;
    Divisor per, tokens, page;  // threads of a token (hkv HD / 8), tokens, page size
};

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true);  // lanes 1 0 3 2
    x = a > x ? a : x;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true);  // lanes 2 3 0 1
    return b > x ? b : x;
}

// The block's exponent byte from its largest magnitude's bits: 255 where it is no
// finite number.
template <bool BF>
__device__ __forceinline__ uint32_t fp4_byte(uint32_t top) {
    if (top >= (BF ? 0x7f80u : 0x7c00u)) return 255;
    const uint32_t bits = BF ? top << 16 : as_u32((float)__builtin_bit_cast(_Float16, (uint16_t)top));
    const int byte = (int)((bits + 0x200000u) >> 23) - 2;
    return (uint32_t)(byte < kFp4Least ? kFp4Least : byte > kFp4Most ? kFp4Most : byte);
}

template <bool BF>
__device__ __forceinline__ uint32_t fp4_codes(u32x4_t x, float scale) {
    const uint32_t a = x.x, b = x.y, c = x.z, d = x.w;
    uint32_t r = 0;
    if constexpr (BF) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, a), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, b), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, c), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, d), scale, 3);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, a), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, b), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, c), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, d), scale, 3);
    }
    return r;
}

// Eight elements in the 16-bit type; FP16 holds what is finite to its largest number.
template <bool BF>
__device__ __forceinline__ u32x4_t fp4_elements(uint32_t codes, float scale) {
    if constexpr (BF) return __builtin_bit_cast(u32x4_t, fp4_to_bf16(codes, scale));
    f32x2_t f[4];
    f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
    f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
    f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
    f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f16x2_t h;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float x = f[i][e];
            h[e] = (_Float16)(x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x);  // NaN stays
        }
        r[i] = __builtin_bit_cast(uint32_t, h);
    }
    return r;
}

// A thread's eight elements of a key and of its value: token, head and the row in the
// cache.
template <int HD>
struct Fp4Place {
    uint32_t bt, b, t, h, chunk;
    int page, row;

    __device__ __forceinline__ Fp4Place(const Fp4Pages& p, const Fp4Rows& r, uint32_t i) {
        constexpr uint32_t kChunks = HD / 8;
        bt = r.per.divide(i);
        const uint32_t rest = i - bt * r.per.d;
        chunk = rest % kChunks;
        h = rest / kChunks;
        b = r.tokens.divide(bt);
        t = bt - b * r.tokens.d;
        const int pos = p.len(b) - (int)r.tokens.d + (int)t;
        const int entry = pos < 0 ? -1 : (int)r.page.divide((uint32_t)pos);
        page = p.page_of(b, entry);
        row = pos - entry * p.page_size;
    }
    __device__ __forceinline__ uint8_t* head(const Fp4Pages& p, int kv) const {
        return const_cast<uint8_t*>(p.head(page, kv, (int)h));
    }
    __device__ __forceinline__ uint32_t codes() const { return (uint32_t)row * (HD / 2) + chunk * 4; }
    __device__ __forceinline__ uint32_t byte(const Fp4Pages& p) const {
        return (uint32_t)(p.page_size * (HD / 2) + row * (HD / kFp4Block)) + chunk / 4;
    }
};

template <bool BF>
__device__ __forceinline__ uint32_t largest(u32x4_t x) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t lo = x[w] & 0x7fffu, hi = (x[w] >> 16) & 0x7fffu;
        top = lo > top ? lo : top;
        top = hi > top ? hi : top;
    }
    return fp4_byte<BF>(quad_max(top));
}

template <int HD, bool BF>
__global__ void __launch_bounds__(256) fp4_store_kernel(Fp4Pages p, Fp4Rows r) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= r.threads) return;
    const Fp4Place<HD> at(p, r, i);
    if (at.page < 0) return;
    const u32x4_t k = *reinterpret_cast<const u32x4_t*>(r.k + at.b * r.ks.b + at.t * r.ks.s + at.h * r.ks.h + at.chunk * 8);
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(r.v + at.b * r.vs.b + at.t * r.vs.s + at.h * r.vs.h + at.chunk * 8);
    const uint32_t kb = largest<BF>(k), vb = largest<BF>(v);
    uint8_t *kh = at.head(p, 0), *vh = at.head(p, 1);
    const uint32_t codes = at.codes();
    *reinterpret_cast<uint32_t*>(kh + codes) = kb == 255 ? 0 : fp4_codes<BF>(k, as_f32(kb << 23));
    *reinterpret_cast<uint32_t*>(vh + codes) = vb == 255 ? 0 : fp4_codes<BF>(v, as_f32(vb << 23));
    if ((at.chunk & 3) == 0) {
        kh[at.byte(p)] = (uint8_t)kb;
        vh[at.byte(p)] = (uint8_t)vb;
    }
}

template <int HD, bool BF>
__global__ void __launch_bounds__(256) fp4_load_kernel(Fp4Pages p, Fp4Rows r, uint16_t* k, uint16_t* v) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= r.threads) return;
    const Fp4Place<HD> at(p, r, i);
    u32x4_t kx = {0, 0, 0, 0}, vx = kx;
    if (at.page >= 0) {
        const uint8_t *kh = at.head(p, 0), *vh = at.head(p, 1);
        const uint32_t codes = at.codes(), byte = at.byte(p);
        kx = fp4_elements<BF>(*reinterpret_cast<const uint32_t*>(kh + codes), fp4_scale(kh[byte]));
        vx = fp4_elements<BF>(*reinterpret_cast<const uint32_t*>(vh + codes), fp4_scale(vh[byte]));
    }
    const int64_t out = (int64_t)i * 8;
    *reinterpret_cast<u32x4_t*>(k + out) = kx;
    *reinterpret_cast<u32x4_t*>(v + out) = vx;
}

// ---- pages of several sequences ------------------------------------------------
//
// A table [rows, entries] names each sequence's pages.  A page is in use where a row
// names it, so that there is no count of references beside the table that could
// differ from it.
//
// Fork: new row i continues old row parents[i] with its first lens keys.  Pages that
// they fill are shared.  The page that the next key goes to belongs to one row: the
// first new row whose last page it is keeps it, unless another row holds it as a
// full one; every other row gets a copy.  Pages for `grow` more keys are added.
// New pages are the lowest free ones, in the order of rows and entries.
//
// Compact: of n pages in use those with ids from n on move to the free ones
// below, both in ascending order.
//
// Four launches: the marks are cleared, every entry marks its page, one block counts
// (a bitmap of the pages, 32 to a thread and step, and the rows' wishes), and the last
// writes the table and copies the pages, which is what takes the time.  With few pages and
// entries one block does all but the copies, its marks in LDS: 16 rows of 25
// entries 12.4 us, 17 in four launches.

constexpr int kNoRow = 0x7fffffff;
constexpr int kScan = 1024;
constexpr int kMostCaches = 64;  // of a launch

struct PagePlan {
    const int32_t *table, *lens, *parents;
    int64_t table_stride;
    int32_t *out, *out_lens, *out_count;  // [rows, entries], [rows], short or used
    int rows, old_rows, entries, pages, page_size, grow;
    uint32_t *used, *full;  // bitmaps
    int32_t* first;         // [pages] the first row whose last page it is
    int32_t* ids;           // [pages] free pages; compact: holes
    int32_t* place;         // [pages] compact: a moved page's number
    int32_t* base;          // [rows] a row's first wish
    int2* moves;            // [rows] or [pages]
    int32_t* count;         // moves, free pages
};

__device__ __forceinline__ int words_of(int pages) { return (pages + 31) / 32; }

__device__ __forceinline__ void clear_marks(const PagePlan& p, bool fork, int i) {
    if (i < words_of(p.pages)) {
        p.used[i] = 0;
        if (fork) p.full[i] = 0;
    }
    if (fork && i < p.pages) p.first[i] = kNoRow;
}

// What a new row continues.
struct ForkRow {
    int parent, len, full, held, end;  // full pages; pages with keys; pages with room

    __device__ __forceinline__ ForkRow(const PagePlan& p, int row) {
        parent = p.parents ? p.parents[row] : row;
        if ((unsigned)parent >= (unsigned)p.old_rows) parent = -1;
        const int most = p.entries * p.page_size;  // below 2^30
        len = parent < 0 ? 0 : p.lens[parent];
        len = len < 0 ? 0 : len < most ? len : most;
        full = len / p.page_size;
        held = (len + p.page_size - 1) / p.page_size;
        end = parent < 0 ? 0 : (len + p.grow + p.page_size - 1) / p.page_size;
    }
    __device__ __forceinline__ int page(const PagePlan& p, int entry) const {
        const int id = p.table[parent * p.table_stride + entry];
        return (unsigned)id < (unsigned)p.pages ? id : -1;
    }
    __device__ __forceinline__ bool copies(const PagePlan& p, int row) const {
        if (full == held) return false;
        const int id = page(p, full);
        return id >= 0 && ((p.full[id >> 5] >> (id & 31) & 1) || p.first[id] != row);
    }
};

__device__ __forceinline__ void fork_mark(const PagePlan& p, int64_t i) {
    const int row = (int)(i / p.entries), entry = (int)(i - (int64_t)row * p.entries);
    const ForkRow r(p, row);
    if (entry >= r.held) return;
    const int id = r.page(p, entry);
    if (id < 0) return;
    atomicOr(&p.used[id >> 5], 1u << (id & 31));
    if (entry < r.full) atomicOr(&p.full[id >> 5], 1u << (id & 31));
    else atomicMin(&p.first[id], row);
}
__device__ __forceinline__ void compact_mark(const PagePlan& p, int64_t i) {
    const int64_t row = i / p.entries;
    const int id = p.table[row * p.table_stride + (i - row * p.entries)];
    if ((unsigned)id < (unsigned)p.pages) atomicOr(&p.used[id >> 5], 1u << (id & 31));
}
template <bool FORK>
__global__ void __launch_bounds__(256) clear_marks_kernel(PagePlan p) {
    clear_marks(p, FORK, (int)(blockIdx.x * 256u + threadIdx.x));
}
template <bool FORK>
__global__ void __launch_bounds__(256) mark_kernel(PagePlan p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.rows * p.entries) return;
    if constexpr (FORK) fork_mark(p, i);
    else compact_mark(p, i);
}

// The sum of the threads ahead, and of all.
__device__ __forceinline__ int block_scan(int x, int& total) {
    __shared__ int sums[kScan / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(inc, d);
        inc += lane >= d ? y : 0;
    }
    __syncthreads();  // the sums of the scan before are read
    if (lane == 63) sums[wave] = inc;
    __syncthreads();
    int ahead = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kScan / 64; ++w) {
        ahead += w < wave ? sums[w] : 0;
        total += sums[w];
    }
    return ahead + inc - x;
}

// A thread's words of a bitmap.
struct WordRange {
    int from, to;
    __device__ __forceinline__ explicit WordRange(int words) {
        const int each = (words + kScan - 1) / kScan;
        from = min((int)threadIdx.x * each, words);
        to = min(from + each, words);
    }
};
// Pages of a word, those past the last one left out.
__device__ __forceinline__ uint32_t valid_bits(const PagePlan& p, int word) {
    const int left = p.pages - word * 32;
    return left >= 32 ? ~0u : (1u << left) - 1;
}

__device__ __forceinline__ void fork_plan(const PagePlan& p) {
    const int words = words_of(p.pages);
    const WordRange w(words);
    int n = 0, free = 0;
    for (int i = w.from; i < w.to; ++i) n += __popc(~p.used[i] & valid_bits(p, i));
    int at = block_scan(n, free);
    for (int i = w.from; i < w.to; ++i)
        for (uint32_t m = ~p.used[i] & valid_bits(p, i); m; m &= m - 1) p.ids[at++] = i * 32 + __builtin_ctz(m);
    __syncthreads();
    int wishes = 0, moves = 0, lost = 0;
    for (int row0 = 0; row0 < p.rows; row0 += kScan) {
        const int row = row0 + (int)threadIdx.x;
        int wish = 0, copy = 0, beyond = 0, len = 0, source = -1;
        if (row < p.rows) {
            const ForkRow r(p, row);
            len = r.len;
            copy = r.copies(p, row);
            if (copy) source = r.page(p, r.full);
            const int end = r.end < p.entries ? r.end : p.entries;
            wish = copy + (end > r.held ? end - r.held : 0);
            // keys with no place: past the table, or on a page that the row lacks
            beyond = r.end - end;
            if (r.full < r.held && p.grow > 0 && r.len % p.page_size != 0 && r.page(p, r.full) < 0) ++beyond;
        }
        int all;
        const int first = wishes + block_scan(wish, all);
        wishes += all;
        if (row < p.rows) {
            p.base[row] = first;
            p.out_lens[row] = len;
        }
        const bool moved = copy && first < free;
        const int k = moves + block_scan(moved, all);
        moves += all;
        if (moved) p.moves[k] = make_int2(source, p.ids[first]);
        block_scan(beyond, all);
        lost += all;
    }
    if (threadIdx.x == 0) {
        p.count[0] = moves;
        p.count[1] = free;
        p.out_count[0] = lost + (wishes > free ? wishes - free : 0);
    }
}

__device__ __forceinline__ void compact_plan(const PagePlan& p) {
    const int words = words_of(p.pages);
    const WordRange w(words);
    int n = 0, used = 0, holes = 0, moves = 0;
    for (int i = w.from; i < w.to; ++i) n += __popc(p.used[i] & valid_bits(p, i));
    block_scan(n, used);
    // bits of a word that lie below `used`
    auto below = [&](int i) { return used >= i * 32 + 32 ? ~0u : used <= i * 32 ? 0u : (1u << (used - i * 32)) - 1; };
    int hole = 0, move = 0;
    for (int i = w.from; i < w.to; ++i) {
        hole += __popc(~p.used[i] & below(i));
        move += __popc(p.used[i] & valid_bits(p, i) & ~below(i));
    }
    hole = block_scan(hole, holes);
    move = block_scan(move, moves);
    for (int i = w.from; i < w.to; ++i) {
        for (uint32_t m = ~p.used[i] & below(i); m; m &= m - 1) p.ids[hole++] = i * 32 + __builtin_ctz(m);
        for (uint32_t m = p.used[i] & valid_bits(p, i) & ~below(i); m; m &= m - 1) {
            const int id = i * 32 + __builtin_ctz(m);
            p.moves[move].x = id;
            p.place[id] = move++;
        }
    }
    if (threadIdx.x == 0) {
        p.count[0] = moves;
        p.out_count[0] = used;
    }
}

template <bool FORK>
__global__ void __launch_bounds__(kScan) plan_kernel(PagePlan p) {
    if constexpr (FORK) fork_plan(p);
    else compact_plan(p);
}

// An entry of the new table.
template <bool FORK>
__device__ __forceinline__ void write_entry(const PagePlan& p, int64_t i) {
    const int row = (int)(i / p.entries), entry = (int)(i - (int64_t)row * p.entries);
    int id = -1;
    if constexpr (FORK) {
        const ForkRow r(p, row);
        const int copy = r.copies(p, row);
        const int wish = p.base[row] + (entry == r.full && copy ? 0 : copy + entry - r.held);
        if (entry < r.held && !(entry == r.full && copy)) id = r.page(p, entry);
        else if (entry < r.end) id = wish < p.count[1] ? p.ids[wish] : -1;
    } else {
        id = p.table[row * p.table_stride + entry];
        if ((unsigned)id >= (unsigned)p.pages) id = -1;
        else if (id >= p.out_count[0]) id = p.ids[p.place[id]];
    }
    p.out[i] = id;
}

constexpr int kSmallPages = 8192, kSmallCells = 4096;

template <bool FORK>
__global__ void __launch_bounds__(kScan) small_plan_kernel(PagePlan p) {
    __shared__ uint32_t used[kSmallPages / 32], full[FORK ? kSmallPages / 32 : 1];
    __shared__ int32_t ids[kSmallPages], other[kSmallPages];  // first or place
    p.used = used;
    p.full = full;
    (FORK ? p.first : p.place) = other;
    int32_t* const holes = p.ids;  // what the copies look up
    p.ids = ids;
    for (int i = threadIdx.x; i < p.pages; i += kScan) clear_marks(p, FORK, i);
    __syncthreads();
    const int cells = p.rows * p.entries;
    for (int i = threadIdx.x; i < cells; i += kScan) {
        if constexpr (FORK) fork_mark(p, i);
        else compact_mark(p, i);
    }
    __syncthreads();
    if constexpr (FORK) fork_plan(p);
    else compact_plan(p);
    __syncthreads();
    for (int i = threadIdx.x; i < cells; i += kScan) write_entry<FORK>(p, i);
    if constexpr (!FORK)
        for (int i = threadIdx.x; i < p.count[0]; i += kScan) holes[i] = ids[i];
}

struct PageCaches {
    unsigned char* at[kMostCaches];
    int64_t bytes[kMostCaches];  // of a page
};

// Blocks of y = the last write the table (small plans have), those of the others copy
// their cache's pages, 8 KB a block and step.  ONCE: more than the caches hold, past which
// the copies go (1024 pages of 557 KB, 1.14 GB read and written: 203 us, 5.6 TB/s; 239 us through the
// caches; 213 with 8192 blocks, 222 in steps of 16 KB).
template <bool FORK, bool ONCE>
__global__ void __launch_bounds__(256) move_pages_kernel(PagePlan p, PageCaches c, int caches) {
    if ((int)blockIdx.y == caches) {
        const int64_t n = (int64_t)p.rows * p.entries;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) write_entry<FORK>(p, i);
        return;
    }
    unsigned char* cache = c.at[blockIdx.y];
    const int64_t bytes = c.bytes[blockIdx.y];
    // parts of 8 KB
    const uint32_t steps = (uint32_t)((bytes + 8191) / 8192);
    const uint64_t all = (uint64_t)p.count[0] * steps;
    for (uint64_t i = blockIdx.x; i < all; i += gridDim.x) {
        const uint32_t k = (uint32_t)(i / steps), step = (uint32_t)(i - (uint64_t)k * steps);
        const int2 m = FORK ? p.moves[k] : make_int2(p.moves[k].x, p.ids[k]);
        const int64_t off = (int64_t)step * 8192 + threadIdx.x * 16;
        const unsigned char* src = cache + m.x * bytes + off;
        unsigned char* dst = cache + m.y * bytes + off;
        u32x4_t v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (off + u * 4096 < bytes) {
                const u32x4_t* x = reinterpret_cast<const u32x4_t*>(src + u * 4096);
                v[u] = ONCE ? __builtin_nontemporal_load(x) : *x;
            }
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (off + u * 4096 < bytes) {
                u32x4_t* x = reinterpret_cast<u32x4_t*>(dst + u * 4096);
                if constexpr (ONCE) __builtin_nontemporal_store(v[u], x);
                else *x = v[u];
            }
    }
}

// ---- host side -----------------------------------------------------------------

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool rows_ok(const void* x, const int64_t* s) {
    bool ok = x != nullptr && aligned16(x) && s != nullptr;
    for (int i = 0; ok && i < 3; ++i) ok = s[i] >= 0 && s[i] % 8 == 0;
    return ok;
}

// Fills the rows of a store or load; 0: nothing to do, -1: refused.
int64_t blocks_of(const spline_hip_fp4_cache* c, int64_t tokens, Fp4Rows& r) {
    if (!fp4_sizes_ok(c, tokens)) return -1;
    if (c->batch == 0 || tokens == 0) return 0;
    if (!fp4_pointers_ok(c)) return -1;
    const int64_t per = c->kv_heads * c->head_dim / 8;
    if (c->batch * tokens > 0x7fffff00ll / per) return -1;
    r.per = Divisor((uint32_t)per);
    r.tokens = Divisor((uint32_t)tokens);
    r.page = Divisor((uint32_t)c->page_size);
    r.threads = (uint32_t)(c->batch * tokens * per);
    return ceil_div(r.threads, 256);
}

template <bool BF>
int store(const spline_hip_fp4_cache* c, const void* k, const void* v, const int64_t* ks, const int64_t* vs,
          int64_t tokens, void* stream) {
    Fp4Rows r{};
    const int64_t blocks = blocks_of(c, tokens, r);
    if (blocks <= 0) return blocks < 0 ? hipErrorInvalidValue : hipSuccess;
    if (!rows_ok(k, ks) || !rows_ok(v, vs)) return hipErrorInvalidValue;
    r.k = static_cast<const uint16_t*>(k);
    r.v = static_cast<const uint16_t*>(v);
    r.ks = {ks[0], ks[2], ks[1]};
    r.vs = {vs[0], vs[2], vs[1]};
    const Fp4Pages p = fp4_pages(c);
    const dim3 grid((unsigned)blocks), block(256);
    if (c->head_dim == 128) hipLaunchKernelGGL((fp4_store_kernel<128, BF>), grid, block, 0, hs(stream), p, r);
    else hipLaunchKernelGGL((fp4_store_kernel<64, BF>), grid, block, 0, hs(stream), p, r);
    return hipGetLastError();
}

template <bool BF>
int load(const spline_hip_fp4_cache* c, void* k, void* v, int64_t tokens, void* stream) {
    Fp4Rows r{};
    const int64_t blocks = blocks_of(c, tokens, r);
    if (blocks <= 0) return blocks < 0 ? hipErrorInvalidValue : hipSuccess;
    if (!k || !v || !aligned16(k) || !aligned16(v)) return hipErrorInvalidValue;
    const Fp4Pages p = fp4_pages(c);
    const dim3 grid((unsigned)blocks), block(256);
    uint16_t *k16 = static_cast<uint16_t*>(k), *v16 = static_cast<uint16_t*>(v);
    if (c->head_dim == 128) hipLaunchKernelGGL((fp4_load_kernel<128, BF>), grid, block, 0, hs(stream), p, r, k16, v16);
    else hipLaunchKernelGGL((fp4_load_kernel<64, BF>), grid, block, 0, hs(stream), p, r, k16, v16);
    return hipGetLastError();
}

// The workspace's parts: bytes in all, or -1.
int64_t lay_out(const spline_hip_pages* a, bool fork, PagePlan& p, char* ws) {
    const int64_t limit = 1 << 24;  // rows, pages, entries
    if (!a || a->rows < 0 || a->rows > limit || a->old_rows < 0 || a->old_rows > limit || a->pages < 0 ||
        a->pages > 0x7fffffff - 32 || a->entries < 0 || a->entries > limit || a->num_caches < 0)
        return -1;
    if (fork ? a->page_size <= 0 || a->page_size > 65536 || a->entries > kFp4MostKeys / a->page_size || a->grow < 0 ||
                   a->grow > kFp4MostKeys / 2
             : a->rows != a->old_rows)
        return -1;
    // entries, and the pages that all rows may want, are counted in 32 bits
    if (a->rows * (a->entries + 2 + (fork ? ceil_div(a->grow, a->page_size) : 0)) > 0x7fffffff) return -1;
    int64_t bytes = 0;
    auto take = [&](int64_t n) {
        char* at = ws + bytes;
        bytes += ceil_div(n, 16) * 16;
        return at;
    };
    const int64_t words = ceil_div(a->pages, 32);
    p.used = reinterpret_cast<uint32_t*>(take(4 * words));
    if (fork) {
        p.full = reinterpret_cast<uint32_t*>(take(4 * words));
        p.first = reinterpret_cast<int32_t*>(take(4 * a->pages));
        p.base = reinterpret_cast<int32_t*>(take(4 * a->rows));
    } else {
        p.place = reinterpret_cast<int32_t*>(take(4 * a->pages));
    }
    p.ids = reinterpret_cast<int32_t*>(take(4 * a->pages));
    p.moves = reinterpret_cast<int2*>(take(8 * (fork ? a->rows : a->pages)));
    p.count = reinterpret_cast<int32_t*>(take(16));
    return bytes;
}

template <bool FORK>
void move(const spline_hip_pages* a, const PagePlan& p, hipStream_t st) {
    const dim3 block(256);
    const int64_t cells = ceil_div(a->rows * a->entries, 256);
    const bool small = a->pages <= kSmallPages && a->rows * a->entries <= kSmallCells;
    if (small) {
        hipLaunchKernelGGL((small_plan_kernel<FORK>), dim3(1), dim3(kScan), 0, st, p);
    } else {
        const int64_t marks = ceil_div(FORK ? a->pages : ceil_div(a->pages, 32), 256);
        if (marks > 0) hipLaunchKernelGGL((clear_marks_kernel<FORK>), dim3((unsigned)marks), block, 0, st, p);
        if (cells > 0) hipLaunchKernelGGL((mark_kernel<FORK>), dim3((unsigned)cells), block, 0, st, p);
        hipLaunchKernelGGL((plan_kernel<FORK>), dim3(1), dim3(kScan), 0, st, p);
    }
    // A page goes to one place.  A fork seldom copies as many pages as it has rows, and
    // blocks without one cost their launch.
    const int64_t most_moves = FORK ? (a->rows < a->pages ? a->rows : a->pages) : a->pages / 2;
    double bytes = 0;
    for (int64_t i = 0; i < a->num_caches; ++i) bytes += (double)a->cache_page_bytes[i] * most_moves;
    const bool once = bytes >= kMallBytes;
    int64_t at = 0;
    do {
        const int n = (int)(a->num_caches - at < kMostCaches ? a->num_caches - at : kMostCaches);
        const bool table = at == 0 && !small;
        PageCaches c{};
        int64_t steps = 0;
        for (int i = 0; i < n; ++i) {
            c.at[i] = static_cast<unsigned char*>(a->caches[at + i]);
            c.bytes[i] = a->cache_page_bytes[at + i];
            steps = c.bytes[i] > steps ? c.bytes[i] : steps;
        }
        steps = ceil_div(steps, 8192) * most_moves;
        int64_t x = ceil_div(FORK ? 8192 : 32768, n + 1);
        const int64_t need = table && cells > steps ? cells : steps;
        x = x < need ? x : need;
        if (x > 0 && n + table > 0) {
            const dim3 grid((unsigned)x, (unsigned)(n + table));
            if (once) hipLaunchKernelGGL((move_pages_kernel<FORK, true>), grid, block, 0, st, p, c, n);
            else hipLaunchKernelGGL((move_pages_kernel<FORK, false>), grid, block, 0, st, p, c, n);
        }
        at += n;
    } while (at < a->num_caches);
}

int rearrange(const spline_hip_pages* a, bool fork, void* stream) {
    PagePlan p{};
    if (lay_out(a, fork, p, static_cast<char*>(a ? a->workspace : nullptr)) < 0) return hipErrorInvalidValue;
    auto ints = [](const void* x) { return x != nullptr && ((uintptr_t)x & 3) == 0; };
    const bool any = a->rows > 0 && a->entries > 0, old = a->old_rows > 0 && a->entries > 0;
    if (!a->workspace || !aligned16(a->workspace) || !ints(a->out_count) || (any && !ints(a->out_table)) ||
        (old && (!ints(a->table) || a->table_stride < 0)))
        return hipErrorInvalidValue;
    if (fork && ((a->rows > 0 && !ints(a->out_lens)) || (a->old_rows > 0 && !ints(a->lens)) ||
                 (a->parents ? ((uintptr_t)a->parents & 3) != 0 : a->rows != 0 && a->rows != a->old_rows)))
        return hipErrorInvalidValue;
    if (a->num_caches > 0 && (!a->caches || !a->cache_page_bytes)) return hipErrorInvalidValue;
    for (int64_t i = 0; i < a->num_caches; ++i)
        if (a->cache_page_bytes[i] < 0 || a->cache_page_bytes[i] % 16 != 0 || a->cache_page_bytes[i] > (int64_t)1 << 40 ||
            (a->pages > 0 && a->cache_page_bytes[i] > 0 && (!a->caches[i] || !aligned16(a->caches[i]))))
            return hipErrorInvalidValue;
    p.table = a->table;
    p.lens = a->lens;
    p.parents = a->parents;
    p.table_stride = a->table_stride;
    p.out = a->out_table;
    p.out_lens = a->out_lens;
    p.out_count = a->out_count;
    p.rows = (int)a->rows;
    p.old_rows = (int)a->old_rows;
    p.entries = (int)a->entries;
    p.pages = (int)a->pages;
    p.page_size = (int)a->page_size;
    p.grow = (int)a->grow;
    fork ? move<true>(a, p, hs(stream)) : move<false>(a, p, hs(stream));
    return hipGetLastError();
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" int launch_paged_fp4_store_bf16(const spline_hip_fp4_cache* cache, const void* k, const void* v,
                                           const int64_t* k_strides, const int64_t* v_strides, int64_t tokens,
                                           void* stream) {
    return store<true>(cache, k, v, k_strides, v_strides, tokens, stream);
}
extern "C" int launch_paged_fp4_store_fp16(const spline_hip_fp4_cache* cache, const void* k, const void* v,
                                           const int64_t* k_strides, const int64_t* v_strides, int64_t tokens,
                                           void* stream) {
    return store<false>(cache, k, v, k_strides, v_strides, tokens, stream);
}
extern "C" int launch_paged_fp4_load_bf16(const spline_hip_fp4_cache* cache, void* k, void* v, int64_t tokens,
                                          void* stream) {
    return load<true>(cache, k, v, tokens, stream);
}
extern "C" int launch_paged_fp4_load_fp16(const spline_hip_fp4_cache* cache, void* k, void* v, int64_t tokens,
                                          void* stream) {
    return load<false>(cache, k, v, tokens, stream);
}
extern "C" int64_t spline_hip_fork_pages_workspace_bytes(const spline_hip_pages* args) {
    PagePlan p{};
    return lay_out(args, true, p, nullptr);
}
extern "C" int64_t spline_hip_compact_pages_workspace_bytes(const spline_hip_pages* args) {
    PagePlan p{};
    return lay_out(args, false, p, nullptr);
}
extern "C" int launch_fork_pages(const spline_hip_pages* args, void* stream) { return rearrange(args, true, stream); }
extern "C" int launch_compact_pages(const spline_hip_pages* args, void* stream) {
    return rearrange(args, false, stream);
}
