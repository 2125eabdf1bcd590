// fp4.hpp -- the pages of a 4-bit cache: E2M1 numbers in blocks of 32 that share a
// power of two.
//
// A page holds, for keys (0) and values (1) and each KV head, page_size rows of
// codes, two to a byte with the even element in the low half, and behind them
// page_size rows of HD / 32 exponents: byte e of a block stands for 2^(e - 127),
// bytes above 252 for NaN in the whole block.  A key and its value take 17 / 16
// bytes an element pair.  Code c stands for {0, 1/2, 1, 3/2, 2, 3, 4, 6}[c & 7],
// negative with bit 3.  Products of a code and its block's power of two have three
// significant bits, so that BF16 holds them exactly: v_cvt_scalef32_pk_bf16_fp4
// makes two of them (all codes and exponents were compared on MI355X).
#pragma once

#include <hip/hip_runtime.h>

#include "flash_attn.hpp"
#include "spline_ops_hip.h"

namespace pt {

constexpr int kFp4Block = 32;
constexpr int kFp4Least = 27, kFp4Most = 252;  // exponents that are stored: 2^-100 to 2^125
constexpr int kFp4Group = 16;                  // page sizes are multiples of it

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// The power of two of a block's byte, as an FP32 factor: Inf, which the conversions
// answer with NaN, above kFp4Most.
__device__ __forceinline__ float fp4_scale(uint32_t byte) {
    return as_f32((byte > (uint32_t)kFp4Most ? 255u : byte) << 23);
}

// Elements 0..7 of a word of codes.
__device__ __forceinline__ bf16x8_t fp4_to_bf16(uint32_t codes, float scale) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return (bf16x8_t){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Where a cache's bytes lie.
struct Fp4Pages {
    uint8_t* cache;
    const int32_t* table;
    const int32_t* lens;
    int64_t table_stride;
    int64_t page_bytes, head_bytes;  // of a page; of a head's keys or values in it
    int pages, page_size, entries, hkv;

    // The page of an entry of a sequence's table, or -1.
    __device__ __forceinline__ int page_of(int64_t b, int entry) const {
        if ((unsigned)entry >= (unsigned)entries) return -1;
        const int page = table[b * table_stride + entry];
        return (unsigned)page < (unsigned)pages ? page : -1;
    }
    __device__ __forceinline__ const uint8_t* head(int page, int kv, int h) const {
        return cache + page * page_bytes + (kv * hkv + h) * head_bytes;
    }
    // Valid keys of a sequence (the table's end may cut them off).
    __device__ __forceinline__ int len(int64_t b) const {
        const int n = lens[b];
        return n < 0 ? 0 : n;
    }
};

// ---- host side -----------------------------------------------------------------

constexpr int64_t kFp4MostKeys = 1 << 30;    // of a sequence's table: positions are 32-bit
constexpr int64_t kFp4LooseTokens = 1 << 14;   // more have to fit the table

inline bool fp4_sizes_ok(const spline_hip_fp4_cache* c, int64_t tokens) {
    return c && c->batch >= 0 && c->batch <= 0x7fffffff && c->kv_heads > 0 && c->kv_heads <= 65536 &&
           (c->head_dim == 64 || c->head_dim == 128) && c->page_size > 0 && c->page_size % kFp4Group == 0 &&
           c->page_size <= 65536 && c->pages >= 0 && c->pages <= 0x7fffffff && c->entries >= 0 &&
           c->entries <= kFp4MostKeys / c->page_size && tokens >= 0 &&
           (tokens <= kFp4LooseTokens || tokens <= c->entries * c->page_size);
}

inline bool fp4_pointers_ok(const spline_hip_fp4_cache* c) {
    return (c->pages == 0 || (c->cache && aligned16(c->cache))) &&
           (c->entries == 0 || (c->table && ((uintptr_t)c->table & 3) == 0 && c->table_stride >= 0)) && c->lens &&
           ((uintptr_t)c->lens & 3) == 0;
}

inline Fp4Pages fp4_pages(const spline_hip_fp4_cache* c) {
    Fp4Pages p{};
    p.cache = static_cast<uint8_t*>(c->cache);
    p.table = c->table;
    p.lens = c->lens;
    p.table_stride = c->table_stride;
    p.head_bytes = c->page_size * (c->head_dim / 2 + c->head_dim / kFp4Block);
    p.page_bytes = 2 * c->kv_heads * p.head_bytes;
    p.pages = (int)c->pages;
    p.page_size = (int)c->page_size;
    p.entries = (int)c->entries;
    p.hkv = (int)c->kv_heads;
    return p;
}

}  // namespace pt
