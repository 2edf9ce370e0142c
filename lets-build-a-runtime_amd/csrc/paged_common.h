// paged_common.h — the paged key/value cache as its kernels see it.
//
// A page of the cache holds, for each K/V head in turn, the K rows [page][hdp], the V rows
// in groups of eight positions [page/8][hdp][8], and a float scale for each K row and each V
// row (hdp: head_dim rounded up to 16).  A stored value stands for itself times its row's
// scale; a row with an infinity or a NaN is stored as zeros with a NaN scale.
#pragma once

#include "lbr_device.h"

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// Element types (OpNode.extra[3]).
#define LBR_CACHE_F32 0
#define LBR_CACHE_F16 1
#define LBR_CACHE_I8 2
#define LBR_CACHE_E4M3 3

constexpr int cache_elem(int type) { return type == LBR_CACHE_F32 ? 4 : type == LBR_CACHE_F16 ? 2 : 1; }

struct PagedCache {
    char* base;
    const int* table;         // [B][wide]
    const int* start;         // [B]
    const int* count;         // [B]
    long long page_bytes;     // all heads
    int head_bytes;           // one head of a page
    int part;                 // bytes of the K rows of a head, and of the V rows
    int heads, hd, hdp;
    int shift;                // log2 of the positions of a page
    int pages, wide;          // pages of the cache, of a table row
};

// First byte of head h in the page that holds position pos of sequence b; null where the table does
// not reach or names no page of the cache.
__device__ __forceinline__ char* cache_head(const PagedCache& c, int b, int h, long long pos) {
    const long long at = pos >> c.shift;
    if (pos < 0 || at >= c.wide) return nullptr;
    const int page = c.table[(long long)b * c.wide + at];
    if (page < 0 || page >= c.pages) return nullptr;
    return c.base + page * c.page_bytes + (long long)h * c.head_bytes;
}

// Max over the aligned groups of G lanes that hold a row.
template <int G>
__device__ __forceinline__ unsigned row_max_bits(unsigned v) {
    static_assert(G == 8 || G == 16 || G == 32 || G == 64, "lanes of a row");
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));
    if (G >= 16) v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));
    if (G >= 32) {
        auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max((unsigned)a[0], (unsigned)a[1]);
    }
    if (G == 64) {
        auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max((unsigned)a[0], (unsigned)a[1]);
    }
    return v;
}

// Fields of Step for the cache ops: in[0] = cache, in[1] = table, in[2] = start, in[3] = count, in[4]
// = K or Q, in[5] = V; i[0] = type, i[1] = B, i[2] = heads, i[3] = head_dim, i[4] = log2 page_size,
// i[5] = pages, i[6] = pages of a table row, i[7] = S or T, i[8] = query heads, i[9] = 16-byte rows;
// f[0] = score scale.
inline PagedCache paged_cache(const Step& s) {
    PagedCache c;
    c.base = (char*)s.in[0];
    c.table = (const int*)s.in[1];
    c.start = (const int*)s.in[2];
    c.count = (const int*)s.in[3];
    c.heads = (int)s.i[2];
    c.hd = (int)s.i[3];
    c.hdp = (c.hd + 15) / 16 * 16;
    c.shift = (int)s.i[4];
    c.part = (1 << c.shift) * c.hdp * cache_elem((int)s.i[0]);
    c.head_bytes = 2 * c.part + 8 * (1 << c.shift);
    c.page_bytes = (long long)c.heads * c.head_bytes;
    c.pages = (int)s.i[5];
    c.wide = (int)s.i[6];
    return c;
}

// Checks what all cache ops have in common and fills the Step's fields above except in[4], in[5],
// i[7..9]; `first` is the index of the table among the node's inputs.
int decode_paged_common(const OpNode* n, Step* s, int cache, int first, long long B);
