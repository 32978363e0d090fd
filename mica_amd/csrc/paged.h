// The paged key/value cache of csrc/kv_cache.hip and csrc/attn_paged.hip, head dim 256.
//
// A sequence's tokens lie in blocks of 32.  A finished block is a page: int8 keys and values, x = scale q, with one fp32 scale
// for each head and side.  The block that a sequence has not filled yet (its rest) stays in bf16, in a place of its own, and is
// quantized as a whole when its last token comes: every value is rounded once, and what the cache holds depends on the tokens
// alone, not on the calls that brought them.
//
//   data   int8 [pages][2][HK][8192]      side 0: keys, [8 groups of 32 dims][32 tokens][32 dims]
//                                         side 1: values, [256 dims][32 tokens in fours, in the order 0 4 2 6 1 5 3 7]
//   scales fp32 [pages][2][HK]
//   recent bf16 [slots][2][HK][32][256]   the rest of the sequence in a slot, rows as they come
//
// Both sides are in the order in which the matrix cores' operands take them: 16 bytes a lane, 1 KB a wave, one behind the
// other (a lane's score rows are tokens 4 (0 .. 7 in bit-reversed order) apart, hence the order of the fours).
#pragma once

#include "ragged.h"

constexpr int kPage = 32;              // tokens of a block
constexpr int kPagedDim = 256;         // head dim
constexpr int kPageBytes = kPage * kPagedDim;

struct Pages {
    int8_t *data;
    float *scales;
    uint16_t *recent;
    const int *table; // [B][width], rows ldt apart: the page of each finished block
    long long ldt;
    const int *lens;  // [B]
    const int *slots; // [B] or null: b
    int width, pages, n_slots, HK;

    // a sequence's tokens, never more than its row of the table and a rest hold
    MICA_DEVICE int len(int b) const { return min(max(lens[b], 0), width * kPage + kPage - 1); }
    // the page of block `block`, -1 where there is none
    MICA_DEVICE int page(int b, int block) const {
        if (block < 0 || block >= width) return -1;
        const int id = table[b * ldt + block];
        return id >= 0 && id < pages ? id : -1;
    }
    MICA_DEVICE int slot(int b) const {
        const int s = slots ? slots[b] : b;
        return s >= 0 && s < n_slots ? s : -1;
    }
    MICA_DEVICE long long index(int page, int side, int hk) const { return ((long long)page * 2 + side) * HK + hk; }
    MICA_DEVICE int8_t *block(int page, int side, int hk) const { return data + index(page, side, hk) * kPageBytes; }
    // the scale of a block; NaN without a page, and for one that is not finite
    MICA_DEVICE float scale(int page, int side, int hk) const {
        const float s = page >= 0 ? scales[index(page, side, hk)] : __builtin_nanf("");
        return __builtin_fabsf(s) < __builtin_inff() ? s : __builtin_nanf("");
    }
    MICA_DEVICE uint16_t *rest(int slot, int side, int hk) const {
        return recent + index(slot, side, hk) * (kPage * kPagedDim);
    }
};

// where the four tokens 4 i .. 4 i + 3 lie in a value page's row: i's three bits reversed
MICA_DEVICE constexpr int page_four(int i) { return ((i & 1) << 2) | (i & 2) | (i >> 2); }

// The cache's own arguments; 0 when they hold.
static inline int mica_paged_check(Pages &c, void *data, void *scales, void *recent, int pages, int n_slots, int HK, int head_dim,
                                   const int *table, long long ldt, int width, const int *lens, const int *slots, int B) {
    if (head_dim != kPagedDim || HK <= 0 || HK > (1 << 16) || pages < 0 || n_slots < 0 || width < 0 ||
        width > (1 << 24))
        return MICA_MISS_SHAPE;
    if (B > 0 && (!lens || !recent || (pages > 0 && (!data || !scales)) || (width > 0 && !table))) return MICA_MISS_ARG;
    if (B > 1 && ldt < width) return MICA_MISS_STRIDE;
    if (!mica_aligned16(data) || !mica_aligned16(recent) || ((uintptr_t)scales & 3) || ((uintptr_t)table & 3) ||
        ((uintptr_t)lens & 3) || ((uintptr_t)slots & 3))
        return MICA_MISS_ALIGN;
    c.data = (int8_t *)data; c.scales = (float *)scales; c.recent = (uint16_t *)recent;
    c.table = table; c.ldt = B > 1 ? ldt : width; c.width = width; c.lens = lens; c.slots = slots;
    c.pages = pages; c.n_slots = n_slots; c.HK = HK;
    return 0;
}
