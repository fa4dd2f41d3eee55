// The paged 4-bit KV cache: format and addressing, shared by the kernels that write and read it.
//
// Values are symmetric INT4 with one binary16 scale per (token, KV head, group of gs dimensions):
//   s = fp16(max|x| / 7), q = clamp(round_half_even(x / s), -7, 7), value q s.
// A group that holds a value that is not finite gets that scale (infinity or NaN) with codes 0 and so reads back as
// NaN. A page holds `page` tokens (a power of two from 16 up) of every KV head; sequence b's token t is in slot
// t % page of page block_table[b, t / page].
//   k_pages [P, NKV, page, hd / 2]   a token's hd / 8 words; word W g + i (W = hd / 32, g < 4) holds dimensions
//                                    8 (4 i + g) .. + 7 in AWQ nibble order. A lane that reads W consecutive words
//                                    from word W g has, for every i, the k slots (g, 0 .. 7) of an MFMA over dimensions
//                                    32 i .. 32 i + 31, and such an MFMA lies inside one quantization group.
//   v_pages [P, NKV, page, hd / 2]   16-bit units [page / 4][16][hd / 64][4 tokens]; nibble n of unit (m, u) is
//                                    dimension 64 u + 16 n + m. One lane's load holds four tokens of the same
//                                    dimensions, paired in 32-bit words as the MFMA's k slots want them, and the 16
//                                    lanes m of one nibble are 16 consecutive dimensions: inside one group again.
//   k_scale, v_scale [P, NKV, hd / gs, page]
#pragma once

#include "soi_device.h"
#include "soi_host.h"

namespace soi {

struct Kv4Cache {
    uint8_t* k_pages;
    uint16_t* k_scale;
    uint8_t* v_pages;
    uint16_t* v_scale;
    const int32_t* table;  // [B, max_blocks]
    const int32_t* lens;   // [B]: tokens of each sequence, the new ones of an append included
    int B, max_blocks, P, NKV, page, page_shift;
};

// The page that holds position pos of sequence b, or -1: a position outside the table, or an entry that names no page.
__device__ __forceinline__ int kv4_page(const Kv4Cache& c, int b, int pos) {
    const int blk = pos >> c.page_shift;
    if (pos < 0 || blk >= c.max_blocks) return -1;
    const int id = ldg(c.table + static_cast<int64_t>(b) * c.max_blocks + blk);
    return id >= 0 && id < c.P ? id : -1;
}

// host: the argument checks that every call over a cache shares, and its device form
int kv4_check(const soi_kv4_cache* c, const char* what);
Kv4Cache kv4_device(const soi_kv4_cache* c);

}  // namespace soi

// X(hd, gs) for the head_dim `hd` and group_size `gs` that kv4_check has passed
#define SOI_KV4_SHAPES(X)                                                                    \
    if (hd == 64 && gs == 32) X(64, 32);                                                     \
    else if (hd == 64) X(64, 64);                                                            \
    else if (hd == 128 && gs == 32) X(128, 32);                                              \
    else if (hd == 128 && gs == 64) X(128, 64);                                              \
    else if (hd == 128) X(128, 128);                                                         \
    else if (gs == 32) X(256, 32);                                                           \
    else if (gs == 64) X(256, 64);                                                           \
    else X(256, 128)
