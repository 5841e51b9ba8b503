// Layout of the 4-bit paged cache.
//
// A pool holds pages of 64 tokens; a page has a part for every KV head, a part four blocks of 16 tokens, and a block both
// sides of its tokens:
//
//     keys:   codes [16 tokens][64 bytes], parameters [16 tokens][8 bytes]
//     values: the same
//
// so that whatever runs along the tokens of a head is contiguous (9216 bytes per page, 2304 per block, multiples of 16: one
// bulk copy).  A token's parameters are scale of coordinates 0..63, scale of 64..127, offset of either, in the type of the
// model; a code is 4 bits, eight of them in a word, coordinate i of the eight at bit 4 i.  Where a token's sixteen words lie
// follows from how the attention kernel's lanes read them:
//   * keys: word c (coordinates 8c..8c+7) at byte 16 (c % 4) + 4 (c / 4): lane t of a quad takes 16 bytes, words t, t + 4,
//     t + 8, t + 12, two of either group;
//   * values: word c at byte 8 (c % 8) + 4 (c / 8), i.e. eight coordinates of one group beside the same eight of the other; in
//     rows 2, 3, 6, 7, 10, 11, 14, 15 of a block the two halves of the 64 bytes are exchanged, which puts the rows that are read
//     together on different banks.
#pragma once

#include "pairs.cuh"

namespace reskv {

constexpr int kPageTokens = 64;
constexpr int kBlockTokens = 16;
constexpr int kBlockCodes = kBlockTokens * 64, kBlockParams = kBlockTokens * 8;
constexpr int kBlockSide = kBlockCodes + kBlockParams;
constexpr int kBlockBytes = 2 * kBlockSide;                                     // 2304
constexpr int kPageHeadBytes = kPageTokens / kBlockTokens * kBlockBytes;        // 9216
constexpr int kPagedGroup = 8;                                                  // most query heads per KV head

// Byte of word c (0..15) of the token in row `row` of a block's codes.
__host__ __device__ __forceinline__ int key_word(int row, int c) { return row * 64 + 16 * (c & 3) + 4 * (c >> 2); }
__host__ __device__ __forceinline__ int value_word(int row, int c) {
    return row * 64 + 8 * ((c & 7) ^ ((row >> 1 & 1) << 2)) + 4 * (c >> 3);
}

// Where the tokens of a step lie: token i of the packed tensors belongs to the sequence s with cu[s] <= i < cu[s + 1] and is
// number starts[s] + i - cu[s] of it; its page is table[s, number / 64].
struct PagedPlace {
    const int *cu, *starts, *table;
    int sequences, width, pages;
};

}  // namespace reskv
