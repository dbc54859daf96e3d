// The 4-bit key / value cache: its layout in memory, what a call says about it, and how kernels walk it.
//
// A group is 32 neighbouring values of a head vector: a scale d and 32 codes c of 4 bits stand for d (c - 8).  d is an fp16
// number of at most 8 significant bits and |d| <= 8160, c - 8 has at most 3: every value that the cache can hold is an fp16
// number, normal or not, so that keys and values are exact operands of the fp16 matrix instructions.
//
// A tile is 32 tokens of one key head, 36 D bytes in one piece, in the order in which a wavefront wants it as operands of
// v_mfma_f32_16x16x32_f16 (lane (r = lane % 16, j = lane / 16) holds 8 values of the contraction of operand row r):
//     key codes    dwords [w / 4][lane][w % 4], w = u G + g (G = D / 32 groups): token 8 (r / 4) + 4 u + r % 4, values 32 g + 8 j + e
//     value codes  dwords [w / 4][lane][w % 4]: value 16 w + r, tokens 8 j + e
//     key scales   [token][g], value scales [g][token]
// Element e = 0 .. 7 of a dword lies in nibble e / 2 + 4 (e % 2): masking the dword (shifted by 0, 4, 8, 12) leaves the pairs
// (0, 1), (2, 3), ... in its two halves.  With these token orders the scores that a lane gets out of the two key operands
// (u = 0, 1) of a tile are those of the tokens 8 j .. 8 j + 7 for query r: its share of the second product's operand, in place.
#pragma once

#include "common.hpp"

namespace gq {

namespace {

constexpr int kTileTokens = 32;

// Byte offsets in a tile of head vectors of D values.
template <int D> struct KvTile {
    static constexpr int G = D / 32;
    static constexpr int kKeys = 0, kValues = 16 * D, kKeyScales = 32 * D, kValueScales = 34 * D, kBytes = 36 * D;
    // dword w of a lane, of key or value codes
    __host__ __device__ static constexpr int code(int w, int lane) { return ((w >> 2) * 64 + lane) * 16 + (w & 3) * 4; }
};

// row of the key operand that token t of a tile is: lane r of operand u
__device__ __forceinline__ int key_row(int t) { return (t >> 3) * 4 + (t & 3); }
__device__ __forceinline__ int key_half(int t) { return (t >> 2) & 1; }

// What sequence b of a call has: tokens 0 .. length - 1 that its pages have room for, and `news` rows from `row0` on, of which row n is token first + n
// (a negative one, or one from `length` on, is absent).
struct KvSeq { int length, news, row0, first; };

// The lanes' values up to and with each, combined by f, by data-parallel moves: 1, 2, 4, 8 lanes within rows of sixteen, then from the last lane
// of a row into the next one, and of the first half into the second.  `none` combines to nothing.
template <class F> __device__ __forceinline__ int lane_scan(int v, int none, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xA, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xC, 0xF, false));
    return v;
}
__device__ __forceinline__ int lane_scan(int v) {
    return lane_scan(v, 0, [](int a, int b) { return a + b; });
}

// A load that is the same for the whole wavefront, through the scalar cache (of what no kernel of this launch writes).
__device__ __forceinline__ int32_t uniform_load(const int32_t *p) { return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p; }

// Tokens beyond the page table and rows beyond the call's are left out, so that no device value leads a kernel out of its buffers.  The places of
// the others go by the length and the starts as they are.
__device__ __forceinline__ KvSeq kv_seq(const KvCall &kv, int b) {
    KvSeq s;
    const int64_t room = (int64_t)kv.max_pages * kv.page_tokens;
    int length = kv.lengths[b];
    length = length < 0 ? 0 : length;
    s.length = length > room ? (int)room : length;
    int from = b, to = b + 1;
    if (kv.starts) { from = kv.starts[b]; to = kv.starts[b + 1]; }
    from = from < 0 ? 0 : from > kv.rows ? kv.rows : from;
    to = to < from ? from : to;
    const int first = length - (to - from);
    to = to > kv.rows ? kv.rows : to;
    s.row0 = from;
    s.news = to - from > kv.max_new ? kv.max_new : to - from;
    s.first = first < -s.news ? -s.news : first;  // (every place is in front of the sequence either way)
    return s;
}

__device__ __forceinline__ KvSeq seq_of_lane(const KvSeq &s, int lane) {
    return KvSeq{__builtin_amdgcn_readlane(s.length, lane), __builtin_amdgcn_readlane(s.news, lane), __builtin_amdgcn_readlane(s.row0, lane),
                 __builtin_amdgcn_readlane(s.first, lane)};
}

// the place in the page table of a sequence's tile
__device__ __forceinline__ int page_slot(const KvCall &kv, int tile) {
    return kv.page_magic ? (int)__umulhi((uint32_t)tile, kv.page_magic) : tile / (kv.page_tokens >> 5);
}

// Tile `tile` of sequence b and key head h; null where the page table names no page of the cache.
__device__ __forceinline__ uint8_t *kv_tile(const KvCall &kv, int b, int h, int tile, int tile_bytes) {
    const int per_page = kv.page_tokens >> 5;
    const int slot = page_slot(kv, tile);
    const int page = kv.table[b * kv.table_stride + slot];
    if ((uint32_t)page >= (uint32_t)kv.pages) return nullptr;
    return kv.cache + (((int64_t)page * kv.kv_heads + h) * per_page + (tile - slot * per_page)) * tile_bytes;
}

// The account of token p of sequence b and key head h; null as above.
__device__ __forceinline__ float *kv_account(const KvCall &kv, float *accounts, int b, int h, int p) {
    const int slot = page_slot(kv, p >> 5);
    const int page = kv.table[b * kv.table_stride + slot];
    if ((uint32_t)page >= (uint32_t)kv.pages) return nullptr;
    return accounts + ((int64_t)page * kv.kv_heads + h) * kv.page_tokens + (p - slot * kv.page_tokens);
}

}  // namespace

}  // namespace gq
