// What the kernels of attention over a 4-bit cache share: queries, keys and values as operands of the matrix instructions, a row's reference of
// its exponents, the way from a page table to tiles in LDS.
#pragma once

#include "kv.hpp"
#include "lds_dma.hpp"

namespace gq {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_huge_valf();
// A row's largest weight when its reference is set, and what it stays under, as powers of two.  (fp32: little room to spare, for the sake of the smallest weights; a
// reference that moves more often costs 1 % up to D = 128.  At D = 256, where results have to leave the accumulation registers for it, 64 rows of 5 sequences over
// 4000 to 16000 tokens take 105 108 112 123 us with 2^6 2^9 2^10 2^12.)
template <int D, bool TWO> struct Weights { static constexpr float kSet = !TWO ? 6.0f : D == 256 ? 9.0f : 12.0f, kMost = TWO ? 15.5f : 14.0f; };
// Whether a score asks for a new reference: by their difference, for a sum with the reference is rounded where scores are large.
template <int D, bool TWO> __device__ __forceinline__ bool passes(float score, float ref) { return score - ref > Weights<D, TWO>::kMost; }
// The reference that a row's largest score asks for.  (From scores of 2^26 on the difference can round to more than there is room for.)
template <int D, bool TWO> __device__ __forceinline__ float reference(float most) {
    const float set = most - Weights<D, TWO>::kSet;
    return passes<D, TWO>(most, set) ? most : set;
}
// With many rows a weight comes from a score's exact product with the scale, less a reference that is a rounded one: one instruction, and from references of
// this size on an error of a 2^-8 th and more of a factor of 2 (at 2^27, of more than fp16 numbers have room for).  There the product is rounded as the reference was.
// (bfloat16 alone: float32 queries take all of the scale but a power of two, by which products are exact.)
constexpr float kCoarse = 65536.0f;

__device__ __forceinline__ h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ h2 both(float v) { h2 r = {(_Float16)v, (_Float16)v}; return r; }
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) { h8 r = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; return r; }

// Eight codes -> c - 8, exact: the nibbles become the low mantissa bits of 1024 (or, four places up, of 1024 + 16 c).  The constants
// are kept out of the compiler's sight in registers, for an instruction that masks and sets in one takes no literals.
struct Unpack {
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, base = 0x64006400u;
    __device__ __forceinline__ Unpack() { asm("" : "+s"(low), "+s"(high), "+v"(base)); }
    __device__ __forceinline__ void operator()(uint32_t w, h2 (&v)[4]) const {
        const h2 sixteenth = both(0.0625f), less = both(-1032.0f), less16 = both(-72.0f);
        const uint32_t x = w >> 8;
        v[0] = as_h2((w & low) | base) + less;
        v[1] = __builtin_elementwise_fma(as_h2((w & high) | base), sixteenth, less16);
        v[2] = as_h2((x & low) | base) + less;
        v[3] = __builtin_elementwise_fma(as_h2((x & high) | base), sixteenth, less16);
    }
};

// ROWS (16 or 32) query rows as operands of the matrix instructions of that size: lane (r, j), r = lane % ROWS, gets the values
// 8 (64 / ROWS) g + 8 j + 0..7 of row r for g = 0, 1, ..., times 2^e with the largest of the row in [2^11, 2^12), and the sign of the scale, so that what is left to multiply scores by, to_log2, is
// not negative.  TWO: a second operand with what the first has rounded off; both with the scale's mantissa (1/2 to 1; a rounding in 24 bits), so that to_log2 is a power of two.
template <int D, int ROWS, bool BF16, bool TWO>
__device__ __forceinline__ void load_queries(const HeadRows &q, int64_t at, bool live, int wide, float scale_log2, h8 (&hi)[D * ROWS / 512], h8 (&lo)[TWO ? D * ROWS / 512 : 1], float &to_log2) {
    constexpr int N = D * ROWS / 512;
    const int j = ((int)threadIdx.x & 63) / ROWS;
    float x[N][8];
    float most = 0.0f;
#pragma unroll
    for (int g = 0; g < N; g++) {
        const int64_t p = at + 512 / ROWS * g + 8 * j;
        if (!live) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[g][e] = 0.0f;
        } else if constexpr (BF16) {
            const uint16_t *u = static_cast<const uint16_t *>(q.p) + p;
            u4 w;
            if (wide) w = *reinterpret_cast<const u4 *>(u);
            else w = u4{u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[g][2 * e] = __uint_as_float(w[e] << 16);
                x[g][2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
            }
        } else {
            const float *u = static_cast<const float *>(q.p) + p;
            if (wide) {
                const f4 a = *reinterpret_cast<const f4 *>(u), b = *reinterpret_cast<const f4 *>(u + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) { x[g][e] = a[e]; x[g][4 + e] = b[e]; }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[g][e] = u[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(x[g][e]));
    }
#pragma unroll
    for (int m = ROWS; m < 64; m <<= 1) most = fmaxf(most, __shfl_xor(most, m));
    int e = 0;
    if (most > 0.0f && most < __builtin_huge_valf()) e = 12 - __builtin_amdgcn_frexp_expf(most);
    e = e > 100 ? 100 : e;  // (below 2^-88 the scores of a row are nothing)
    const float up = TWO ? ldexpf(__builtin_amdgcn_frexp_mantf(scale_log2), e) : copysignf(ldexpf(1.0f, e), scale_log2);
    to_log2 = TWO ? ldexpf(1.0f, __builtin_amdgcn_frexp_expf(scale_log2) - e) : ldexpf(1.0f, -e) * fabsf(scale_log2);
#pragma unroll
    for (int g = 0; g < N; g++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float v = x[g][i] * up;
            if constexpr (TWO) asm("" : "+v"(v));  // (or the first operand may be made of the product before its rounding, and what is left of it after)
            const _Float16 a = (_Float16)v;
            hi[g][i] = a;
            if constexpr (TWO) lo[g][i] = (_Float16)(v - (float)a);
        }
    }
}

// One tile of the cache in registers, as loaded.
template <int D> struct KeyWords {
    u4 code[D / 64], scale[2];  // (scale: the first D / 64 dwords of each)
    __device__ __forceinline__ void load(const uint8_t *tile) {
        const int lane = (int)threadIdx.x & 63, r = lane & 15;
#pragma unroll
        for (int c = 0; c < D / 64; c++) code[c] = *reinterpret_cast<const u4 *>(tile + KvTile<D>::kKeys + (c * 64 + lane) * 16);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint8_t *p = tile + KvTile<D>::kKeyScales + (8 * (r >> 2) + 4 * u + (r & 3)) * (D / 16);
            if constexpr (D == 64) {
                scale[u].x = *reinterpret_cast<const uint32_t *>(p);
            } else if constexpr (D == 128) {
                const u2 v = *reinterpret_cast<const u2 *>(p);
                scale[u].x = v.x;
                scale[u].y = v.y;
            } else {
                scale[u] = *reinterpret_cast<const u4 *>(p);
            }
        }
    }
    // operand of the sixteen tokens u for group g
    __device__ __forceinline__ h8 operand(const Unpack &unpack, int u, int g) const {
        const int w = u * (D / 32) + g;
        h2 v[4];
        unpack(code[w >> 2][w & 3], v);
        const h2 pair = as_h2(scale[u][g >> 1]);
        const _Float16 one = (g & 1) ? pair.y : pair.x;
        const h2 d = {one, one};
        return join(v[0] * d, v[1] * d, v[2] * d, v[3] * d);
    }
};
template <int D> struct ValueWords {
    u4 code[D / 64], scale[D / 32];
    __device__ __forceinline__ void load(const uint8_t *tile) {
        const int lane = (int)threadIdx.x & 63, j = lane >> 4;
#pragma unroll
        for (int c = 0; c < D / 64; c++) code[c] = *reinterpret_cast<const u4 *>(tile + KvTile<D>::kValues + (c * 64 + lane) * 16);
#pragma unroll
        for (int g = 0; g < D / 32; g++) scale[g] = *reinterpret_cast<const u4 *>(tile + KvTile<D>::kValueScales + g * 64 + j * 16);
    }
    // operand of the sixteen values 16 w ..
    __device__ __forceinline__ h8 operand(const Unpack &unpack, int w) const {
        h2 v[4];
        unpack(code[w >> 2][w & 3], v);
        const u4 d = scale[w >> 1];
        return join(v[0] * as_h2(d[0]), v[1] * as_h2(d[1]), v[2] * as_h2(d[2]), v[3] * as_h2(d[3]));
    }
};

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The scores of a tile's 32 tokens for sixteen rows: lane (r, j) gets those of the tokens 8 j + 0..7 for row r.
template <int D, bool TWO>
__device__ __forceinline__ void tile_scores(const Unpack &unpack, const KeyWords<D> &k, const h8 (&hi)[D / 32], const h8 (&lo)[TWO ? D / 32 : 1], float (&s)[8]) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < D / 32; g++) {
            const h8 a = k.operand(unpack, u, g);
            acc = mfma(a, hi[g], acc);
            if constexpr (TWO) acc = mfma(a, lo[g], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[4 * u + i] = acc[i];
    }
}

constexpr int kSplitWaves = 4;

// The addresses of every STEP-th tile of a sequence and key head from `tile` to `end`; the page of the next one is asked for a call ahead.
template <int BYTES, int STEP> struct TileWalk {
    const KvCall &kv;
    const int32_t *table;
    int head, per_page, slot, in, left, page;
    __device__ __forceinline__ TileWalk(const KvCall &call, int b, int h, int tile, int end)
        : kv(call), table(call.table + b * call.table_stride), head(h), per_page(call.page_tokens >> 5) {
        start(tile, end);
    }
    __device__ __forceinline__ void start(int tile, int end) {
        left = tile < end ? (end - tile + STEP - 1) / STEP : 0;
        page = -1;
        slot = page_slot(kv, tile);
        in = tile - slot * per_page;
        if (left) page = uniform_load(table + slot);
    }
    // null behind the last one, and where the page is none of the cache's
    __device__ __forceinline__ const uint8_t *next() {
        if (left == 0) return nullptr;
        const uint8_t *at = (uint32_t)page < (uint32_t)kv.pages ? kv.cache + (((int64_t)page * kv.kv_heads + head) * per_page + in) * BYTES : nullptr;
        left--;
        in += STEP;
        while (in >= per_page) { in -= per_page; slot++; }
        if (left) page = uniform_load(table + slot);
        return at;
    }
};

template <bool BF16> __device__ __forceinline__ void store_result(void *out, int64_t at, f4 sum, float all) {
    sum *= all == 0.0f ? 0.0f : 1.0f / all;  // (a row that has seen nothing)
    if (all != all) sum = f4{all, all, all, all};
    if constexpr (BF16) {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        const bf16x4 y = {(__bf16)sum.x, (__bf16)sum.y, (__bf16)sum.z, (__bf16)sum.w};
        *reinterpret_cast<bf16x4 *>(static_cast<uint16_t *>(out) + at) = y;
    } else {
        *reinterpret_cast<f4 *>(static_cast<float *>(out) + at) = sum;
    }
}
constexpr int kSplitSlots = 2;

template <int D> struct SplitLds {
    static constexpr int kLoads = (KvTile<D>::kBytes + 1023) / 1024, kSlot = kLoads * 1024;  // DMA instructions of a tile
    static constexpr int kSums = kSplitWaves * 16 * (D + 4) * 4, kJoin = kSums + 2 * kSplitWaves * 16 * 4;
    static constexpr int kRing = kSplitWaves * kSplitSlots * kSlot, kBytes = kRing > kJoin ? kRing : kJoin;
};

// A tile to LDS, past the registers.  (The wait: nothing is read any more from where it goes; the s_nop: a vector instruction may have
// written the descriptor's scalar registers just before.)
template <int D> __device__ __forceinline__ void fetch_tile(uint32_t lds_at, const uint8_t *tile) {
    const i32x4 rsrc = make_rsrc(tile, KvTile<D>::kBytes);  // (what the last instruction asks for behind the tile's end is not read)
    const uint32_t lane = ((uint32_t)threadIdx.x & 63u) * 16u;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_nop 4" ::: "memory");
#pragma unroll
    for (int i = 0; i < SplitLds<D>::kLoads; i++)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds_at + (uint32_t)i * 1024u), "v"(lane), "s"(rsrc), "s"((uint32_t)i * 1024u) : "memory");
}

}  // namespace

}  // namespace gq
