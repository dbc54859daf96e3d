// Softmax attention of the new tokens of every sequence over a 4-bit cache (layout: kv.hpp).
//
//     s_ij = scale q_i . k_j for the tokens j that row i sees (j <= p_i, and j > p_i - window where there is a window; p_i its own place)
//     o_i  = sum_j P_ij v_j,  P_i = softmax(s_i);  a row that sees nothing gets zeros
//     account_j += sum of P_ij over the rows and the query heads of the key head (where asked for)
//
// Both products run on the fp16 matrix instructions (16x16x32 for few rows, 32x32x16 for many).  Keys and values are fp16 numbers as they stand (kv.hpp), q is scaled by a power
// of two per row (fp32: and by the scale's mantissa) and taken as one fp16 number (bf16: exact) or as the sum of two (fp32: 22 bits), P likewise as one (bf16) or
// two; scores, running maximum, sums and results are fp32.
//
// The first product is formed transposed, S^T = K Q^T: a lane holds one query (its column) and eight neighbouring tokens of the
// tile, so that maximum and sum are plain lane arithmetic and the weights are the second product's operand, O^T = V^T P^T,
// where they lie.  The reference of a row's exponents is set so that its largest weight so far is 2^6 (fp32: 2^12, 2^9 at D = 256), and moves only when
// a weight would pass 2^14 (2^15.5; fp16's largest number is 2^16): the lanes of the row then agree on a new one.  fp16 numbers are 2^-24 apart at least, so that a
// weight is rounded to 2^-31 (2^-37, 2^-34) of its row's largest where that is more than its 11 (22) bits: of 100000 weights that small together 5e-5 (7e-7, 6e-6) may be lost.
#include "kv.hpp"
#include "lds_dma.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

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

struct AttendArgs {
    KvCall kv;
    HeadRows q;
    int heads, group, window, wide;
    float scale_log2;        // scale * log2(e)
    void *out;               // [rows, heads, D]
    float *lse;              // [rows, heads], in powers of two; null where nobody asks
    float *part, *part_ml;   // of kv_split_kernel's workgroups: sums [rows, D], (reference, sum) [rows, 2]
    int workgroups, rows;    // of kv_split_kernel; (new token, head) pairs of a key head that it has, at most
    int few;                 // sequences of so many such pairs or fewer are kv_split_kernel's, the others kv_rows_kernel's
    int2 *pieces;            // per unit of kv_split_kernel: the first workgroup that works on it, and how many do
    float *accounts;
    float *scores;           // of kv_split_kernel, in powers of two: [units, rows, score_tiles * 32] from the first tile that a unit sees; null: not kept
    int score_tiles;
    int row_pieces;          // of kv_rows_kernel: pieces that a row tile's tokens are cut into (> 1: sums [line, pieces, D], (reference, sum) [line, pieces, 2])
    uint8_t *operands;       // of kv_rows_kernel, for the accounts: 32 rows' queries as it has them, [key heads, operand tiles]; null: not kept
    float *row_scales;       // and what their scores are multiplied by, [key heads, operand tiles, 32]
    int operand_tiles;
};

// The tiles that the rows of a row tile (sixteen neighbouring (new token, head of the group) pairs) see, and where its chunk of them lies.
struct Span { int first_row, rows, lo, hi; };  // rows in the tile; tokens [lo, hi) that one of them sees
__device__ __forceinline__ Span row_tile_span(const KvSeq &s, int group, int window, int row_tile, int tile_rows) {
    Span r;
    r.first_row = row_tile * tile_rows;
    const int all = s.news * group;
    r.rows = all - r.first_row;
    r.rows = r.rows < 0 ? 0 : r.rows > tile_rows ? tile_rows : r.rows;
    r.lo = r.hi = 0;
    if (r.rows > 0) {
        const int hi = s.first + (r.first_row + r.rows - 1) / group + 1, first = s.first + r.first_row / group + 1;
        r.hi = hi < 0 ? 0 : min(hi, s.length);
        r.lo = window && first > window ? min(first - window, r.hi) : 0;
    }
    return r;
}

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

constexpr int kSplitWaves = 4, kSplitRows = 16;

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

// How the tiles of a call are shared out over its workgroups.  A unit is a sequence and key head (all rows of it: sixteen at most),
// with the tiles that its rows see (one at least, so that rows that see nothing are written too).  Units are cut into pieces
// of one length, of which all units together have about a.workgroups, one piece a workgroup: the lengths are known on the device only, so
// every wavefront finds its place by a sum over them, 64 sequences at a time, one a lane.  (All tiles together: less than 2^31.)
struct Piece {
    int b, h, nth;       // sequence, key head, number of the piece in its unit; b < 0: there is none
    int share, tiles;    // tiles of a piece, of the unit
    KvSeq seq;
    Span span;
    __device__ __forceinline__ int pieces() const { return (tiles + share - 1) / share; }
};
// (a sequence of more rows than `few` has none here)
__device__ __forceinline__ Span span_of(const AttendArgs &a, const KvSeq &seq) {
    Span span = row_tile_span(seq, a.group, a.window, 0, kSplitRows);
    if (seq.news * a.group > a.few) span.rows = 0;
    return span;
}
__device__ __forceinline__ int tiles_of(const Span &span) { return span.rows ? max(1, ((span.hi + 31) >> 5) - (span.lo >> 5)) : 0; }

__device__ __forceinline__ Piece piece_of(const AttendArgs &a, int index) {
    const int lane = (int)threadIdx.x & 63, seqs = a.kv.seqs, heads = a.kv.kv_heads;
    Piece p;
    p.b = -1;
    KvSeq mine{};
    int tiles = 0, total = 0;
    for (int base = (seqs - 1) & ~63; base >= 0; base -= 64) {  // (the first 64 last: they stay)
        mine = KvSeq{};
        if (base + lane < seqs) mine = kv_seq(a.kv, base + lane);
        tiles = tiles_of(span_of(a, mine));
        total += __builtin_amdgcn_readlane(lane_scan(tiles), 63) * heads;
    }
    // (a multiple of the wavefronts: each of them the same number of tiles)
    const int least = (total + a.workgroups - 1) / a.workgroups;
    p.share = max(1, (least + kSplitWaves - 1) / kSplitWaves) * kSplitWaves;
    int front = 0;  // pieces in front
    for (int base = 0; base < seqs; base += 64) {
        if (base) {
            mine = KvSeq{};
            if (base + lane < seqs) mine = kv_seq(a.kv, base + lane);
            tiles = tiles_of(span_of(a, mine));
        }
        const int unit = (tiles + p.share - 1) / p.share;
        const int upto = lane_scan(unit * heads);
        const uint64_t past = __ballot(front + upto > index);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            p.b = base + l;
            p.seq = seq_of_lane(mine, l);
            p.span = span_of(a, p.seq);
            p.tiles = __builtin_amdgcn_readlane(tiles, l);
            const int each = __builtin_amdgcn_readlane(unit, l), in = index - (front + __builtin_amdgcn_readlane(upto, l) - each * heads);
            p.h = in / each;
            p.nth = in - p.h * each;
            break;
        }
        front += __builtin_amdgcn_readlane(upto, 63);
    }
    return p;
}

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
__device__ __forceinline__ float lse_of(float top, float all) { return all == 0.0f ? kNegInf : top + __builtin_amdgcn_logf(all); }

constexpr int kSplitSlots = 2, kMostWorkgroups = 2048;

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

// A piece of a unit: up to sixteen rows, (new token, head) pairs, over `share` tiles.  Each wavefront takes every fourth tile, with a
// maximum, sums and results of its own, and they meet in LDS.  A unit of one piece is finished here; the others leave their sums, by
// workgroup, for kv_join_kernel.
//
// One pass over the cache bounds it: 32 sequences of 2048 to 8192 tokens, 8 heads of D = 128, 193 MB: 42 us, 4.5 TB/s (a copy reaches 4.8).  One
// sequence of 2047 tokens, 2.4 MB: 6.2 us, most of it the way from lengths to table to tiles, each a load that waits for the one in front.
// Tiles by DMA because two of them a wavefront in flight would take a third of its registers (through registers the call took 48 to 55 us, one sequence of 131072 tokens 40 instead of 38).
template <int D, bool BF16>
__global__ __launch_bounds__(64 * kSplitWaves, D == 256 ? 2 : BF16 ? 4 : 3) void kv_split_kernel(const AttendArgs a) {
    constexpr bool TWO = !BF16;
    constexpr int W = D / 16;
    typedef SplitLds<D> Lds;
    __shared__ __align__(16) uint8_t lds[Lds::kBytes];
    // (the results take the place of the tiles once all of these are done with)
    float(*sums)[16][D + 4] = reinterpret_cast<float(*)[16][D + 4]>(lds);
    float(*refs)[16] = reinterpret_cast<float(*)[16]>(lds + Lds::kSums), (*totals)[16] = reinterpret_cast<float(*)[16]>(lds + Lds::kSums + kSplitWaves * 64);
    const KvCall &kv = a.kv;
    const int lane = (int)threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Piece piece = piece_of(a, (int)blockIdx.x);
    if (piece.b < 0) return;
    const int b = piece.b, h = piece.h;
    const KvSeq &seq = piece.seq;
    const Span &span = piece.span;
    const int tile0 = (span.lo >> 5) + piece.nth * piece.share, tile1 = (span.lo >> 5) + min((piece.nth + 1) * piece.share, piece.tiles);
    const Unpack unpack;
    const bool live = r < span.rows;
    const int nth = live ? r / a.group : 0;              // new token of the row
    const int head = h * a.group + (live ? r - nth * a.group : 0);
    const int64_t row = seq.row0 + nth;
    const int base = seq.first, place = base + nth;  // its own token
    const int see_hi = live ? place + 1 : 0, see_lo = a.window ? place + 1 - a.window : 0;
    // tokens that every row sees (the operand rows that stand for none have scores of 0 and go nowhere)
    const int all_hi = base + 1, all_lo = a.window ? base + (span.rows - 1) / a.group + 1 - a.window : 0;

    f4 o[W];
#pragma unroll
    for (int w = 0; w < W; w++) o[w] = f4{0.f, 0.f, 0.f, 0.f};
    float ref = kNegInf, total = 0.0f;  // the row's reference, and the lane's share of its sum

    const int last = min(tile1, (span.hi + 31) >> 5);  // (a unit that sees nothing has a tile in name only)
    TileWalk<KvTile<D>::kBytes, kSplitWaves> walk(kv, b, h, tile0 + wave, last);
    // the wavefront's ring of tiles: one is worked on while the next is on its way
    uint8_t *ring = lds + wave * kSplitSlots * Lds::kSlot;
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)ring);
    const uint8_t *mem = walk.next();
    if (mem) fetch_tile<D>(ring_at, mem);
    h8 qh[D / 32], ql[TWO ? D / 32 : 1];
    float to_log2;
    load_queries<D, 16, BF16, TWO>(a.q, row * a.q.row + head * a.q.head, live, a.wide, a.scale_log2, qh, ql, to_log2);
    int turn = 0;
    for (int tile = tile0 + wave; tile < last; tile += kSplitWaves) {
        const uint8_t *mem_next = walk.next();
        if (mem_next) {
            fetch_tile<D>(ring_at + (uint32_t)(turn ^ 1) * Lds::kSlot, mem_next);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Lds::kLoads) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (mem) {
            KeyWords<D> k;
            k.load(ring + turn * Lds::kSlot);
            float s[8];
            tile_scores<D, TWO>(unpack, k, qh, ql, s);
            const int t0 = tile * 32;
            float most = kNegInf;
            if (t0 >= all_lo && t0 + 32 <= all_hi) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    s[e] *= to_log2;
                    most = fmaxf(most, s[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int t = t0 + 8 * j + e;
                    s[e] = t < see_hi && t >= see_lo ? s[e] * to_log2 : kNegInf;
                    most = fmaxf(most, s[e]);
                }
            }
            if (a.scores && live) {
                float *to = a.scores + ((int64_t)(b * kv.kv_heads + h) * a.rows + r) * a.score_tiles * 32 + (t0 + 8 * j - (span.lo & ~31));
                *reinterpret_cast<f4 *>(to) = f4{s[0], s[1], s[2], s[3]};
                *reinterpret_cast<f4 *>(to + 4) = f4{s[4], s[5], s[6], s[7]};
            }
            if (__any(passes<D, TWO>(most, ref))) {  // (the first score of a row among them: its reference is -infinity)
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                const float next = fmaxf(ref, reference<D, TWO>(most));
                const float shrink = next == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ref - next);
                ref = next;
                total *= shrink;
#pragma unroll
                for (int w = 0; w < W; w++) o[w] *= shrink;
            }
            const float less = ref == kNegInf ? 0.0f : ref;
            h8 ph, pl;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = __builtin_amdgcn_exp2f(s[e] - less);
                total += p;
                ph[e] = (_Float16)p;
                if constexpr (TWO) pl[e] = (_Float16)(p - (float)ph[e]);
            }
            ValueWords<D> v;
            v.load(ring + turn * Lds::kSlot);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const h8 x = v.operand(unpack, w);
                o[w] = mfma(x, ph, o[w]);
                if constexpr (TWO) o[w] = mfma(x, pl, o[w]);
            }
        }
        mem = mem_next;
        turn ^= 1;
    }
    __syncthreads();
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
#pragma unroll
    for (int w = 0; w < W; w++) *reinterpret_cast<f4 *>(&sums[wave][r][16 * w + 4 * j]) = o[w];
    if (j == 0) {
        refs[wave][r] = ref;
        totals[wave][r] = total;
    }
    __syncthreads();

    const int pieces = piece.pieces();
    if (a.pieces && piece.nth == 0 && threadIdx.x == 0) a.pieces[b * kv.kv_heads + h] = make_int2((int)blockIdx.x, pieces);
    for (int i = (int)threadIdx.x; i < span.rows * (D / 4); i += 64 * kSplitWaves) {
        const int rr = i / (D / 4), d = (i - rr * (D / 4)) * 4;
        float top = kNegInf;
#pragma unroll
        for (int w = 0; w < kSplitWaves; w++) top = fmaxf(top, refs[w][rr]);
        f4 sum = {0.f, 0.f, 0.f, 0.f};
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < kSplitWaves; w++) {
            const float f = refs[w][rr] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(refs[w][rr] - top);
            // (a wavefront without a reference has seen no number: its sum is zero, or NaN)
            all += refs[w][rr] == kNegInf ? totals[w][rr] : totals[w][rr] * f;
            sum += *reinterpret_cast<const f4 *>(&sums[w][rr][d]) * f;
        }
        if (pieces == 1) {
            const int n = rr / a.group;
            const int64_t out = (int64_t)(seq.row0 + n) * a.heads + h * a.group + (rr - n * a.group);
            store_result<BF16>(a.out, out * D + d, sum, all);
            if (a.lse && d == 0) a.lse[out] = lse_of(top, all);
        } else {
            *reinterpret_cast<f4 *>(a.part + ((int64_t)blockIdx.x * a.rows + rr) * D + d) = sum;
            if (d == 0) {
                a.part_ml[((int64_t)blockIdx.x * a.rows + rr) * 2] = top;
                a.part_ml[((int64_t)blockIdx.x * a.rows + rr) * 2 + 1] = all;
            }
        }
    }
}

// Joins the pieces of the units that more than one workgroup has worked on: one workgroup per unit and row.  4 to 5 us, the chain from the
// unit's pieces to their references to their sums.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttendArgs a) {
    constexpr int L = D / 4, S = 256 / L;  // lanes of a row's values, and the shares into which the pieces are divided
    __shared__ f4 sums[S][L];
    __shared__ float factors[kMostWorkgroups], tops[4], alls[4];
    const int rr = (int)blockIdx.x, h = (int)blockIdx.y, b = (int)blockIdx.z, tid = (int)threadIdx.x;
    const int2 piece = a.pieces[b * a.kv.kv_heads + h];
    const KvSeq seq = kv_seq(a.kv, b);
    if (rr >= span_of(a, seq).rows) return;  // (without rows nobody has written the unit's pieces)
    const int first = piece.x, pieces = piece.y;
    if (pieces == 1) return;
    const auto line = [&](int i) { return (int64_t)(first + i) * a.rows + rr; };
    float top = kNegInf;
    for (int i = tid; i < pieces; i += 256) top = fmaxf(top, a.part_ml[line(i) * 2]);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    float all = 0.0f;
    for (int i = tid; i < pieces; i += 256) {
        const float ref = a.part_ml[line(i) * 2], t = a.part_ml[line(i) * 2 + 1];
        const float f = ref == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ref - top);
        factors[i] = f;
        all += ref == kNegInf ? t : t * f;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) all += __shfl_xor(all, m);
    if ((tid & 63) == 0) alls[tid >> 6] = all;
    __syncthreads();
    all = (alls[0] + alls[1]) + (alls[2] + alls[3]);
    const int l = tid % L, part = tid / L;
    f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = part; i < pieces; i += S) sum += *reinterpret_cast<const f4 *>(a.part + line(i) * D + l * 4) * factors[i];
    sums[part][l] = sum;
    __syncthreads();
    if (part) return;
    sum = sums[0][l];
    for (int i = 1; i < S; i++) sum += sums[i][l];
    const int n = rr / a.group;
    const int64_t out = (int64_t)(seq.row0 + n) * a.heads + h * a.group + (rr - n * a.group);
    store_result<BF16>(a.out, out * D + l * 4, sum, all);
    if (a.lse && l == 0) a.lse[out] = lse_of(top, all);
}

// Many rows: a workgroup takes 128 neighbouring (new token, head) pairs of a key head, 32 a wavefront, over all the tokens that they
// see, and widens the cache's codes once for all of them: 8192 values of keys and values each (64 tokens at D = 128) at a time go through LDS as fp16 operands of
// v_mfma_f32_32x32x16_f16, written in the order in which lanes read them, into the one of two buffers that is not worked on.
// The instruction's results lie in a lane (r, half) as the operand rows 8 (i / 4) + 4 half + i % 4; operand row m is token m with bits 2
// and 3 exchanged, so that a lane's results 8 s + 0..7 are the scores of tokens 16 s + 8 half + 0..7: the eight of one dword of value
// codes, and its share of the second product's operand where they lie.
//
// Matrix instructions, exponentials and the widening run side by side, two workgroups a CU (2048 rows of 32 heads over 2049 to 4096
// tokens, D = 128).  With a causal bound workgroups differ in length: the second half of them goes from short to long, so that the two of a CU
// add up to the same.  That call: 121 us in bfloat16 (float32: 199), 850 TFLOP/s (a library product of 8192^3: 1193): a stage of 64 tokens
// has 1024 cycles of matrix instructions a wavefront and 1270 of others, which overlap little, and takes 2600.
constexpr int kRowsWaves = 4, kRowsTile = 32 * kRowsWaves, kRowsPiece = 12;  // rows of a workgroup; tiles of the cache, at least, in a piece of its tokens

template <int D> struct RowsLds {
    static constexpr int kTiles = 256 / D;                         // of the cache, at a time: a chunk of codes of keys and one of values a thread
    static constexpr int kKeys = 64 * D, kTile = 2 * kKeys;        // bytes of a tile's key operands; of all its operands
    static constexpr int kStage = kTiles * kTile;
};

// The codes and scales that a thread widens, as loaded: chunk c (four dwords a lane) of a tile's keys or values.
struct Chunk {
    u4 code, scale[2];
    template <int D> __device__ __forceinline__ void load(const uint8_t *tile, bool values, int c) {
        constexpr int G = D / 32;
        const int lane = c & 63, r = lane & 15, j = lane >> 4, w = (c >> 6) * 4;
        code = *reinterpret_cast<const u4 *>(tile + (values ? KvTile<D>::kValues : KvTile<D>::kKeys) + c * 16);
        if (values) {
            const uint8_t *p = tile + KvTile<D>::kValueScales + (w >> 1) * 64 + j * 16;
            scale[0] = *reinterpret_cast<const u4 *>(p);
            scale[1] = *reinterpret_cast<const u4 *>(p + 64);
        } else {
            const uint8_t *p = tile + KvTile<D>::kKeyScales + (8 * (r >> 2) + (r & 3)) * (2 * G);  // of the first of the two tokens of row r
            if constexpr (D == 64) {
                scale[0].x = *reinterpret_cast<const uint32_t *>(p);
                scale[0].y = *reinterpret_cast<const uint32_t *>(p + 4 * 2 * G);
            } else {
                const u2 v = *reinterpret_cast<const u2 *>(p + (w / G) * 4 * 2 * G + (w % G) * 2);
                scale[0].x = v.x;
                scale[0].y = v.y;
            }
        }
    }
    template <int D> __device__ __forceinline__ void widen(const Unpack &unpack, uint8_t *stage, bool values, int c) const {
        constexpr int G = D / 32;
        const int lane = c & 63, r = lane & 15, j = lane >> 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int w = (c >> 6) * 4 + i;
            h2 v[4];
            unpack(code[i], v);
            if (values) {
                const u4 d = scale[i >> 1];
                const h8 x = join(v[0] * as_h2(d[0]), v[1] * as_h2(d[1]), v[2] * as_h2(d[2]), v[3] * as_h2(d[3]));
                // [32 values][tokens 16 s ..][lane]
                *reinterpret_cast<h8 *>(stage + RowsLds<D>::kKeys + (((w >> 1) * 2 + (j >> 1)) * 64 + (w & 1) * 16 + r + 32 * (j & 1)) * 16) = x;
            } else {
                const h2 pair = as_h2((i >> 1) ? scale[0].y : scale[0].x);
                const _Float16 one = (i & 1) ? pair.y : pair.x;
                const h2 d = {one, one};
                const h8 x = join(v[0] * d, v[1] * d, v[2] * d, v[3] * d);
                const int g = w % G, u = w / G, m = (r >> 3) * 16 + u * 8 + ((r >> 2) & 1) * 4 + (r & 3);  // token 8 (r / 4) + 4 u + r % 4, bits 2 and 3 exchanged
                *reinterpret_cast<h8 *>(stage + ((2 * g + (j >> 1)) * 64 + m + 32 * (j & 1)) * 16) = x;
            }
        }
    }
    template <int D> __device__ __forceinline__ static void clear(uint8_t *stage, bool values, int c) {  // (no such tile: numbers, which nobody sees)
        const u4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<u4 *>(stage + (values ? RowsLds<D>::kKeys : 0) + (c * 4 + i) * 16) = zero;
    }
};

__device__ __forceinline__ f16 mfma32(h8 a, h8 b, f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The sequence and its row tile that number `index` of all row tiles is; b < 0: there is none.
struct RowTile { int b, tile, tiles; KvSeq seq; };
__device__ __forceinline__ RowTile row_tile_of(const AttendArgs &a, int index) {
    const int lane = (int)threadIdx.x & 63, seqs = a.kv.seqs;
    RowTile t;
    t.b = -1;
    int front = 0;
    for (int base = 0; base < seqs; base += 64) {
        KvSeq mine{};
        if (base + lane < seqs) mine = kv_seq(a.kv, base + lane);
        const int rows = mine.news * a.group, tiles = rows > a.few ? (rows + kRowsTile - 1) / kRowsTile : 0, upto = lane_scan(tiles);
        const uint64_t past = __ballot(front + upto > index);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            t.b = base + l;
            t.seq = seq_of_lane(mine, l);
            t.tiles = __builtin_amdgcn_readlane(tiles, l);
            t.tile = index - (front + __builtin_amdgcn_readlane(upto, l) - t.tiles);
            break;
        }
        front += __builtin_amdgcn_readlane(upto, 63);
    }
    return t;
}
// The first operand tile of sequence b: tiles of 32 rows, of which no two sequences share one.
__device__ __forceinline__ int first_operand_tile(const AttendArgs &a, const KvSeq &seq, int b) { return (int)((int64_t)seq.row0 * a.group / 32) + b; }

// Results that live in accumulation registers, in which nothing but matrix instructions computes.  Written out, because the compiler would copy all of them to
// ordinary registers and back in every stage for a multiplication that next to none of them needs.  (us a call, D = 256, 8 heads of 2 key heads: 64 rows
// of 5 sequences over 4000 to 16000 tokens in float32 117 108, 1714 rows of 2 over themselves in bfloat16 95 82.)  (The waits: it does not know what matrix instruction
// the reads are behind and the writes in front of.)
template <int N> __device__ __forceinline__ void scale_accumulators(f16 (&v)[N], float by) {
    asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
    for (int w = 0; w < N; w++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float x, y;
            asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(v[w][i]));
            x *= by;
            asm volatile("v_accvgpr_write_b32 %0, %1" : "=a"(y) : "v"(x));
            v[w][i] = y;
        }
    asm volatile("s_nop 7");
}

template <int D, bool BF16, bool ACCOUNTS>
__global__ __launch_bounds__(64 * kRowsWaves, D == 256 ? 1 : 2) void kv_rows_kernel(const AttendArgs a) {
    constexpr bool TWO = !BF16;
    typedef RowsLds<D> Lds;
    constexpr int KS = D / 16, VS = D / 32, T = Lds::kTiles;
    __shared__ __align__(16) uint8_t stage[2][Lds::kStage];
    __shared__ __align__(4) uint8_t there[2][4];  // which tiles of a stage's keys the cache has
    constexpr uint32_t ALL = 0x01010101u >> (8 * (4 - T));
    const KvCall &kv = a.kv;
    // (the key head goes round fastest: with eight of them, one to an XCD and its L2)
    const int rest = (int)blockIdx.x / kv.kv_heads, h = (int)blockIdx.x - rest * kv.kv_heads;
    const int index = rest / a.row_pieces, piece = rest - index * a.row_pieces;
    const RowTile unit = row_tile_of(a, index);
    if (unit.b < 0) return;
    const int b = unit.b;
    const KvSeq &seq = unit.seq;
    const int row_tile = unit.tile < (unit.tiles + 1) / 2 ? unit.tiles - 1 - unit.tile : unit.tile - (unit.tiles + 1) / 2;
    const Span span = row_tile_span(seq, a.group, a.window, row_tile, kRowsTile);
    const int stages = (((span.hi + 31) >> 5) - (span.lo >> 5) + T - 1) / T;
    const int tile0 = (span.lo >> 5) + T * (int)((int64_t)stages * piece / a.row_pieces);
    const int tile1 = min((span.hi + 31) >> 5, (span.lo >> 5) + T * (int)((int64_t)stages * (piece + 1) / a.row_pieces));

    const int tid = (int)threadIdx.x, lane = tid & 63, r = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int in = wave * 32 + r, idx = span.first_row + in;
    const bool live = in < span.rows;
    const int nth = live ? idx / a.group : 0;
    const int head = h * a.group + (live ? idx - nth * a.group : 0);
    const int64_t row = seq.row0 + nth;
    const int base = seq.first, place = base + nth;
    const int own = live ? place : -1;  // (a row that is none, or without tokens, sees nothing)
    const uint32_t most_behind = a.window ? (uint32_t)a.window : 0x80000000u;
    // what every row of the wavefront sees
    const int first_in = span.first_row + wave * 32, last_in = min(first_in + 31, span.first_row + span.rows - 1);
    const int all_hi = __builtin_amdgcn_readfirstlane(base + first_in / a.group + 1);
    const int all_lo = __builtin_amdgcn_readfirstlane(a.window ? base + last_in / a.group + 1 - a.window : 0);

    const Unpack unpack;
    // A wavefront widens the same tile of every stage, a thread one chunk of its keys and one of its values.
    const int part = tid % D, tile_in = __builtin_amdgcn_readfirstlane(tid / D);
    TileWalk<KvTile<D>::kBytes, T> walk(kv, b, h, tile0 + tile_in, tile1);
    struct Fetched {  // of a stage, on its way
        const uint8_t *mem;
        Chunk keys, values;
    } fetched[2];
    const auto load = [&](Fetched &f) __attribute__((always_inline)) {
        f.mem = walk.next();
        if (f.mem) {
            f.keys.template load<D>(f.mem, false, part);
            f.values.template load<D>(f.mem, true, part);
        }
    };
    const auto widen = [&](const Fetched &f, int to) __attribute__((always_inline)) {
        uint8_t *at = stage[to] + tile_in * Lds::kTile;
        if (f.mem) {
            f.keys.template widen<D>(unpack, at, false, part);
            f.values.template widen<D>(unpack, at, true, part);
        } else {
            Chunk::template clear<D>(at, false, part);
            Chunk::template clear<D>(at, true, part);
        }
        if (part == 0) there[to][tile_in] = f.mem ? 1 : 0;
    };

    load(fetched[0]);
    load(fetched[1]);
    h8 qh[KS], ql[TWO ? KS : 1];
    float to_log2;
    load_queries<D, 32, BF16, TWO>(a.q, row * a.q.row + head * a.q.head, live, a.wide, a.scale_log2, qh, ql, to_log2);
    to_log2 = to_log2 < 0x1p-122f ? 0x1p-122f : to_log2;  // (not 0, so that its product with -infinity stays that; a scale of NaN stays one)
    if constexpr (D == 256) {  // (512 registers: the rows' operands in accumulation registers, beside the results)
#pragma unroll
        for (int k = 0; k < KS; k++) {
            asm("" : "+a"(qh[k]));
            if constexpr (TWO) asm("" : "+a"(ql[k]));
        }
    }
    if (ACCOUNTS && piece == 0 && wave * 32 < span.rows) {
        const int64_t tile = (int64_t)h * a.operand_tiles + first_operand_tile(a, seq, b) + row_tile * kRowsWaves + wave;
        h8 *to = reinterpret_cast<h8 *>(a.operands) + tile * (TWO ? 2 : 1) * KS * 64 + lane;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            to[k * 64] = qh[k];
            if constexpr (TWO) to[(KS + k) * 64] = ql[k];
        }
        if (half == 0) a.row_scales[tile * 32 + r] = to_log2;
    }

    f16 o[VS];
    float ref, total;     // the row's reference, and the lane's share of its sum
    bool coarse = false;  // one of the wavefront's references has been large

    // One stage, from buffer `mine`; the next one, which has been on its way for a stage, goes into `other`.  (Making the next stage's scores in front of these weights, so that one wavefront has
    // both kinds of work to issue, was no faster: the second workgroup of the CU does as well.)
    const auto attend_stage = [&](auto mode, int tile, int mine) __attribute__((always_inline)) {
        constexpr bool COARSE = decltype(mode)::value;  // (the rows' scores may be large: they are multiplied first)
        const float by = COARSE ? 1.0f : to_log2;
        f16 s[T];
#pragma unroll
        for (int t = 0; t < T; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const h8 x = *reinterpret_cast<const h8 *>(stage[mine] + t * Lds::kTile + (k * 64 + lane) * 16);
                s[t] = mfma32(x, qh[k], s[t]);
                if constexpr (TWO) s[t] = mfma32(x, ql[k], s[t]);
            }
        }
        // (operands are read four instructions ahead)
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < T * KS - 4; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, TWO ? 2 : 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, TWO ? 8 : 4, 0);
        if constexpr (COARSE) {
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[t][i] *= to_log2;
        }
        const int t0 = tile * 32;
        const uint32_t known = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t *>(there[mine])) & ALL;
        if (!(t0 >= all_lo && t0 + 32 * T <= all_hi && known == ALL)) {
#pragma unroll
            for (int t = 0; t < T; t++) {
                const uint32_t window = (known >> (8 * t)) & 1u ? most_behind : 0u;
                const int behind = own - t0 - 32 * t - 8 * half;  // the tokens from the lane's first one to the row's own
#pragma unroll
                for (int i = 0; i < 16; i++) s[t][i] = (uint32_t)(behind - 16 * (i >> 3) - (i & 7)) < window ? s[t][i] : kNegInf;
            }
        }
        float most = kNegInf;  // (scores as the products left them: what they are multiplied by is not negative)
#pragma unroll
        for (int t = 0; t < T; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) most = fmaxf(most, s[t][i]);
        if (__any(passes<D, TWO>(most * by, ref))) {
            most *= by;
            most = fmaxf(most, __shfl_xor(most, 32));
            const float set = fmaxf(ref, reference<D, TWO>(most));
            const float shrink = set == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ref - set);
            ref = set;
            if constexpr (!TWO && !COARSE) coarse = coarse || __any(fabsf(ref) >= kCoarse && ref != kNegInf);
            total *= shrink;
            if constexpr (D == 256) {
                scale_accumulators(o, shrink);
            } else {
#pragma unroll
                for (int w = 0; w < VS; w++) o[w] *= shrink;
            }
        }
        const float less = ref == kNegInf ? 0.0f : -ref;
#pragma unroll
        for (int t = 0; t < T; t++) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                h8 ph, pl;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][8 * k + e], by, less)), p1 = __builtin_amdgcn_exp2f(fmaf(s[t][8 * k + e + 1], by, less));
                    ph[e] = (_Float16)p0;
                    ph[e + 1] = (_Float16)p1;
                    if constexpr (TWO) {
                        pl[e] = (_Float16)(p0 - (float)ph[e]);
                        pl[e + 1] = (_Float16)(p1 - (float)ph[e + 1]);
                    }
                    if constexpr (TWO || ACCOUNTS) {  // (accounts are kept to fp32's accuracy whatever the type)
                        total += p0;
                        total += p1;
                    } else {  // the weights as they are used, two in one instruction
                        const h2 pair = {ph[e], ph[e + 1]}, ones = {(_Float16)1.0f, (_Float16)1.0f};
                        total = __builtin_amdgcn_fdot2(pair, ones, total, false);
                    }
                }
#pragma unroll
                for (int w = 0; w < VS; w++) {
                    const h8 x = *reinterpret_cast<const h8 *>(stage[mine] + t * Lds::kTile + Lds::kKeys + ((w * 2 + k) * 64 + lane) * 16);
                    o[w] = mfma32(x, ph, o[w]);
                    if constexpr (TWO) o[w] = mfma32(x, pl, o[w]);
                }
            }
        }
        // (the weights of sixteen tokens are made while the products with those in front run)
        __builtin_amdgcn_sched_group_barrier(0x002, 26, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
        for (int i = 0; i < 2 * T * VS - 4; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, TWO ? 2 : 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x002, 6, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, TWO ? 8 : 4, 1);
    };
    // (a wavefront without rows widens for the others; at D = 256 the branch would move accumulators about: 56 us become 65)
    const bool rows_here = D == 256 || wave * 32 < span.rows;
    const auto step = [&](auto mode, int tile, int mine, int other) __attribute__((always_inline)) {
        load(fetched[mine]);
        if (rows_here) attend_stage(mode, tile, mine);
        if (tile + T < tile1) widen(fetched[other], other);
        __syncthreads();
    };
    const auto attend_all = [&](auto mode) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < VS; w++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[w][i] = 0.0f;
        ref = kNegInf;
        total = 0.0f;
        if (tile0 < tile1) widen(fetched[0], 0);
        __syncthreads();
        for (int tile = tile0; tile < tile1; tile += 2 * T) {
            step(mode, tile, 0, 1);
            if (tile + T < tile1) step(mode, tile + T, 1, 0);
        }
    };
    attend_all(std::false_type{});
    // Again from the start with scores that are large: what was summed is not theirs.  (A branch for them in the stage would cost all others: at D = 256, 1714
    // rows of 2 sequences over themselves 81 us, with it 90.)
    if constexpr (!TWO) {
        if (__syncthreads_or(coarse)) {
            walk.start(tile0 + tile_in, tile1);
            load(fetched[0]);
            load(fetched[1]);
            attend_all(std::true_type{});
        }
    }
    total += __shfl_xor(total, 32);
    if (!live) return;
    const int64_t out = row * a.heads + head;
    if (a.row_pieces > 1) {
        const int64_t line = out * a.row_pieces + piece;
#pragma unroll
        for (int w = 0; w < VS; w++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<f4 *>(a.part + line * D + 32 * w + 2 * i + 4 * half) = f4{o[w][i], o[w][i + 1], o[w][i + 2], o[w][i + 3]};
        if (half == 0) {
            a.part_ml[line * 2] = ref;
            a.part_ml[line * 2 + 1] = total;
        }
        return;
    }
#pragma unroll
    for (int w = 0; w < VS; w++)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            store_result<BF16>(a.out, out * D + 32 * w + 2 * i + 4 * half, f4{o[w][i], o[w][i + 1], o[w][i + 2], o[w][i + 3]}, total);
    if (ACCOUNTS && half == 0) a.lse[out] = lse_of(ref, total);
}

// Joins the pieces of kv_rows_kernel: a thread makes four values of a line, (row, head).  (Rows of sequences that kv_split_kernel has get what was in the
// scratch memory, until that kernel writes them.)
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_rows_join_kernel(const AttendArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, line = at / (D / 4);
    const int d = (int)(at - line * (D / 4)) * 4, n = a.row_pieces;
    if (line >= (int64_t)a.kv.rows * a.heads) return;
    const float *ml = a.part_ml + line * n * 2;
    float top = kNegInf, all = 0.0f;
#pragma unroll 8
    for (int i = 0; i < n; i++) top = fmaxf(top, ml[2 * i]);
    f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int i = 0; i < n; i++) {
        const float f = ml[2 * i] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml[2 * i] - top);
        all += ml[2 * i] == kNegInf ? ml[2 * i + 1] : ml[2 * i + 1] * f;
        sum += *reinterpret_cast<const f4 *>(a.part + (line * n + i) * D + d) * f;
    }
    store_result<BF16>(a.out, line * D + d, sum, all);
    if (a.lse && d == 0) a.lse[line] = lse_of(top, all);
}

// The accounts from the scores that kv_split_kernel has kept: one thread a token, which adds up the unit's rows.
__global__ __launch_bounds__(256) void kv_score_account_kernel(const AttendArgs a) {
    __shared__ float lse[16];
    const KvCall &kv = a.kv;
    const int h = (int)blockIdx.y, b = (int)blockIdx.z, tid = (int)threadIdx.x;
    const KvSeq seq = kv_seq(kv, b);
    const Span span = span_of(a, seq);
    const int first = span.lo & ~31, t = first + (int)blockIdx.x * 256 + tid;
    if (span.rows == 0 || first + (int)blockIdx.x * 256 >= span.hi) return;
    if (tid < span.rows) {
        const int n = tid / a.group;
        lse[tid] = a.lse[(int64_t)(seq.row0 + n) * a.heads + h * a.group + (tid - n * a.group)];
    }
    __syncthreads();
    if (t < span.lo || t >= span.hi) return;
    float *to = kv_account(kv, a.accounts, b, h, t);
    if (!to) return;
    const float *s = a.scores + (int64_t)(b * kv.kv_heads + h) * a.rows * a.score_tiles * 32 + (t - first);
    float sum = 0.0f;
    for (int r = 0; r < span.rows; r++) {
        const float v = s[(int64_t)r * a.score_tiles * 32];
        sum += v == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(v - lse[r]);  // (a token that the row does not see)
    }
    *to += sum;
}

// The accounts of many rows: a workgroup owns one or two neighbouring tiles of a sequence and key head, their keys in registers as operands, and goes over
// all rows that see them, as kv_rows_kernel has left them, 32 at a time and every fourth such tile a wavefront: every account is added to once, in
// one order.  The way of the rows' operands from the other XCDs' memory side bounds it where there are few, matrix instructions
// and one exponential a (row, token) where there are many: 78 us for 2048 rows of 32 heads over 2049 to 4096 tokens, D = 128, bfloat16, 12 for 301 rows and
// fewer of 5 sequences, 12 heads of D = 64, float32, 500 tokens in a window.
//
// Two tiles where their operands fit the registers of two wavefronts a SIMD, for the rows' operands are then read half as often (the first of these calls with its
// attention 200 us, with one tile a workgroup 223; at D = 64 a third wavefront does more than the second tile: the other call 38 us, with two tiles 44 to 50).
template <int D, bool BF16> constexpr int account_tiles() { return D == 128 && BF16 ? 2 : 1; }
template <int D, bool BF16>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 ? 2 : 3) void kv_rows_account_kernel(const AttendArgs a) {
    constexpr bool TWO = !BF16;
    constexpr int AHEAD = 2;  // row tiles of a wavefront on their way or worked on
    constexpr int KS = D / 16, G = D / 32, N = TWO ? 2 * KS : KS, NT = account_tiles<D, BF16>();
    __shared__ float sums[4][32 * NT];
    const KvCall &kv = a.kv;
    const int h = (int)blockIdx.y, b = (int)blockIdx.z;
    const KvSeq seq = kv_seq(kv, b);
    const int base = seq.first;
    const int tile = (a.window && base + 1 > a.window ? (base + 1 - a.window) >> 5 : 0) + (int)blockIdx.x * NT;
    if (tile >= (seq.length + 31) >> 5 || seq.news * a.group <= a.few) return;
    const int t0 = tile * 32;
    const int lane = (int)threadIdx.x & 63, r = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // the new tokens that see one of the tiles', and their operand tiles
    const int n0 = max(0, t0 - base), n1 = a.window ? (int)min((int64_t)seq.news, (int64_t)t0 + 32 * NT - 1 + a.window - base) : seq.news;
    const int from = n0 * a.group / 32 + wave, to = (n1 * a.group + 31) / 32;
    const int64_t first = (int64_t)h * a.operand_tiles + first_operand_tile(a, seq, b);
    struct Rows {  // 32 rows
        h8 q[N];
        float scale, lse;
        int place;  // -1: no row
    };
    const auto load = [&](int n, Rows &rows) __attribute__((always_inline)) {
        const int idx = n * 32 + r;
        const bool live = idx < seq.news * a.group;
        const int nth = live ? idx / a.group : 0, head = h * a.group + (live ? idx - nth * a.group : 0);
        rows.place = live ? base + nth : -1;
        rows.lse = a.lse[(int64_t)(seq.row0 + nth) * a.heads + head];
        rows.scale = a.row_scales[(first + n) * 32 + r];
        const h8 *q = reinterpret_cast<const h8 *>(a.operands) + (first + n) * N * 64 + lane;
#pragma unroll
        for (int k = 0; k < N; k++) rows.q[k] = q[k * 64];
    };
    Rows ring[AHEAD];
#pragma unroll
    for (int p = 0; p < AHEAD; p++)
        if (from + 4 * p < to) load(from + 4 * p, ring[p]);
    // the tiles' keys: operand row r is token r, values 16 k + 8 half + 0..7 (of a tile that the cache does not have: zeros)
    h8 keys[NT][KS];
    {
        const Unpack unpack;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const uint8_t *mem = t0 + 32 * t < seq.length ? kv_tile(kv, b, h, tile + t, KvTile<D>::kBytes) : nullptr;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int g = k >> 1, j = 2 * (k & 1) + half;
                uint32_t code = 0x88888888u;
                _Float16 one = (_Float16)0.0f;
                if (mem) {
                    code = *reinterpret_cast<const uint32_t *>(mem + KvTile<D>::kKeys + KvTile<D>::code(key_half(r) * G + g, key_row(r) + 16 * j));
                    one = reinterpret_cast<const _Float16 *>(mem + KvTile<D>::kKeyScales)[r * G + g];
                }
                h2 v[4];
                unpack(code, v);
                const h2 d = {one, one};
                keys[t][k] = join(v[0] * d, v[1] * d, v[2] * d, v[3] * d);
            }
        }
    }
    const uint32_t window = a.window ? (uint32_t)a.window : 0x80000000u;
    float sum[NT][16] = {};
    for (int n = from; n < to; n += 4 * AHEAD) {
#pragma unroll
        for (int p = 0; p < AHEAD; p++) {
            if (n + 4 * p >= to) break;
            Rows &now = ring[p];
            const bool open = __all(now.place >= t0 + 32 * NT - 1 && (!a.window || now.place - a.window < t0) && (TWO || fabsf(now.lse) < kCoarse));
#pragma unroll
            for (int t = 0; t < NT; t++) {
                f16 s;
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    s = mfma32(keys[t][k], now.q[k], s);
                    if constexpr (TWO) s = mfma32(keys[t][k], now.q[KS + k], s);
                }
                if (open) {
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[t][i] += __builtin_amdgcn_exp2f(fmaf(s[i], now.scale, -now.lse));
                } else {
                    const int behind = now.place - t0 - 32 * t - 4 * half;  // tokens of the tile's first for the lane to the row's own
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float w = __builtin_amdgcn_exp2f(s[i] * now.scale - now.lse);
                        sum[t][i] += (uint32_t)(behind - 8 * (i >> 2) - (i & 3)) < window ? w : 0.0f;
                    }
                }
            }
            if (n + 4 * (p + AHEAD) < to) load(n + 4 * (p + AHEAD), now);
        }
    }
    // over the 32 rows: lanes that differ in one bit pass each other half of what they have left, until each pair of lanes has one token's sum
#pragma unroll
    for (int t = 0; t < NT; t++) {
        int count = 16;
#pragma unroll
        for (int m = 16; m > 1; m >>= 1) {
            count >>= 1;
            const bool upper = lane & m;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (i >= count) break;
                const float give = upper ? sum[t][i] : sum[t][i + count], keep = upper ? sum[t][i + count] : sum[t][i];
                sum[t][i] = keep + __shfl_xor(give, m);
            }
        }
        const float all = sum[t][0] + __shfl_xor(sum[t][0], 1);
        const int i = r >> 1;
        if (!(r & 1)) sums[wave][32 * t + 8 * (i >> 2) + 4 * half + (i & 3)] = all;
    }
    __syncthreads();
    const int i = (int)threadIdx.x, token = t0 + i;
    if (i < 32 * NT && token < seq.length) {
        float *p = kv_account(kv, a.accounts, b, h, token);
        if (p) *p += (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
    }
}

// The accounts of few rows over so many tokens that their scores are not kept: as above, by sixteen rows.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_account_kernel(const AttendArgs a) {
    constexpr bool TWO = !BF16;
    const KvCall &kv = a.kv;
    const int h = (int)blockIdx.y, b = (int)blockIdx.z;
    const KvSeq seq = kv_seq(kv, b);
    const Span span = span_of(a, seq);
    const int tile = __builtin_amdgcn_readfirstlane((span.lo >> 5) + (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6));
    if (span.rows == 0 || tile * 32 >= span.hi) return;
    const uint8_t *mem = kv_tile(kv, b, h, tile, KvTile<D>::kBytes);
    if (!mem) return;
    KeyWords<D> k;
    k.load(mem);
    const int lane = (int)threadIdx.x & 63, r = lane & 15, j = lane >> 4, t0 = tile * 32;
    const bool live = r < span.rows;
    const int nth = live ? r / a.group : 0, head = h * a.group + (live ? r - nth * a.group : 0);
    const int64_t row = seq.row0 + nth;
    const int place = seq.first + nth, see_hi = live ? place + 1 : 0, see_lo = a.window ? place + 1 - a.window : 0;
    const Unpack unpack;
    h8 qh[D / 32], ql[TWO ? D / 32 : 1];
    float to_log2, s[8];
    load_queries<D, 16, BF16, TWO>(a.q, row * a.q.row + head * a.q.head, live, a.wide, a.scale_log2, qh, ql, to_log2);
    const float lse = live ? a.lse[row * a.heads + head] : 0.0f;
    tile_scores<D, TWO>(unpack, k, qh, ql, s);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int t = t0 + 8 * j + e;
        float sum = t < see_hi && t >= see_lo ? __builtin_amdgcn_exp2f(s[e] * to_log2 - lse) : 0.0f;
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) sum += __shfl_xor(sum, m);
        if (r == 0 && t < span.hi) {
            float *p = kv_account(kv, a.accounts, b, h, t);
            if (p) *p += sum;
        }
    }
}

// Scores that are kept for the accounts, at most; beyond, the keys are read a second time (16 sequences of up to 4096 tokens, 8 heads of 4
// queries: 5.8 us from 10 MB of scores, 34 us from the keys).
constexpr size_t kMostScoreBytes = (size_t)256 << 20;

// Pieces that all units together are cut into.  Per CU at D = 64 / 128 / 256: four, three, two, as many as run there at a time by LDS or one
// fewer.  (us a call at 1, 2, 3, 4, 6 a CU, D = 128: 32 sequences of up to 8192 tokens 65 55 52 53 50, one of 131072 39 38 39 39 42,
// one of 16384 14 15 15 17 17; D = 64, 16 of up to 8192 28 22 20 19 20; D = 256, 8 of up to 8192 38 30 36 36 42.)
int split_workgroups(int D) { return std::min(kMostWorkgroups, device_cu_count() * (D == 256 ? 2 : D == 128 ? 3 : 4)); }

// One call may hold prompts beside single tokens: where its sequences have on average, but for the longest, under half of the largest number of new tokens,
// and the page table has room for this many tiles, those of few rows are taken by the kernel for them, in launches of their own.  (With more than sixteen query heads a
// key head even single tokens have too many rows for it.)  (us a call with one kernel and with
// both, D = 128: 512 new tokens beside 31 single ones over 2000 to 8192, 8192 tiles: 185 75; 300 beside one over 131072: 585 59; 256 beside 31 over 1500, 1536
// tiles: 46 36; beside 31 over 500, 512 tiles: 23 30; 512 beside 7 over 1000, 256 tiles: 36 42.)
constexpr int64_t kMixedTiles = 1024;

// Row tiles that the sequences of a call have, at most.
int64_t row_tiles_of(const AttendArgs &a) { return (int64_t)a.kv.rows * a.group / kRowsTile + a.kv.seqs; }

template <int D, bool BF16> int attend(const AttendArgs &a, int max_tiles, hipStream_t s) {
    const KvCall &kv = a.kv;
    const unsigned heads = (unsigned)kv.kv_heads, seqs = (unsigned)kv.seqs;
    constexpr int NT = account_tiles<D, BF16>();
    // (workgroups for the accounts are laid out by the page table's width; a launch has fewer than 2^24 of them)
    if (a.accounts && ((a.row_pieces && (max_tiles + NT - 1) / NT >= 1 << 24) || (a.workgroups && !a.scores && (max_tiles + 3) / 4 >= 1 << 24)))
        return fail(GQ_ERR_INVALID, "kv_attention: accounts of up to %d tiles of a sequence: too many (pass the page table's first columns)", max_tiles);
    if (a.row_pieces) {
        const unsigned grid = (unsigned)(row_tiles_of(a) * kv.kv_heads * a.row_pieces);
        if (int rc = launch(a.accounts ? kv_rows_kernel<D, BF16, true> : kv_rows_kernel<D, BF16, false>, dim3(grid), dim3(64 * kRowsWaves), 0, s, a)) return rc;
        if (a.row_pieces > 1)
            if (int rc = launch(kv_rows_join_kernel<D, BF16>, dim3((unsigned)(((int64_t)kv.rows * a.heads * (D / 4) + 255) / 256)), dim3(256), 0, s, a)) return rc;
        if (a.accounts)
            if (int rc = launch(kv_rows_account_kernel<D, BF16>, dim3((unsigned)((max_tiles + NT - 1) / NT), heads, seqs), dim3(256), 0, s, a)) return rc;
    }
    if (a.workgroups) {
        const int grid = a.workgroups + kv.seqs * kv.kv_heads;  // (a unit's last piece may be short)
        if (int rc = launch(kv_split_kernel<D, BF16>, dim3((unsigned)grid), dim3(64 * kSplitWaves), 0, s, a)) return rc;
        if (a.pieces)
            if (int rc = launch(kv_join_kernel<D, BF16>, dim3((unsigned)a.rows, heads, seqs), dim3(256), 0, s, a)) return rc;
        if (!a.accounts) return GQ_OK;
        if (a.scores) return launch(kv_score_account_kernel, dim3((unsigned)((a.score_tiles + 7) / 8), heads, seqs), dim3(256), 0, s, a);
        return launch(kv_account_kernel<D, BF16>, dim3((unsigned)((max_tiles + 3) / 4), heads, seqs), dim3(256), 0, s, a);
    }
    return GQ_OK;
}

}  // namespace

int launch_kv_attention(const KvCall &kv, const HeadRows &q, int heads, float scale, int window, float *accounts, void *out, hipStream_t s) {
    AttendArgs a{};
    a.kv = kv;
    a.q = q;
    a.heads = heads;
    a.group = heads / kv.kv_heads;
    a.window = window;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.out = out;
    a.accounts = accounts;
    const int64_t size = q.bf16 ? 2 : 4;
    a.wide = ((reinterpret_cast<uintptr_t>(q.p) | (uintptr_t)(q.row * size) | (uintptr_t)(q.head * size)) & 15) == 0;
    // tiles that a unit's rows see, at most, and those that see any of the new tokens
    const int64_t room = (int64_t)kv.max_pages * kv.page_tokens / 32;
    const int64_t tiles = std::max<int64_t>(1, window ? std::min<int64_t>(room, ((int64_t)window + kv.max_new + 31) / 32 + 1) : room);
    const int64_t most_rows = (int64_t)kv.max_new * a.group;
    const bool many = most_rows > kSplitRows;
    const size_t line = (size_t)kv.rows * heads;
    size_t row_lines = 0, split_lines = 0;  // of sums that are joined
    a.few = many ? 0 : kSplitRows;
    if (many) {
        if (a.group <= kSplitRows && kv.starts && kv.seqs * tiles >= kMixedTiles && 2 * ((int64_t)kv.rows - kv.max_new) < (int64_t)(kv.seqs - 1) * kv.max_new) a.few = kSplitRows;
        // Pieces of a row tile's tokens: as many workgroups as run at a time (row tiles as if sequences had the same number of new tokens), each with enough
        // tokens for its start (us a call with 8, 12, 16, 32 tiles at least, D = 128: 512 tokens over 600 27 22 22 22, 64 of 4 sequences over 2000 31 29 30 36, 32 of
        // 2 over 8000 36 34 35 40; D = 64, 301 of 5 over 1111 in a window 43 43 48 49), and no more than pay for a launch and for the sums' way to memory and back: at
        // two pieces 8 tokens of 32 sequences over 4000 take 56 us for 94, 300 of 4 over 1000 59 for 52.
        const int64_t units = (((int64_t)kv.rows * a.group + kv.seqs - 1) / kv.seqs + kRowsTile - 1) / kRowsTile * kv.seqs * kv.kv_heads;
        const double tile_us = (kv.head_dim == 64 ? 0.5 : kv.head_dim == 128 ? 0.62 : 1.3) * (q.bf16 ? 1.0 : 1.6), sums_us = 2.0 * line * kv.head_dim * 4 / 4.5e6;  // (as measured, two workgroups a CU where they fit)
        int64_t pieces = std::min<int64_t>((kv.head_dim == 256 ? 1 : 2) * device_cu_count() / units, tiles / kRowsPiece);
        while (pieces > 1 && tiles * tile_us * (pieces - 1) < (4.0 + sums_us * pieces) * pieces) pieces--;
        a.row_pieces = (int)std::max<int64_t>(1, pieces);
        if (a.row_pieces > 1) row_lines = line * a.row_pieces;
        if (accounts) a.operand_tiles = (int)((int64_t)kv.rows * a.group / 32 + kv.seqs + 1);
    }
    if (a.few) {
        a.rows = (int)std::min<int64_t>(most_rows, kSplitRows);
        const int64_t all = (int64_t)kv.seqs * kv.kv_heads * tiles;
        a.workgroups = (int)std::min<int64_t>(split_workgroups(kv.head_dim), (all + kSplitWaves - 1) / kSplitWaves);
        if (tiles > kSplitWaves) split_lines = (size_t)(a.workgroups + kv.seqs * kv.kv_heads) * a.rows;
    }
    const size_t lines = std::max(row_lines, split_lines);  // (kv_split_kernel runs when the others' sums are done with)
    // scratch memory, each part on a line of its own
    size_t at = 0;
    const auto part = [&at](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t score_bytes = a.workgroups && accounts ? (size_t)kv.seqs * kv.kv_heads * a.rows * tiles * 128 : 0;
    const bool keep_scores = score_bytes > 0 && score_bytes <= kMostScoreBytes;
    const size_t operand_tiles = (size_t)a.operand_tiles * kv.kv_heads;
    const size_t lse = part(accounts ? line * 4 : 0), ml = part(lines * 8), sums = part(lines * (size_t)kv.head_dim * 4);
    const size_t pieces = part(split_lines ? (size_t)kv.seqs * kv.kv_heads * 8 : 0), scores = part(keep_scores ? score_bytes : 0);
    const size_t operands = part(operand_tiles * 32 * kv.head_dim * (q.bf16 ? 2 : 4)), row_scales = part(operand_tiles * 128);
    if (at) {
        void *ws = nullptr;
        if (int rc = stream_workspace(s, at, &ws)) return rc;
        unsigned char *p = static_cast<unsigned char *>(ws);
        if (accounts) a.lse = reinterpret_cast<float *>(p + lse);
        if (lines) {
            a.part_ml = reinterpret_cast<float *>(p + ml);
            a.part = reinterpret_cast<float *>(p + sums);
        }
        if (split_lines) a.pieces = reinterpret_cast<int2 *>(p + pieces);
        if (keep_scores) {
            a.scores = reinterpret_cast<float *>(p + scores);
            a.score_tiles = (int)tiles;
        }
        if (operand_tiles) {
            a.operands = p + operands;
            a.row_scales = reinterpret_cast<float *>(p + row_scales);
        }
    }
    switch (kv.head_dim) {
    case 64: return q.bf16 ? attend<64, true>(a, (int)tiles, s) : attend<64, false>(a, (int)tiles, s);
    case 128: return q.bf16 ? attend<128, true>(a, (int)tiles, s) : attend<128, false>(a, (int)tiles, s);
    default: return q.bf16 ? attend<256, true>(a, (int)tiles, s) : attend<256, false>(a, (int)tiles, s);
    }
}

}  // namespace gq
