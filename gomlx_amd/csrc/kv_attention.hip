// Softmax attention of the new tokens of every sequence over a 4-bit cache (layout: kv.hpp).
//
//     s_ij = scale q_i . k_j for the tokens j that row i sees (j <= p_i, and j > p_i - window where there is a window; p_i its own place)
//     o_i  = sum_j P_ij v_j,  P_i = softmax(s_i);  a row that sees nothing gets zeros
//     account_j += sum of P_ij over the rows and the query heads of the key head (where asked for)
//
// Both products run on v_mfma_f32_16x16x32_f16.  Keys and values are fp16 numbers as they stand (kv.hpp), q is scaled by a power
// of two per row and taken as one fp16 number (bf16: exact) or as the sum of two (fp32: 22 bits), P likewise as one (bf16) or
// two; scores, running maximum, sums and results are fp32.
//
// The first product is formed transposed, S^T = K Q^T: a lane holds one query (its column) and eight neighbouring tokens of the
// tile, so that maximum and sum are plain lane arithmetic and the weights are the second product's operand, O^T = V^T P^T,
// where they lie.  The reference of a row's exponents is set so that its largest weight so far is 2^6, and moves only when a weight
// would pass 2^14 (below fp16's largest number; small weights stay clear of its denormals): the lanes of the row then agree on a new one.
#include "kv.hpp"

#include <algorithm>
#include <cmath>

namespace gq {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kHeadroom = 6.0f;   // a row's largest weight is 2^6 when its reference is set ...
constexpr float kMostLog2 = 14.0f;  // ... and stays under 2^14

__device__ __forceinline__ h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ h2 both(float v) { h2 r = {(_Float16)v, (_Float16)v}; return r; }
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) { h8 r = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y}; return r; }

// Eight codes -> c - 8, exact: the nibbles become the low mantissa bits of 1024 (or, four places up, of 1024 + 16 c).
__device__ __forceinline__ void unpack(uint32_t w, h2 (&v)[4]) {
    const h2 sixteenth = both(0.0625f), low = both(-1032.0f), high = both(-72.0f);
    const uint32_t x = w >> 8;
    v[0] = as_h2((w & 0x000F000Fu) | 0x64006400u) + low;
    v[1] = __builtin_elementwise_fma(as_h2((w & 0x00F000F0u) | 0x64006400u), sixteenth, high);
    v[2] = as_h2((x & 0x000F000Fu) | 0x64006400u) + low;
    v[3] = __builtin_elementwise_fma(as_h2((x & 0x00F000F0u) | 0x64006400u), sixteenth, high);
}

struct AttendArgs {
    KvCall kv;
    HeadRows q;
    int heads, group, window, chunk_tiles, row_tiles, wide;
    float scale_log2;        // scale * log2(e)
    void *out;               // [rows, heads, D]
    float *lse;              // [rows, heads], in powers of two; null where nobody asks
    float *part, *part_ml;   // chunks > 1: sums [rows * heads, chunks, D], (reference, sum) [rows * heads, chunks, 2]
    int chunks;
    float *accounts;
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
        const int base = s.length - s.news;
        const int hi = base + (r.first_row + r.rows - 1) / group + 1;
        const int lo = window ? base + r.first_row / group + 1 - window : 0;
        r.hi = hi < 0 ? 0 : hi;
        r.lo = lo < 0 ? 0 : lo;
    }
    return r;
}

// Sixteen query rows as operands: lane (r, j) gets the values 32 g + 8 j + 0..7 of row r, times 2^e with the largest of the row in
// [2^11, 2^12); `back` is 2^-e.  TWO: a second operand with what the first has rounded off.
template <int D, bool BF16, bool TWO>
__device__ __forceinline__ void load_queries(const HeadRows &q, int64_t at, bool live, int wide, h8 (&hi)[D / 32], h8 (&lo)[TWO ? D / 32 : 1], float &back) {
    const int j = ((int)threadIdx.x & 63) >> 4;
    float x[D / 32][8];
    float most = 0.0f;
#pragma unroll
    for (int g = 0; g < D / 32; g++) {
        const int64_t p = at + 32 * g + 8 * j;
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
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    int e = 0;
    if (most > 0.0f && most < __builtin_huge_valf()) e = 12 - __builtin_amdgcn_frexp_expf(most);
    e = e > 100 ? 100 : e;  // (below 2^-88 the scores of a row are nothing)
    const float up = ldexpf(1.0f, e);
    back = ldexpf(1.0f, -e);
#pragma unroll
    for (int g = 0; g < D / 32; g++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = x[g][i] * up;
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
    __device__ __forceinline__ h8 operand(int u, int g) const {
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
    __device__ __forceinline__ h8 operand(int w) const {
        h2 v[4];
        unpack(code[w >> 2][w & 3], v);
        const u4 d = scale[w >> 1];
        return join(v[0] * as_h2(d[0]), v[1] * as_h2(d[1]), v[2] * as_h2(d[2]), v[3] * as_h2(d[3]));
    }
};

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The scores of a tile's 32 tokens for sixteen rows: lane (r, j) gets those of the tokens 8 j + 0..7 for row r.
template <int D, bool TWO>
__device__ __forceinline__ void tile_scores(const KeyWords<D> &k, const h8 (&hi)[D / 32], const h8 (&lo)[TWO ? D / 32 : 1], float (&s)[8]) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < D / 32; g++) {
            const h8 a = k.operand(u, g);
            acc = mfma(a, hi[g], acc);
            if constexpr (TWO) acc = mfma(a, lo[g], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[4 * u + i] = acc[i];
    }
}

constexpr int kSplitWaves = 4;

// Sixteen rows of one key head over one chunk of the tokens that they see.  Each wavefront takes every fourth tile with a
// maximum, sums and results of its own; they meet in LDS at the end.
template <int D, bool BF16>
__global__ __launch_bounds__(64 * kSplitWaves) void kv_split_kernel(const AttendArgs a) {
    constexpr bool TWO = !BF16;
    constexpr int W = D / 16;
    __shared__ float sums[kSplitWaves][16][D + 4];
    __shared__ float refs[kSplitWaves][16], totals[kSplitWaves][16];
    const KvCall &kv = a.kv;
    const int b = (int)blockIdx.z, h = (int)blockIdx.y;
    const int row_tile = (int)blockIdx.x / a.chunks, chunk = (int)blockIdx.x - row_tile * a.chunks;
    const KvSeq seq = kv_seq(kv, b);
    const Span span = row_tile_span(seq, a.group, a.window, row_tile, 16);
    if (span.rows == 0) return;
    const int tile0 = (span.lo >> 5) + chunk * a.chunk_tiles, tiles_end = (span.hi + 31) >> 5;
    if (chunk > 0 && tile0 >= tiles_end) return;
    const int tile1 = min(tile0 + a.chunk_tiles, tiles_end);

    const int lane = (int)threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int idx = span.first_row + r;
    const bool live = r < span.rows;
    const int nth = live ? idx / a.group : 0;            // new token of the row
    const int head = h * a.group + (live ? idx - nth * a.group : 0);
    const int64_t row = seq.row0 + nth;
    const int place = seq.length - seq.news + nth;       // its own token
    const int see_hi = live ? place + 1 : 0, see_lo = a.window ? place + 1 - a.window : 0;
    // tokens that every row of the tile sees
    const int all_hi = __builtin_amdgcn_readfirstlane(seq.length - seq.news + span.first_row / a.group + 1);
    const int all_lo = a.window ? seq.length - seq.news + (span.first_row + span.rows - 1) / a.group + 1 - a.window : 0;
    const bool full_rows = span.rows == 16;

    h8 qh[D / 32], ql[TWO ? D / 32 : 1];
    float back;
    load_queries<D, BF16, TWO>(a.q, row * a.q.row + head * a.q.head, live, a.wide, qh, ql, back);
    const float to_log2 = back * a.scale_log2;

    f4 o[W];
#pragma unroll
    for (int w = 0; w < W; w++) o[w] = f4{0.f, 0.f, 0.f, 0.f};
    float ref = kNegInf, total = 0.0f;  // the row's reference, and the lane's share of its sum

    for (int tile = tile0 + wave; tile < tile1; tile += kSplitWaves) {
        const uint8_t *at = kv_tile(kv, b, h, tile, KvTile<D>::kBytes);
        if (!at) continue;
        KeyWords<D> k;
        ValueWords<D> v;
        k.load(at);
        v.load(at);
        float s[8];
        tile_scores<D, TWO>(k, qh, ql, s);
        const int t0 = tile * 32;
        float most = kNegInf;
        if (full_rows && t0 >= all_lo && t0 + 32 <= all_hi) {
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
        if (__any(most > ref + kMostLog2)) {  // (the first score of a row among them: its reference is -infinity)
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float next = fmaxf(ref, most - kHeadroom);
            const float shrink = next == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ref - next);
            ref = next;
            total *= shrink;
#pragma unroll
            for (int w = 0; w < W; w++) o[w] *= shrink;
        }
        const float from = ref == kNegInf ? 0.0f : ref;
        h8 ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = __builtin_amdgcn_exp2f(s[e] - from);
            total += p;
            ph[e] = (_Float16)p;
            if constexpr (TWO) pl[e] = (_Float16)(p - (float)ph[e]);
        }
#pragma unroll
        for (int w = 0; w < W; w++) {
            const h8 x = v.operand(w);
            o[w] = mfma(x, ph, o[w]);
            if constexpr (TWO) o[w] = mfma(x, pl, o[w]);
        }
    }
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
#pragma unroll
    for (int w = 0; w < W; w++) *reinterpret_cast<f4 *>(&sums[wave][r][16 * w + 4 * j]) = o[w];
    if (j == 0) {
        refs[wave][r] = ref;
        totals[wave][r] = total;
    }
    __syncthreads();

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
        const int ii = span.first_row + rr, n = ii / a.group;
        const int64_t to = (int64_t)(seq.row0 + n) * a.heads + h * a.group + (ii - n * a.group);
        if (a.chunks > 1) {
            *reinterpret_cast<f4 *>(a.part + (to * a.chunks + chunk) * D + d) = sum;
            if (d == 0) {
                a.part_ml[(to * a.chunks + chunk) * 2] = top;
                a.part_ml[(to * a.chunks + chunk) * 2 + 1] = all;
            }
        } else {
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
            sum *= inv;
            if (all != all) sum = f4{all, all, all, all};
            if constexpr (BF16) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                bf16x4 y = {(__bf16)sum.x, (__bf16)sum.y, (__bf16)sum.z, (__bf16)sum.w};
                *reinterpret_cast<bf16x4 *>(static_cast<uint16_t *>(a.out) + to * D + d) = y;
            } else {
                *reinterpret_cast<f4 *>(static_cast<float *>(a.out) + to * D + d) = sum;
            }
            if (a.lse && d == 0) a.lse[to] = all == 0.0f ? kNegInf : top + __builtin_amdgcn_logf(all);
        }
    }
}

// Joins the chunks of a row: one workgroup per row and head.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttendArgs a) {
    constexpr int L = D / 4, S = 256 / L;  // lanes of a row's values, and the shares into which the chunks are divided
    __shared__ f4 sums[S][L];
    __shared__ float refs[S], totals[S];
    const int64_t row = blockIdx.x / a.heads;
    const int head = (int)(blockIdx.x - row * a.heads);
    int b = 0;
    if (a.kv.starts) {  // the sequence of the row
        int lo = 0, hi = a.kv.seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.kv.starts[mid] <= row) lo = mid;
            else hi = mid - 1;
        }
        b = lo;
    } else {
        b = (int)row;
    }
    const KvSeq seq = kv_seq(a.kv, b);
    const int n = (int)row - seq.row0;
    if (n < 0 || n >= seq.news) return;
    const Span span = row_tile_span(seq, a.group, a.window, (n * a.group + head % a.group) >> 4, 16);
    const int tiles = ((span.hi + 31) >> 5) - (span.lo >> 5);
    const int used = max(1, min(a.chunks, (tiles + a.chunk_tiles - 1) / a.chunk_tiles));
    const int l = (int)threadIdx.x % L, share = (int)threadIdx.x / L;
    const int64_t to = row * a.heads + head;
    float top = kNegInf, all = 0.0f;
    f4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int c = share; c < used; c += S) {
        const float ref = a.part_ml[(to * a.chunks + c) * 2], t = a.part_ml[(to * a.chunks + c) * 2 + 1];
        const f4 v = *reinterpret_cast<const f4 *>(a.part + (to * a.chunks + c) * D + l * 4);
        const float next = fmaxf(top, ref);
        const float fo = top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(top - next), fn = ref == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ref - next);
        sum = sum * fo + v * fn;
        all = (top == kNegInf ? all : all * fo) + (ref == kNegInf ? t : t * fn);
        top = next;
    }
    sums[share][l] = sum;
    if (l == 0) { refs[share] = top; totals[share] = all; }
    __syncthreads();
    if (share) return;
    top = kNegInf;
    for (int i = 0; i < S; i++) top = fmaxf(top, refs[i]);
    sum = f4{0.f, 0.f, 0.f, 0.f};
    all = 0.0f;
    for (int i = 0; i < S; i++) {
        const float f = refs[i] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(refs[i] - top);
        sum += sums[i][l] * f;
        all += refs[i] == kNegInf ? totals[i] : totals[i] * f;
    }
    sum *= all == 0.0f ? 0.0f : 1.0f / all;
    if (all != all) sum = f4{all, all, all, all};
    if constexpr (BF16) {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        bf16x4 y = {(__bf16)sum.x, (__bf16)sum.y, (__bf16)sum.z, (__bf16)sum.w};
        *reinterpret_cast<bf16x4 *>(static_cast<uint16_t *>(a.out) + to * D + l * 4) = y;
    } else {
        *reinterpret_cast<f4 *>(static_cast<float *>(a.out) + to * D + l * 4) = sum;
    }
    if (a.lse && l == 0) a.lse[to] = all == 0.0f ? kNegInf : top + __builtin_amdgcn_logf(all);
}

// The accounts: a wavefront owns a tile of a sequence and key head and goes over all rows that see it, so that every account is
// added to once, in one order.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_account_kernel(const AttendArgs a) {
    constexpr bool TWO = !BF16;
    const KvCall &kv = a.kv;
    const int h = (int)blockIdx.y, b = (int)blockIdx.z;
    const KvSeq seq = kv_seq(kv, b);
    const int base = seq.length - seq.news;
    const int first_tile = a.window ? max(0, base + 1 - a.window) >> 5 : 0;
    const int tile = __builtin_amdgcn_readfirstlane(first_tile + (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6));
    if (tile * 32 >= seq.length || seq.news == 0) return;
    const uint8_t *at = kv_tile(kv, b, h, tile, KvTile<D>::kBytes);
    if (!at) return;
    KeyWords<D> k;
    k.load(at);
    const int lane = (int)threadIdx.x & 63, r = lane & 15, j = lane >> 4, t0 = tile * 32;
    // the new tokens that see one of the tile's
    const int n0 = max(0, t0 - base), n1 = a.window ? min(seq.news, t0 + 31 + a.window - base) : seq.news;
    float sum[8] = {};
    for (int i0 = n0 * a.group; i0 < n1 * a.group; i0 += 16) {
        const int idx = i0 + r;
        const bool live = idx < n1 * a.group;
        const int nth = live ? idx / a.group : 0, head = h * a.group + (live ? idx - nth * a.group : 0);
        const int64_t row = seq.row0 + nth;
        const int place = base + nth, see_hi = live ? place + 1 : 0, see_lo = a.window ? place + 1 - a.window : 0;
        h8 qh[D / 32], ql[TWO ? D / 32 : 1];
        float back, s[8];
        load_queries<D, BF16, TWO>(a.q, row * a.q.row + head * a.q.head, live, a.wide, qh, ql, back);
        const float lse = live ? a.lse[row * a.heads + head] : 0.0f;
        tile_scores<D, TWO>(k, qh, ql, s);
        const float to_log2 = back * a.scale_log2;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int t = t0 + 8 * j + e;
            sum[e] += t < see_hi && t >= see_lo ? __builtin_amdgcn_exp2f(s[e] * to_log2 - lse) : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) sum[e] += __shfl_xor(sum[e], m);
        const int t = t0 + 8 * j + e;
        if (r == 0 && t < seq.length) {
            float *p = kv_account(kv, a.accounts, b, h, t);
            if (p) *p += sum[e];
        }
    }
}

template <int D, bool BF16> int attend(const AttendArgs &a, int max_tiles, hipStream_t s) {
    const KvCall &kv = a.kv;
    const dim3 grid((unsigned)(a.chunks * a.row_tiles), (unsigned)kv.kv_heads, (unsigned)kv.seqs);
    if (int rc = launch(kv_split_kernel<D, BF16>, grid, dim3(64 * kSplitWaves), 0, s, a)) return rc;
    if (a.chunks > 1)
        if (int rc = launch(kv_join_kernel<D, BF16>, dim3((unsigned)((int64_t)kv.rows * a.heads)), dim3(256), 0, s, a)) return rc;
    if (!a.accounts) return GQ_OK;
    return launch(kv_account_kernel<D, BF16>, dim3((unsigned)((max_tiles + 3) / 4), (unsigned)kv.kv_heads, (unsigned)kv.seqs), dim3(256), 0, s, a);
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
    a.row_tiles = (int)(((int64_t)kv.max_new * a.group + 15) / 16);
    // tiles that a row tile's chunks have to cover, and those that see any of the new tokens
    const int64_t room = (int64_t)kv.max_pages * kv.page_tokens / 32;
    const int span_new = 15 / a.group + 1;  // new tokens of a row tile, less one
    const int64_t tiles = std::max<int64_t>(1, window ? std::min<int64_t>(room, ((int64_t)window + span_new + 31) / 32 + 1) : room);
    const int64_t max_tiles = std::max<int64_t>(1, window ? std::min<int64_t>(room, ((int64_t)window + kv.max_new + 31) / 32 + 1) : room);
    const int64_t units = (int64_t)kv.seqs * kv.kv_heads * a.row_tiles;
    // about 1024 workgroups, each with a tile per wavefront at least
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>((1024 + units - 1) / units, (tiles + kSplitWaves - 1) / kSplitWaves));
    a.chunk_tiles = (int)((tiles + chunks - 1) / chunks + kSplitWaves - 1) / kSplitWaves * kSplitWaves;
    a.chunks = (int)((tiles + a.chunk_tiles - 1) / a.chunk_tiles);
    const size_t line = (size_t)kv.rows * heads;
    const size_t lse_bytes = accounts ? (line * 4 + 255) / 256 * 256 : 0, ml_bytes = a.chunks > 1 ? (line * a.chunks * 8 + 255) / 256 * 256 : 0;
    const size_t part_bytes = a.chunks > 1 ? line * a.chunks * (size_t)kv.head_dim * 4 : 0;
    if (lse_bytes + ml_bytes + part_bytes) {
        void *ws = nullptr;
        if (int rc = stream_workspace(s, lse_bytes + ml_bytes + part_bytes, &ws)) return rc;
        unsigned char *p = static_cast<unsigned char *>(ws);
        if (lse_bytes) a.lse = reinterpret_cast<float *>(p);
        a.part_ml = reinterpret_cast<float *>(p + lse_bytes);
        a.part = reinterpret_cast<float *>(p + lse_bytes + ml_bytes);
    }
    switch (kv.head_dim) {
    case 64: return q.bf16 ? attend<64, true>(a, (int)max_tiles, s) : attend<64, false>(a, (int)max_tiles, s);
    case 128: return q.bf16 ? attend<128, true>(a, (int)max_tiles, s) : attend<128, false>(a, (int)max_tiles, s);
    default: return q.bf16 ? attend<256, true>(a, (int)max_tiles, s) : attend<256, false>(a, (int)max_tiles, s);
    }
}

}  // namespace gq
