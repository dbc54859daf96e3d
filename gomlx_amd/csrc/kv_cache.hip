// The 4-bit cache's writer and reader, and the eviction of the tokens that attention has least looked at (layout: kv.hpp).
#include "kv.hpp"

#include <algorithm>

namespace gq {

namespace {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLargest = 65408.0f;  // from here on -m / 8 rounds to more than 8160, and 8 d is no fp16 number
constexpr uint32_t kNanHalf = 0x7E00u;

__device__ __forceinline__ uint32_t half_bits(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ float half_value(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }
__device__ __forceinline__ float round_to_bf16(float v) {  // of finite v, to nearest even
    const uint32_t u = __float_as_uint(v);
    return __uint_as_float((u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u);
}
// where element e of a dword lies
__device__ __forceinline__ int nibble_shift(int e) { return ((e >> 1) + 4 * (e & 1)) * 4; }

// Eight neighbouring values.
template <bool BF16> __device__ __forceinline__ void load8(float (&v)[8], const void *p, int64_t at, int wide) {
    if constexpr (BF16) {
        const uint16_t *x = static_cast<const uint16_t *>(p) + at;
        u4 w;
        if (wide) w = *reinterpret_cast<const u4 *>(x);
        else w = u4{x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
        const float *x = static_cast<const float *>(p) + at;
        if (wide) {
            const float4 lo = *reinterpret_cast<const float4 *>(x), hi = *reinterpret_cast<const float4 *>(x + 4);
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
            v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = x[i];
        }
    }
}

// A group's scale, from the eight values of each of its four lanes: minus an eighth of the value of largest magnitude (the
// first of those), rounded to 8 significant bits.  The value itself then has code 0 and none is more than 8 steps away.
__device__ __forceinline__ float group_scale(const float (&v)[8]) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < 8; i++) m = fabsf(v[i]) > fabsf(m) ? v[i] : m;
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
        const float o = __shfl_xor(m, s);
        const bool take = fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && ((int)threadIdx.x & s));
        m = take ? o : m;
    }
    return half_value(half_bits(round_to_bf16(m * -0.125f)));
}
// floor(v / d + 8.5) within 0 .. 15, the quotient rounded once: inv is 1 / d rounded to nearest, and a product with it, corrected by its
// exact remainder, is then the rounded quotient (quotients so small that the remainder leaves fp32's range give 8 either way).
__device__ __forceinline__ uint32_t code_of(float v, float d, float inv) {
    const float q = v * inv, quotient = fmaf(fmaf(-q, d, v), inv, q);
    return (uint32_t)fminf(fmaxf(floorf(quotient + 8.5f), 0.0f), 15.0f);
}

// How the writer and the reader share out a call: a wavefront takes a block of eight tokens of a sequence and key head.  They are laid out for the longest of a call's
// sequences, `blocks` a sequence; or, `together`, `blocks` a key head for all sequences, as many as the rows can need, which wavefronts look up by a sum over the
// sequences, 64 at a time, one a lane.  That is taken where the first layout would be more than run at a time, and more than the second by what the sums cost.  (us a call of
// the writer with either, 8 heads of D = 128, new tokens: 512 beside 31 single ones 8.4 6.1, beside 7 6.0 6.0; 8192 beside 255 365 19; 128 beside 255 14 7.9; 100
// beside 2047 60 47; 32 beside 1023 22 27; 300 of 4 sequences 6.3 6.6.  The reader 4.8 4.5, 4.6 4.4, 295 12, 7.9 5.3, 39 32, 11 18, 4.7 4.9.)
struct Layout { int blocks, together; };
Layout layout_of(const KvCall &kv) {
    // blocks that a sequence's rows touch at most, and all rows: one row one, up to nine two, ...
    const int64_t each = (kv.max_new + 14) / 8, all = std::min<int64_t>(kv.rows, 2 * (int64_t)kv.seqs) + kv.rows / 8;
    const bool together = kv.starts && kv.seqs * each * kv.kv_heads > 32 * device_cu_count() && kv.seqs * each > all * (256 + kv.seqs) / 256;
    return Layout{(int)(together ? all : each), together};
}
// Threads of a launch are counted in 32 bits.
int wavefronts_of(const char *fn, const KvCall &kv, const Layout &layout, unsigned *workgroups) {
    const int64_t units = (int64_t)kv.kv_heads * layout.blocks * (layout.together ? 1 : kv.seqs);
    if (units >= (int64_t)1 << 26) return fail(GQ_ERR_INVALID, "%s: %d rows of %d sequences and %d key heads: too many", fn, kv.rows, kv.seqs, kv.kv_heads);
    *workgroups = (unsigned)((units + 3) / 4);
    return GQ_OK;
}

struct Block { int b, h, nth; KvSeq s; };  // of the sequence's blocks; b < 0: there is none
// COUNT(sequence): the blocks that its rows touch
template <class COUNT> __device__ __forceinline__ Block block_of(const KvCall &kv, const Layout &layout, int unit, COUNT count) {
    Block r;
    if (!layout.together) {
        const int per = kv.kv_heads * layout.blocks;
        r.b = unit / per;
        if (r.b >= kv.seqs) { r.b = -1; return r; }
        const int rest = unit - r.b * per;
        r.h = rest / layout.blocks;
        r.nth = rest - r.h * layout.blocks;
        r.s = kv_seq(kv, r.b);
        if (r.nth >= count(r.s)) r.b = -1;
        return r;
    }
    const int index = unit / kv.kv_heads, lane = (int)threadIdx.x & 63;
    r.h = unit - index * kv.kv_heads;
    r.b = -1;
    int front = 0;
    for (int base = 0; base < kv.seqs; base += 64) {
        KvSeq mine{};
        if (base + lane < kv.seqs) mine = kv_seq(kv, base + lane);
        const int blocks = count(mine), upto = lane_scan(blocks);
        const uint64_t past = __ballot(front + upto > index);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            r.b = base + l;
            r.s = seq_of_lane(mine, l);
            r.nth = index - (front + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(blocks, l));
            break;
        }
        front += __builtin_amdgcn_readlane(upto, 63);
    }
    return r;
}

// Eight tokens of one block (a lane's share of a value operand: their codes share dwords) per wavefront, key head and sequence.
// A lane takes eight values of a token, D / 8 lanes a token, and D / 64 rounds the block: a lane's key codes are one dword.  Its
// value codes are eight dwords that other lanes hold other tokens of; the lanes of equal values exchange halves until each has
// D / 64 whole ones.  A dword belongs to one lane of one wavefront of the launch, so that tokens that share bytes need no atomics.
//
// A few new tokens: the chain length -> page -> bytes of a partly filled dword bounds it (5.6 us for one token of each of 32 sequences, 8 heads
// of D = 128); many: the inputs' bytes (2653 tokens of 7 prompts in float32, 25 MB read and written: 10.7 us, 2.3 TB/s).
struct AppendArgs {
    KvCall kv;
    HeadRows k, v;
    float *accounts;
    Layout layout;
    int wide;
};

template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
    typedef KvTile<D> T;
    constexpr int G = T::G, L = D / 8, ROUNDS = D / 64, PER = 8 / ROUNDS;  // lanes of a token, rounds, tokens of a round
    const KvCall &kv = a.kv;
    const int unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int lane = (int)threadIdx.x & 63, l = lane % L, x = l * 8, mine = lane / L;  // the lane's values; its token of a round
    const int g = x >> 5;
    float k[ROUNDS][8], v[ROUNDS][8];
    if (!kv.starts) {  // one row, which is known before the sequence's length is: whichever of the eight tokens it turns out to be
        const int b = unit / kv.kv_heads, h = unit - b * kv.kv_heads;
        if (b >= kv.seqs) return;
        load8<BF16>(k[0], a.k.p, (int64_t)b * a.k.row + h * a.k.head + x, a.wide);
        load8<BF16>(v[0], a.v.p, (int64_t)b * a.v.row + h * a.v.head + x, a.wide);
    }
    const Block block = block_of(kv, a.layout, unit, [](const KvSeq &s) {
        const int from = max(s.first, 0), end = min(s.first + s.news, s.length);
        return end > from ? ((end + 7) >> 3) - (from >> 3) : 0;
    });
    if (block.b < 0) return;
    const KvSeq &s = block.s;
    const int b = block.b, h = block.h;
    const int first = s.first, from = max(first, 0), end = min(first + s.news, s.length);  // new tokens that have a place: from .. end - 1
    const int p0 = (from & ~7) + block.nth * 8;
    uint8_t *tile = kv_tile(kv, b, h, p0 >> 5, T::kBytes);
    if (!tile) return;
    const int j = (p0 >> 3) & 3;
    const bool account = a.accounts && l == 0;
    const int live_from = from > p0 ? from - p0 : 0, live_to = end - p0 < 8 ? end - p0 : 8;  // new tokens of the block
    uint32_t live_mask = 0;
    for (int e = live_from; e < live_to; e++) live_mask |= 0xFu << nibble_shift(e);
    // the dwords of value codes that the lane will finish, where other tokens share them
    uint32_t *value_at[ROUNDS], old[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int c = x + mine * ROUNDS + i;
        value_at[i] = reinterpret_cast<uint32_t *>(tile + T::kValues + T::code(c >> 4, (c & 15) + 16 * j));
        old[i] = live_mask == 0xFFFFFFFFu ? 0u : *value_at[i];
    }
    if (kv.starts) {
#pragma unroll
        for (int n = 0; n < ROUNDS; n++) {
            const int e = n * PER + mine;
            const int64_t row = s.row0 + min(max(p0 + e - first, 0), s.news - 1);
            load8<BF16>(k[n], a.k.p, row * a.k.row + h * a.k.head + x, a.wide);
            load8<BF16>(v[n], a.v.p, row * a.v.row + h * a.v.head + x, a.wide);
        }
    } else {
#pragma unroll
        for (int n = 1; n < ROUNDS; n++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                k[n][i] = k[0][i];
                v[n][i] = v[0][i];
            }
    }
    uint32_t bits[8] = {};
#pragma unroll
    for (int n = 0; n < ROUNDS; n++) {
        const int e = n * PER + mine, p = p0 + e;
        const bool live = e >= live_from && e < live_to;
        bool good = true;
#pragma unroll
        for (int i = 0; i < 8; i++) good = good && fabsf(k[n][i]) < kLargest && fabsf(v[n][i]) < kLargest;
        const uint64_t token = (L == 64 ? ~0ull : ((1ull << (L & 63)) - 1)) << (mine * L);
        good = (__ballot(good) & token) == token;
        if (!good) {
#pragma unroll
            for (int i = 0; i < 8; i++) k[n][i] = v[n][i] = 0.0f;
        }
        const float dk = group_scale(k[n]), dv = group_scale(v[n]);
        const float ik = dk == 0.0f ? 0.0f : 1.0f / dk, iv = dv == 0.0f ? 0.0f : 1.0f / dv;  // (no scale: every code is 8)
        uint32_t word = 0;
        const int at = nibble_shift(e);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            word |= code_of(k[n][i], dk, ik) << nibble_shift(i);
            bits[i] |= (live ? code_of(v[n][i], dv, iv) : 0u) << at;
        }
        if (live) {
            const int t = p & 31;
            *reinterpret_cast<uint32_t *>(tile + T::kKeys + T::code(key_half(t) * G + g, key_row(t) + 16 * (l & 3))) = word;
            if ((l & 3) == 0) {
                reinterpret_cast<uint16_t *>(tile + T::kKeyScales)[t * G + g] = (uint16_t)(good ? half_bits(dk) : kNanHalf);
                reinterpret_cast<uint16_t *>(tile + T::kValueScales)[g * 32 + t] = (uint16_t)half_bits(dv);
            }
            if (account) {
                float *q = kv_account(kv, a.accounts, b, h, p);
                if (q) *q = 0.0f;
            }
        }
    }
    // Lanes of equal values, L, 2 L, ... apart, pass each other the dwords that the other one finishes: lane `mine` of them those from mine * ROUNDS on.
    int count = 8;
#pragma unroll
    for (int m = 32; m >= L; m >>= 1) {
        count >>= 1;
        const bool upper = lane & m;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i >= count) break;
            const uint32_t give = upper ? bits[i] : bits[i + count], keep = upper ? bits[i + count] : bits[i];
            bits[i] = keep | (uint32_t)__shfl_xor((int)give, m);
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) *value_at[i] = (old[i] & ~live_mask) | bits[i];
}

// What the cache stands for at the last tokens of every sequence, in the fp16 numbers that it holds; zeros in front of a
// sequence's first token, behind the page table's end and where it names no page.  A wavefront takes its eight tokens one behind the other, each with loads of its own under a branch: for few tokens these
// round trips bound it (7.4 us for the 17 MB of the 7 prompts above, 2.3 TB/s), for many HBM's rate (16 sequences of 4096 tokens, 342 MB: 70 us, 4.9 TB/s).
template <int D>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvCall kv, uint16_t *__restrict__ K, uint16_t *__restrict__ V, const Layout layout) {
    typedef KvTile<D> T;
    constexpr int NE = D / 64, G = T::G;
    // (blocks of eight also in front of the first token)
    const Block block = block_of(kv, layout, __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6))),
                                 [](const KvSeq &s) { return s.news ? ((s.first + s.news + 7) >> 3) - (s.first >> 3) : 0; });
    if (block.b < 0) return;
    const KvSeq &s = block.s;
    const int b = block.b, h = block.h;
    const int first = s.first, end = first + s.news;
    const int p0 = (first & ~7) + block.nth * 8;
    const uint8_t *tile = p0 >= 0 && p0 < s.length ? kv_tile(kv, b, h, p0 >> 5, T::kBytes) : nullptr;
    const int lane = (int)threadIdx.x & 63, x = lane * NE, j = (p0 >> 3) & 3, g = x >> 5;
    uint32_t vw[NE] = {};
    if (tile) {
#pragma unroll
        for (int i = 0; i < NE; i++) vw[i] = *reinterpret_cast<const uint32_t *>(tile + T::kValues + T::code((x + i) >> 4, ((x + i) & 15) + 16 * j));
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int p = p0 + e;
        if (p < first || p >= end) continue;
        uint16_t k[NE] = {}, v[NE] = {};
        if (tile) {
            const int t = p & 31, w = key_half(t) * G + g, l = key_row(t) + 16 * ((x >> 3) & 3);
            const uint32_t kw = *reinterpret_cast<const uint32_t *>(tile + T::kKeys + T::code(w, l));
            const float dk = half_value(reinterpret_cast<const uint16_t *>(tile + T::kKeyScales)[t * G + g]);
            const float dv = half_value(reinterpret_cast<const uint16_t *>(tile + T::kValueScales)[g * 32 + t]);
#pragma unroll
            for (int i = 0; i < NE; i++) {
                k[i] = (uint16_t)half_bits(((float)((kw >> nibble_shift((x + i) & 7)) & 15u) - 8.0f) * dk);
                v[i] = (uint16_t)half_bits(((float)((vw[i] >> nibble_shift(e)) & 15u) - 8.0f) * dv);
            }
        }
        const int64_t to = ((int64_t)(s.row0 + (p - first)) * kv.kv_heads + h) * D + x;
        if constexpr (NE == 1) {
            K[to] = k[0];
            V[to] = v[0];
        } else if constexpr (NE == 2) {
            *reinterpret_cast<uint32_t *>(K + to) = k[0] | (uint32_t)k[1] << 16;
            *reinterpret_cast<uint32_t *>(V + to) = v[0] | (uint32_t)v[1] << 16;
        } else {
            *reinterpret_cast<u2 *>(K + to) = u2{k[0] | (uint32_t)k[1] << 16, k[2] | (uint32_t)k[3] << 16};
            *reinterpret_cast<u2 *>(V + to) = u2{v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16};
        }
    }
}

// ---- eviction ---------------------------------------------------------------------------------------------------------
//
// kept[b][h] = the last `recent` tokens and the keep - recent others of largest account, in order; ties go to the lower token.
// The account's order as whole numbers: NaN above everything, -0 equal to 0.
__device__ __forceinline__ uint32_t account_key(float f) {
    if (f != f) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(f + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048, kFew = 512;

// The sum of v over the threads in front, and over all.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *waves, uint32_t &total) {
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    const uint32_t inc = (uint32_t)lane_scan((int)v);
    __syncthreads();  // (the previous use of `waves` is over)
    if (lane == 63) waves[w] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelectWaves; i++) {
        const uint32_t n = waves[i];
        before += i < w ? n : 0;
        all += n;
    }
    total = all;
    return before + inc - v;
}

// One workgroup per sequence and key head.  A wavefront owns a run of neighbouring tokens, 64 at a time, and holds their keys in
// registers where IT rounds of them suffice, in LDS where kLdsRounds do (IT = kInLds; IT = 0: reads them again for every pass).  The smallest kept key is found digit by
// digit, eleven bits at a time of its distance from the smallest key there is, so that keys of similar size spread over the
// histogram (those that equal the smallest, zeros mostly, are left out of it), until so few are left that each is held against all of them; a wavefront then counts what it keeps, and
// writes its tokens behind those of the wavefronts in front.
// The passes' barriers bound it, one behind the other: 10 us for 8 heads of one sequence of 4096 tokens, 28 us for those of 16 sequences of 4096 to 16384.  20
// heads of 7000 to 28000 tokens: the keys in LDS 40 us, read again for every pass 71.
constexpr int kInLds = -1, kLdsRounds = 32;
template <int IT>
__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(const KvCall kv, const float *__restrict__ accounts, int keep, int recent, int32_t *__restrict__ kept) {
    __shared__ uint32_t hist[kBins], waves[kSelectWaves], found[2], ends[3][kSelectWaves], few[kFew], count;
    const int h = (int)blockIdx.x, b = (int)blockIdx.y, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const KvSeq s = kv_seq(kv, b);
    int32_t *out = kept + ((int64_t)b * kv.kv_heads + h) * keep;
    if (s.length <= keep) {
        for (int i = tid; i < keep; i += kSelectThreads) out[i] = i < s.length ? i : -1;
        return;
    }
    const int n = s.length - recent;
    uint32_t want = (uint32_t)(keep - recent);  // of the first n tokens (n > want)
    for (int i = tid; i < recent; i += kSelectThreads) out[want + i] = n + i;
    if (want == 0) return;
    const int rounds = IT > 0 ? IT : (n + kSelectThreads - 1) / kSelectThreads;
    const int t0 = wave * rounds * 64 + lane;
    // (an account without a page counts as the smallest)
    const auto key_at = [&](int t) {
        const float *p = kv_account(kv, const_cast<float *>(accounts), b, h, t);
        return p ? account_key(*p) : 0u;
    };
    uint32_t keys[IT > 0 ? IT : 1];
    extern __shared__ uint32_t lds_keys[];  // [round][thread]: a thread reads what it has written
    if constexpr (IT > 0) {
        // (loads without branches between them, of the last token where there is none: they go out together)
        int64_t at[IT];
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int t = min(t0 + 64 * i, n - 1), slot = page_slot(kv, t >> 5), page = kv.table[b * kv.table_stride + slot];
            at[i] = (uint32_t)page < (uint32_t)kv.pages ? ((int64_t)page * kv.kv_heads + h) * kv.page_tokens + (t - slot * kv.page_tokens) : -1;
        }
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const uint32_t u = kv.pages ? account_key(accounts[max(at[i], (int64_t)0)]) : 0u;
            keys[i] = at[i] < 0 ? 0u : u;
        }
    } else if constexpr (IT == kInLds) {
#pragma unroll 8
        for (int i = 0; i < rounds; i++) {
            const int t = min(t0 + 64 * i, n - 1), slot = page_slot(kv, t >> 5), page = kv.table[b * kv.table_stride + slot];
            const bool there = (uint32_t)page < (uint32_t)kv.pages;
            const int64_t at = there ? ((int64_t)page * kv.kv_heads + h) * kv.page_tokens + (t - slot * kv.page_tokens) : 0;
            const uint32_t u = kv.pages ? account_key(accounts[at]) : 0u;
            lds_keys[i * kSelectThreads + tid] = there ? u : 0u;
        }
    }
    const auto each = [&](auto f) {  // f(token, key) for the thread's tokens
        if constexpr (IT > 0) {
#pragma unroll
            for (int i = 0; i < IT; i++)
                if (t0 + 64 * i < n) f(t0 + 64 * i, keys[i]);
        } else if constexpr (IT == kInLds) {
#pragma unroll 4
            for (int i = 0; i < rounds; i++)
                if (t0 + 64 * i < n) f(t0 + 64 * i, lds_keys[i * kSelectThreads + tid]);
        } else {
            for (int i = 0; i < rounds; i++)
                if (t0 + 64 * i < n) f(t0 + 64 * i, key_at(t0 + 64 * i));
        }
    };
    // the smallest key, the smallest but for accounts of 0, and the largest
    uint32_t low = 0xFFFFFFFFu, next = 0xFFFFFFFFu, high = 0;
    const uint32_t zero = account_key(0.0f);
    each([&](int, uint32_t u) {
        low = min(low, u);
        next = min(next, u == zero ? 0xFFFFFFFFu : u);
        high = max(high, u);
    });
    const auto least = [](int a, int b) { return (int)min((uint32_t)a, (uint32_t)b); };
    const auto most = [](int a, int b) { return (int)max((uint32_t)a, (uint32_t)b); };
    low = (uint32_t)lane_scan((int)low, -1, least);
    next = (uint32_t)lane_scan((int)next, -1, least);
    high = (uint32_t)lane_scan((int)high, 0, most);
    if (lane == 63) { ends[0][wave] = low; ends[1][wave] = high; ends[2][wave] = next; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSelectWaves; i++) {
        low = i ? min(low, ends[0][i]) : ends[0][0];
        high = i ? max(high, ends[1][i]) : ends[1][0];
        next = i ? min(next, ends[2][i]) : ends[2][0];
    }
    __syncthreads();
    // Digits of the distance from the smallest key (zeros, which many are, lie far below the others: from the next one then); `want` counts down to
    // how many of the tokens that equal the key are kept.
    uint32_t key = low == zero && next != 0xFFFFFFFFu ? next : low;  // the smallest key that the open bits allow
    int width = 32 - __clz(high - min(key, high));  // bits that are open (0: every key is the same, or one more than the smallest)
    if (key != low && width == 0) width = 1;
    while (width > 0) {
        const int shift = width > 11 ? width - 11 : 0;
        const uint32_t top = width < 32 ? 1u << width : 0u;  // keys from key to key + top - 1 are looked at (0: all)
        for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        each([&](int, uint32_t u) {
            const uint32_t at = u - key;
            if (u > low && u >= key && (top == 0 || at < top)) atomicAdd(&hist[at >> shift], 1u);
        });
        __syncthreads();
        const int bin = kBins - 1 - 2 * tid;  // the largest digits first, two a thread
        const uint32_t first = hist[bin], second = hist[bin - 1];
        uint32_t total;
        const uint32_t before = block_scan(first + second, waves, total);
        if (before < want && want <= before + first) { found[0] = (uint32_t)bin; found[1] = want - before; }
        else if (before + first < want && want <= before + first + second) { found[0] = (uint32_t)bin - 1; found[1] = want - before - first; }
        if (tid == 0 && want > total) { found[0] = 0xFFFFFFFFu; found[1] = want - total; }  // down to those that equal the smallest
        __syncthreads();
        const uint32_t digit = found[0], left = digit == 0xFFFFFFFFu ? 0u : hist[digit];
        want = found[1];
        __syncthreads();  // (from here on the next pass may clear hist and set found)
        if (digit == 0xFFFFFFFFu) {
            key = low;
            break;
        }
        key += digit << shift;
        width = shift;
        if (width == 0 || left > kFew) continue;
        // few are left: each against all of them
        if (tid == 0) count = 0;
        __syncthreads();
        each([&](int, uint32_t u) {
            if (u > low && u >= key && u - key < (1u << width)) few[atomicAdd(&count, 1u)] = u;
        });
        __syncthreads();
        const uint32_t all = count, mine = (uint32_t)tid < all ? few[tid] : 0;
        if ((uint32_t)tid < all) {
            uint32_t above = 0, same = 0;
            for (uint32_t i = 0; i < all; i++) {
                above += few[i] > mine;
                same += few[i] == mine;
            }
            if (above < want && want <= above + same) { found[0] = mine; found[1] = want - above; }  // (all that equal it write the same)
        }
        __syncthreads();
        key = found[0];
        want = found[1];
        break;
    }
    // u > key stay, and the first `want` that equal it
    uint32_t more = 0, same = 0;
    each([&](int, uint32_t u) {
        more += u > key;
        same += u == key;
    });
    const uint32_t mores = (uint32_t)lane_scan((int)more), sames = (uint32_t)lane_scan((int)same);
    if (lane == 63) { ends[0][wave] = mores; ends[1][wave] = sames; }
    __syncthreads();
    uint32_t at = 0, equal = 0;  // kept, and equal to the key, in front
    for (int i = 0; i < wave; i++) {
        const uint32_t e = ends[1][i];
        at += ends[0][i] + (equal < want ? min(e, want - equal) : 0);
        equal += e;
    }
    const auto place = [&](int t, uint32_t u) {  // the whole wavefront, tokens in order of lanes
        const uint64_t below = (1ull << lane) - 1;
        const bool here = t < n, is = here && u == key;
        const uint64_t equals = __ballot(is);
        const bool stays = here && (u > key || (is && equal + (uint32_t)__popcll(equals & below) < want));
        const uint64_t stay = __ballot(stays);
        if (stays) out[at + (uint32_t)__popcll(stay & below)] = t;
        at += (uint32_t)__popcll(stay);
        equal += (uint32_t)__popcll(equals);
    };
    if constexpr (IT > 0) {
#pragma unroll
        for (int i = 0; i < IT; i++) place(t0 + 64 * i, keys[i]);
    } else {
        for (int i = 0; i < rounds; i++) place(t0 + 64 * i, IT == kInLds ? lds_keys[i * kSelectThreads + tid] : t0 + 64 * i < n ? key_at(t0 + 64 * i) : 0u);
    }
}

// Moves the kept tokens of a sequence and key head to its front, in place.  kept[i] >= i, so that a workgroup that reads its next
// tokens before it writes the present ones, and goes from the front to the back, never overwrites what it has yet to read.
// Workgroups share a head by what they move, not by tokens: blockIdx.z = 0 .. 3 the key codes of lanes 16 j .. 16 j + 15, then four
// for every 64 values (the value codes of every fourth operand row's neighbours), and one for scales and accounts.
// 9 us for 2048 tokens of 8 heads; 84 us for 16 sequences of 4096 of up to 16384 (8 heads, D = 128, 74 MB to write): single tokens are picked out of
// tiles whose lines hold four of them (key codes) or eight (value codes), and the steps of a head follow each other.
constexpr int kMoveThreads = 256, kMoveTokens = 1024;

// Every thread's loads are back: what the workgroup writes from here on is not what one of its wavefronts still reads.
__device__ __forceinline__ void all_read() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

template <int D>
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(const KvCall kv, float *accounts, int keep, const int32_t *__restrict__ kept, int32_t *new_lengths) {
    typedef KvTile<D> T;
    constexpr int G = T::G, R = kMoveTokens / kMoveThreads;
    __shared__ int64_t sources[2][kMoveTokens];  // tile * 32 + token in it
    const int h = (int)blockIdx.x, b = (int)blockIdx.y, part = (int)blockIdx.z, tid = (int)threadIdx.x;
    const int32_t *list = kept + ((int64_t)b * kv.kv_heads + h) * keep;
    // (new_lengths may be kv.lengths: nobody else reads them in this launch)
    if (h == 0 && part == 0 && tid == 0) new_lengths[b] = min(kv_seq(kv, b).length, keep);
    if (list[keep - 1] < keep || kv.pages == 0) return;  // nothing to move: as many tokens as places, or fewer (-1)
    const int per_page = kv.page_tokens >> 5;
    const auto tile_number = [&](int tile) -> int64_t {
        const int slot = min(page_slot(kv, tile), kv.max_pages - 1), page = kv.table[b * kv.table_stride + slot];
        return (uint32_t)page < (uint32_t)kv.pages && tile - slot * per_page < per_page ? ((int64_t)page * kv.kv_heads + h) * per_page + (tile - slot * per_page) : -1;
    };
    // Where the tokens of a step come from, found out a step ahead.  (-1 behind the last one, and where the page table names no page: nothing is written there;
    // what is read for it is the cache's first tile, so that loads need no branches between them and go out together.)
    int entry[R];
    bool stay;  // the thread's tokens of the step are where they belong
    const auto ask = [&](int i0) {
#pragma unroll
        for (int n = 0; n < R; n++) {
            const int i = i0 + n * kMoveThreads + tid;
            entry[n] = i < keep ? list[i] : -1;
        }
    };
    const auto found = [&](int64_t *to, int at) {
        int64_t tile[R];
#pragma unroll
        for (int n = 0; n < R; n++) tile[n] = tile_number(max(entry[n], 0) >> 5);
#pragma unroll
        for (int n = 0; n < R; n++) to[n * kMoveThreads + tid] = entry[n] < 0 || tile[n] < 0 ? -1 : tile[n] * 32 + (entry[n] & 31);
        stay = true;
#pragma unroll
        for (int n = 0; n < R; n++) stay = stay && (entry[n] < 0 || entry[n] == at + n * kMoveThreads + tid);
    };
    ask(0);
    found(sources[0], 0);
    for (int i0 = 0, turn = 0; i0 < keep; i0 += kMoveTokens, turn ^= 1) {
        const int64_t *source = sources[turn];
        const bool all_stay = __syncthreads_and(stay);
        ask(i0 + kMoveTokens);
        if (all_stay) {
            found(sources[turn ^ 1], i0 + kMoveTokens);
            continue;
        }
        if (part < 4) {  // one token a thread and round: its dwords of lane part
            u4 code[R][(G + 3) / 4];
            int64_t from[R], to[R];
#pragma unroll
            for (int n = 0; n < R; n++) to[n] = tile_number(min(i0 + n * kMoveThreads + tid, keep - 1) >> 5);
#pragma unroll
            for (int n = 0; n < R; n++) {
                from[n] = source[n * kMoveThreads + tid];
                const int64_t some = max(from[n], (int64_t)0);
                const int t = (int)some & 31;
                const uint8_t *at = kv.cache + (some >> 5) * T::kBytes + T::kKeys + T::code(key_half(t) * G, key_row(t) + 16 * part);
                if constexpr (G == 2) {
                    const u2 w = *reinterpret_cast<const u2 *>(at);
                    code[n][0] = u4{w.x, w.y, 0, 0};
                } else {
#pragma unroll
                    for (int c = 0; c < G / 4; c++) code[n][c] = *reinterpret_cast<const u4 *>(at + c * 1024);
                }
            }
            found(sources[turn ^ 1], i0 + kMoveTokens);
            all_read();
#pragma unroll
            for (int n = 0; n < R; n++) {
                const int i = i0 + n * kMoveThreads + tid;
                if (from[n] < 0 || to[n] < 0) continue;
                const int t = i & 31;
                uint8_t *at = kv.cache + to[n] * T::kBytes + T::kKeys + T::code(key_half(t) * G, key_row(t) + 16 * part);
                if constexpr (G == 2) {
                    *reinterpret_cast<u2 *>(at) = u2{code[n][0].x, code[n][0].y};
                } else {
#pragma unroll
                    for (int c = 0; c < G / 4; c++) *reinterpret_cast<u4 *>(at + c * 1024) = code[n][c];
                }
            }
        } else if (part < 4 + D / 16) {  // a thread makes the dwords of eight tokens and four values: 16 threads a tile
            constexpr int kRounds = kMoveTokens / 32 * 16 / kMoveThreads;
            const int set = (part - 4) >> 2, r = ((part - 4) & 3) * 4 + (tid & 3), j = (tid >> 2) & 3;
            u4 word[kRounds];
            uint32_t mask[kRounds];
            int64_t to[kRounds];
#pragma unroll
            for (int n = 0; n < kRounds; n++) to[n] = tile_number(min(i0 + (n * (kMoveThreads / 16) + (tid >> 4)) * 32, keep - 1) >> 5);
#pragma unroll
            for (int n = 0; n < kRounds; n++) {
                const int i = (n * (kMoveThreads / 16) + (tid >> 4)) * 32 + j * 8;
                word[n] = u4{0, 0, 0, 0};
                mask[n] = 0;
                u4 w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int64_t some = max(source[i + e], (int64_t)0);
                    w[e] = *reinterpret_cast<const u4 *>(kv.cache + (some >> 5) * T::kBytes + T::kValues + (set * 64 + r + 16 * (((int)some & 31) >> 3)) * 16);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int64_t from = source[i + e];
                    const int down = nibble_shift((int)from & 7);
                    const uint32_t here = from < 0 ? 0u : 15u;
#pragma unroll
                    for (int c = 0; c < 4; c++) word[n][c] |= ((w[e][c] >> down) & here) << nibble_shift(e);
                    mask[n] |= here << nibble_shift(e);
                }
            }
            found(sources[turn ^ 1], i0 + kMoveTokens);
            all_read();
#pragma unroll
            for (int n = 0; n < kRounds; n++) {
                if (!mask[n] || to[n] < 0) continue;
                u4 *at = reinterpret_cast<u4 *>(kv.cache + to[n] * T::kBytes + T::kValues + (set * 64 + r + 16 * j) * 16);
                if (mask[n] != 0xFFFFFFFFu) {
                    const u4 old = *at;
#pragma unroll
                    for (int c = 0; c < 4; c++) word[n][c] |= old[c] & ~mask[n];
                }
                *at = word[n];
            }
        } else {
            uint16_t ks[R][G], vs[R][G];
            float account[R];
            int64_t from[R], to[R];
#pragma unroll
            for (int n = 0; n < R; n++) to[n] = tile_number(min(i0 + n * kMoveThreads + tid, keep - 1) >> 5);
#pragma unroll
            for (int n = 0; n < R; n++) {
                from[n] = source[n * kMoveThreads + tid];
                const int64_t some = max(from[n], (int64_t)0);
                const int t = (int)some & 31;
                const uint8_t *at = kv.cache + (some >> 5) * T::kBytes;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    ks[n][g] = reinterpret_cast<const uint16_t *>(at + T::kKeyScales)[t * G + g];
                    vs[n][g] = reinterpret_cast<const uint16_t *>(at + T::kValueScales)[g * 32 + t];
                }
                account[n] = accounts[some];  // (pages hold their tokens' accounts in the order of their tiles)
            }
            found(sources[turn ^ 1], i0 + kMoveTokens);
            all_read();
#pragma unroll
            for (int n = 0; n < R; n++) {
                const int i = i0 + n * kMoveThreads + tid;
                if (from[n] < 0 || to[n] < 0) continue;
                const int t = i & 31;
                uint8_t *at = kv.cache + to[n] * T::kBytes;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    reinterpret_cast<uint16_t *>(at + T::kKeyScales)[t * G + g] = ks[n][g];
                    reinterpret_cast<uint16_t *>(at + T::kValueScales)[g * 32 + t] = vs[n][g];
                }
                accounts[to[n] * 32 + t] = account[n];
            }
        }
    }
}

// eight values with 16-byte loads
bool wide_rows(const HeadRows &h) {
    const int64_t size = h.bf16 ? 2 : 4;
    return ((reinterpret_cast<uintptr_t>(h.p) | (uintptr_t)(h.row * size) | (uintptr_t)(h.head * size)) & 15) == 0;
}

template <int D> int append(const AppendArgs &a, bool bf16, hipStream_t s) {
    unsigned workgroups;
    if (int rc = wavefronts_of("kv_append", a.kv, a.layout, &workgroups)) return rc;
    const dim3 grid(workgroups), block(256);
    return bf16 ? launch(kv_append_kernel<D, true>, grid, block, 0, s, a) : launch(kv_append_kernel<D, false>, grid, block, 0, s, a);
}
template <int D> int read(const KvCall &kv, uint16_t *k, uint16_t *v, hipStream_t s) {
    const Layout layout = layout_of(kv);
    unsigned workgroups;
    if (int rc = wavefronts_of("kv_read", kv, layout, &workgroups)) return rc;
    return launch(kv_read_kernel<D>, dim3(workgroups), dim3(256), 0, s, kv, k, v, layout);
}

}  // namespace

int launch_kv_append(const KvCall &kv, const HeadRows &k, const HeadRows &v, float *accounts, hipStream_t s) {
    AppendArgs a{kv, k, v, accounts, layout_of(kv), 0};
    a.wide = wide_rows(k) && wide_rows(v);
    switch (kv.head_dim) {
    case 64: return append<64>(a, k.bf16, s);
    case 128: return append<128>(a, k.bf16, s);
    default: return append<256>(a, k.bf16, s);
    }
}

int launch_kv_read(const KvCall &kv, uint16_t *k, uint16_t *v, hipStream_t s) {
    switch (kv.head_dim) {
    case 64: return read<64>(kv, k, v, s);
    case 128: return read<128>(kv, k, v, s);
    default: return read<256>(kv, k, v, s);
    }
}

template <int D> static int move_kept(const KvCall &kv, float *accounts, int keep, const int32_t *kept, int32_t *new_lengths, hipStream_t s) {
    return launch(kv_move_kernel<D>, dim3((unsigned)kv.kv_heads, (unsigned)kv.seqs, 4 + D / 16 + 1), dim3(kMoveThreads), 0, s, kv, accounts, keep, kept, new_lengths);
}

int launch_kv_evict(const KvCall &kv, float *accounts, int keep, int recent, int32_t *kept, int32_t *new_lengths, hipStream_t s) {
    const dim3 grid((unsigned)kv.kv_heads, (unsigned)kv.seqs);
    const int64_t n = (int64_t)kv.max_pages * kv.page_tokens - recent;  // tokens to choose from, at most
    // (32 keys a thread no longer fit the 128 registers of a workgroup of 1024)
    if (n > 16 * kSelectThreads && n <= kLdsRounds * kSelectThreads) {
        constexpr int bytes = kLdsRounds * kSelectThreads * 4;
        static const bool lds_ok = hipFuncSetAttribute(reinterpret_cast<const void *>(kv_select_kernel<kInLds>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
        if (!lds_ok) return fail(GQ_ERR_HIP, "kv_evict: cannot reserve %d bytes of LDS", bytes);
        if (int rc = launch(kv_select_kernel<kInLds>, grid, dim3(kSelectThreads), bytes, s, kv, accounts, keep, recent, kept)) return rc;
    } else {
        const auto select = n <= 4 * kSelectThreads ? kv_select_kernel<4> : n <= 16 * kSelectThreads ? kv_select_kernel<16> : kv_select_kernel<0>;
        if (int rc = launch(select, grid, dim3(kSelectThreads), 0, s, kv, accounts, keep, recent, kept)) return rc;
    }
    switch (kv.head_dim) {
    case 64: return move_kept<64>(kv, accounts, keep, kept, new_lengths, s);
    case 128: return move_kept<128>(kv, accounts, keep, kept, new_lengths, s);
    default: return move_kept<256>(kv, accounts, keep, kept, new_lengths, s);
    }
}

}  // namespace gq
