// A token for every row of logits x, from a temperature T, top-k, top-p, min-p and a given u in [0, 1):
//
//     weights   p_i = exp((x_i - max x) / T)
//     order     by logit, the largest first; of equal ones the lowest index
//     kept      the first k of the order; of these the shortest beginning that weighs top_p of them all, one token at least; of these p_i >= min_p
//     token     the lowest index t with sum of the kept p_i, i <= t, over u times all of them
//     T <= 0    the first of the order
//
// What is kept is a beginning of the order, so that it is known by its last token: a key (a logit's bits, ordered) and how many of the tokens with that key
// are kept, the lowest indices.  Sums over the kept tokens in order of index then find the token, first among the chunks of 2048, then in one.
//
// Weights are formed in 64 bits: next to a border, of which a vocabulary has as many as tokens, 32 would give another token once in some hundred rows.  Where order must
// not matter (histograms, sums that several threads add to) they are whole numbers of 2^-42 of the largest.  The same arguments always give the same token.
//
// The first launch reads the logits once: a wavefront a chunk, which leaves its maximum, its sum and its largest keys (some 90, fewer where many are
// equal, complete from a level on).  In the second a workgroup a row finds the cut among the keys that the chunks have left, and reads a single chunk again.  Where the cut lies
// below what they have left (a flat distribution under top-p) the row is gone over twice more, by all its chunks at a time in launches that find nothing to do otherwise; where the
// call's settings make that unlikely these launches are left out, and the second one does it by itself.
#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace gq {

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 2048, kChunkKeys = 128, kLevelLanes = 48, kMostChunks = 1024;
constexpr int kPickThreads = 512, kPickWaves = kPickThreads / 64, kBins = 2048, kListBins = 512, kListMost = 6144, kFew = 64;
// Flat rows that the launches for them have room for (68 KB each); the others are gone over in the second launch.  Of 512 rows of an output head that is unsure of every eighth some 14 to 25 are flat.
// us for 64, 128, 256 and 512 rows of 128256 that all are, under top-p 0.95: 92 135 312 426, with room for 512 of them 92 134 209 368, for 32 of them 232 247 265 381.
constexpr int kWideRows = 128;
static_assert((kMostLogits + 7 + kChunk - 1) / kChunk <= kMostChunks, "a row's chunks have room in LDS, wherever its first logit lies");
constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -__builtin_huge_valf();

struct Chunk {
    double sum;      // of the weights, the chunk's largest 1
    float most;
    int at;          // the lowest index of the largest
    uint32_t level;  // the list has every key from here on
    int count;
};

// A flat row on its way through the launches for it: the weights of its tokens by bins of 1/32 in powers of two, the keys of the bin with the cut in it, what the chunks weigh above it.
struct Wide {
    int64_t row;
    float most;
    uint32_t floor_key;
    uint32_t listed;
    uint64_t weights[kBins];
    uint32_t counts[kBins];
    uint64_t chunk_weight[kMostChunks];
    uint32_t keys[kListMost];
    uint16_t chunks[kListMost];
};

struct SampleArgs {
    const uint8_t *logits;
    int64_t row_bytes;
    int vocab, chunks;  // of a row, at most
    Sampling how;
    const float *uniform;
    Chunk *chunk;      // [rows, chunks]
    uint32_t *keys;    // [rows, chunks, kChunkKeys]
    Wide *wide;        // [wide_rows]; null: there are no launches for them
    uint32_t *wides;   // how many there are (or would be)
    int wide_rows;
    int32_t *tokens;
    float *probabilities;  // may be null
};

struct Settings {
    double t, top_p, min_p, rate;  // rate: 1 / t in powers of two
    int k;                 // 0: all
    bool first;            // the first of the order
    __device__ __forceinline__ bool cuts() const { return k || top_p < 1.0 || min_p > 0.0; }
    __device__ __forceinline__ bool orders() const { return k || top_p < 1.0; }
};
__device__ __forceinline__ Settings settings_of(const SampleArgs &a, int64_t row) {
    Settings s;
    s.t = a.how.temperatures ? (double)a.how.temperatures[row] : a.how.temperature;
    s.top_p = a.how.top_ps ? (double)a.how.top_ps[row] : a.how.top_p;
    s.min_p = a.how.min_ps ? (double)a.how.min_ps[row] : a.how.min_p;
    s.k = a.how.top_ks ? a.how.top_ks[row] : a.how.top_k;
    s.k = s.k >= a.vocab || s.k < 0 ? 0 : s.k;
    s.top_p = s.top_p < 1.0 ? s.top_p : 1.0;  // (NaN: no bound)
    s.min_p = s.min_p > 0.0 ? fmin(s.min_p, 1.0) : 0.0;
    s.first = !(s.t > 0.0) || s.k == 1 || s.top_p <= 0.0;
    s.rate = 1.4426950408889634 / s.t;
    return s;
}

// Logits in order as whole numbers; a NaN counts as minus infinity, -0 as 0.
__device__ __forceinline__ float clean(float x) { return x == x ? x : kNegInf; }
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// 2^y for -1010 <= y <= 0, to 1e-12 of itself: the nearest whole number to the exponent, for the rest, at most 1/2 either way, 1 + c1 f + ... + c8 f^8 that is nearest
// to 2^f there (a weighted least-squares fit, to 8.2e-13).
__device__ __forceinline__ double power_of_two(double y) {
    const double whole = y + 6755399441055744.0;  // 1.5 * 2^52: the last bits of the sum are the whole number
    const double f = y - (whole - 6755399441055744.0);
    double p = 1.3178930833147116e-06;
    p = fma(p, f, 1.530915726184116e-05);
    p = fma(p, f, 1.5403825484862121e-04);
    p = fma(p, f, 1.333345485557617e-03);
    p = fma(p, f, 9.61812861606663e-03);
    p = fma(p, f, 5.5504109352728245e-02);
    p = fma(p, f, 2.4022650698111078e-01);
    p = fma(p, f, 6.931471805482102e-01);
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(whole) << 20), __double2loint(p));
}
// (what weighs 2^-1000 of the largest, minus infinity and NaN among it, is nothing in any sum)
__device__ __forceinline__ double weight(float x, float most, double rate) { return x == most ? 1.0 : power_of_two(fmax(((double)x - (double)most) * rate, -1000.0)); }
constexpr double kUnit = 4398046511104.0;  // 2^42: a vocabulary of 2^21 tokens of the same weight sums to 2^63
__device__ __forceinline__ uint64_t units(double w) { return (uint64_t)__builtin_rint(w * kUnit); }

// A row as 16-byte blocks, aligned: `lead` places in front of its first logit are no part of it.
template <bool BF16> struct Row {
    static constexpr int kSize = BF16 ? 2 : 4, kBlock = 16 / kSize;
    const uint8_t *base;
    int lead, end;  // logits lie in places lead to end
    __device__ __forceinline__ Row(const SampleArgs &a, int64_t row) {
        const uint8_t *p = a.logits + row * a.row_bytes;
        lead = (int)((uintptr_t)p & 15) / kSize;
        base = p - lead * kSize;
        end = lead + a.vocab;
    }
    __device__ __forceinline__ int chunks() const { return (end + kChunk - 1) / kChunk; }
    __device__ __forceinline__ float one(int place) const {
        if (place < lead || place >= end) return kNegInf;
        if constexpr (BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(base)[place] << 16);
        else return reinterpret_cast<const float *>(base)[place];
    }
    // where value i of lane `lane` of a chunk lies
    __device__ __forceinline__ static int place(int chunk, int lane, int i) { return chunk * kChunk + ((i / kBlock) * 64 + lane) * kBlock + i % kBlock; }
    // values `from` on of a lane, N of them (a multiple of eight)
    template <int N> __device__ __forceinline__ void load(int chunk, int lane, float (&x)[N], int from = 0) const {
        if (chunk * kChunk >= lead && (chunk + 1) * kChunk <= end) {
            constexpr int LOADS = N / kBlock;
            u4 w[LOADS];
#pragma unroll
            for (int i = 0; i < LOADS; i++) w[i] = *reinterpret_cast<const u4 *>(base + (int64_t)place(chunk, lane, from + i * kBlock) * kSize);
#pragma unroll
            for (int i = 0; i < N; i++) {
                if constexpr (BF16) {
                    const uint32_t u = w[i / 8][i % 8 / 2];
                    x[i] = __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16);
                } else {
                    x[i] = __uint_as_float(w[i / 4][i % 4]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = one(place(chunk, lane, from + i));
        }
    }
};

// The lanes' values up to and with each, by data-parallel moves: 1, 2, 4, 8 lanes within rows of sixteen, then from the last lane of a row into the next one, and of
// the first half into the second.  `none` combines to nothing.  (Through LDS, as shuffles go, a scan of 64 bits takes three times as long, and the second launch is a chain of them.)
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t v, uint32_t none) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t moved(uint64_t v, uint64_t none) {
    return (uint64_t)moved<CTRL, ROWS>((uint32_t)(v >> 32), (uint32_t)(none >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)v, (uint32_t)none);
}
template <class T, class F> __device__ __forceinline__ T scan_lanes(T v, T none, F f) {
    v = f(v, moved<0x111, 0xF>(v, none));
    v = f(v, moved<0x112, 0xF>(v, none));
    v = f(v, moved<0x114, 0xF>(v, none));
    v = f(v, moved<0x118, 0xF>(v, none));
    v = f(v, moved<0x142, 0xA>(v, none));
    v = f(v, moved<0x143, 0xC>(v, none));
    return v;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
__device__ __forceinline__ uint64_t last_lane(uint64_t v) { return (uint64_t)last_lane((uint32_t)(v >> 32)) << 32 | last_lane((uint32_t)v); }
struct Sum { template <class T> static constexpr T none = 0; template <class T> __device__ __forceinline__ T operator()(T p, T q) const { return p + q; } };
struct Most { template <class T> static constexpr T none = 0; template <class T> __device__ __forceinline__ T operator()(T p, T q) const { return max(p, q); } };
struct Least { template <class T> static constexpr T none = ~(T)0; template <class T> __device__ __forceinline__ T operator()(T p, T q) const { return min(p, q); } };
template <class F, class T> __device__ __forceinline__ T over_lanes(T v, F f) { return last_lane(scan_lanes(v, F::template none<T>, f)); }
__device__ __forceinline__ double sum_of_lanes(double v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// One wavefront a chunk.  The level: of the lanes' largest keys the 48th (its upper 16 bits), so that 48 keys at least are at or above it and, where the large ones
// lie anywhere, some 90 of 2048, of the 128 that there is room for.  Where more are (by chance in one chunk of thousands; equal ones: a mask by a large negative
// number, padding) the level goes up over them, so that such a chunk takes nothing from the row's other lists: one row of 128256 with 200 numbers among -1e9 takes 22 us under top-k 50
// and top-p 0.9, and 512 rows without a mask 86; with an empty list in the chunk's place, and all of the row gone over by its workgroup, 530 and 285.
//
// 512 rows of 128256 in float32 take 64 us, 4.1 TB/s.  The memory gives 5.9 to a kernel that only reads (123 MB; 45 us for these), and 26 vector instructions a logit, 16 of them in 64 bits for the chunk's sum, take 48:
// each wavefront loads its chunk first and works on it then, so that the two overlap by what other wavefronts do alone.  Keys that are read again come from the memory too (some 90 a chunk, 0.44 times
// as many requests as the logits ask for).  One row: 7 us.
template <bool BF16> __global__ __launch_bounds__(256) void sample_scan_kernel(const SampleArgs a, int64_t waves) {
    const int lane = (int)threadIdx.x & 63;
    const int64_t index = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (index >= waves) return;
    const int64_t row = index / a.chunks;
    const int chunk = (int)(index - row * a.chunks);
    const Row<BF16> r(a, row);
    if (chunk >= r.chunks()) return;
    float x[32];
    r.load(chunk, lane, x);
    const Settings s = settings_of(a, row);
    if (index == 0 && lane == 0) *a.wides = 0;
    float mine = kNegInf;
#pragma unroll
    for (int i = 0; i < 32; i++) mine = fmaxf(mine, x[i]);  // (a NaN is not taken)
    const float most = value_of(over_lanes(key_of(mine), Most{}));
    Chunk c{0.0, most, 0, 0, 0};
    if (s.first) {
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int i = 31; i >= 0; i--) at = x[i] == most ? Row<BF16>::place(chunk, lane, i) - r.lead : at;
        c.at = (int)over_lanes((uint32_t)at, Least{});
    } else if (most > kNegInf) {
        double sum = 0.0;
        const float lowest = (float)((double)most - 693.0 * s.t);  // weighs 2^-999.8; a NaN and minus infinity count as that
        const double least_weight = ((double)lowest - (double)most) * s.rate;
        if (least_weight <= -950.0 && least_weight >= -1010.0) {  // (not so where 32 bits have no such number, near infinity or zero temperature)
#pragma unroll
            for (int i = 0; i < 32; i++) sum += power_of_two(((double)fmaxf(x[i], lowest) - (double)most) * s.rate);
        } else {
#pragma unroll 1
            for (int i = 0; i < 32; i++) sum += x[i] > kNegInf ? weight(x[i], most, s.rate) : 0.0;
        }
        c.sum = sum_of_lanes(sum);
        if (s.cuts()) {
            const uint32_t top = key_of(mine);
            uint32_t level = 0;
#pragma unroll
            for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
                if (__popcll(__ballot(top >= (level | bit))) >= kLevelLanes) level |= bit;
            uint32_t *keys = a.keys + index * kChunkKeys;
            // (a lane has one or two of them, and reads these again: to look for one in each of its registers takes 12 instructions a register)
            uint32_t in, mine_in, upto;
            const auto look = [&] {
                const float least = value_of(max(level, key_of(-3.402823466e38f)));  // (minus infinity is in no list)
                in = 0;
#pragma unroll
                for (int i = 0; i < 32; i++) in |= x[i] >= least ? 1u << i : 0u;
                mine_in = (uint32_t)__popc(in);
                upto = scan_lanes(mine_in, 0u, Sum{});
                return (int)last_lane(upto);
            };
            int count = look();
            if (count > kChunkKeys) {  // many equal ones at the level: the list begins above them
                level += 0x10000u;
                count = look();
                if (count > kChunkKeys) {  // (fewer lanes than the level asks for have all of the large ones: the first step at which they fit)
                    uint32_t over = 0;
#pragma unroll 1
                    for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
                        level = over | bit;
                        if (look() > kChunkKeys) over = level;
                    }
                    level = over + 0x10000u;
                    count = look();
                }
            }
            for (uint32_t to = upto - mine_in; in; in &= in - 1, to++) keys[to] = key_of(r.one(Row<BF16>::place(chunk, lane, __ffs((int)in) - 1)));
            c.level = level;
            c.count = count;
        }
    }
    if (lane == 0) a.chunk[index] = c;
}

// ---- the second launch ------------------------------------------------------------------------------------------------

// Sums of the threads in front of each, in order; `total` of all of them.
__device__ __forceinline__ uint64_t threads_in_front(uint64_t v, uint64_t *waves, uint64_t &total) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint64_t upto = scan_lanes(v, (uint64_t)0, Sum{});
    __syncthreads();
    if (((int)threadIdx.x & 63) == 63) waves[wave] = upto;
    __syncthreads();
    uint64_t front = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; i++) {
        if (i < wave) front += waves[i];
        total += waves[i];
    }
    return front + upto - v;
}

// The last kept token: the kept ones are those of larger key and the first `ties` of this one; how many are above it, or what they weigh.
struct Cut {
    uint32_t key, ties;
    uint64_t above;  // tokens, where the cut is one of tokens, or weight
};

struct PickLds {
    uint64_t weights[kBins];
    uint32_t counts[kBins];
    uint32_t keys[kListMost];
    uint16_t chunks[kListMost];
    uint64_t chunk_weight[kMostChunks];
    uint32_t chunk_ties[kMostChunks];
    uint64_t waves[kPickWaves];
    uint64_t found_above;
    uint32_t few[kFew];
    uint64_t few_weights[kFew];
    uint32_t found, found_key, found_same, listed, fews;
};

template <class T, class F> __device__ __forceinline__ T over_threads(T v, uint64_t *waves, F f) {
    v = over_lanes(v, f);
    __syncthreads();
    if (((int)threadIdx.x & 63) == 0) waves[(int)threadIdx.x >> 6] = (uint64_t)v;
    __syncthreads();
    v = (T)waves[0];
#pragma unroll
    for (int i = 1; i < kPickWaves; i++) v = f(v, (T)waves[i]);
    return v;
}
__device__ __forceinline__ uint64_t sum_of_threads(uint64_t v, uint64_t *waves) { return over_threads(v, waves, Sum{}); }

// The first of the bins, from bin 0 on, up to which `want` is reached, of tokens (by count) or of weight; `above`: what is in front of it.  BINS: none.
template <int BINS> __device__ __forceinline__ uint32_t find_bin(PickLds &l, bool by_count, uint64_t want, uint64_t &above) {
    constexpr int N = BINS / kPickThreads;
    const int first = (int)threadIdx.x * N;
    if (threadIdx.x == 0) l.found = BINS;
    uint64_t bins[N], mine = 0, total;
#pragma unroll
    for (int i = 0; i < N; i++) {
        bins[i] = by_count ? l.counts[first + i] : l.weights[first + i];
        mine += bins[i];
    }
    uint64_t at = threads_in_front(mine, l.waves, total) + above;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (at < want && want <= at + bins[i]) {
            l.found = (uint32_t)(first + i);
            l.found_above = at;
        }
        at += bins[i];
    }
    __syncthreads();
    const uint32_t bin = l.found;
    if (bin < BINS) above = l.found_above;
    __syncthreads();
    return bin;
}

template <int BINS> __device__ __forceinline__ void clear_bins(PickLds &l) {
    __syncthreads();
    for (int i = (int)threadIdx.x; i < BINS; i += kPickThreads) { l.weights[i] = 0; l.counts[i] = 0; }
    __syncthreads();
}
__device__ __forceinline__ void add_to_bin(PickLds &l, uint32_t bin, bool with_weight, uint64_t weight) {
    if (with_weight) atomicAdd(reinterpret_cast<unsigned long long *>(&l.weights[bin]), (unsigned long long)weight);
    atomicAdd(&l.counts[bin], 1u);
}
// how many of the tokens of the cut's key are kept
__device__ __forceinline__ uint32_t ties_of(uint64_t want, uint64_t above, uint64_t each, uint32_t all) {
    const uint64_t ties = (want - above + each - 1) / each;
    return ties < all ? (uint32_t)ties : all;
}

// The cut at `want` tokens (or weight) among the l.listed keys in LDS, with cut.above as what is above all of them: by nine bits at a time of a key's distance from the largest, until so few
// are left that each is held against all of them.  False: they do not reach it.
template <class Weight> __device__ __forceinline__ bool cut_of_list(PickLds &l, Weight weight_of, bool by_count, uint64_t want, Cut &cut) {
    const int tid = (int)threadIdx.x, n = (int)l.listed;
    uint32_t top = kAll, left = (uint32_t)n;
    int width = 32;  // keys from top down to top - 2^width + 1 are looked at
    if (n == 0) return false;
    if (n > kFew) {
        uint32_t low = kAll;
        top = 0;
        for (int i = tid; i < n; i += kPickThreads) { low = min(low, l.keys[i]); top = max(top, l.keys[i]); }
        low = over_threads(low, l.waves, Least{});
        top = over_threads(top, l.waves, Most{});
        width = 32 - __clz((int)(top - low));
        do {
            const uint32_t last = width < 32 ? (1u << width) - 1u : kAll;
            const int shift = width > 9 ? width - 9 : 0;
            clear_bins<kListBins>(l);
            for (int i = tid; i < n; i += kPickThreads) {
                const uint32_t key = l.keys[i], d = top - key;
                if (key <= top && d <= last) add_to_bin(l, d >> shift, !by_count, by_count ? 0 : weight_of(key));
            }
            __syncthreads();
            const uint32_t bin = find_bin<kListBins>(l, by_count, want, cut.above);
            if (bin >= kListBins) return false;  // (the first time, or never)
            left = l.counts[bin];
            top -= bin << shift;
            width = shift;
        } while (width && left > kFew);
        if (width == 0) {
            cut.key = top;
            cut.ties = ties_of(want, cut.above, by_count ? 1 : weight_of(top), left);
            __syncthreads();
            return true;
        }
    }
    __syncthreads();
    if (tid == 0) { l.fews = 0; l.found_same = 0; }
    __syncthreads();
    for (int i = tid; i < n; i += kPickThreads) {
        const uint32_t key = l.keys[i];
        if (key <= top && (width == 32 || top - key < (1u << width))) l.few[atomicAdd(&l.fews, 1u)] = key;
    }
    __syncthreads();
    if (tid < (int)left) l.few_weights[tid] = by_count ? 1 : weight_of(l.few[tid]);
    __syncthreads();
    // eight threads a key, an eighth of the others each
    const int mine = tid / 8;
    if (mine < (int)left) {
        const uint32_t key = l.few[mine];
        uint64_t above = 0;
        uint32_t same = 0;
#pragma unroll
        for (int i = 0; i < kFew / 8; i++) {
            const int other = tid % 8 + 8 * i;
            const uint32_t k = l.few[other];
            const bool there = other < (int)left;
            above += there && k > key ? l.few_weights[other] : 0;
            same += there && k == key;
        }
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) {
            above += __shfl_xor(above, m);
            same += __shfl_xor(same, m);
        }
        above += cut.above;
        const uint64_t w = l.few_weights[mine];
        if (above < want && want <= above + same * w) {  // (all of one key write the same)
            l.found_key = key;
            l.found_above = above;
            l.found_same = ties_of(want, above, w, same);
        }
    }
    __syncthreads();
    cut.key = l.found_key;
    cut.above = l.found_above;
    cut.ties = l.found_same;
    __syncthreads();
    return cut.ties != 0;
}

// What the cut keeps of the list weighs; only keys from the cut's on stay in it.
template <class Weight> __device__ __forceinline__ uint64_t keep_of_list(PickLds &l, Weight weight_of, const Cut &cut) {
    constexpr int N = kListMost / kPickThreads;
    const int tid = (int)threadIdx.x, lane = tid & 63, n = (int)l.listed;
    uint32_t keys[N], kept = 0;
    uint16_t chunks[N];
    uint64_t sum = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int at = tid + i * kPickThreads;
        keys[i] = at < n ? l.keys[at] : 0u;
        chunks[i] = at < n ? l.chunks[at] : 0;
        kept += keys[i] >= cut.key;
    }
    __syncthreads();
    if (tid == 0) l.listed = 0;
    __syncthreads();
    const uint32_t upto = scan_lanes(kept, 0u, Sum{}), all = last_lane(upto);
    uint32_t to = 0;
    if (lane == 0 && all) to = atomicAdd(&l.listed, all);
    to = __builtin_amdgcn_readfirstlane(to) + upto - kept;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (keys[i] < cut.key) continue;
        l.keys[to] = keys[i];
        l.chunks[to++] = chunks[i];
    }
    __syncthreads();
    for (int i = tid; i < (int)l.listed; i += kPickThreads) sum += l.keys[i] > cut.key ? weight_of(l.keys[i]) : 0;
    return sum_of_threads(sum, l.waves) + cut.ties * weight_of(cut.key);
}

// The same among the keys that `each` passes on, however many: digit by digit, 11, 11 and 10 bits.
template <class Each, class Weight> __device__ __forceinline__ bool cut_of_many(PickLds &l, Each each, Weight weight_of, bool by_count, uint64_t want, Cut &cut) {
    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, done = pass == 0 ? 32 : pass == 1 ? 21 : 10;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        clear_bins<kBins>(l);
        each([&](uint32_t key, int) {
            if (done < 32 && key >> done != prefix >> done) return;
            add_to_bin(l, digits - (key >> shift & digits), !by_count, by_count ? 0 : weight_of(key));  // (the largest first)
        });
        __syncthreads();
        const uint32_t bin = find_bin<kBins>(l, by_count, want, cut.above);
        if (bin >= kBins) return false;
        prefix |= (digits - bin) << shift;
        if (pass == 2) cut.ties = ties_of(want, cut.above, by_count ? 1 : weight_of(prefix), l.counts[bin]);
    }
    cut.key = prefix;
    __syncthreads();
    return true;
}

// Bins of 1/32 in powers of two below the largest logit.
__device__ __forceinline__ uint32_t bin_of(uint32_t key, float most, uint32_t most_key, float rate) {
    const float d = (most - value_of(key)) * rate * 32.0f;
    return key == most_key ? 0u : (uint32_t)fminf(d, (float)(kBins - 1));
}
// the weight that top-p asks for
__device__ __forceinline__ uint64_t share_of(const Settings &s, uint64_t w) {
    const double p = ceil(s.top_p * (double)w);
    return p < 1.0 ? (uint64_t)1 : (uint64_t)p;
}

// A token's weight and what min-p asks of keys, given the row's largest.
__device__ __forceinline__ uint32_t floor_of(const Settings &s, float most, uint32_t most_key) {
    if (!(s.min_p > 0.0)) return 0;
    const double least = (double)most + s.t * log(s.min_p);
    float f = (float)least;
    if ((double)f < least) f = value_of(key_of(f) + 1);
    return most == __builtin_huge_valf() ? most_key : min(most_key, key_of(clean(f)));
}

// The token, once the cut is known: chunks in l.chunk_weight (without the cut's ties) and l.chunk_ties.
template <bool BF16>
__device__ __forceinline__ void draw(const SampleArgs &a, PickLds &l, const Row<BF16> &r, const Settings &s, int64_t row, int chunks, float most, const Cut &cut) {
    const int tid = (int)threadIdx.x;
    const bool cuts = s.cuts();
    // the chunk: two neighbouring ones a thread
    const uint64_t cut_weight = cuts ? units(weight(value_of(cut.key), most, s.rate)) : 0;
    constexpr int N = kMostChunks / kPickThreads;
    uint64_t kept[N], tie_at[N], mine = 0, total, tie_total;
    uint32_t ties[N], my_ties = 0;
    const int c0 = tid * N;
#pragma unroll
    for (int i = 0; i < N; i++) {
        kept[i] = c0 + i < chunks ? l.chunk_weight[c0 + i] : 0;
        ties[i] = c0 + i < chunks ? l.chunk_ties[c0 + i] : 0;
        my_ties += ties[i];
    }
    uint64_t tie_front = threads_in_front((uint64_t)my_ties, l.waves, tie_total);
#pragma unroll
    for (int i = 0; i < N; i++) {
        tie_at[i] = tie_front;
        const uint64_t left = cut.ties > tie_front ? cut.ties - tie_front : 0;
        kept[i] += min((uint64_t)ties[i], left) * cut_weight;
        tie_front += ties[i];
        mine += kept[i];
    }
    uint64_t front = threads_in_front(mine, l.waves, total);
    const double u = (double)a.uniform[row];
    uint64_t want = u > 0.0 ? (uint64_t)fmin(u * (double)total, (double)total) : 0;  // (NaN: 0)
    want = want < total ? want : total - 1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (front <= want && want < front + kept[i]) {
            l.found = (uint32_t)(c0 + i);
            l.found_above = front;
            l.chunk_weight[0] = kept[i];
            l.found_same = (uint32_t)min(tie_at[i], (uint64_t)kAll);
        }
        front += kept[i];
    }
    __syncthreads();

    // the token: four neighbouring ones a thread
    const int c = (int)l.found;
    want -= l.found_above;
    const uint64_t of_chunk = l.chunk_weight[0];
    uint32_t rank = l.found_same;
    // (with nothing cut off the chunk's weight is a sum in 64 bits, not one of these units, of which its tokens may have none: in parts of the chunk then)
    const float unit_most = cuts ? most : a.chunk[row * a.chunks + c].most;
    constexpr int M = kChunk / kPickThreads;
    float x[M];
    my_ties = 0;
#pragma unroll
    for (int i = 0; i < M; i++) {
        x[i] = clean(r.one(c * kChunk + tid * M + i));
        my_ties += cuts && x[i] > kNegInf && key_of(x[i]) == cut.key;
    }
    rank += (uint32_t)threads_in_front((uint64_t)my_ties, l.waves, tie_total);
    mine = 0;
    uint64_t w[M];
#pragma unroll
    for (int i = 0; i < M; i++) {
        const uint32_t key = key_of(x[i]);
        const bool tie = cuts && key == cut.key;
        const bool keep = x[i] > kNegInf && (!cuts || key > cut.key || (tie && rank < cut.ties));
        if (tie && x[i] > kNegInf) rank++;
        w[i] = keep ? units(weight(x[i], unit_most, s.rate)) : 0;
        mine += w[i];
    }
    uint64_t in_chunk;
    front = threads_in_front(mine, l.waves, in_chunk);
    if (!cuts) want = (uint64_t)((double)want / (double)of_chunk * (double)in_chunk);
    want = min(want, in_chunk - 1);
#pragma unroll
    for (int i = 0; i < M; i++) {
        if (front <= want && want < front + w[i]) {
            a.tokens[row] = c * kChunk + tid * M + i - r.lead;
            if (a.probabilities) a.probabilities[row] = (float)(weight(x[i], most, s.rate) * kUnit / (double)total);
        }
        front += w[i];
    }
}

// The kept weight of every chunk from the list in LDS, added to what is in l.chunk_weight, and its tokens that equal the cut's.
template <class Weight> __device__ __forceinline__ void chunks_of_list(PickLds &l, Weight weight_of, const Cut &cut, int chunks, bool clear) {
    __syncthreads();
    for (int c = (int)threadIdx.x; c < chunks; c += kPickThreads) {
        if (clear) l.chunk_weight[c] = 0;
        l.chunk_ties[c] = 0;
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < (int)l.listed; i += kPickThreads) {
        const uint32_t key = l.keys[i];
        const int c = l.chunks[i];
        if (key > cut.key) atomicAdd(reinterpret_cast<unsigned long long *>(&l.chunk_weight[c]), (unsigned long long)weight_of(key));
        else if (key == cut.key) atomicAdd(&l.chunk_ties[c], 1u);
    }
    __syncthreads();
}

// All of a flat row in one workgroup: its bins, the keys of the one with the cut in it, then its chunks.
template <bool BF16>
__device__ __forceinline__ void draw_alone(const SampleArgs &a, PickLds &l, const Row<BF16> &r, const Settings &s, int64_t row, int chunks, float most, uint32_t most_key, uint32_t floor_key) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float rate = (float)s.rate;
    const auto weight_of = [&](uint32_t key) { return units(weight(value_of(key), most, s.rate)); };
    const auto each_of_row = [&](auto f) {
#pragma unroll 1
        for (int at = wave * 4; at < chunks * 4; at += at % 4 == 3 ? (kPickWaves - 1) * 4 + 1 : 1) {  // (a quarter of a chunk at a time: few registers)
            float x[8];
            r.load(at / 4, lane, x, at % 4 * 8);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (x[i] > kNegInf) f(key_of(x[i]), at / 4);
        }
    };
    Cut cut{0u, kAll, 0};
    uint64_t all = 0;
#pragma unroll 1
    for (int turn = s.k ? 0 : 1; turn < (s.top_p < 1.0 ? 2 : 1); turn++) {
        const bool by_count = turn == 0;
        Cut c{0u, 0u, 0};
        clear_bins<kBins>(l);
        each_of_row([&](uint32_t key, int) { add_to_bin(l, bin_of(key, most, most_key, rate), true, weight_of(key)); });
        __syncthreads();
        if (turn == (s.k ? 0 : 1)) {  // (what all of the row weighs, where fewer numbers than k are there too)
            uint64_t mine = 0;
            for (int i = tid; i < kBins; i += kPickThreads) mine += l.weights[i];
            all = sum_of_threads(mine, l.waves);
        }
        const uint64_t want = by_count ? (uint64_t)s.k : share_of(s, all);
        const uint32_t bin = find_bin<kBins>(l, by_count, want, c.above);
        if (bin >= kBins) continue;
        const uint32_t in_bin = l.counts[bin];
        __syncthreads();
        if (in_bin > (uint32_t)kListMost) {
            cut_of_many(l, [&](auto f) { each_of_row([&](uint32_t key, int at) { if (bin_of(key, most, most_key, rate) == bin) f(key, at); }); }, weight_of, by_count, want, c);
        } else {
            if (tid == 0) l.listed = 0;
            __syncthreads();
            each_of_row([&](uint32_t key, int at) {
                if (bin_of(key, most, most_key, rate) != bin) return;
                const uint32_t to = atomicAdd(&l.listed, 1u);
                l.keys[to] = key;
                l.chunks[to] = (uint16_t)at;
            });
            __syncthreads();
            cut_of_list(l, weight_of, by_count, want, c);
        }
        cut = c;
        if (by_count && s.top_p < 1.0) {
            uint64_t mine = 0;
            each_of_row([&](uint32_t key, int) { mine += key > cut.key ? weight_of(key) : 0; });
            all = sum_of_threads(mine, l.waves) + cut.ties * weight_of(cut.key);
        }
    }
    if (floor_key > cut.key) cut = Cut{floor_key, kAll, 0};
    __syncthreads();
#pragma unroll 1
    for (int c = wave; c < chunks; c += kPickWaves) {
        uint64_t sum = 0;
        uint32_t ties = 0;
#pragma unroll 1
        for (int from = 0; from < 32; from += 8) {
            float x[8];
            r.load(c, lane, x, from);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t key = key_of(x[i]);
                if (x[i] > kNegInf && key > cut.key) sum += weight_of(key);
                ties += x[i] > kNegInf && key == cut.key;
            }
        }
        sum = over_lanes(sum, Sum{});
        ties = over_lanes(ties, Sum{});
        if (lane == 0) { l.chunk_weight[c] = sum; l.chunk_ties[c] = ties; }
    }
    __syncthreads();
    draw(a, l, r, s, row, chunks, most, cut);
}

// A chain of passes over the lists behind barriers: 17 us for one row of 128256 under top-k and top-p, 25 for 512 (two a CU).  Keys by bins of their distance from the largest and few keys held
// against each other took the first of these from 31; the lists' loads sixteen at a time, scans by lane moves and the list cut down to what top-k keeps are in it.
template <bool BF16> __global__ __launch_bounds__(kPickThreads, 4) void sample_pick_kernel(const SampleArgs a) {
    __shared__ PickLds l;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int64_t row = blockIdx.x;
    const Row<BF16> r(a, row);
    const Settings s = settings_of(a, row);
    const int chunks = r.chunks();
    const Chunk *chunk = a.chunk + row * a.chunks;

    // the row's largest logit, and the level from which on the lists have every key
    uint32_t most_key = 0, level = 0;
    for (int c = tid; c < chunks; c += kPickThreads) {
        const float m = chunk[c].most;
        const bool some = m > kNegInf;
        most_key = max(most_key, some ? key_of(m) : 0u);
        level = max(level, some ? chunk[c].level : 0u);
        l.chunk_ties[c] = some ? (uint32_t)chunk[c].count : 0u;
    }
    most_key = over_threads(most_key, l.waves, Most{});
    level = over_threads(level, l.waves, Most{});
    const float most = value_of(most_key);
    if (most_key == 0 || s.first) {  // (a row without a number has no token)
        uint32_t at = kAll;
        for (int c = tid; c < chunks; c += kPickThreads)
            if (most_key && key_of(chunk[c].most) == most_key) at = min(at, (uint32_t)chunk[c].at);
        at = over_threads(at, l.waves, Least{});
        if (tid == 0) {
            a.tokens[row] = (int32_t)at;
            if (a.probabilities) a.probabilities[row] = most_key ? 1.0f : 0.0f;
        }
        return;
    }
    const auto weight_of = [&](uint32_t key) { return units(weight(value_of(key), most, s.rate)); };
    if (!s.cuts()) {
        for (int c = tid; c < chunks; c += kPickThreads) {
            l.chunk_weight[c] = chunk[c].most > kNegInf ? units(chunk[c].sum * weight(chunk[c].most, most, s.rate)) : 0;
            l.chunk_ties[c] = 0;
        }
        __syncthreads();
        draw(a, l, r, s, row, chunks, most, Cut{0u, kAll, 0});
        return;
    }
    const uint32_t floor_key = floor_of(s, most, most_key);
    Cut cut{0u, kAll, 0};
    bool from_lists = s.orders() || floor_key >= level;
    if (from_lists) {
        if (tid == 0) l.listed = 0;
        __syncthreads();
        // (sixteen loads on their way at a time)
        constexpr int AHEAD = 16;
        const uint32_t *keys = a.keys + row * a.chunks * kChunkKeys;
        const int slots = chunks * kChunkKeys;
#pragma unroll 1
        for (int i0 = tid; i0 < slots + lane; i0 += AHEAD * kPickThreads) {  // (whole wavefronts)
            uint32_t key[AHEAD], in = 0;
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int at = i0 + i * kPickThreads;
                key[i] = at < slots && at % kChunkKeys < (int)l.chunk_ties[at / kChunkKeys] ? keys[at] : 0u;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) in += key[i] >= level && key[i];
            const uint32_t upto = scan_lanes(in, 0u, Sum{}), all = last_lane(upto);
            uint32_t to = 0;
            if (lane == 0 && all) to = atomicAdd(&l.listed, all);
            to = __builtin_amdgcn_readfirstlane(to) + upto - in;
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (key[i] < level || !key[i]) continue;
                if (to < (uint32_t)kListMost) { l.keys[to] = key[i]; l.chunks[to] = (uint16_t)((i0 + i * kPickThreads) / kChunkKeys); }
                to++;
            }
        }
        __syncthreads();
        from_lists = l.listed <= (uint32_t)kListMost;
    }
    uint64_t all = 0;
    if (from_lists && s.k) {
        cut = Cut{0u, 0u, 0};
        // (Fewer than k: all of them stay, and what the lists do not have adds nothing where it weighs nothing.  A mask that leaves ten tokens of 128256 under top-k 50 and
        // top-p 0.9: 19 us for minus infinity, 20 for -1e9; 74 and 836 with the row gone over for more.)
        if (!cut_of_list(l, weight_of, true, (uint64_t)s.k, cut)) {
            from_lists = level < most_key && weight_of(level) == 0;
            cut = Cut{level, kAll, 0};
        }
        if (from_lists && s.top_p < 1.0) all = keep_of_list(l, weight_of, cut);
    } else if (from_lists && s.top_p < 1.0) {
        double sum = 0.0;
        for (int c = tid; c < chunks; c += kPickThreads)
            if (chunk[c].most > kNegInf) sum += chunk[c].sum * weight(chunk[c].most, most, s.rate);
        all = sum_of_threads(units(sum), l.waves);
    }
    if (from_lists && s.top_p < 1.0) {
        cut = Cut{0u, 0u, 0};
        from_lists = cut_of_list(l, weight_of, false, share_of(s, all), cut);
    }
    if (from_lists) {
        if (floor_key > cut.key) cut = Cut{floor_key, kAll, 0};
        chunks_of_list(l, weight_of, cut, chunks, true);
        draw(a, l, r, s, row, chunks, most, cut);
        return;
    }
    // a flat row: into the launches for those, where there are any and they have room
    __syncthreads();
    if (a.wide) {
        if (tid == 0) l.found = atomicAdd(a.wides, 1u);
        __syncthreads();
        const uint32_t slot = l.found;
        if (slot < (uint32_t)a.wide_rows) {
            Wide &w = a.wide[slot];
            for (int i = tid; i < kBins; i += kPickThreads) { w.weights[i] = 0; w.counts[i] = 0; }
            if (tid == 0) { w.row = row; w.most = most; w.floor_key = floor_key; w.listed = 0; }
            return;
        }
    }
    draw_alone(a, l, r, s, row, chunks, most, most_key, floor_key);
}

// ---- the launches for flat rows: eight chunks a workgroup ------------------------------------------------------------------
// 10 + 16 + 14 us for a few rows of 50257 in bfloat16, 14 + 19 + 16 for some 20 of 128256 in float32: loads, 64-bit exponentials and barriers one behind the other.  (One workgroup a row, as in draw_alone,
// took 70 us more than these for the first, 100 to 200 for the second.)

__device__ __forceinline__ Wide *wide_of(const SampleArgs &a, int slot) { return slot < a.wide_rows && (uint32_t)slot < *a.wides ? a.wide + slot : nullptr; }

template <bool BF16> __global__ __launch_bounds__(kPickThreads) void sample_bins_kernel(const SampleArgs a, int parts) {
    __shared__ uint64_t weights[kBins];
    __shared__ uint32_t counts[kBins];
    const int slot = (int)blockIdx.x / parts, tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Wide *w = wide_of(a, slot);
    if (!w) return;
    const int64_t row = w->row;
    const Row<BF16> r(a, row);
    const Settings s = settings_of(a, row);
    const int c = ((int)blockIdx.x - slot * parts) * kPickWaves + wave;
    if (!s.orders()) return;
    float x[32];
    if (c < r.chunks()) r.load(c, lane, x);
    for (int i = tid; i < kBins; i += kPickThreads) { weights[i] = 0; counts[i] = 0; }
    __syncthreads();
    const float most = w->most;
    const uint32_t most_key = key_of(most);
    if (c < r.chunks()) {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (!(x[i] > kNegInf)) continue;
            const uint32_t bin = bin_of(key_of(x[i]), most, most_key, (float)s.rate);
            if (s.top_p < 1.0) atomicAdd(reinterpret_cast<unsigned long long *>(&weights[bin]), (unsigned long long)units(weight(x[i], most, s.rate)));
            atomicAdd(&counts[bin], 1u);
        }
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kPickThreads) {
        if (!counts[i]) continue;
        if (s.top_p < 1.0) atomicAdd(reinterpret_cast<unsigned long long *>(&w->weights[i]), (unsigned long long)weights[i]);
        atomicAdd(&w->counts[i], counts[i]);
    }
}

// The bins in which a row's cuts lie: that of its top-k in the last of them, that of its top-p in one of them (with both it depends on what the first k weigh, of which the
// bins in front of the last tell the least).  What is above them, and their tokens.  first == kBins: everything is kept.
struct CutBins {
    uint32_t first, last;
    uint64_t above, above_weight;  // tokens and weight
    uint32_t tokens;
    bool counted;  // the top-k cuts something off
    uint64_t all;  // without a top-k that does: the weight of the row
};
__device__ __forceinline__ CutBins bins_of_cuts(PickLds &l, const Settings &s, const Wide &w) {
    const int tid = (int)threadIdx.x;
    CutBins c{kBins, kBins, 0, 0, 0, false, 0};
    if (!s.orders()) return c;
    const bool weighs = s.top_p < 1.0;
    for (int i = tid; i < kBins; i += kPickThreads) {
        if (s.k) l.counts[i] = w.counts[i];
        if (weighs) l.weights[i] = w.weights[i];
    }
    __syncthreads();
    if (s.k) c.last = find_bin<kBins>(l, true, (uint64_t)s.k, c.above);
    c.counted = c.last < kBins;
    c.first = c.last;
    if (weighs) {
        uint64_t mine = 0;
        for (int i = tid; i < (int)c.last; i += kPickThreads) mine += l.weights[i];
        c.all = sum_of_threads(mine, l.waves);
        c.first = find_bin<kBins>(l, false, share_of(s, c.all), c.above_weight);
        if (!c.counted) c.last = c.first;
    }
    if (c.first >= kBins) return c;
    if (c.first == c.last) {
        c.tokens = w.counts[c.first];
    } else {
        uint64_t in = 0, above = 0;
        for (int i = tid; i <= (int)c.last; i += kPickThreads) (i < (int)c.first ? above : in) += l.counts[i];
        c.above = sum_of_threads(above, l.waves);
        c.tokens = (uint32_t)sum_of_threads(in, l.waves);
    }
    return c;
}

template <bool BF16> __global__ __launch_bounds__(kPickThreads) void sample_gather_kernel(const SampleArgs a, int parts) {
    __shared__ PickLds l;
    const int slot = (int)blockIdx.x / parts, tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Wide *w = wide_of(a, slot);
    if (!w) return;
    const int64_t row = w->row;
    const Row<BF16> r(a, row);
    const Settings s = settings_of(a, row);
    const int c = ((int)blockIdx.x - slot * parts) * kPickWaves + wave;
    float x[32];
    if (c < r.chunks()) r.load(c, lane, x);
    const CutBins bins = bins_of_cuts(l, s, *w);
    if (c >= r.chunks() || bins.tokens > (uint32_t)kListMost) return;
    const float most = w->most;
    const uint32_t most_key = key_of(most), floor_key = w->floor_key;
    uint64_t sum = 0;
    uint32_t in = 0, found = 0;  // which of the lane's are in the bins; how many of the wavefront's
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const uint32_t key = key_of(x[i]);
        const uint32_t mine = x[i] > kNegInf ? bin_of(key, most, most_key, (float)s.rate) : kAll;
        if (mine < bins.first && key >= floor_key) sum += units(weight(x[i], most, s.rate));
        const bool listed = mine >= bins.first && mine <= bins.last && mine < kBins;  // (whatever min-p says: top-p goes by all of the first k)
        in |= (uint32_t)listed << i;
        found += __popcll(__ballot(listed));
    }
    if (found) {
        uint32_t to = 0;
        if (lane == 0) to = atomicAdd(&w->listed, found);
        to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const uint64_t all = __ballot(in >> i & 1u);
            if (in >> i & 1u) {
                const uint32_t at = to + __popcll(all & ((1ull << lane) - 1));
                w->keys[at] = key_of(x[i]);
                w->chunks[at] = (uint16_t)c;
            }
            to += __popcll(all);
        }
    }
    sum = over_lanes(sum, Sum{});
    if (lane == 0) w->chunk_weight[c] = sum;
}

template <bool BF16> __global__ __launch_bounds__(kPickThreads, 4) void sample_wide_kernel(const SampleArgs a) {
    __shared__ PickLds l;
    const int tid = (int)threadIdx.x;
    const Wide *w = wide_of(a, (int)blockIdx.x);
    if (!w) return;
    const int64_t row = w->row;
    const Row<BF16> r(a, row);
    const Settings s = settings_of(a, row);
    const int chunks = r.chunks();
    const float most = w->most;
    const uint32_t most_key = key_of(most), floor_key = w->floor_key;
    const auto weight_of = [&](uint32_t key) { return units(weight(value_of(key), most, s.rate)); };
    const CutBins bins = bins_of_cuts(l, s, *w);
    if (bins.tokens > (uint32_t)kListMost) {
        __syncthreads();
        draw_alone(a, l, r, s, row, chunks, most, most_key, floor_key);
        return;
    }
    __syncthreads();
    const int n = bins.first < kBins ? (int)w->listed : 0;
    for (int i = tid; i < n; i += kPickThreads) { l.keys[i] = w->keys[i]; l.chunks[i] = w->chunks[i]; }
    for (int i = tid; i < chunks; i += kPickThreads) l.chunk_weight[i] = w->chunk_weight[i];
    if (tid == 0) l.listed = (uint32_t)n;
    __syncthreads();
    Cut cut{0u, kAll, 0};
    uint64_t all = bins.all;
    if (n && bins.counted) {
        Cut c{0u, 0u, bins.above};
        if (cut_of_list(l, weight_of, true, (uint64_t)s.k, c)) cut = c;
        all = bins.above_weight;
        if (s.top_p < 1.0) all += keep_of_list(l, weight_of, cut);
    }
    if (n && s.top_p < 1.0) {
        Cut c{0u, 0u, bins.above_weight};
        if (cut_of_list(l, weight_of, false, share_of(s, all), c)) cut = c;
    }
    if (floor_key > cut.key) cut = Cut{floor_key, kAll, 0};
    chunks_of_list(l, weight_of, cut, chunks, false);
    draw(a, l, r, s, row, chunks, most, cut);
}

}  // namespace

int launch_sample(const void *logits, bool bf16, int64_t rows, int64_t vocab, int64_t row_stride, const float *uniform, const Sampling &how, int32_t *tokens,
                  float *probabilities, hipStream_t s) {
    SampleArgs a{};
    a.row_bytes = row_stride * (bf16 ? 2 : 4);
    a.vocab = (int)vocab;
    a.chunks = (int)((vocab + 7 + kChunk - 1) / kChunk);
    // as many rows at a time as 256 MB of workspace hold
    const size_t a_row = (size_t)a.chunks * (sizeof(Chunk) + kChunkKeys * 4);
    const int64_t batch = std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)(((size_t)256 << 20) / a_row)));
    // Flat rows have launches of their own where a bound may lead below a chunk's list (not a small top-k, which the lists hold: 48 keys of a chunk and more, where not too many of them are equal) and a workgroup
    // would go over a row in several rounds.  Where they find nothing to do they add 6 us: one row of 128256 under top-k 50 and top-p 0.9 23 us without them and 29 with them, 512 rows 100 and 104; a row that
    // needs them and has none takes 70 to 200 more.
    const bool cuts = how.top_ks || how.top_ps || how.min_ps || how.top_k > 0 || how.top_p < 1.0 || how.min_p > 0.0;
    const bool wide = cuts && (how.top_ks || how.top_k <= 0 || how.top_k > 64) && a.chunks > kPickWaves;
    a.wide_rows = (int)std::min<int64_t>(batch, kWideRows);
    const size_t lists = (size_t)batch * a_row, wides = (lists + 255) / 256 * 256, flat = wides + 256;
    void *ws = nullptr;
    if (int rc = stream_workspace(s, flat + (wide ? a.wide_rows * sizeof(Wide) : 0), &ws)) return rc;
    unsigned char *at = static_cast<unsigned char *>(ws);
    a.chunk = reinterpret_cast<Chunk *>(at);
    a.keys = reinterpret_cast<uint32_t *>(a.chunk + batch * a.chunks);
    a.wides = reinterpret_cast<uint32_t *>(at + wides);
    a.wide = wide ? reinterpret_cast<Wide *>(at + flat) : nullptr;
    const int parts = (a.chunks + kPickWaves - 1) / kPickWaves;
    for (int64_t row = 0; row < rows; row += batch) {
        const int64_t n = std::min(batch, rows - row), waves = n * a.chunks;
        a.logits = static_cast<const uint8_t *>(logits) + row * a.row_bytes;
        a.how = how;
        if (how.temperatures) a.how.temperatures += row;
        if (how.top_ks) a.how.top_ks += row;
        if (how.top_ps) a.how.top_ps += row;
        if (how.min_ps) a.how.min_ps += row;
        a.uniform = uniform + row;
        a.tokens = tokens + row;
        a.probabilities = probabilities ? probabilities + row : nullptr;
        const dim3 block(kPickThreads), slices((unsigned)(a.wide_rows * parts));
        if (int rc = launch(bf16 ? sample_scan_kernel<true> : sample_scan_kernel<false>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, a, waves)) return rc;
        if (int rc = launch(bf16 ? sample_pick_kernel<true> : sample_pick_kernel<false>, dim3((unsigned)n), block, 0, s, a)) return rc;
        if (!wide) continue;
        if (int rc = launch(bf16 ? sample_bins_kernel<true> : sample_bins_kernel<false>, slices, block, 0, s, a, parts)) return rc;
        if (int rc = launch(bf16 ? sample_gather_kernel<true> : sample_gather_kernel<false>, slices, block, 0, s, a, parts)) return rc;
        if (int rc = launch(bf16 ? sample_wide_kernel<true> : sample_wide_kernel<false>, dim3((unsigned)a.wide_rows), block, 0, s, a)) return rc;
    }
    return GQ_OK;
}

}  // namespace gq
