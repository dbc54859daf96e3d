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
// Two launches.  The first reads the logits once: a wavefront a chunk, which leaves its maximum, its sum and its largest keys (32 at least, some 45, complete from
// a level on).  In the second a workgroup a row finds the cut among the keys that the chunks have left, and reads a single chunk again.  Where the cut lies
// below what they have left (a flat distribution under top-p) it goes over the row again, three times or more.
#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace gq {

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 2048, kChunkKeys = 128, kMostChunks = 1024;
constexpr int kPickThreads = 512, kPickWaves = kPickThreads / 64, kBins = 2048, kListMost = 6144;
constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr float kNegInf = -__builtin_huge_valf();

struct Chunk {
    double sum;      // of the weights, the chunk's largest 1
    float most;
    int at;          // the lowest index of the largest
    uint32_t level;  // the list has every key from here on
    int count;
};

struct SampleArgs {
    const uint8_t *logits;
    int64_t row_bytes;
    int vocab, chunks;  // of a row, at most
    Sampling how;
    const float *uniform;
    Chunk *chunk;      // [rows, chunks]
    uint32_t *keys;    // [rows, chunks, kChunkKeys]
    int32_t *tokens;
    float *probabilities;  // may be null
};

struct Settings {
    double t, top_p, min_p, rate;  // rate: 1 / t in powers of two
    int k;                 // 0: all
    bool first;            // the first of the order
    __device__ __forceinline__ bool cuts() const { return k || top_p < 1.0 || min_p > 0.0; }
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
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : kNegInf; }
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// 2^y for y <= 0, to 1e-11 of itself: the series of exp(f ln 2) for |f| <= 1/2 up to its ninth power.
__device__ __forceinline__ double power_of_two(double y) {
    y = fmax(y, -1100.0);  // (a NaN too: 0)
    const double n = __builtin_rint(y), f = y - n;
    double p = 1.01780860092396997e-7;   // ln(2)^k / k!, k = 9, 8, ...
    p = fma(p, f, 1.32154867901443095e-6);
    p = fma(p, f, 1.52527338040598403e-5);
    p = fma(p, f, 1.54035303933816099e-4);
    p = fma(p, f, 1.33335581464284434e-3);
    p = fma(p, f, 9.61812910762847716e-3);
    p = fma(p, f, 5.55041086648215800e-2);
    p = fma(p, f, 2.40226506959100712e-1);
    p = fma(p, f, 6.93147180559945309e-1);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}
__device__ __forceinline__ double weight(float x, float most, double rate) { return x == most ? 1.0 : power_of_two(((double)x - (double)most) * rate); }
constexpr double kUnit = 4398046511104.0;  // 2^42: a vocabulary of 2^21 tokens of the same weight sums to 2^63
__device__ __forceinline__ uint64_t units(double w) { return (uint64_t)__builtin_rint(w * kUnit); }

// A row as 16-byte blocks, aligned: `lead` places in front of its first logit are no part of it.
template <bool BF16> struct Row {
    static constexpr int kSize = BF16 ? 2 : 4, kBlock = 16 / kSize, kLoads = kChunk / 64 / kBlock;
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
        if constexpr (BF16) return clean(__uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(base)[place] << 16));
        else return clean(reinterpret_cast<const float *>(base)[place]);
    }
    // where value i of lane `lane` of a chunk lies
    __device__ __forceinline__ static int place(int chunk, int lane, int i) { return chunk * kChunk + ((i / kBlock) * 64 + lane) * kBlock + i % kBlock; }
    __device__ __forceinline__ void load(int chunk, int lane, float (&x)[32]) const {
        if (chunk * kChunk >= lead && (chunk + 1) * kChunk <= end) {
            u4 w[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; i++) w[i] = *reinterpret_cast<const u4 *>(base + (int64_t)place(chunk, lane, i * kBlock) * kSize);
#pragma unroll
            for (int i = 0; i < 32; i++) {
                if constexpr (BF16) {
                    const uint32_t u = w[i / 8][i % 8 / 2];
                    x[i] = clean(__uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16));
                } else {
                    x[i] = clean(__uint_as_float(w[i / 4][i % 4]));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = one(place(chunk, lane, i));
        }
    }
};

template <class T, class F> __device__ __forceinline__ T over_lanes(T v, F f) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = f(v, __shfl_xor(v, m));
    return v;
}

// One wavefront a chunk.  The level: of the lanes' largest keys the 32nd (its upper 16 bits), so that 32 keys at least are at or above it and, where the large ones
// lie anywhere, some 45 of 2048.
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
    float mine = kNegInf;
#pragma unroll
    for (int i = 0; i < 32; i++) mine = fmaxf(mine, x[i]);
    const float most = over_lanes(mine, [](float p, float q) { return fmaxf(p, q); });
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 31; i >= 0; i--) at = x[i] == most ? Row<BF16>::place(chunk, lane, i) - r.lead : at;
    at = over_lanes(at, [](int p, int q) { return min(p, q); });
    Chunk c{0.0, most, at, kAll, 0};
    if (!s.first && most > kNegInf) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 32; i++) sum += weight(x[i], most, s.rate);
        c.sum = over_lanes(sum, [](double p, double q) { return p + q; });
        if (s.cuts()) {
            const uint32_t top = key_of(mine);
            uint32_t level = 0;
#pragma unroll
            for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
                if (__popcll(__ballot(top >= (level | bit))) >= 32) level |= bit;
            uint32_t *keys = a.keys + index * kChunkKeys;
            int count = 0;
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const uint32_t key = key_of(x[i]);
                const bool in = key >= level && x[i] > kNegInf;
                const uint64_t all = __ballot(in);
                const int to = count + __popcll(all & ((1ull << lane) - 1));
                if (in && to < kChunkKeys) keys[to] = key;
                count += __popcll(all);
            }
            if (count <= kChunkKeys) { c.level = level; c.count = count; }
        }
    }
    if (lane == 0) a.chunk[index] = c;
}

// ---- the second launch ------------------------------------------------------------------------------------------------

// Sums of the threads in front of each, in order; `total` of all of them.
template <class T> __device__ __forceinline__ T threads_in_front(T v, T *waves, T &total) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    T upto = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const T o = __shfl_up(upto, m);
        if (lane >= m) upto += o;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    T front = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; i++) {
        if (i < wave) front += waves[i];
        total += waves[i];
    }
    return front + upto - v;
}

// The last kept token: the kept ones are those of larger key and the first `ties` of this one; how many are above it, and their weight.
struct Cut {
    uint32_t key, ties;
    uint32_t above;
    uint64_t above_weight;
};

struct PickLds {
    uint64_t weights[kBins];
    uint32_t counts[kBins];
    uint32_t keys[kListMost];
    uint16_t chunks[kListMost];
    uint64_t chunk_weight[kMostChunks];
    uint32_t chunk_ties[kMostChunks];
    uint64_t waves[kPickWaves];
    uint64_t found_weight;
    uint32_t found, found_count, listed;
};

// The first of the bins, from bin 0 on, up to which `want` is reached, of tokens (by count) or of weight; what is in front of it.  kBins: none.
__device__ __forceinline__ uint32_t find_bin(PickLds &l, bool by_count, uint64_t want, uint32_t &above, uint64_t &above_weight) {
    constexpr int N = kBins / kPickThreads;
    const int first = (int)threadIdx.x * N;
    uint64_t weights = 0, counts = 0, total;
    if (threadIdx.x == 0) l.found = kBins;
#pragma unroll
    for (int i = 0; i < N; i++) { weights += l.weights[first + i]; counts += l.counts[first + i]; }
    uint64_t w = threads_in_front(weights, l.waves, total) + above_weight, c = threads_in_front(counts, l.waves, total) + above;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint64_t bw = l.weights[first + i], bc = l.counts[first + i];
        const uint64_t before = by_count ? c : w, after = by_count ? c + bc : w + bw;
        if (before < want && want <= after) {
            l.found = (uint32_t)(first + i);
            l.found_count = (uint32_t)c;
            l.found_weight = w;
        }
        w += bw;
        c += bc;
    }
    __syncthreads();
    const uint32_t bin = l.found;
    if (bin < kBins) { above = l.found_count; above_weight = l.found_weight; }
    __syncthreads();
    return bin;
}

__device__ __forceinline__ void clear_bins(PickLds &l) {
    __syncthreads();
    for (int i = (int)threadIdx.x; i < kBins; i += kPickThreads) { l.weights[i] = 0; l.counts[i] = 0; }
    __syncthreads();
}
__device__ __forceinline__ void add_to_bin(PickLds &l, uint32_t bin, uint64_t weight) {
    atomicAdd(reinterpret_cast<unsigned long long *>(&l.weights[bin]), (unsigned long long)weight);
    atomicAdd(&l.counts[bin], 1u);
}

// The cut at `want` tokens (or weight) among the keys that `each` passes on, with `cut` as what is above all of these: digit by digit, 11, 11 and 10 bits.  False: they
// do not reach it.
template <class Each, class Weight> __device__ __forceinline__ bool find_cut(PickLds &l, Each each, Weight weight_of, bool by_count, uint64_t want, Cut &cut) {
    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, done = pass == 0 ? 32 : pass == 1 ? 21 : 10;
        clear_bins(l);
        each([&](uint32_t key, int) {
            if (done < 32 && key >> done != prefix >> done) return;
            const uint32_t digits = pass == 2 ? 1023u : 2047u;
            add_to_bin(l, digits - (key >> shift & digits), weight_of(key));  // (the largest first)
        });
        __syncthreads();
        const uint32_t bin = find_bin(l, by_count, want, cut.above, cut.above_weight);
        if (bin >= kBins) return false;
        prefix |= ((pass == 2 ? 1023u : 2047u) - bin) << shift;
        if (pass == 2) {
            const uint32_t all = l.counts[bin];
            const uint64_t left = want - (by_count ? cut.above : cut.above_weight), w = by_count ? 1 : weight_of(prefix);
            const uint64_t ties = (left + w - 1) / w;
            cut.ties = ties < all ? (uint32_t)ties : all;
        }
    }
    cut.key = prefix;
    __syncthreads();
    return true;
}

template <bool BF16> __global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(const SampleArgs a) {
    __shared__ PickLds l;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x;
    const Row<BF16> r(a, row);
    const Settings s = settings_of(a, row);
    const int chunks = r.chunks();
    const Chunk *chunk = a.chunk + row * a.chunks;

    // the row's largest logit; where; the level from which on the lists have every key; their length
    float most = kNegInf;
    int at = 0x7FFFFFFF;
    uint32_t level = 0;
    for (int c = tid; c < chunks; c += kPickThreads) {
        const float m = chunk[c].most;
        if (m > most) { most = m; at = chunk[c].at; }
        if (m > kNegInf) level = max(level, chunk[c].level);
    }
    const float wave_most = over_lanes(most, [](float p, float q) { return fmaxf(p, q); });
    at = over_lanes(most == wave_most ? at : 0x7FFFFFFF, [](int p, int q) { return min(p, q); });
    level = over_lanes(level, [](uint32_t p, uint32_t q) { return max(p, q); });
    if (lane == 0) {
        l.weights[wave] = key_of(wave_most);
        l.counts[wave] = (uint32_t)at;
        l.counts[kPickWaves + wave] = level;
    }
    __syncthreads();
    uint32_t most_key = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; i++) {
        const uint32_t k = (uint32_t)l.weights[i];
        at = k > most_key ? (int)l.counts[i] : k == most_key ? min(at, (int)l.counts[i]) : at;
        most_key = max(most_key, k);
        level = max(level, l.counts[kPickWaves + i]);
    }
    most = value_of(most_key);
    if (s.first || most == kNegInf) {  // (a row without a number has no token)
        if (tid == 0) {
            a.tokens[row] = most == kNegInf ? -1 : at;
            if (a.probabilities) a.probabilities[row] = most == kNegInf ? 0.0f : 1.0f;
        }
        return;
    }
    const auto weight_of = [&](uint32_t key) { return units(weight(value_of(key), most, s.rate)); };
    const auto each_listed = [&](auto f) {
        for (int i = tid; i < (int)l.listed; i += kPickThreads) f(l.keys[i], (int)l.chunks[i]);
    };
    const auto each_of_row = [&](auto f) {
#pragma unroll 1
        for (int c = wave; c < chunks; c += kPickWaves) {
            float x[32];
            r.load(c, lane, x);
#pragma unroll
            for (int i = 0; i < 32; i++)
                if (x[i] > kNegInf) f(key_of(x[i]), c);
        }
    };

    // the cut: nothing, to begin with
    Cut cut{0u, kAll, 0u, 0u};
    uint32_t floor_key = 0;  // what min-p asks for
    if (s.min_p > 0.0) {
        const double least = (double)most + s.t * log(s.min_p);
        float f = (float)least;
        if ((double)f < least) f = value_of(key_of(f) + 1);
        floor_key = most == __builtin_huge_valf() ? most_key : min(most_key, key_of(clean(f)));
    }
    const bool orders = s.k || s.top_p < 1.0;
    bool from_lists = s.cuts() && level != kAll && (orders || floor_key >= level);
    if (from_lists) {
        if (tid == 0) l.listed = 0;
        __syncthreads();
#pragma unroll 1
        for (int c = wave; c < chunks; c += kPickWaves) {
            const int count = chunk[c].most > kNegInf ? chunk[c].count : 0;
            const uint32_t *keys = a.keys + (row * a.chunks + c) * kChunkKeys;
            for (int i = lane; i < count; i += 64) {
                const uint32_t key = keys[i];
                if (key < level) continue;
                const uint32_t to = atomicAdd(&l.listed, 1u);
                if (to < (uint32_t)kListMost) { l.keys[to] = key; l.chunks[to] = (uint16_t)c; }
            }
        }
        __syncthreads();
        from_lists = l.listed <= (uint32_t)kListMost;
    }
    // the weight of the row, for top-p without top-k
    uint64_t all = 0;
    if (!s.k && s.top_p < 1.0) {
        double sum = 0.0;
        for (int c = tid; c < chunks; c += kPickThreads)
            if (chunk[c].most > kNegInf) sum += chunk[c].sum * weight(chunk[c].most, most, s.rate);
        uint64_t total;
        threads_in_front(units(sum), l.waves, total);
        all = total;
    }
    const auto share = [&](uint64_t w) {
        const double p = ceil(s.top_p * (double)w);
        return p < 1.0 ? (uint64_t)1 : (uint64_t)p;
    };
    if (from_lists && orders) {
        if (s.k) {
            Cut c{0u, 0u, 0u, 0u};
            from_lists = find_cut(l, each_listed, weight_of, true, (uint64_t)s.k, c);
            if (from_lists) {
                cut = c;
                all = c.above_weight + c.ties * weight_of(c.key);
            }
        }
        if (from_lists && s.top_p < 1.0) {
            Cut c{0u, 0u, 0u, 0u};
            from_lists = find_cut(l, each_listed, weight_of, false, share(all), c);
            if (from_lists) cut = c;
        }
    }
    if (s.cuts() && !from_lists && orders) {
        // over the row again: bins of 1/32 in powers of two, then the keys of the one with the cut in it
        const auto bin_of = [&](uint32_t key) {
            const float d = (most - value_of(key)) * (float)s.rate * 32.0f;
            return key == most_key ? 0u : (uint32_t)fminf(d, (float)(kBins - 1));
        };
        const auto cut_at = [&](bool by_count, uint64_t want, Cut &c) {
            clear_bins(l);
            each_of_row([&](uint32_t key, int) { add_to_bin(l, bin_of(key), weight_of(key)); });
            __syncthreads();
            if (!by_count && !s.k) {  // (the sum of these very numbers)
                uint64_t mine = 0;
                for (int i = tid; i < kBins; i += kPickThreads) mine += l.weights[i];
                threads_in_front(mine, l.waves, all);
                want = share(all);
            }
            const uint32_t bin = find_bin(l, by_count, want, c.above, c.above_weight);
            if (bin >= kBins) return false;
            const bool fits = l.counts[bin] <= (uint32_t)kListMost;
            __syncthreads();
            if (!fits)
                return find_cut(l, [&](auto f) { each_of_row([&](uint32_t key, int at_chunk) { if (bin_of(key) == bin) f(key, at_chunk); }); }, weight_of, by_count, want, c);
            if (tid == 0) l.listed = 0;
            __syncthreads();
            each_of_row([&](uint32_t key, int at_chunk) {
                if (bin_of(key) != bin) return;
                const uint32_t to = atomicAdd(&l.listed, 1u);
                l.keys[to] = key;
                l.chunks[to] = (uint16_t)at_chunk;
            });
            __syncthreads();
            return find_cut(l, each_listed, weight_of, by_count, want, c);
        };
        if (s.k) {
            Cut c{0u, 0u, 0u, 0u};
            if (cut_at(true, (uint64_t)s.k, c)) {
                cut = c;
                all = c.above_weight + c.ties * weight_of(c.key);
            } else if (s.top_p < 1.0) {  // (fewer numbers than k: all of them)
                uint64_t mine = 0;
                for (int i = tid; i < kBins; i += kPickThreads) mine += l.weights[i];
                threads_in_front(mine, l.waves, all);
            }
        }
        if (s.top_p < 1.0) {
            Cut c{0u, 0u, 0u, 0u};
            if (cut_at(false, share(all), c)) cut = c;
        }
    }
    if (floor_key > cut.key) cut = Cut{floor_key, kAll, 0u, 0u};

    // the kept weight of every chunk, and its tokens that equal the cut's
    if (from_lists) {
        __syncthreads();
        for (int c = tid; c < chunks; c += kPickThreads) { l.chunk_weight[c] = 0; l.chunk_ties[c] = 0; }
        __syncthreads();
        each_listed([&](uint32_t key, int c) {
            if (key > cut.key) atomicAdd(reinterpret_cast<unsigned long long *>(&l.chunk_weight[c]), (unsigned long long)weight_of(key));
            else if (key == cut.key) atomicAdd(&l.chunk_ties[c], 1u);
        });
    } else if (s.cuts()) {
#pragma unroll 1
        for (int c = wave; c < chunks; c += kPickWaves) {
            float x[32];
            r.load(c, lane, x);
            uint64_t sum = 0;
            uint32_t ties = 0;
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const uint32_t key = key_of(x[i]);
                if (x[i] > kNegInf && key > cut.key) sum += weight_of(key);
                ties += x[i] > kNegInf && key == cut.key;
            }
            sum = over_lanes(sum, [](uint64_t p, uint64_t q) { return p + q; });
            ties = over_lanes(ties, [](uint32_t p, uint32_t q) { return p + q; });
            if (lane == 0) { l.chunk_weight[c] = sum; l.chunk_ties[c] = ties; }
        }
    } else {
        for (int c = tid; c < chunks; c += kPickThreads) {
            l.chunk_weight[c] = chunk[c].most > kNegInf ? units(chunk[c].sum * weight(chunk[c].most, most, s.rate)) : 0;
            l.chunk_ties[c] = 0;
        }
    }
    __syncthreads();

    // the chunk: two neighbouring ones a thread
    const uint64_t cut_weight = s.cuts() ? weight_of(cut.key) : 0;
    constexpr int N = kMostChunks / kPickThreads;
    uint64_t kept[N], mine = 0, total;
    uint32_t ties[N], my_ties = 0;
    const int c0 = tid * N;
#pragma unroll
    for (int i = 0; i < N; i++) {
        kept[i] = c0 + i < chunks ? l.chunk_weight[c0 + i] : 0;
        ties[i] = c0 + i < chunks ? l.chunk_ties[c0 + i] : 0;
        my_ties += ties[i];
    }
    uint64_t tie_total;
    uint64_t tie_front = threads_in_front((uint64_t)my_ties, l.waves, tie_total);
    uint64_t tie_at[N];
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
            l.found_weight = front;
            l.chunk_weight[0] = kept[i];
            l.found_count = (uint32_t)min(tie_at[i], (uint64_t)kAll);
        }
        front += kept[i];
    }
    __syncthreads();

    // the token: four neighbouring ones a thread
    const int c = (int)l.found;
    want -= l.found_weight;
    const uint64_t of_chunk = l.chunk_weight[0];
    uint32_t rank = l.found_count;
    // (with nothing cut off the chunk's weight is a sum in 64 bits, not one of these units, of which its tokens may have none: in parts of the chunk then)
    const float unit_most = s.cuts() ? most : chunk[c].most;
    __syncthreads();
    constexpr int M = kChunk / kPickThreads;
    float x[M];
    my_ties = 0;
#pragma unroll
    for (int i = 0; i < M; i++) {
        x[i] = r.one(c * kChunk + tid * M + i);
        my_ties += s.cuts() && x[i] > kNegInf && key_of(x[i]) == cut.key;
    }
    rank += (uint32_t)threads_in_front((uint64_t)my_ties, l.waves, tie_total);
    mine = 0;
    uint64_t w[M];
#pragma unroll
    for (int i = 0; i < M; i++) {
        const uint32_t key = key_of(x[i]);
        const bool tie = s.cuts() && key == cut.key;
        const bool keep = x[i] > kNegInf && (!s.cuts() || key > cut.key || (tie && rank < cut.ties));
        if (tie && x[i] > kNegInf) rank++;
        w[i] = keep ? units(weight(x[i], unit_most, s.rate)) : 0;
        mine += w[i];
    }
    uint64_t in_chunk;
    front = threads_in_front(mine, l.waves, in_chunk);
    if (!s.cuts()) want = (uint64_t)((double)want / (double)of_chunk * (double)in_chunk);
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

}  // namespace

int launch_sample(const void *logits, bool bf16, int64_t rows, int64_t vocab, int64_t row_stride, const float *uniform, const Sampling &how, int32_t *tokens,
                  float *probabilities, hipStream_t s) {
    SampleArgs a{};
    a.row_bytes = row_stride * (bf16 ? 2 : 4);
    a.vocab = (int)vocab;
    a.chunks = (int)((vocab + 7 + kChunk - 1) / kChunk);
    if (a.chunks > kMostChunks) return fail(GQ_ERR_INVALID, "sample: a vocabulary of %lld tokens: at most %d", (long long)vocab, kMostChunks * kChunk - 7);
    // as many rows at a time as 256 MB of workspace hold
    const size_t a_row = (size_t)a.chunks * (sizeof(Chunk) + kChunkKeys * 4);
    const int64_t batch = std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)(((size_t)256 << 20) / a_row)));
    void *ws = nullptr;
    if (int rc = stream_workspace(s, (size_t)batch * a_row, &ws)) return rc;
    a.chunk = static_cast<Chunk *>(ws);
    a.keys = reinterpret_cast<uint32_t *>(a.chunk + batch * a.chunks);
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
        if (int rc = launch(bf16 ? sample_scan_kernel<true> : sample_scan_kernel<false>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, a, waves)) return rc;
        if (int rc = launch(bf16 ? sample_pick_kernel<true> : sample_pick_kernel<false>, dim3((unsigned)n), dim3(kPickThreads), 0, s, a)) return rc;
    }
    return GQ_OK;
}

}  // namespace gq
