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

template <int NE, bool BF16> __device__ __forceinline__ void load_values(float (&v)[NE], const void *p, int64_t at, int wide) {
    if constexpr (BF16) {
        const uint16_t *x = static_cast<const uint16_t *>(p) + at;
        uint32_t u[NE];
        if (NE == 2 && wide) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(x);
            u[0] = w & 0xFFFFu;
            u[NE - 1] = w >> 16;
        } else if (NE == 4 && wide) {
            const u2 w = *reinterpret_cast<const u2 *>(x);
            u[0] = w.x & 0xFFFFu;
            u[1 % NE] = w.x >> 16;
            u[2 % NE] = w.y & 0xFFFFu;
            u[NE - 1] = w.y >> 16;
        } else {
#pragma unroll
            for (int i = 0; i < NE; i++) u[i] = x[i];
        }
#pragma unroll
        for (int i = 0; i < NE; i++) v[i] = __uint_as_float(u[i] << 16);
    } else {
        const float *x = static_cast<const float *>(p) + at;
        if (NE == 2 && wide) {
            const float2 w = *reinterpret_cast<const float2 *>(x);
            v[0] = w.x;
            v[NE - 1] = w.y;
        } else if (NE == 4 && wide) {
            const float4 w = *reinterpret_cast<const float4 *>(x);
            v[0] = w.x;
            v[1 % NE] = w.y;
            v[2 % NE] = w.z;
            v[NE - 1] = w.w;
        } else {
#pragma unroll
            for (int i = 0; i < NE; i++) v[i] = x[i];
        }
    }
}

// A group's scale, from the NE values of each of its 32 / NE lanes: minus an eighth of the value of largest magnitude (the
// first of those), rounded to 8 significant bits.  The value itself then has code 0 and none is more than 8 steps away.
template <int NE> __device__ __forceinline__ float group_scale(const float (&v)[NE]) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < NE; i++) m = fabsf(v[i]) > fabsf(m) ? v[i] : m;
#pragma unroll
    for (int s = 1; s < 32 / NE; s <<= 1) {
        const float o = __shfl_xor(m, s);
        const bool take = fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && ((int)threadIdx.x & s));
        m = take ? o : m;
    }
    return half_value(half_bits(round_to_bf16(m * -0.125f)));
}
__device__ __forceinline__ uint32_t code_of(float v, float d) {
    return d == 0.0f ? 8u : (uint32_t)fminf(fmaxf(floorf(v / d + 8.5f), 0.0f), 15.0f);
}

// Eight tokens of one block (a lane's share of a value operand: their codes share dwords) per wavefront, key head and sequence;
// a lane holds D / 64 values of every token.  A dword of value codes belongs to one lane of one wavefront of the launch, so
// that tokens that share bytes need no atomics.
struct AppendArgs {
    KvCall kv;
    HeadRows k, v;
    float *accounts;
    int blocks, wide;  // blocks of eight tokens that the new ones of a sequence can touch
};

template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
    typedef KvTile<D> T;
    constexpr int NE = D / 64, G = T::G;
    const KvCall &kv = a.kv;
    const int64_t unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int per = kv.kv_heads * a.blocks;
    const int b = (int)(unit / per);
    if (b >= kv.seqs) return;
    const int rest = (int)(unit - (int64_t)b * per), h = rest / a.blocks, nth = rest - h * a.blocks;
    const KvSeq s = kv_seq(kv, b);
    const int first = s.length - s.news, from = first < 0 ? 0 : first;
    const int block = (from >> 3) + nth, p0 = block * 8;
    if (p0 >= s.length || s.news == 0) return;
    uint8_t *tile = kv_tile(kv, b, h, p0 >> 5, T::kBytes);
    if (!tile) return;
    const int lane = (int)threadIdx.x & 63, x = lane * NE;  // first value of the lane
    const int j = (p0 >> 3) & 3, g = x >> 5;

    float k[8][NE], v[8][NE];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int p = p0 + e;
        const bool live = p >= from && p < s.length;
        const int64_t row = live ? s.row0 + (p - first) : s.row0;
        load_values<NE, BF16>(k[e], a.k.p, row * a.k.row + h * a.k.head + x, a.wide);
        load_values<NE, BF16>(v[e], a.v.p, row * a.v.row + h * a.v.head + x, a.wide);
    }
    uint32_t bits[NE] = {}, live_mask = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int p = p0 + e;
        if (p < from || p >= s.length) continue;
        bool good = true;
#pragma unroll
        for (int i = 0; i < NE; i++) good = good && fabsf(k[e][i]) < kLargest && fabsf(v[e][i]) < kLargest;
        good = __all(good);
        if (!good) {
#pragma unroll
            for (int i = 0; i < NE; i++) k[e][i] = v[e][i] = 0.0f;
        }
        const float dk = group_scale<NE>(k[e]), dv = group_scale<NE>(v[e]);
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < NE; i++) {
            word |= code_of(k[e][i], dk) << nibble_shift((x + i) & 7);
            bits[i] |= code_of(v[e][i], dv) << nibble_shift(e);
        }
        live_mask |= 0xFu << nibble_shift(e);
#pragma unroll
        for (int m = 1; m < 8 / NE; m <<= 1) word |= (uint32_t)__shfl_xor((int)word, m);
        const int t = p & 31;
        if ((x & 7) == 0) {
            const int w = key_half(t) * G + g, l = key_row(t) + 16 * ((x >> 3) & 3);
            *reinterpret_cast<uint32_t *>(tile + T::kKeys + T::code(w, l)) = word;
        }
        if ((x & 31) == 0) {
            reinterpret_cast<uint16_t *>(tile + T::kKeyScales)[t * G + g] = (uint16_t)(good ? half_bits(dk) : kNanHalf);
            reinterpret_cast<uint16_t *>(tile + T::kValueScales)[g * 32 + t] = (uint16_t)half_bits(dv);
        }
        if (a.accounts && lane == 0) {
            float *at = kv_account(kv, a.accounts, b, h, p);
            if (at) *at = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const int c = x + i;
        uint32_t *at = reinterpret_cast<uint32_t *>(tile + T::kValues + T::code(c >> 4, (c & 15) + 16 * j));
        *at = live_mask == 0xFFFFFFFFu ? bits[i] : (*at & ~live_mask) | bits[i];
    }
}

// What the cache stands for at the last tokens of every sequence, in the fp16 numbers that it holds; zeros in front of a
// sequence's first token and where the page table names no page.
template <int D>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvCall kv, uint16_t *__restrict__ K, uint16_t *__restrict__ V, int blocks) {
    typedef KvTile<D> T;
    constexpr int NE = D / 64, G = T::G;
    const int64_t unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int per = kv.kv_heads * blocks;
    const int b = (int)(unit / per);
    if (b >= kv.seqs) return;
    const int rest = (int)(unit - (int64_t)b * per), h = rest / blocks, nth = rest - h * blocks;
    const KvSeq s = kv_seq(kv, b);
    const int first = s.length - s.news;
    const int p0 = (first >> 3) * 8 + nth * 8;  // (an arithmetic shift: blocks of eight also in front of the first token)
    if (p0 >= s.length) return;
    const uint8_t *tile = p0 >= 0 ? kv_tile(kv, b, h, p0 >> 5, T::kBytes) : nullptr;
    const int lane = (int)threadIdx.x & 63, x = lane * NE, j = (p0 >> 3) & 3, g = x >> 5;
    uint32_t vw[NE] = {};
    if (tile) {
#pragma unroll
        for (int i = 0; i < NE; i++) vw[i] = *reinterpret_cast<const uint32_t *>(tile + T::kValues + T::code((x + i) >> 4, ((x + i) & 15) + 16 * j));
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int p = p0 + e;
        if (p < first || p >= s.length) continue;
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

constexpr int kSelectThreads = 1024;

// The sum of v over the threads in front, and over all.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *waves, uint32_t &total) {
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    uint32_t inc = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)inc, s);
        if (lane >= s) inc += o;
    }
    __syncthreads();  // (the previous use of `waves` is over)
    if (lane == 63) waves[w] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelectThreads / 64; i++) {
        const uint32_t n = waves[i];
        before += i < w ? n : 0;
        all += n;
    }
    total = all;
    return before + inc - v;
}

__global__ __launch_bounds__(kSelectThreads) void kv_select_kernel(const KvCall kv, float *__restrict__ accounts, int keep, int recent, int32_t *__restrict__ kept) {
    __shared__ uint32_t hist[256], waves[kSelectThreads / 64], found[2];
    const int h = (int)blockIdx.x, b = (int)blockIdx.y, tid = (int)threadIdx.x;
    const KvSeq s = kv_seq(kv, b);
    int32_t *out = kept + ((int64_t)b * kv.kv_heads + h) * keep;
    if (s.length <= keep) {
        for (int i = tid; i < keep; i += kSelectThreads) out[i] = i < s.length ? i : -1;
        return;
    }
    const int n = s.length - recent;
    uint32_t want = (uint32_t)(keep - recent);  // of the first n tokens (n > want)
    // (an account without a page counts as the smallest)
    const auto key_at = [&](int t) {
        const float *p = kv_account(kv, accounts, b, h, t);
        return p ? account_key(*p) : 0u;
    };
    // the want-th largest key, eight bits at a time; `want` counts down to how many of the tokens that equal it are kept
    uint32_t key = 0;
    for (int shift = 24; shift >= 0 && want; shift -= 8) {
        for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += kSelectThreads) {
            const uint32_t u = key_at(t);
            if (shift == 24 || (u >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255u], 1u);
        }
        __syncthreads();
        const uint32_t mine = tid < 256 ? hist[255 - tid] : 0;  // the largest digits first
        uint32_t total;
        const uint32_t before = block_scan(mine, waves, total);
        if (tid < 256 && before < want && want <= before + mine) { found[0] = 255u - tid; found[1] = want - before; }
        __syncthreads();
        key |= found[0] << shift;
        want = found[1];
        __syncthreads();
    }
    const bool some = keep > recent;
    uint32_t at = 0, equal = 0;  // kept so far; tokens equal to the key so far
    for (int t0 = 0; t0 < s.length; t0 += kSelectThreads) {
        const int t = t0 + tid;
        const uint32_t u = t < n && some ? key_at(t) : 0;
        const bool same = t < n && some && u == key;
        uint32_t sames, all;
        const uint32_t rank = equal + block_scan(same ? 1u : 0u, waves, sames);
        const bool keeps = t < n ? some && (u > key || (same && rank < want)) : t < s.length;
        const uint32_t place = at + block_scan(keeps ? 1u : 0u, waves, all);
        if (keeps) out[place] = t;
        equal += sames;
        at += all;
    }
}

// Moves the kept tokens of a sequence and key head to its front.  kept[i] >= i, so that a workgroup that reads its next tokens
// before it writes the present ones, and goes from the front to the back, never overwrites what it has yet to read.
// blockIdx.z: 0 the keys, their scales and the accounts, 1 the values and theirs.
constexpr int kMoveTokens = 128;

// Every thread's loads are back: what the workgroup writes from here on is not what one of its wavefronts still reads.
__device__ __forceinline__ void all_read() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

template <int D>
__global__ __launch_bounds__(512) void kv_move_kernel(const KvCall kv, float *accounts, int keep, const int32_t *__restrict__ kept, int32_t *new_lengths) {
    typedef KvTile<D> T;
    constexpr int G = T::G;
    const int h = (int)blockIdx.x, b = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int32_t *list = kept + ((int64_t)b * kv.kv_heads + h) * keep;
    // (new_lengths may be kv.lengths: nobody else reads them in this launch)
    if (h == 0 && blockIdx.z == 0 && tid == 0) new_lengths[b] = min(kv_seq(kv, b).length, keep);
    if (list[keep - 1] < keep) return;  // nothing to move: as many tokens as places, or fewer (-1)
    if (blockIdx.z == 0) {
        const int i_in = tid >> 2, j = tid & 3;
        for (int i0 = 0; i0 < keep; i0 += kMoveTokens) {
            const int i = i0 + i_in;
            uint32_t code[G], scale = 0;
            float account = 0.0f;
            const bool live = i < keep;
            const uint8_t *from = nullptr;
            if (live) {
                const int t = list[i];
                from = kv_tile(kv, b, h, t >> 5, T::kBytes);
                if (from) {
                    const int in = t & 31, l = key_row(in) + 16 * j;
#pragma unroll
                    for (int g = 0; g < G; g++) code[g] = *reinterpret_cast<const uint32_t *>(from + T::kKeys + T::code(key_half(in) * G + g, l));
#pragma unroll
                    for (int g = j; g < G; g += 4) scale |= (uint32_t)reinterpret_cast<const uint16_t *>(from + T::kKeyScales)[in * G + g] << (16 * (g >> 2));
                    if (j == 0) {
                        const float *p = kv_account(kv, accounts, b, h, t);
                        account = p ? *p : 0.0f;
                    }
                }
            }
            all_read();
            if (live && from) {
                uint8_t *to = kv_tile(kv, b, h, i >> 5, T::kBytes);
                if (to) {
                    const int in = i & 31, l = key_row(in) + 16 * j;
#pragma unroll
                    for (int g = 0; g < G; g++) *reinterpret_cast<uint32_t *>(to + T::kKeys + T::code(key_half(in) * G + g, l)) = code[g];
#pragma unroll
                    for (int g = j; g < G; g += 4) reinterpret_cast<uint16_t *>(to + T::kKeyScales)[in * G + g] = (uint16_t)(scale >> (16 * (g >> 2)));
                    if (j == 0) {
                        float *p = kv_account(kv, accounts, b, h, i);
                        if (p) *p = account;
                    }
                }
            }
            __syncthreads();
        }
    } else {
        // one thread: the dword of eight tokens for four values (64 lanes x D / 64 sets of them a tile), and the scales of one token
        constexpr int kSets = D / 64, kTiles = 512 / (64 * kSets);
        const int tile_in = tid / (64 * kSets), set = (tid >> 6) % kSets, lane = tid & 63, r = lane & 15, j = lane >> 4;
        for (int i0 = 0; i0 < keep; i0 += kTiles * 32) {
            const int i1 = i0 + tile_in * 32 + j * 8;  // the first of the eight
            u4 word = {0, 0, 0, 0};
            uint32_t mask = 0;
            uint16_t scale[8] = {};
            const int sg = set * 16 + r;  // (of the lanes, the first G of a value set's share move the scales)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int i = i1 + e;
                if (i >= keep) continue;
                const int t = list[i];
                const uint8_t *from = kv_tile(kv, b, h, t >> 5, T::kBytes);
                if (!from) continue;
                const int in = t & 31, sh = nibble_shift(in & 7);
                const u4 w = *reinterpret_cast<const u4 *>(from + T::kValues + ((set * 64) + r + 16 * (in >> 3)) * 16);
#pragma unroll
                for (int c = 0; c < 4; c++) word[c] |= ((w[c] >> sh) & 15u) << nibble_shift(e);
                mask |= 0xFu << nibble_shift(e);
                if (sg < G) scale[e] = reinterpret_cast<const uint16_t *>(from + T::kValueScales)[sg * 32 + in];
            }
            all_read();
            if (mask) {
                uint8_t *to = kv_tile(kv, b, h, i1 >> 5, T::kBytes);
                if (to) {
                    u4 *at = reinterpret_cast<u4 *>(to + T::kValues + (set * 64 + lane) * 16);
                    if (mask != 0xFFFFFFFFu) {
                        const u4 old = *at;
#pragma unroll
                        for (int c = 0; c < 4; c++) word[c] |= old[c] & ~mask;
                    }
                    *at = word;
                    if (sg < G) {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if ((mask >> nibble_shift(e)) & 1u) reinterpret_cast<uint16_t *>(to + T::kValueScales)[sg * 32 + ((i1 + e) & 31)] = scale[e];
                    }
                }
            }
            __syncthreads();
        }
    }
}

bool pairs_aligned(const HeadRows &h, int n) {
    const int64_t size = (h.bf16 ? 2 : 4);
    return ((reinterpret_cast<uintptr_t>(h.p) | (uintptr_t)(h.row * size) | (uintptr_t)(h.head * size)) & (uintptr_t)(n * size - 1)) == 0;
}

template <int D> int append(const AppendArgs &a, bool bf16, hipStream_t s) {
    const int64_t units = (int64_t)a.kv.seqs * a.kv.kv_heads * a.blocks;
    const dim3 grid((unsigned)((units + 3) / 4)), block(256);
    return bf16 ? launch(kv_append_kernel<D, true>, grid, block, 0, s, a) : launch(kv_append_kernel<D, false>, grid, block, 0, s, a);
}
template <int D> int read(const KvCall &kv, uint16_t *k, uint16_t *v, hipStream_t s) {
    const int blocks = (kv.max_new + 14) / 8;
    const int64_t units = (int64_t)kv.seqs * kv.kv_heads * blocks;
    return launch(kv_read_kernel<D>, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, kv, k, v, blocks);
}

}  // namespace

int launch_kv_append(const KvCall &kv, const HeadRows &k, const HeadRows &v, float *accounts, hipStream_t s) {
    AppendArgs a{kv, k, v, accounts, (kv.max_new + 14) / 8, 0};
    const int ne = kv.head_dim / 64;
    a.wide = pairs_aligned(k, ne) && pairs_aligned(v, ne);
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

int launch_kv_evict(const KvCall &kv, float *accounts, int keep, int recent, int32_t *kept, int32_t *new_lengths, hipStream_t s) {
    const dim3 grid((unsigned)kv.kv_heads, (unsigned)kv.seqs);
    if (int rc = launch(kv_select_kernel, grid, dim3(kSelectThreads), 0, s, kv, accounts, keep, recent, kept)) return rc;
    const dim3 both((unsigned)kv.kv_heads, (unsigned)kv.seqs, 2);
    switch (kv.head_dim) {
    case 64: return launch(kv_move_kernel<64>, both, dim3(512), 0, s, kv, accounts, keep, kept, new_lengths);
    case 128: return launch(kv_move_kernel<128>, both, dim3(512), 0, s, kv, accounts, keep, kept, new_lengths);
    default: return launch(kv_move_kernel<256>, both, dim3(512), 0, s, kv, accounts, keep, kept, new_lengths);
    }
}

}  // namespace gq
