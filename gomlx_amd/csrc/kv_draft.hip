// Trees of drafted tokens: what every node sees and where it stands, and the path of them that the model's samples follow, kept in the
// 4-bit cache (layout: kv.hpp).
//
// The rows of a sequence are its tree's nodes, the root first and every node behind its parent: parent(i) < i, anything else is none.
//     sees(i) = sees(parent(i)) + {i},  depth(i) = depth(parent(i)) + 1
//     path: node 0, then the first child of the path's end whose token is the end's sample, until there is none
#include "kv.hpp"

namespace gq {

namespace {

// Each node walks up to its root, in LDS: nodes of a path descend, so that the bits of a word of the mask come one behind the other and every word is
// written once.  Latency bounds it: 3.2 us for 256 trees of 32 to 64 nodes, and for one of 8.
__global__ __launch_bounds__(256) void draft_tree_kernel(const TreeCall c, int32_t *tree, int words, int32_t *positions) {
    __shared__ int up[kMostNodes];
    const int b = (int)blockIdx.x, tid = (int)threadIdx.x, threads = (int)blockDim.x;
    int row0, n;
    c.rows_of(b, row0, n);
    for (int i = tid; i < n; i += threads) up[i] = c.parents[row0 + i];
    const int first = c.first[b];
    __syncthreads();
    for (int i = tid; i < n; i += threads) {
        int32_t *out = tree + (int64_t)(row0 + i) * words;
        int word = words - 1, depth = -1;
        uint32_t bits = 0;
        for (int at = i, below = n; (uint32_t)at < (uint32_t)below; depth++) {  // (a parent that is not in front of its child: none)
            for (; word > at >> 5; word--) {
                out[word] = (int32_t)bits;
                bits = 0;
            }
            bits |= 1u << (at & 31);
            below = at;
            at = up[at];
        }
        for (; word >= 0; word--) {
            out[word] = (int32_t)bits;
            bits = 0;
        }
        positions[row0 + i] = first + depth;
    }
}

// where element e of a dword lies
__device__ __forceinline__ int nibble_shift(int e) { return ((e >> 1) + 4 * (e & 1)) * 4; }

// Every thread's loads are back: what the workgroup writes from here on is not what one of its wavefronts still reads.
__device__ __forceinline__ void all_read() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

struct AcceptArgs {
    KvCall kv;
    const int32_t *parents, *tokens, *sampled;
    float *accounts;
    int32_t *path, *next, *new_lengths;
    int path_columns;
};

// The path from the root: its nodes in `path`, how many they are, and how many of the first are where they belong (path[i] == i).
struct Walk { int count, stay; };
__device__ __forceinline__ Walk walk_down(int n, const int *up, const int *word, const int *drawn, int *path) {
    const int lane = (int)threadIdx.x & 63;
    Walk w{0, 0};
    if (n == 0) return w;
    // (the first 64 nodes in registers: a step is a compare and a few scalar instructions)
    const int up0 = lane < n ? up[lane] : -1, word0 = lane < n ? word[lane] : -1, drawn0 = lane < n ? drawn[lane] : -1;
    for (int at = 0;;) {
        if (lane == 0) path[w.count] = at;
        if (w.stay == w.count && at == w.count) w.stay++;
        w.count++;
        const int token = at < 64 ? __builtin_amdgcn_readlane(drawn0, at) : __builtin_amdgcn_readfirstlane(drawn[at]);
        if (token < 0) break;
        uint64_t child = __ballot(lane > at && lane < n && up0 == at && word0 == token);
        int base = 0;
        while (!child && (base += 64) < n) {
            const int i = base + lane;
            child = __ballot(i > at && i < n && up[min(i, n - 1)] == at && word[min(i, n - 1)] == token);
        }
        if (!child) break;
        at = base + __ffsll((unsigned long long)child) - 1;
    }
    return w;
}

// One workgroup per sequence and key head; each walks down the tree for itself.  path[i] >= i and grows, so that a workgroup that reads what comes
// into a tile before it writes the tile, and goes from the front to the back, never overwrites what it has yet to read.  A chain of dependent loads
// bounds it (lengths and starts, nodes, pages, codes): 5.3 us for one sequence of 16 nodes, 9.2 us for 64 of 32 to 64, 8 key heads of D = 128.
template <int D>
__global__ __launch_bounds__(256) void kv_accept_kernel(const AcceptArgs a) {
    typedef KvTile<D> T;
    constexpr int G = T::G, N = G / 2;  // dwords of a tile's key or value codes that a thread moves
    __shared__ int up[kMostNodes], word[kMostNodes], drawn[kMostNodes], path[kMostNodes], walked[2];
    __shared__ int64_t from[32];  // of the tile's tokens: tile * 32 + token in it; -1: nothing comes there
    const KvCall &kv = a.kv;
    const int h = (int)blockIdx.x, b = (int)blockIdx.y, tid = (int)threadIdx.x;
    const KvSeq s = kv_seq(kv, b);
    const int n = s.news;
    for (int i = tid; i < n; i += 256) {
        up[i] = a.parents[s.row0 + i];
        word[i] = a.tokens[s.row0 + i];
        drawn[i] = a.sampled[s.row0 + i];
    }
    __syncthreads();
    if (tid < 64) {
        const Walk w = walk_down(n, up, word, drawn, path);
        if (tid == 0) { walked[0] = w.count; walked[1] = w.stay; }
    }
    __syncthreads();
    const int count = walked[0], stay = max(walked[1], -s.first);  // (tokens in front of the sequence's first are none)
    if (h == 0) {
        for (int i = tid; i < a.path_columns; i += 256) a.path[(int64_t)b * a.path_columns + i] = i < count ? path[i] : -1;
        if (tid == 0) {
            a.next[b] = count ? drawn[path[count - 1]] : -1;
            a.new_lengths[b] = n ? max(0, s.first + count) : max(0, kv.lengths[b]);
        }
    }
    const int per_page = kv.page_tokens >> 5;
    const auto tile_number = [&](int tile) -> int64_t {
        const int slot = page_slot(kv, tile), page = kv.table[b * kv.table_stride + slot];
        return (uint32_t)page < (uint32_t)kv.pages ? ((int64_t)page * kv.kv_heads + h) * per_page + (tile - slot * per_page) : -1;
    };
    if (kv.pages == 0) return;
    const int end = min(s.first + count, s.length);
    for (int p0 = s.first + stay; p0 < end; p0 = (p0 | 31) + 1) {
        const int64_t here = tile_number(p0 >> 5);
        if (tid < 32) {
            const int p = (p0 & ~31) + tid;
            int64_t f = -1;
            if (p >= p0 && p < end) {
                const int source = s.first + path[p - s.first];
                const int64_t tile = source < s.length ? tile_number(source >> 5) : -1;
                if (tile >= 0) f = tile * 32 + (source & 31);
            }
            from[tid] = f;
        }
        __syncthreads();
        uint32_t keys[N], values[N], masks[N], scales = 0;
        float account = 0.0f;
        // (for tokens that come from nowhere the tile itself is read, so that loads need no branches between them and go out together)
        const int64_t some = max(here, (int64_t)0) * 32;
        uint8_t *const to = kv.cache + (some >> 5) * T::kBytes;
        const auto tile_of = [&](int64_t f) { return kv.cache + (f >> 5) * T::kBytes; };
#pragma unroll
        for (int i = 0; i < N; i++) {  // token, lane of its row, group
            const int at = tid + 256 * i, t = at / (4 * G), j = at / G & 3, g = at % G;
            const int64_t f = from[t] < 0 ? some : from[t];
            const int u = (int)f & 31;
            keys[i] = *reinterpret_cast<const uint32_t *>(tile_of(f) + T::kKeys + T::code(key_half(u) * G + g, key_row(u) + 16 * j));
        }
#pragma unroll
        for (int i = 0; i < N; i++) {  // eight tokens, value
            const int at = tid + 256 * i, j = at / D, v = at % D;
            const auto word = [&](const uint8_t *tile, int octet) { return *reinterpret_cast<const uint32_t *>(tile + T::kValues + T::code(v >> 4, (v & 15) + 16 * octet)); };
            const uint32_t old = word(to, j);  // with the tokens beside them
            uint32_t w[8];
            values[i] = masks[i] = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int64_t f = from[8 * j + e] < 0 ? some : from[8 * j + e];
                w[e] = word(tile_of(f), ((int)f & 31) >> 3);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int64_t f = from[8 * j + e];
                const uint32_t code = f < 0 ? 0u : 15u;
                values[i] |= (w[e] >> nibble_shift((int)f & 7) & code) << nibble_shift(e);
                masks[i] |= code << nibble_shift(e);
            }
            values[i] |= old & ~masks[i];
        }
        const int t = tid / G, g = tid % G;  // of scales (32 G of each) and accounts
        const int64_t f = t < 32 ? from[t] : -1;
        if (f >= 0) {
            const int u = (int)f & 31;
            scales = reinterpret_cast<const uint16_t *>(tile_of(f) + T::kKeyScales)[u * G + g] | (uint32_t)reinterpret_cast<const uint16_t *>(tile_of(f) + T::kValueScales)[g * 32 + u] << 16;
            if (a.accounts && g == 0) account = a.accounts[f];  // (pages hold their tokens' accounts in the order of their tiles)
        }
        all_read();
        if (here >= 0) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int at = tid + 256 * i, u = at / (4 * G), j = at / G & 3, g = at % G;
                if (from[u] >= 0) *reinterpret_cast<uint32_t *>(to + T::kKeys + T::code(key_half(u) * G + g, key_row(u) + 16 * j)) = keys[i];
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int at = tid + 256 * i, j = at / D, v = at % D;
                if (masks[i]) *reinterpret_cast<uint32_t *>(to + T::kValues + T::code(v >> 4, (v & 15) + 16 * j)) = values[i];
            }
            if (f >= 0) {
                reinterpret_cast<uint16_t *>(to + T::kKeyScales)[t * G + g] = (uint16_t)scales;
                reinterpret_cast<uint16_t *>(to + T::kValueScales)[g * 32 + t] = (uint16_t)(scales >> 16);
                if (a.accounts && g == 0) a.accounts[here * 32 + t] = account;
            }
        }
        all_read();  // (and written, for the next tile's sources; `from` is free)
    }
}

}  // namespace

int launch_draft_tree(const TreeCall &c, int32_t *tree, int words, int32_t *positions, hipStream_t s) {
    return launch(draft_tree_kernel, dim3((unsigned)c.seqs), dim3(c.max_new > 128 ? 256 : c.max_new > 64 ? 128 : 64), 0, s, c, tree, words, positions);
}

int launch_kv_accept(const KvCall &kv, const int32_t *parents, const int32_t *tokens, const int32_t *sampled, float *accounts, int32_t *path, int path_columns, int32_t *next,
                     int32_t *new_lengths, hipStream_t s) {
    const AcceptArgs a{kv, parents, tokens, sampled, accounts, path, next, new_lengths, path_columns};
    const dim3 grid((unsigned)kv.kv_heads, (unsigned)kv.seqs), block(256);
    switch (kv.head_dim) {
    case 64: return launch(kv_accept_kernel<64>, grid, block, 0, s, a);
    case 128: return launch(kv_accept_kernel<128>, grid, block, 0, s, a);
    default: return launch(kv_accept_kernel<256>, grid, block, 0, s, a);
    }
}

}  // namespace gq
