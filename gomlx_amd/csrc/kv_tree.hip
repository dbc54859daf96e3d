// Softmax attention of a tree of drafted tokens over a 4-bit cache (layout: kv.hpp; operands, references and formats: kv_attend.hpp, kv_attention.hip).
//
//     s_ij = scale q_i . k_j for the tokens j that row i sees: those in front of the tree, and token j of the tree where bit j of the row's mask is set;
//            with a window the last `window` of all these
//     o_i  = sum_j P_ij v_j,  P_i = softmax(s_i);  a row that sees nothing gets zeros
//
// Every row of a sequence sees the same long context, so that a key head's (node, query head) pairs, 16 RG of them, go over the cache together: a wavefront widens a tile's
// codes once, in registers, and contracts them with all of these rows (queries in LDS, as operands; results in registers).  Widening costs 208 vector instructions a
// tile of 32 tokens at D = 128, every 16 rows 32 matrix instructions of 16 cycles (twice that in float32) and some 75 vector instructions for their weights: at 64 rows a tile's share of the
// memory's rate and of the vector units' about meet.
#include "kv_attend.hpp"

#include <algorithm>
#include <cmath>

namespace gq {

namespace {

constexpr int kMostTreeWorkgroups = 2048;

struct TreeArgs {
    KvCall kv;
    HeadRows q;
    int heads, group, window, wide;
    float scale_log2;       // scale * log2(e)
    const int32_t *tree;    // [rows, words]
    int words;
    void *out;              // [rows, heads, D]
    float *part, *part_ml;  // of workgroups whose unit has several: sums [rows, D], (reference, sum) [rows, 2]
    int workgroups;         // that all units together are cut into, about
    int blocks, rows;       // row blocks of a sequence and rows of a block, at most
    int2 *pieces;           // per unit: the first workgroup that works on it, and how many do
};

// A unit is a block of ROWS neighbouring (node, head of the group) pairs of a sequence and key head, with the tiles that one of them may see (one at least, so
// that rows that see nothing are written too).
__device__ __forceinline__ int blocks_of(const TreeArgs &a, const KvSeq &s, int block_rows) { return (s.news * a.group + block_rows - 1) / block_rows; }
__device__ __forceinline__ void tokens_of(const TreeArgs &a, const KvSeq &s, int &lo, int &hi) {
    hi = max(0, min(s.first + s.news, s.length));
    lo = a.window && s.first > a.window ? min(s.first - a.window, hi) : 0;  // (a row sees one token of the tree at least, or none and one more of the context)
}
__device__ __forceinline__ int tree_tiles(const TreeArgs &a, const KvSeq &s) {
    int lo, hi;
    tokens_of(a, s, lo, hi);
    return s.news ? max(1, ((hi + 31) >> 5) - (lo >> 5)) : 0;
}

// Pieces of one length, a multiple of the wavefronts, of which all units together have about a.workgroups; the lengths are known on the device only, so that every
// wavefront finds its place by a sum over them, 64 sequences at a time, one a lane.  (All tiles together: less than 2^31.)
struct TreePiece {
    int b, h, block, nth;  // b < 0: there is none
    int share, tiles;      // tiles of a piece, of the unit
    KvSeq seq;
    __device__ __forceinline__ int pieces() const { return (tiles + share - 1) / share; }
};
__device__ __forceinline__ TreePiece tree_piece_of(const TreeArgs &a, int index, int block_rows) {
    const int lane = (int)threadIdx.x & 63, seqs = a.kv.seqs, heads = a.kv.kv_heads;
    TreePiece p;
    p.b = -1;
    KvSeq mine{};
    int tiles = 0, units = 0, total = 0;
    for (int base = (seqs - 1) & ~63; base >= 0; base -= 64) {  // (the first 64 last: they stay)
        mine = KvSeq{};
        if (base + lane < seqs) mine = kv_seq(a.kv, base + lane);
        tiles = tree_tiles(a, mine);
        units = blocks_of(a, mine, block_rows) * heads;
        total += __builtin_amdgcn_readlane(lane_scan(tiles * units), 63);
    }
    const int least = (total + a.workgroups - 1) / a.workgroups;
    p.share = max(1, (least + kSplitWaves - 1) / kSplitWaves) * kSplitWaves;
    int front = 0;  // pieces in front
    for (int base = 0; base < seqs; base += 64) {
        if (base) {
            mine = KvSeq{};
            if (base + lane < seqs) mine = kv_seq(a.kv, base + lane);
            tiles = tree_tiles(a, mine);
            units = blocks_of(a, mine, block_rows) * heads;
        }
        const int each = (tiles + p.share - 1) / p.share, upto = lane_scan(each * units);
        const uint64_t past = __ballot(front + upto > index);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            p.b = base + l;
            p.seq = seq_of_lane(mine, l);
            p.tiles = __builtin_amdgcn_readlane(tiles, l);
            const int all = __builtin_amdgcn_readlane(each * units, l), in = index - (front + __builtin_amdgcn_readlane(upto, l) - all);
            const int blocks = blocks_of(a, p.seq, block_rows), per_head = all / heads;
            p.h = in / per_head;
            const int rest = in - p.h * per_head;
            p.nth = rest / blocks;
            p.block = rest - p.nth * blocks;  // (blocks of one piece of the tokens are neighbours)
            break;
        }
        front += __builtin_amdgcn_readlane(upto, 63);
    }
    return p;
}

// What a row sees: context tokens from `lo` on, and from there the tokens of the tree whose bit is set.
struct Sight { int lo; const int32_t *mask; };
__device__ __forceinline__ Sight sight_of(const TreeArgs &a, const KvSeq &s, int node) {
    Sight v;
    v.mask = a.tree + (int64_t)(s.row0 + node) * a.words;
    v.lo = 0;
    if (a.window) {
        const int words = (s.news + 31) >> 5;
        const auto word = [&](int w) { return (uint32_t)v.mask[w] & (s.news - 32 * w < 32 ? (1u << (s.news - 32 * w)) - 1u : 0xFFFFFFFFu); };  // (bits behind the last node are none)
        int left = a.window;
        for (int w = words - 1; w >= 0; w--) {
            uint32_t bits = word(w);
            const int n = __popc(bits);
            if (n >= left) {  // the last `left` of these, and nothing in front
                for (int drop = n - left; drop > 0; drop--) bits &= bits - 1;
                v.lo = s.first + 32 * w + __ffs((int)bits) - 1;
                return v;
            }
            left -= n;
        }
        v.lo = s.first - left;
    }
    return v;
}
// eight bits of a row's mask from token `at` of the tree on (nothing is looked up outside its words)
__device__ __forceinline__ uint32_t mask_bits(const int32_t *mask, int words, int at) {
    const int w = at >> 5, shift = at & 31;
    const uint32_t low = (uint32_t)w < (uint32_t)words ? (uint32_t)mask[w] : 0u, high = (uint32_t)(w + 1) < (uint32_t)words ? (uint32_t)mask[w + 1] : 0u;
    return (uint32_t)((((uint64_t)high << 32) | low) >> shift) & 255u;
}

template <int D, bool BF16, int RG> struct TreeLds {
    static constexpr int kOperands = RG * (D / 32) * 1024, kQueries = kOperands * (BF16 ? 1 : 2);  // bytes
    static constexpr int kRing = kSplitWaves * kSplitSlots * SplitLds<D>::kSlot;
    static constexpr int kSums = kSplitWaves * 16 * (D + 4) * 4;
    static constexpr int kBytes = (kQueries + kRing > kSums ? kQueries + kRing : kSums);
};

template <int D, bool BF16, int RG>
__global__ __launch_bounds__(64 * kSplitWaves, D == 256 ? 1 : 2) void kv_tree_kernel(const TreeArgs a) {
    constexpr bool TWO = !BF16;
    constexpr int W = D / 16, G = D / 32, ROWS = 16 * RG;
    typedef TreeLds<D, BF16, RG> Lds;
    __shared__ __align__(16) uint8_t lds[Lds::kBytes];
    __shared__ float refs[kSplitWaves][ROWS], totals[kSplitWaves][ROWS], scales[ROWS];
    __shared__ int lows[ROWS];
    const KvCall &kv = a.kv;
    const int tid = (int)threadIdx.x, lane = tid & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const TreePiece piece = tree_piece_of(a, (int)blockIdx.x, ROWS);
    if (piece.b < 0) return;
    const int b = piece.b, h = piece.h;
    const KvSeq &seq = piece.seq;
    const int row_first = piece.block * ROWS, rows = min(ROWS, seq.news * a.group - row_first);
    int lo, hi;
    tokens_of(a, seq, lo, hi);
    const int tile0 = (lo >> 5) + piece.nth * piece.share, tile1 = min((lo >> 5) + min((piece.nth + 1) * piece.share, piece.tiles), (hi + 31) >> 5);
    const Unpack unpack;

    TileWalk<KvTile<D>::kBytes, kSplitWaves> walk(kv, b, h, tile0 + wave, tile1);
    uint8_t *ring = lds + Lds::kQueries + wave * kSplitSlots * SplitLds<D>::kSlot;
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)ring);
    const uint8_t *mem = walk.next();
    if (mem) fetch_tile<D>(ring_at, mem);
    // the rows' queries, sixteen rows a wavefront at a time
    h8 *operands = reinterpret_cast<h8 *>(lds);
#pragma unroll 1
    for (int m = wave; m < RG; m += kSplitWaves) {
        const int idx = row_first + 16 * m + r;
        const bool live = 16 * m + r < rows;
        const int node = live ? idx / a.group : 0, head = h * a.group + (live ? idx - node * a.group : 0);
        h8 qh[G], ql[TWO ? G : 1];
        float to_log2;
        load_queries<D, 16, BF16, TWO>(a.q, (int64_t)(seq.row0 + node) * a.q.row + head * a.q.head, live, a.wide, a.scale_log2, qh, ql, to_log2);
#pragma unroll
        for (int g = 0; g < G; g++) {
            operands[(m * G + g) * 64 + lane] = qh[g];
            if constexpr (TWO) operands[Lds::kOperands / 16 + (m * G + g) * 64 + lane] = ql[g];
        }
        if (j == 0) {
            scales[16 * m + r] = to_log2;
            lows[16 * m + r] = live ? sight_of(a, seq, node).lo : 0;
        }
    }
    __syncthreads();
    float to_log2[RG];
    int all_lo = 0;  // from here on every row sees the context
#pragma unroll
    for (int m = 0; m < RG; m++) {
        to_log2[m] = scales[16 * m + r];
        all_lo = max(all_lo, lows[16 * m + r]);
    }
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) all_lo = max(all_lo, __shfl_xor(all_lo, m));
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);

    f4 o[RG][W];
    float ref[RG], total[RG];  // the rows' references, and the lane's share of their sums
#pragma unroll
    for (int m = 0; m < RG; m++) {
        ref[m] = kNegInf;
        total[m] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) o[m][w] = f4{0.f, 0.f, 0.f, 0.f};
    }

    int turn = 0;
    for (int tile = tile0 + wave; tile < tile1; tile += kSplitWaves) {
        const uint8_t *mem_next = walk.next();
        if (mem_next) {
            fetch_tile<D>(ring_at + (uint32_t)(turn ^ 1) * SplitLds<D>::kSlot, mem_next);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(SplitLds<D>::kLoads) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (mem) {
            const int t0 = tile * 32;
            float s[RG][8];
            {
                KeyWords<D> k;
                k.load(ring + turn * SplitLds<D>::kSlot);
                f4 acc[RG][2];
#pragma unroll
                for (int m = 0; m < RG; m++) acc[m][0] = acc[m][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const h8 k0 = k.operand(unpack, 0, g), k1 = k.operand(unpack, 1, g);
#pragma unroll
                    for (int m = 0; m < RG; m++) {
                        const h8 q = operands[(m * G + g) * 64 + lane];
                        acc[m][0] = mfma(k0, q, acc[m][0]);
                        acc[m][1] = mfma(k1, q, acc[m][1]);
                        if constexpr (TWO) {
                            const h8 rest = operands[Lds::kOperands / 16 + (m * G + g) * 64 + lane];
                            acc[m][0] = mfma(k0, rest, acc[m][0]);
                            acc[m][1] = mfma(k1, rest, acc[m][1]);
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < RG; m++)
#pragma unroll
                    for (int e = 0; e < 8; e++) s[m][e] = acc[m][e >> 2][e & 3] * to_log2[m];
            }
            if (t0 < all_lo || t0 + 32 > seq.first) {
#pragma unroll
                for (int m = 0; m < RG; m++) {
                    const int idx = row_first + 16 * m + r;
                    const bool live = 16 * m + r < rows;
                    const int from = live ? lows[16 * m + r] : hi, at = t0 + 8 * j;
                    const uint32_t bits = live ? mask_bits(a.tree + (int64_t)(seq.row0 + idx / a.group) * a.words, a.words, at - seq.first) : 0u;
#pragma unroll
                    for (int e = 0; e < 8; e++) s[m][e] = at + e >= from && at + e < hi && (at + e < seq.first || (bits >> e & 1u)) ? s[m][e] : kNegInf;
                }
            }
            float most[RG];
            bool beyond = false;
#pragma unroll
            for (int m = 0; m < RG; m++) {
                most[m] = fmaxf(fmaxf(fmaxf(s[m][0], s[m][1]), fmaxf(s[m][2], s[m][3])), fmaxf(fmaxf(s[m][4], s[m][5]), fmaxf(s[m][6], s[m][7])));
                beyond = beyond || passes<D, TWO>(most[m], ref[m]);
            }
            if (__any(beyond)) {  // (the first score of a row among them: its reference is -infinity)
#pragma unroll
                for (int m = 0; m < RG; m++) {
                    if (!__any(passes<D, TWO>(most[m], ref[m]))) continue;
                    most[m] = fmaxf(most[m], __shfl_xor(most[m], 16));
                    most[m] = fmaxf(most[m], __shfl_xor(most[m], 32));
                    const float next = fmaxf(ref[m], reference<D, TWO>(most[m]));
                    const float shrink = next == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ref[m] - next);
                    ref[m] = next;
                    total[m] *= shrink;
#pragma unroll
                    for (int w = 0; w < W; w++) o[m][w] *= shrink;
                }
            }
            h8 ph[RG], pl[TWO ? RG : 1];
#pragma unroll
            for (int m = 0; m < RG; m++) {
                const float less = ref[m] == kNegInf ? 0.0f : ref[m];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p = __builtin_amdgcn_exp2f(s[m][e] - less);
                    total[m] += p;
                    ph[m][e] = (_Float16)p;
                    if constexpr (TWO) pl[m][e] = (_Float16)(p - (float)ph[m][e]);
                }
            }
            ValueWords<D> v;
            v.load(ring + turn * SplitLds<D>::kSlot);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const h8 x = v.operand(unpack, w);
#pragma unroll
                for (int m = 0; m < RG; m++) {
                    o[m][w] = mfma(x, ph[m], o[m][w]);
                    if constexpr (TWO) o[m][w] = mfma(x, pl[m], o[m][w]);
                }
            }
        }
        mem = mem_next;
        turn ^= 1;
    }

    // the wavefronts' results, sixteen rows at a time, in the place of queries and tiles
    float(*sums)[16][D + 4] = reinterpret_cast<float(*)[16][D + 4]>(lds);
    const int pieces = piece.pieces();
    if (a.pieces && piece.nth == 0 && tid == 0) a.pieces[(b * kv.kv_heads + h) * a.blocks + piece.block] = make_int2((int)blockIdx.x, pieces);
#pragma unroll
    for (int m = 0; m < RG; m++) {
        total[m] += __shfl_xor(total[m], 16);
        total[m] += __shfl_xor(total[m], 32);
        if (j == 0) {
            refs[wave][16 * m + r] = ref[m];
            totals[wave][16 * m + r] = total[m];
        }
    }
#pragma unroll
    for (int m = 0; m < RG; m++) {
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; w++) *reinterpret_cast<f4 *>(&sums[wave][r][16 * w + 4 * j]) = o[m][w];
        __syncthreads();
        const int here = min(16, rows - 16 * m);
        for (int i = tid; i < here * (D / 4); i += 64 * kSplitWaves) {
            const int in = i / (D / 4), rr = 16 * m + in, d = (i - in * (D / 4)) * 4;
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
                sum += *reinterpret_cast<const f4 *>(&sums[w][in][d]) * f;
            }
            if (pieces == 1) {
                const int node = (row_first + rr) / a.group;
                const int64_t out = (int64_t)(seq.row0 + node) * a.heads + h * a.group + (row_first + rr - node * a.group);
                store_result<BF16>(a.out, out * D + d, sum, all);
            } else {
                const int64_t line = (int64_t)blockIdx.x * a.rows + rr;
                *reinterpret_cast<f4 *>(a.part + line * D + d) = sum;
                if (d == 0) {
                    a.part_ml[line * 2] = top;
                    a.part_ml[line * 2 + 1] = all;
                }
            }
        }
    }
}

// Joins the pieces of the units that more than one workgroup has worked on: one workgroup per unit and row.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void kv_tree_join_kernel(const TreeArgs a, int block_rows) {
    constexpr int L = D / 4, S = 256 / L;  // lanes of a row's values, and the shares into which the pieces are divided
    __shared__ f4 sums[S][L];
    __shared__ float factors[kMostTreeWorkgroups], tops[4], alls[4];
    const int block = (int)blockIdx.x / a.rows, rr = (int)blockIdx.x - block * a.rows, h = (int)blockIdx.y, b = (int)blockIdx.z, tid = (int)threadIdx.x;
    const KvSeq seq = kv_seq(a.kv, b);
    if (block * block_rows + rr >= seq.news * a.group) return;  // (without rows nobody has written the unit's pieces)
    const int unit = (b * a.kv.kv_heads + h) * a.blocks + block;
    const int2 piece = a.pieces[unit];
    const int first = piece.x, pieces = piece.y, stride = blocks_of(a, seq, block_rows);  // (between the pieces of a unit lie its neighbours')
    if (pieces == 1) return;
    const auto line = [&](int i) { return (int64_t)(first + i * stride) * a.rows + rr; };
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
    const int node = (block * block_rows + rr) / a.group;
    const int64_t out = (int64_t)(seq.row0 + node) * a.heads + h * a.group + (block * block_rows + rr - node * a.group);
    store_result<BF16>(a.out, out * D + l * 4, sum, all);
}

template <int D, bool BF16, int RG> int tree_attend(const TreeArgs &a, hipStream_t s) {
    const KvCall &kv = a.kv;
    const unsigned grid = (unsigned)(a.workgroups + (int64_t)kv.seqs * kv.kv_heads * a.blocks);  // (a unit's last piece may be short)
    if (int rc = launch(kv_tree_kernel<D, BF16, RG>, dim3(grid), dim3(64 * kSplitWaves), 0, s, a)) return rc;
    if (!a.pieces) return GQ_OK;
    return launch(kv_tree_join_kernel<D, BF16>, dim3((unsigned)(a.blocks * a.rows), (unsigned)kv.kv_heads, (unsigned)kv.seqs), dim3(256), 0, s, a, 16 * RG);
}
template <int D, bool BF16> int tree_attend(const TreeArgs &a, int row_groups, hipStream_t s) {
    switch (row_groups) {
    case 1: return tree_attend<D, BF16, 1>(a, s);
    case 2: return tree_attend<D, BF16, 2>(a, s);
    default:
        if constexpr (D == 256) return tree_attend<D, BF16, 2>(a, s);
        else return tree_attend<D, BF16, 4>(a, s);
    }
}

}  // namespace

// How a call's rows are cut into blocks: 16 RG (node, query head) pairs of a key head.
struct TreePlan { int row_groups, rows; int64_t blocks, tiles; };
static TreePlan tree_plan(const KvCall &kv, int heads, int window) {
    TreePlan p;
    const int64_t most_rows = (int64_t)kv.max_new * (heads / kv.kv_heads), room = (int64_t)kv.max_pages * kv.page_tokens / 32;
    p.row_groups = most_rows <= 16 ? 1 : most_rows <= 32 || kv.head_dim == 256 ? 2 : 4;
    p.rows = (int)std::min<int64_t>(most_rows, 16 * p.row_groups);
    p.blocks = (most_rows + 16 * p.row_groups - 1) / (16 * p.row_groups);
    p.tiles = std::max<int64_t>(1, window ? std::min<int64_t>(room, ((int64_t)window + kv.max_new + 31) / 32 + 1) : room);
    return p;
}

int check_kv_tree_attention(const char *fn, const KvCall &kv, int heads, int window) {
    const TreePlan p = tree_plan(kv, heads, window);
    const int64_t units = (int64_t)kv.seqs * kv.kv_heads * p.blocks;
    // (threads of a launch are counted in 32 bits, and so are the tiles of all units)
    if (p.blocks > INT32_MAX / kv.kv_heads / kv.seqs || units * p.rows > (1 << 24) - 4096 || units > (INT32_MAX - 4096) / p.tiles)
        return fail(GQ_ERR_INVALID, "%s: %d sequences of up to %d rows of %d heads over up to %lld tiles: too many (pass the page table's first columns)", fn, kv.seqs, kv.max_new, heads,
                    (long long)p.tiles);
    return GQ_OK;
}

int launch_kv_tree_attention(const KvCall &kv, const HeadRows &q, int heads, float scale, int window, const int32_t *tree, int words, void *out, hipStream_t s) {
    TreeArgs a{};
    a.kv = kv;
    a.q = q;
    a.heads = heads;
    a.group = heads / kv.kv_heads;
    a.window = window;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.tree = tree;
    a.words = words;
    a.out = out;
    const int64_t size = q.bf16 ? 2 : 4;
    a.wide = ((reinterpret_cast<uintptr_t>(q.p) | (uintptr_t)(q.row * size) | (uintptr_t)(q.head * size)) & 15) == 0;
    const TreePlan p = tree_plan(kv, heads, window);
    a.rows = p.rows;
    a.blocks = (int)p.blocks;
    const int64_t tiles = p.tiles, units = (int64_t)kv.seqs * kv.kv_heads * a.blocks;
    const int per_cu = kv.head_dim == 256 ? 1 : 2;
    a.workgroups = (int)std::min<int64_t>(std::min(kMostTreeWorkgroups, device_cu_count() * per_cu), (units * tiles + kSplitWaves - 1) / kSplitWaves);
    if (tiles > kSplitWaves) {
        const size_t lines = (size_t)(a.workgroups + units) * a.rows;
        const auto up = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
        const size_t ml = up(lines * kv.head_dim * 4), pieces = ml + up(lines * 8), all = pieces + (size_t)units * 8;
        void *ws = nullptr;
        if (int rc = stream_workspace(s, all, &ws)) return rc;
        unsigned char *at = static_cast<unsigned char *>(ws);
        a.part = reinterpret_cast<float *>(at);
        a.part_ml = reinterpret_cast<float *>(at + ml);
        a.pieces = reinterpret_cast<int2 *>(at + pieces);
    }
    switch (kv.head_dim) {
    case 64: return q.bf16 ? tree_attend<64, true>(a, p.row_groups, s) : tree_attend<64, false>(a, p.row_groups, s);
    case 128: return q.bf16 ? tree_attend<128, true>(a, p.row_groups, s) : tree_attend<128, false>(a, p.row_groups, s);
    default: return q.bf16 ? tree_attend<256, true>(a, p.row_groups, s) : tree_attend<256, false>(a, p.row_groups, s);
    }
}

}  // namespace gq
