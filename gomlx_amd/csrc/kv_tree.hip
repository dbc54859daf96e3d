// Softmax attention of a tree of drafted tokens over a 4-bit cache (layout: kv.hpp; operands, references and formats: kv_attend.hpp, kv_attention.hip).
//
//     s_ij = scale q_i . k_j for the tokens j that row i sees: those in front of the tree, and token j of the tree where bit j of the row's mask is set;
//            with a window the last `window` of all these
//     o_i  = sum_j P_ij v_j,  P_i = softmax(s_i);  a row that sees nothing gets zeros
//
// Every row of a sequence sees the same long context, so that a key head's (node, query head) pairs, up to 64 of them, go over the cache together: a wavefront widens a tile's
// codes once, in registers, and contracts them with all of these rows (queries in LDS, as operands; results in registers).  Widening costs 208 vector instructions a
// tile of 32 tokens at D = 128, every 16 rows 16 matrix instructions of 16 cycles (in float32 32) and some 47 vector instructions, eight of them exponentials of four times the
// usual length, for their weights.  These bound it, for next to matrix instructions little else is issued: at 64 rows some 2000 cycles of the one and 1000 of the other a
// tile, 3100 as measured (two wavefronts a SIMD; one alone takes 3500).  us a call, D = 128, bfloat16, 8 key heads of 4 queries: 32 sequences of 2048 to 8192 tokens with 8
// to 16 nodes each 80 (450 TFLOP/s, 2.5 TB/s of cache); 32 nodes over 131072 tokens 96 (720 TFLOP/s); 16 sequences of 2048 to 8192 tokens with 32 to 64 nodes 124 (580).  (One of hundreds of
// calls behind one another; of the first ten, before the clock has risen, 86, 104 and 138.)
#include "kv_attend.hpp"

#include <algorithm>
#include <cmath>

namespace gq {

namespace {

constexpr int kLeastShare = 4;  // tiles of a workgroup, at least: one a wavefront

struct TreeArgs {
    KvCall kv;
    HeadRows q;
    int heads, group, window, wide;
    float scale_log2;       // scale * log2(e)
    const int32_t *tree;    // [rows, words]
    int words;
    void *out;              // [rows, heads, D]
    float *part, *part_ml;  // of units that several workgroups work on: sums [workgroups, 2, rows, D], (reference, sum) [workgroups, 2, rows, 2]
    int blocks, rows;       // row blocks of a sequence and rows of a block, at most
    int all_blocks;         // of all sequences, at most, where the join finds them by number; 0: it is laid out by `blocks`
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

// The tiles of all units stand in one line, and every workgroup takes the same number of them: the end of a unit, perhaps some whole ones, the beginning of another.  (Pieces
// of units, one a workgroup, take as long as the longest: 32 sequences of 2048 to 8192 tokens, 16 nodes, 8 heads of 4 queries, D = 128, 104 us for 84.)  The lengths are known on the device only, so that every wavefront finds
// its place by a sum over them, 64 sequences at a time, one a lane.  (All tiles together: less than 2^31.)
struct TreePlace {
    int b, unit, tile;  // sequence; of its units; tile of the unit
    int left, share;    // tiles of the workgroup; b < 0: it has none
    KvSeq seq;
    // (the same for the whole wavefront: in scalar registers)
    __device__ __forceinline__ void uniform() {
        for (int *v : {&b, &unit, &tile, &left, &share, &seq.length, &seq.news, &seq.row0, &seq.first}) *v = __builtin_amdgcn_readfirstlane(*v);
    }
};
__device__ __forceinline__ TreePlace tree_place_of(const TreeArgs &a, int index, int workgroups, int block_rows) {
    const int lane = (int)threadIdx.x & 63, seqs = a.kv.seqs, heads = a.kv.kv_heads;
    TreePlace p;
    p.b = -1;
    KvSeq mine{};
    int each = 0, units = 0, total = 0, wide = 0;  // tiles of a unit of the lane's sequence, and such units; of all; with every unit's rounded up to the least share
    const auto up = [](int n) { return (n + kLeastShare - 1) / kLeastShare * kLeastShare; };
    const auto look = [&](int base) {
        mine = KvSeq{};
        if (base + lane < seqs) mine = kv_seq(a.kv, base + lane);
        each = tree_tiles(a, mine);
        units = blocks_of(a, mine, block_rows) * heads;
    };
    for (int base = (seqs - 1) & ~63; base >= 0; base -= 64) {  // (the first 64 last: they stay)
        look(base);
        total += __builtin_amdgcn_readlane(lane_scan(each * units), 63);
        const int mine_up = (int)min((int64_t)up(each) * units, (int64_t)1 << 18);
        wide = min(wide + __builtin_amdgcn_readlane(lane_scan(mine_up), 63), 1 << 24);  // (so many do not fit)
    }
    // Where the workgroups are more than enough none works on two units.
    const bool apart = wide <= workgroups * kLeastShare;
    p.share = apart ? kLeastShare : (total + workgroups - 1) / workgroups;
    if (apart) total = wide;
    const int at = index * p.share;
    if (index > (total - 1) / p.share) return p;
    p.left = min(p.share, total - at);
    int front = 0;
    for (int base = 0; base < seqs; base += 64) {
        if (base) look(base);
        const int tiles = (apart ? up(each) : each) * units, upto = lane_scan(tiles);
        const uint64_t past = __ballot(front + upto > at);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            p.b = base + l;
            p.seq = seq_of_lane(mine, l);
            const int in = at - (front + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l)), own = __builtin_amdgcn_readlane(each, l), line = apart ? up(own) : own;
            p.unit = in / line;
            p.tile = in - p.unit * line;
            if (apart) p.left = min(p.left, own - p.tile);
            break;
        }
        front += __builtin_amdgcn_readlane(upto, 63);
    }
    return p;
}

// What a row sees: tokens of the context from this one on, and from there on those of the tree whose bit is set.
__device__ __forceinline__ int sight_of(const TreeArgs &a, const KvSeq &s, int node) {
    if (!a.window) return 0;
    const int32_t *mask = a.tree + (int64_t)(s.row0 + node) * a.words;
    int left = a.window;
    for (int w = ((s.news + 31) >> 5) - 1; w >= 0; w--) {
        uint32_t bits = (uint32_t)mask[w];
        if (s.news - 32 * w < 32) bits &= (1u << (s.news - 32 * w)) - 1u;  // (those behind the last node are none)
        const int n = __popc(bits);
        if (n >= left) {  // the last `left` of these, and nothing in front
            for (int drop = n - left; drop > 0; drop--) bits &= bits - 1;
            return s.first + 32 * w + __ffs((int)bits) - 1;
        }
        left -= n;
    }
    return s.first > left ? s.first - left : 0;
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
    static constexpr int kJoin = RG < 256 / D ? RG : D == 256 ? (RG < 2 ? RG : 2) : 256 / D;  // groups of sixteen rows whose results meet at a time
    static constexpr int kSums = kSplitWaves * 16 * kJoin * (D + 4) * 4;
    static constexpr int kBytes = (kQueries + kRing > kSums ? kQueries + kRing : kSums);
};

template <int D, bool BF16, int RG>
__global__ __launch_bounds__(64 * kSplitWaves, D == 256 ? 1 : 2) void kv_tree_kernel(const TreeArgs a) {
    constexpr bool TWO = !BF16;
    constexpr int W = D / 16, G = D / 32, ROWS = 16 * RG;
    typedef TreeLds<D, BF16, RG> Lds;
    __shared__ __align__(16) uint8_t lds[Lds::kBytes];
    __shared__ float refs[kSplitWaves][ROWS], totals[kSplitWaves][ROWS], scales[ROWS];
    __shared__ float factors[kSplitWaves][ROWS];  // what a wavefront multiplies its scores by as it takes their exponentials
    __shared__ int lows[ROWS], mask_rows[ROWS];  // (read where a tile needs masks: in registers they would take what the results need)
    const KvCall &kv = a.kv;
    const int tid = (int)threadIdx.x, lane = tid & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TreePlace at = tree_place_of(a, (int)blockIdx.x, (int)gridDim.x, ROWS);
    if (at.b < 0) return;
    const Unpack unpack;
    uint8_t *ring = lds + Lds::kQueries + wave * kSplitSlots * SplitLds<D>::kSlot;
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)ring);
    h8 *operands = reinterpret_cast<h8 *>(lds);

#pragma unroll 1
    for (;;) {
        at.uniform();
        const KvSeq seq = at.seq;
        const int blocks = blocks_of(a, seq, ROWS), h = at.unit / blocks, block = at.unit - h * blocks;
        const int row_first = block * ROWS, rows = min(ROWS, seq.news * a.group - row_first);
        int lo, hi;
        tokens_of(a, seq, lo, hi);
        const int tiles = tree_tiles(a, seq), here = min(at.left, tiles - at.tile);
        const int tile0 = (lo >> 5) + at.tile, tile1 = min(tile0 + here, (hi + 31) >> 5);

        TileWalk<KvTile<D>::kBytes, kSplitWaves> walk(kv, at.b, h, tile0 + wave, tile1);
        const uint8_t *mem = walk.next();
        if (mem) fetch_tile<D>(ring_at, mem);
        // the rows' queries, sixteen rows a wavefront at a time
#pragma unroll 1
        for (int m = wave; m < RG; m += kSplitWaves) {
            const int idx = row_first + 16 * m + r;
            const bool live = 16 * m + r < rows;
            const int node = live ? idx / a.group : 0, head = h * a.group + (live ? idx - node * a.group : 0);
            h8 qh[G], ql[TWO ? G : 1];
            float to_log2;
            load_queries<D, 16, BF16, TWO>(a.q, (int64_t)(seq.row0 + node) * a.q.row + head * a.q.head, live, a.wide, a.scale_log2, qh, ql, to_log2);
            to_log2 = to_log2 < 0x1p-122f ? 0x1p-122f : to_log2;  // (not 0, so that its product with -infinity stays that; a scale of NaN stays one)
#pragma unroll
            for (int g = 0; g < G; g++) {
                operands[(m * G + g) * 64 + lane] = qh[g];
                if constexpr (TWO) operands[Lds::kOperands / 16 + (m * G + g) * 64 + lane] = ql[g];
            }
            if (j == 0) {
                scales[16 * m + r] = to_log2;
                lows[16 * m + r] = live ? sight_of(a, seq, node) : 0;
                mask_rows[16 * m + r] = live ? seq.row0 + node : -1;
            }
        }
        __syncthreads();
        int all_lo = 0;  // from here on every row sees the context
#pragma unroll
        for (int m = 0; m < RG; m++) {
            factors[wave][16 * m + r] = scales[16 * m + r];
            all_lo = max(all_lo, lows[16 * m + r]);
        }
        if (a.window) {
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) all_lo = max(all_lo, __shfl_xor(all_lo, m));
        }
        all_lo = __builtin_amdgcn_readfirstlane(all_lo);

        f4 o[RG][W];
        float ref[RG], total[RG];  // the rows' references, and the lane's share of their sums
        bool coarse = false;       // one of the references is large: scores are multiplied by their scale first, and the factors are 1
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
                f4 s[RG][2];  // scores as the products leave them: what they are multiplied by is not negative
                {
                    // The rows' operands are read three steps (of sixteen rows and a group) ahead, and the next group's codes widened between the matrix instructions.
                    constexpr int AHEAD = TWO ? 1 : 3, STEPS = G * RG;
                    h8 q[AHEAD + 1], rest[TWO ? 2 : 1], keys[2][2];
                    const auto read = [&](int i) __attribute__((always_inline)) {
                        q[i % (AHEAD + 1)] = operands[(i % RG * G + i / RG) * 64 + lane];
                        if constexpr (TWO) rest[i % 2] = operands[Lds::kOperands / 16 + (i % RG * G + i / RG) * 64 + lane];
                    };
                    KeyWords<D> k;
                    k.load(ring + turn * SplitLds<D>::kSlot);
#pragma unroll
                    for (int i = 0; i < AHEAD; i++)
                        if (i < STEPS) read(i);
                    keys[0][0] = k.operand(unpack, 0, 0);
                    keys[0][1] = k.operand(unpack, 1, 0);
#pragma unroll
                    for (int m = 0; m < RG; m++) s[m][0] = s[m][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < STEPS; i++) {
                        const int g = i / RG, m = i % RG;
                        __builtin_amdgcn_sched_barrier(0);  // (the order as written: left alone the compiler widens everything first and reads an operand as it needs it)
                        if (i + AHEAD < STEPS) read(i + AHEAD);
                        if (g + 1 < G) {
                            if (m == 0) keys[(g + 1) & 1][0] = k.operand(unpack, 0, g + 1);
                            if (m == RG / 2) keys[(g + 1) & 1][1] = k.operand(unpack, 1, g + 1);
                        }
                        s[m][0] = mfma(keys[g & 1][0], q[i % (AHEAD + 1)], s[m][0]);
                        s[m][1] = mfma(keys[g & 1][1], q[i % (AHEAD + 1)], s[m][1]);
                        if constexpr (TWO) {
                            s[m][0] = mfma(keys[g & 1][0], rest[i % 2], s[m][0]);
                            s[m][1] = mfma(keys[g & 1][1], rest[i % 2], s[m][1]);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (t0 < all_lo || t0 + 32 > seq.first) {
#pragma unroll
                    for (int m = 0; m < RG; m++) {
                        const int row = mask_rows[16 * m + r], from = row < 0 ? hi : lows[16 * m + r], first = t0 + 8 * j;
                        uint32_t bits = row < 0 ? 0u : mask_bits(a.tree + (int64_t)row * a.words, a.words, first - seq.first);
                        // bit e: token first + e is seen
                        const int context = seq.first - first, behind = from - first, end = hi - first;
                        bits |= context >= 8 ? 255u : context > 0 ? (1u << context) - 1u : 0u;
                        bits &= behind >= 8 ? 0u : behind > 0 ? 255u << behind : 255u;
                        bits &= end >= 8 ? 255u : end > 0 ? (1u << end) - 1u : 0u;
#pragma unroll
                        for (int e = 0; e < 8; e++) s[m][e >> 2][e & 3] = bits >> e & 1u ? s[m][e >> 2][e & 3] : kNegInf;
                    }
                }
                if (!TWO && coarse) {
#pragma unroll
                    for (int m = 0; m < RG; m++) { s[m][0] *= scales[16 * m + r]; s[m][1] *= scales[16 * m + r]; }
                }
                float by[RG], most[RG];
                bool beyond = false;
#pragma unroll
                for (int m = 0; m < RG; m++) by[m] = factors[wave][16 * m + r];
#pragma unroll
                for (int m = 0; m < RG; m++) {
                    // (the maximum that takes a NaN, which makes the row one anyway: the other would first have to make sure of every score's kind)
                    const auto larger = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
                    most[m] = larger(larger(larger(s[m][0].x, s[m][0].y), larger(s[m][0].z, s[m][0].w)), larger(larger(s[m][1].x, s[m][1].y), larger(s[m][1].z, s[m][1].w)));
                    most[m] *= by[m];
                    beyond = beyond || passes<D, TWO>(most[m], ref[m]);
                }
                if (__any(beyond)) {  // (the first score of a row among them: its reference is -infinity)
                    bool large = false;
#pragma unroll
                    for (int m = 0; m < RG; m++) {
                        if (!__any(passes<D, TWO>(most[m], ref[m]))) continue;
                        most[m] = fmaxf(most[m], __shfl_xor(most[m], 16));
                        most[m] = fmaxf(most[m], __shfl_xor(most[m], 32));
                        const float next = fmaxf(ref[m], reference<D, TWO>(most[m]));
                        const float shrink = next == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ref[m] - next);
                        ref[m] = next;
                        large = large || (fabsf(next) >= kCoarse && next != kNegInf);
                        total[m] *= shrink;
#pragma unroll
                        for (int w = 0; w < W; w++) o[m][w] *= shrink;
                    }
                    if (!TWO && !coarse && __any(large)) {  // (this tile's scores too)
                        coarse = true;
#pragma unroll
                        for (int m = 0; m < RG; m++) {
                            s[m][0] *= scales[16 * m + r];
                            s[m][1] *= scales[16 * m + r];
                            factors[wave][16 * m + r] = by[m] = 1.0f;
                        }
                    }
                }
                h8 ph[RG], pl[TWO ? RG : 1];
#pragma unroll
                for (int m = 0; m < RG; m++) {
                    const float less = ref[m] == kNegInf ? 0.0f : -ref[m];
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[m][e >> 2][e & 3], by[m], less)), p1 = __builtin_amdgcn_exp2f(fmaf(s[m][e >> 2][(e & 3) + 1], by[m], less));
                        ph[m][e] = (_Float16)p0;
                        ph[m][e + 1] = (_Float16)p1;
                        if constexpr (TWO) {
                            total[m] += p0;
                            total[m] += p1;
                            pl[m][e] = (_Float16)(p0 - (float)ph[m][e]);
                            pl[m][e + 1] = (_Float16)(p1 - (float)ph[m][e + 1]);
                        } else {  // the weights as they are used, two in one instruction
                            const h2 pair = {ph[m][e], ph[m][e + 1]}, ones = {(_Float16)1.0f, (_Float16)1.0f};
                            total[m] = __builtin_amdgcn_fdot2(pair, ones, total[m], false);
                        }
                    }
                }
                ValueWords<D> v;
                v.load(ring + turn * SplitLds<D>::kSlot);
                h8 x[2];
                x[0] = v.operand(unpack, 0);
#pragma unroll
                for (int w = 0; w < W; w++) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (w + 1 < W) x[(w + 1) & 1] = v.operand(unpack, w + 1);
#pragma unroll
                    for (int m = 0; m < RG; m++) {
                        o[m][w] = mfma(x[w & 1], ph[m], o[m][w]);
                        if constexpr (TWO) o[m][w] = mfma(x[w & 1], pl[m], o[m][w]);
                    }
                }
            }
            mem = mem_next;
            turn ^= 1;
        }

        // the wavefronts' results, a few groups of rows at a time, in the place of queries and tiles
        constexpr int JOIN = Lds::kJoin;
        int thread = tid;
        asm volatile("" : "+v"(thread));  // (or what follows from it is made in front of all units, for registers that the tiles need)
        const int in_row = thread & 15, in_four = (thread >> 4) & 3;
        float(*sums)[16 * JOIN][D + 4] = reinterpret_cast<float(*)[16 * JOIN][D + 4]>(lds);
        const bool begins = at.tile == 0, whole = begins && here == tiles;
        if (a.pieces && begins && tid == 0) a.pieces[(at.b * kv.kv_heads + h) * a.blocks + block] = make_int2((int)blockIdx.x, 1 + (tiles - here + at.share - 1) / at.share);
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
        for (int m0 = 0; m0 < RG; m0 += JOIN) {
            __syncthreads();
            if (m0 == 0 && thread < ROWS) {  // what each wavefront's sums are multiplied by; the row's reference and sum
                float top = kNegInf, all = 0.0f;
#pragma unroll
                for (int w = 0; w < kSplitWaves; w++) top = fmaxf(top, refs[w][thread]);
#pragma unroll
                for (int w = 0; w < kSplitWaves; w++) {
                    const float by = refs[w][thread], f = by == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(by - top);
                    // (a wavefront without a reference has seen no number: its sum is zero, or NaN)
                    all += by == kNegInf ? totals[w][thread] : totals[w][thread] * f;
                    factors[w][thread] = f;
                }
                refs[0][thread] = top;
                totals[0][thread] = all;
            }
#pragma unroll
            for (int m = m0; m < m0 + JOIN && m < RG; m++)
#pragma unroll
                for (int w = 0; w < W; w++) *reinterpret_cast<f4 *>(&sums[wave][16 * (m - m0) + in_row][16 * w + 4 * in_four]) = o[m][w];
            __syncthreads();
            const int count = min(16 * JOIN, rows - 16 * m0);
            for (int i = thread; i < count * (D / 4); i += 64 * kSplitWaves) {
                const int in = i / (D / 4), rr = 16 * m0 + in, d = (i - in * (D / 4)) * 4;
                f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kSplitWaves; w++) sum += *reinterpret_cast<const f4 *>(&sums[w][in][d]) * factors[w][rr];
                if (whole) {
                    const int node = (row_first + rr) / a.group;
                    const int64_t out = (int64_t)(seq.row0 + node) * a.heads + h * a.group + (row_first + rr - node * a.group);
                    store_result<BF16>(a.out, out * D + d, sum, totals[0][rr]);
                } else {
                    const int64_t line = ((int64_t)blockIdx.x * 2 + begins) * a.rows + rr;
                    *reinterpret_cast<f4 *>(a.part + line * D + d) = sum;
                    if (d == 0) {
                        a.part_ml[line * 2] = refs[0][rr];
                        a.part_ml[line * 2 + 1] = totals[0][rr];
                    }
                }
            }
        }
        at.left -= here;
        if (at.left <= 0) break;
        // the next unit, of the next sequence that has one where this was the last
        at.tile = 0;
        if (++at.unit == blocks * kv.kv_heads) {
            at.unit = 0;
            do {
                at.seq = kv_seq(kv, ++at.b);
            } while (at.seq.news == 0);  // (tiles are left: there is one)
        }
        __syncthreads();
    }
}

// Joins the pieces of the units that more than one workgroup has worked on: SHARES threads for four values of a row.  4 us for one sequence of 2047 tokens (16 pieces a unit), 7.5 for 32
// of up to 8192 (two or three pieces, 20 MB of sums; with a workgroup a row 20).
template <int D, bool BF16, int SHARES>
__global__ __launch_bounds__(256) void kv_tree_join_kernel(const TreeArgs a, int block_rows) {
    constexpr int L = D / 4, R = 256 / L / SHARES;  // lanes of a row's values; rows of a workgroup
    __shared__ f4 sums[256];
    __shared__ float tops[256 / L], alls[256 / L];
    const int per_block = (a.rows + R - 1) / R, h = (int)blockIdx.y, tid = (int)threadIdx.x;
    int block = (int)blockIdx.x / per_block, b = (int)blockIdx.z;
    const int rr = ((int)blockIdx.x - block * per_block) * R + tid / L / SHARES, share = tid / L % SHARES, d = tid % L * 4;
    KvSeq seq{};
    if (a.all_blocks) {
        const int index = block, lane = tid & 63;
        int front = 0;
        b = -1;
        for (int base = 0; base < a.kv.seqs; base += 64) {
            KvSeq mine{};
            if (base + lane < a.kv.seqs) mine = kv_seq(a.kv, base + lane);
            const int blocks = blocks_of(a, mine, block_rows), upto = lane_scan(blocks);
            const uint64_t past = __ballot(front + upto > index);
            if (past) {
                const int l = __ffsll((unsigned long long)past) - 1;
                b = base + l;
                seq = seq_of_lane(mine, l);
                block = index - (front + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(blocks, l));
                break;
            }
            front += __builtin_amdgcn_readlane(upto, 63);
        }
        if (b < 0) return;
    } else {
        seq = kv_seq(a.kv, b);
    }
    const int unit = (b * a.kv.kv_heads + h) * a.blocks + block;
    if (block * block_rows >= seq.news * a.group) return;  // (without rows nobody has written the unit's pieces)
    const int2 piece = a.pieces[unit];
    const int first = piece.x, pieces = piece.y;
    if (pieces == 1) return;
    const bool live = rr < a.rows && block * block_rows + rr < seq.news * a.group;
    const auto line = [&](int i) { return ((int64_t)(first + i) * 2 + (i == 0)) * a.rows + (live ? rr : 0); };
    float top = kNegInf, all = 0.0f;
    f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = share; i < pieces; i += SHARES) top = fmaxf(top, a.part_ml[line(i) * 2]);
#pragma unroll 4
    for (int i = share; i < pieces; i += SHARES) {
        const float ref = a.part_ml[line(i) * 2], t = a.part_ml[line(i) * 2 + 1];
        const float f = ref == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ref - top);
        all += ref == kNegInf ? t : t * f;
        sum += *reinterpret_cast<const f4 *>(a.part + line(i) * D + d) * f;
    }
    if constexpr (SHARES > 1) {
        sums[tid] = sum;
        if (d == 0) { tops[tid / L] = top; alls[tid / L] = all; }
        __syncthreads();
        if (share) return;
        const int mine = tid / L;
#pragma unroll
        for (int i = 0; i < SHARES; i++) top = fmaxf(top, tops[mine + i]);
        sum = f4{0.f, 0.f, 0.f, 0.f};
        all = 0.0f;
#pragma unroll
        for (int i = 0; i < SHARES; i++) {
            const float f = tops[mine + i] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(tops[mine + i] - top);
            all += tops[mine + i] == kNegInf ? alls[mine + i] : alls[mine + i] * f;
            sum += sums[tid + i * L] * f;
        }
    }
    if (!live) return;
    const int node = (block * block_rows + rr) / a.group;
    const int64_t out = (int64_t)(seq.row0 + node) * a.heads + h * a.group + (block * block_rows + rr - node * a.group);
    store_result<BF16>(a.out, out * D + d, sum, all);
}

template <int D, bool BF16, int SHARES> int tree_join(const TreeArgs &a, int block_rows, hipStream_t s) {
    constexpr int R = 1024 / D / SHARES;
    const int per_block = (a.rows + R - 1) / R;
    const dim3 grid((unsigned)((a.all_blocks ? a.all_blocks : a.blocks) * per_block), (unsigned)a.kv.kv_heads, a.all_blocks ? 1u : (unsigned)a.kv.seqs);
    return launch(kv_tree_join_kernel<D, BF16, SHARES>, grid, dim3(256), 0, s, a, block_rows);
}
template <int D, bool BF16, int RG> int tree_attend(const TreeArgs &a, int workgroups, hipStream_t s) {
    if (int rc = launch(kv_tree_kernel<D, BF16, RG>, dim3((unsigned)workgroups), dim3(64 * kSplitWaves), 0, s, a)) return rc;
    if (!a.pieces) return GQ_OK;
    // (with many pieces a unit the threads of a row share them)
    const int64_t units = (int64_t)a.kv.seqs * a.kv.kv_heads * a.blocks;
    constexpr int most = 1024 / D;
    return workgroups > 8 * units ? tree_join<D, BF16, most>(a, 16 * RG, s) : tree_join<D, BF16, 1>(a, 16 * RG, s);
}
template <int D, bool BF16> int tree_attend(const TreeArgs &a, int row_groups, int workgroups, hipStream_t s) {
    switch (row_groups) {
    case 1: return tree_attend<D, BF16, 1>(a, workgroups, s);
    case 2: return tree_attend<D, BF16, 2>(a, workgroups, s);
    case 3:
        if constexpr (D < 256) return tree_attend<D, BF16, 3>(a, workgroups, s);
    default:
        if constexpr (D == 256) return tree_attend<D, BF16, 2>(a, workgroups, s);
        else return tree_attend<D, BF16, 4>(a, workgroups, s);
    }
}

}  // namespace

// How a call's rows are cut into blocks: 16 RG (node, query head) pairs of a key head.
struct TreePlan { int row_groups, rows; int64_t blocks, tiles, all_blocks; };
static TreePlan tree_plan(const KvCall &kv, int heads, int window) {
    TreePlan p;
    const int64_t most_rows = (int64_t)kv.max_new * (heads / kv.kv_heads), room = (int64_t)kv.max_pages * kv.page_tokens / 32;
    p.row_groups = (int)std::min<int64_t>((most_rows + 15) / 16, kv.head_dim == 256 ? 2 : 4);
    p.rows = (int)std::min<int64_t>(most_rows, 16 * p.row_groups);
    p.blocks = (most_rows + 16 * p.row_groups - 1) / (16 * p.row_groups);
    // (one large tree beside many small ones: nearly all of a grid laid out for the largest would have nothing to do)
    p.all_blocks = (int64_t)kv.rows * (heads / kv.kv_heads) / (16 * p.row_groups) + kv.seqs;
    if (p.blocks * kv.seqs <= 2 * p.all_blocks) p.all_blocks = 0;
    p.tiles = std::max<int64_t>(1, window ? std::min<int64_t>(room, ((int64_t)window + kv.max_new + 31) / 32 + 1) : room);
    return p;
}

int check_kv_tree_attention(const char *fn, const KvCall &kv, int heads, int window) {
    const TreePlan p = tree_plan(kv, heads, window);
    const int64_t units = (int64_t)kv.seqs * kv.kv_heads * p.blocks;
    // (threads of a launch are counted in 32 bits: fewer than 2^24 workgroups, of which a block of rows has one for every 1024 values that are joined; and so are the tiles of all units)
    const int64_t joined = p.all_blocks ? p.all_blocks * kv.kv_heads : units;
    if (p.blocks > INT32_MAX / kv.kv_heads / kv.seqs || joined * ((p.rows * kv.head_dim + 1023) / 1024) > (1 << 24) - 4096 || units > (INT32_MAX - 4096) / p.tiles)
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
    a.all_blocks = (int)p.all_blocks;
    const int64_t tiles = p.tiles, units = (int64_t)kv.seqs * kv.kv_heads * a.blocks;
    // Two workgroups a CU, as many as run at a time with 64 rows (with 16 there is room for more, of whose pieces more have to be joined): 16 nodes of 32 sequences of 2048 to 8192
    // tokens, 1, 2, 3 and 4 a CU: bfloat16 at D = 128 99 80 101 98 us, at D = 64 71 54 68 64, float32 129 110 125 128; 4 nodes at D = 128 65 52 53 60, at D = 64 47 34 31 31; 32 nodes over 131072 tokens
    // 107 95 109 105.  At D = 256 one runs at a time: 130 140 157 175.
    const int per_cu = kv.head_dim == 256 ? 1 : 2;
    const int workgroups = (int)std::min<int64_t>(device_cu_count() * per_cu, units * ((tiles + kLeastShare - 1) / kLeastShare));
    if (tiles > 1) {
        const size_t lines = (size_t)workgroups * 2 * a.rows;
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
    case 64: return q.bf16 ? tree_attend<64, true>(a, p.row_groups, workgroups, s) : tree_attend<64, false>(a, p.row_groups, workgroups, s);
    case 128: return q.bf16 ? tree_attend<128, true>(a, p.row_groups, workgroups, s) : tree_attend<128, false>(a, p.row_groups, workgroups, s);
    default: return q.bf16 ? tree_attend<256, true>(a, p.row_groups, workgroups, s) : tree_attend<256, false>(a, p.row_groups, workgroups, s);
    }
}

}  // namespace gq
