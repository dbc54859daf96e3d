// An RMS norm of every query and key head with the rotation by position behind it, in one pass.
//
//     y = x / sqrt(mean(x^2) + eps) * (gain + offset)           over the D values of a head (where a norm is given)
//     (a, b) -> (a cos - b sin, a sin + b cos)                  for the pairs (i, i + rot / 2) or (2 i, 2 i + 1), i < rot / 2
//
// cos and sin come from a table [position][rot / 2] that a program lays out once: angles of large positions are formed in 64
// bits there, and every way of scaling the rates is a matter of the table.  A position outside the table makes a row of NaN.
//
// A lane holds four neighbouring values, D / 4 lanes a head, so that a wavefront reads and writes whole lines; the partner of a
// value in the other half of the rotation is a lane exchange away.  All arithmetic in 32 bits, one rounding at the store.
//
// HBM bounds it: 2048 rows of 32 + 8 heads of D = 128, float32 to bfloat16, 64 MB: 16.7 us a call, 3.8 TB/s; one row: 3.2 us, a launch and two loads.
#include "common.hpp"

#include <algorithm>

namespace gq {

namespace {

struct RopeArgs {
    HeadRows q, k;
    int q_heads, heads;  // heads: of queries and keys together
    int64_t rows, table_rows, first;  // first: workgroups of the call in front of the launch's
    const int32_t *positions;
    const float *cos, *sin;
    int rot;
    RmsNorm norm[2];
    int has_norm[2];
    void *out[2];
    int wide;  // inputs can be read 16 (bf16: 8) bytes at a time
};

__device__ __forceinline__ float bf16_bits(uint32_t u) { return __uint_as_float(u << 16); }

template <bool BF16> __device__ __forceinline__ float4 load4(const void *p, int64_t at, int wide) {
    float4 v;
    if constexpr (BF16) {
        const uint16_t *x = static_cast<const uint16_t *>(p) + at;
        if (wide) {
            const uint2 u = *reinterpret_cast<const uint2 *>(x);
            v = make_float4(bf16_bits(u.x & 0xFFFFu), __uint_as_float(u.x & 0xFFFF0000u), bf16_bits(u.y & 0xFFFFu), __uint_as_float(u.y & 0xFFFF0000u));
        } else {
            v = make_float4(bf16_bits(x[0]), bf16_bits(x[1]), bf16_bits(x[2]), bf16_bits(x[3]));
        }
    } else {
        const float *x = static_cast<const float *>(p) + at;
        v = wide ? *reinterpret_cast<const float4 *>(x) : make_float4(x[0], x[1], x[2], x[3]);
    }
    return v;
}

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <int D, bool BF16, bool OUT_BF16, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const RopeArgs a) {
    constexpr int L = D / 4;  // lanes of a head
    const int64_t unit = ((a.first + blockIdx.x) * 256 + threadIdx.x) / L;
    const int lane = (int)threadIdx.x & (L - 1);
    const int64_t row = unit / a.heads;
    if (row >= a.rows) return;  // (whole heads leave together: the exchanges below stay inside one head)
    const int head = (int)(unit - row * a.heads);
    const bool key = head >= a.q_heads;
    const HeadRows &in = key ? a.k : a.q;
    const int h = key ? head - a.q_heads : head;
    const int d = lane * 4;

    const int pos = a.positions[row];
    float4 x = load4<BF16>(in.p, row * in.row + h * in.head + d, a.wide);
    if (a.has_norm[key]) {
        const RmsNorm &n = a.norm[key];
        float ss = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, x.w * x.w)));
#pragma unroll
        for (int m = 1; m < L; m <<= 1) ss += __shfl_xor(ss, m);
        const float r = sqrtf(ss * (1.0f / D) + n.eps);
        x.x /= r; x.y /= r; x.z /= r; x.w /= r;
        if (n.gain) {
            x.x *= n.gain[d] + n.gain_offset;
            x.y *= n.gain[d + 1] + n.gain_offset;
            x.z *= n.gain[d + 2] + n.gain_offset;
            x.w *= n.gain[d + 3] + n.gain_offset;
        }
    }
    const int half = a.rot >> 1;
    const bool known = (uint32_t)pos < (uint64_t)a.table_rows;
    const int64_t at = known ? (int64_t)pos * half : 0;
    float4 y = x;
    const bool turns = known && d < a.rot;  // (nothing is read for a position that the table does not have: it may have none, and no memory)
    if constexpr (INTERLEAVED) {
        if (turns) {
            const float2 c = *reinterpret_cast<const float2 *>(a.cos + at + (d >> 1)), s = *reinterpret_cast<const float2 *>(a.sin + at + (d >> 1));
            y.x = fmaf(x.x, c.x, -(x.y * s.x));
            y.y = fmaf(x.x, s.x, x.y * c.x);
            y.z = fmaf(x.z, c.y, -(x.w * s.y));
            y.w = fmaf(x.z, s.y, x.w * c.y);
        }
    } else {
        const bool upper = d >= half;
        const int step = half >> 2;  // lanes to the partner
        const int from = ((int)threadIdx.x & 63) + (d < a.rot ? (upper ? -step : step) : 0);
        const float4 o = make_float4(__shfl(x.x, from), __shfl(x.y, from), __shfl(x.z, from), __shfl(x.w, from));
        if (turns) {
            const int i = upper ? d - half : d;
            const float4 c = *reinterpret_cast<const float4 *>(a.cos + at + i);
            float4 s = *reinterpret_cast<const float4 *>(a.sin + at + i);
            if (!upper) s = make_float4(-s.x, -s.y, -s.z, -s.w);  // the first of a pair: a cos - b sin, the second: b cos + a sin
            y = make_float4(fmaf(x.x, c.x, o.x * s.x), fmaf(x.y, c.y, o.y * s.y), fmaf(x.z, c.z, o.z * s.z), fmaf(x.w, c.w, o.w * s.w));
        }
    }
    if (!known) y.x = y.y = y.z = y.w = __uint_as_float(0x7FC00000u);
    const int64_t to = (row * (key ? a.heads - a.q_heads : a.q_heads) + h) * D + d;
    if constexpr (OUT_BF16) {
        bf16x4 v = {(__bf16)y.x, (__bf16)y.y, (__bf16)y.z, (__bf16)y.w};
        *reinterpret_cast<bf16x4 *>(static_cast<uint16_t *>(a.out[key]) + to) = v;
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out[key]) + to) = y;
    }
}

template <int D, bool BF16, bool OUT_BF16> int launch_rope(RopeArgs a, bool interleaved, hipStream_t s) {
    const int64_t per = 256 / (D / 4), blocks = (a.rows * a.heads + per - 1) / per;
    constexpr int64_t kMost = ((int64_t)1 << 24) - 1;  // (a launch has fewer than 2^32 threads: 2^26 heads of 256 values, 2^28 of 64)
    for (a.first = 0; a.first < blocks; a.first += kMost) {
        const dim3 grid((unsigned)std::min(blocks - a.first, kMost)), block(256);
        if (int rc = interleaved ? launch(qk_norm_rope_kernel<D, BF16, OUT_BF16, true>, grid, block, 0, s, a)
                                 : launch(qk_norm_rope_kernel<D, BF16, OUT_BF16, false>, grid, block, 0, s, a))
            return rc;
    }
    return GQ_OK;
}
template <int D> int launch_rope(const RopeArgs &a, bool interleaved, bool bf16, bool out_bf16, hipStream_t s) {
    if (bf16) return out_bf16 ? launch_rope<D, true, true>(a, interleaved, s) : launch_rope<D, true, false>(a, interleaved, s);
    return out_bf16 ? launch_rope<D, false, true>(a, interleaved, s) : launch_rope<D, false, false>(a, interleaved, s);
}

bool wide_rows(const HeadRows &h, int n) {  // n elements at a time
    const size_t size = h.bf16 ? 2 : 4;
    return ((reinterpret_cast<uintptr_t>(h.p) | (size_t)(h.row * (int64_t)size) | (size_t)(h.head * (int64_t)size)) & (n * size - 1)) == 0;
}

}  // namespace

int launch_qk_norm_rope(const HeadRows &q, int q_heads, const HeadRows &k, int k_heads, int head_dim, int64_t rows, const int32_t *positions, const float *cos,
                        const float *sin, int64_t table_rows, int rot, bool interleaved, const RmsNorm *q_norm, const RmsNorm *k_norm, bool out_bf16, void *q_out,
                        void *k_out, hipStream_t s) {
    RopeArgs a{};
    a.q = q;
    a.k = k;
    a.q_heads = q_heads;
    a.heads = q_heads + k_heads;
    a.rows = rows;
    a.table_rows = table_rows;
    a.positions = positions;
    a.cos = cos;
    a.sin = sin;
    a.rot = rot;
    if (q_norm) { a.norm[0] = *q_norm; a.has_norm[0] = 1; }
    if (k_norm) { a.norm[1] = *k_norm; a.has_norm[1] = 1; }
    a.out[0] = q_out;
    a.out[1] = k_out;
    a.wide = (q_heads == 0 || wide_rows(q, 4)) && (k_heads == 0 || wide_rows(k, 4));
    switch (head_dim) {
    case 64: return launch_rope<64>(a, interleaved, q.bf16, out_bf16, s);
    case 128: return launch_rope<128>(a, interleaved, q.bf16, out_bf16, s);
    default: return launch_rope<256>(a, interleaved, q.bf16, out_bf16, s);
    }
}

}  // namespace gq
