// Rotary positions and the paged cache's writer.
//
//   angle(t, i) = position(t) * f(i);  a pair (x0, x1) of a head becomes (x0 c - x1 s, x1 c + x0 s),
//   c = amplitude * cos(angle), s = amplitude * sin(angle)
//
// Pairs are (i, i + R/2) in the half layout and (2i, 2i + 1) in the interleaved one; values R.. of a head are copied.
// The angle is formed in 64 bits as a count of turns, and its whole turns are dropped there: a 32-bit product
// is off by 0.03 rad at position 500000, the turn's fraction in 32 bits by 4e-7 rad at any position.  cos, sin and the products are
// 32-bit, the result is rounded once.
//
// Memory-bound: every row is read and written once, 16 bytes a lane, and the R/2 angles of a token are formed once by its
// workgroup (LDS) and used by all of its heads.  8192 tokens of 32 heads of 128: 27.7 us (134 MB, 4.8 TB/s; a plain copy reaches 5.1);
// 8000 tokens of 8 heads of 128 into pages of 16: 18.3 us (66 MB, 3.6 TB/s: the 64 bytes that four tokens put side by side are half a
// cache line).  One token: 4 us, the launch.  Loading the next pieces before the angles are formed, or four at a time, was
// slower (30.5 and 22.0 us): more instructions to fetch for a kernel whose workgroups live for two microseconds.
#pragma once
#include "common.hpp"
#include "serving_args.hpp"

namespace smelt {

using smelt_serving::RopeArgs;
using smelt_serving::RopeRows;

__device__ __forceinline__ uint32_t fast_div(uint32_t n, uint32_t d, uint32_t inv) { return d <= 1 ? n : __umulhi(n, inv); }

template <class ActT>
__device__ __forceinline__ void unpack8(uint4_t v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[2 * k] = ActT::widen((uint16_t)(w[k] & 0xFFFFu));
        f[2 * k + 1] = ActT::widen((uint16_t)(w[k] >> 16));
    }
}

template <class ActT>
__device__ __forceinline__ uint4_t pack8(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)ActT::narrow(f[2 * k]) | ((uint32_t)ActT::narrow(f[2 * k + 1]) << 16);
    return uint4_t{w[0], w[1], w[2], w[3]};
}

// cos and sin of the workgroup's tokens, `pairs` a token, into LDS
__device__ __forceinline__ void rope_angles(const RopeArgs& a, uint32_t first, uint32_t count, float2* cs) {
    const uint32_t pairs = a.rot / 2;
    const uint32_t inv = smelt_serving::reciprocal(pairs);
    for (uint32_t i = threadIdx.x; i < count * pairs; i += blockDim.x) {
        const uint32_t tok = fast_div(i, pairs, inv), pair = i - tok * pairs;
        double turns = (double)a.positions[first + tok] * (a.table[pair] * 0.15915494309189533577);
        turns -= __builtin_rint(turns);
        float s, c;
        sincospif(2.0f * (float)turns, &s, &c);
        cs[i] = float2{c * a.amplitude, s * a.amplitude};
    }
}

// Where a token's rows go: rows of their own, or the cache.
enum RopeTarget { kToRows, kToKeys, kToValues };

template <int TARGET>
__device__ __forceinline__ size_t rope_at(const RopeArgs& a, const RopeRows& r, uint32_t token, int32_t slot, uint32_t head, uint32_t d) {
    if (TARGET == kToRows) return (size_t)token * r.dst_stride + (size_t)head * a.dim + d;
    const uint32_t page = (uint32_t)slot >> a.page_shift, off = (uint32_t)slot & ((1u << a.page_shift) - 1u);
    const size_t base = ((size_t)page * r.heads + head) * a.dim << a.page_shift;
    // values: [page][head][offset][dim]; keys: [page][head][dim / 8][offset][8], the operand order of the attention kernels
    if (TARGET == kToValues) return base + (size_t)off * a.dim + d;
    return base + ((((size_t)(d >> 3) << a.page_shift) + off) << 3) + (d & 7u);
}

// What a unit of a token's work is: a pair of 16-byte pieces of a rotated head (half), one piece (interleaved), or a copied piece;
// without VEC one pair of values, or one copied value.
struct RopeUnit {
    int target;
    uint32_t tok, head, d, d2;      // d2: the pair's other piece or value, d where there is none
    bool copied;
};

// unit i of a workgroup's: the tokens' q units, then the k units, then the v units
template <bool VEC, bool APPEND>
__device__ __forceinline__ RopeUnit rope_unit(const RopeArgs& a, uint32_t shift, uint32_t i) {
    RopeUnit x;
    x.target = kToRows;
    uint32_t u;
    if (!APPEND || i < a.q.units << shift) {
        x.tok = fast_div(i, a.q.units, a.q_units_inv);
        u = i - x.tok * a.q.units;
    } else {
        i -= a.q.units << shift;
        x.target = kToKeys;
        x.tok = i & ((1u << shift) - 1u);
        u = i >> shift;
        if (u >= a.k.units) {
            i -= a.k.units << shift;
            x.target = kToValues;
            x.tok = fast_div(i, a.v.units, a.v_units_inv);
            u = i - x.tok * a.v.units;
        }
    }
    const bool value = x.target == kToValues;
    x.head = value ? fast_div(u, a.per_copy, a.per_copy_inv) : fast_div(u, a.per_head, a.per_head_inv);
    const uint32_t unit = u - x.head * (value ? a.per_copy : a.per_head);
    const uint32_t one = VEC ? 8u : 1u, rotated = VEC ? (a.interleaved ? a.rot / 8 : a.rot / 16) : a.rot / 2;
    x.copied = value || unit >= rotated;
    if (x.copied) x.d = x.d2 = value ? unit * one : a.rot + (unit - rotated) * one;
    else if (!a.interleaved) { x.d = unit * one; x.d2 = x.d + a.rot / 2; }
    else if (VEC) x.d = x.d2 = unit * 8;
    else { x.d = 2 * unit; x.d2 = x.d + 1; }
    return x;
}
// (the fields are chosen one by one: a chosen set of rows would have to lie in memory)
template <bool APPEND>
__device__ __forceinline__ const uint16_t* rope_src(const RopeArgs& a, const RopeUnit& x, uint32_t first) {
    const uint16_t* src = a.q.src;
    uint32_t stride = a.q.src_stride;
    if (APPEND && x.target == kToKeys) { src = a.k.src; stride = a.k.src_stride; }
    if (APPEND && x.target == kToValues) { src = a.v.src; stride = a.v.src_stride; }
    return src + (size_t)(first + x.tok) * stride + (size_t)x.head * a.dim;
}
template <bool APPEND>
__device__ __forceinline__ uint16_t* rope_dst(const RopeArgs& a, const RopeUnit& x, uint32_t first, int32_t slot, uint32_t d) {
    if (APPEND && x.target == kToKeys) return a.k.dst + rope_at<kToKeys>(a, a.k, first + x.tok, slot, x.head, d);
    if (APPEND && x.target == kToValues) return a.v.dst + rope_at<kToValues>(a, a.v, first + x.tok, slot, x.head, d);
    return a.q.dst + rope_at<kToRows>(a, a.q, first + x.tok, 0, x.head, d);
}

// One workgroup per `tokens_per_group` (a power of two) tokens.  Its threads take units in turn: along the rows that are stored as they
// are read, and token after token for keys, since the 16-byte pieces that neighbouring tokens put into a key page lie side by side.
template <class ActT, bool VEC, bool APPEND>
__device__ __forceinline__ void rope_body(const RopeArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const uint32_t pairs = a.rot / 2;
    float2* cs = reinterpret_cast<float2*>(smem);
    int32_t* slots = reinterpret_cast<int32_t*>(cs + a.tokens_per_group * pairs);
    const uint32_t first = blockIdx.x * a.tokens_per_group, shift = 31 - __builtin_clz(a.tokens_per_group);
    const uint32_t count = a.tokens - first < a.tokens_per_group ? a.tokens - first : a.tokens_per_group;
    if (APPEND && threadIdx.x < count) slots[threadIdx.x] = a.slots[first + threadIdx.x];
    rope_angles(a, first, count, cs);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.per_token << shift; i += blockDim.x) {
        const RopeUnit x = rope_unit<VEC, APPEND>(a, shift, i);
        if (x.tok >= count) continue;
        int32_t slot = 0;
        if (APPEND && x.target != kToRows) {
            slot = slots[x.tok];
            if (slot < 0 || ((uint32_t)slot >> a.page_shift) >= a.pages) continue;      // nowhere to go
        }
        const uint16_t* src = rope_src<APPEND>(a, x, first);
        uint16_t* to = rope_dst<APPEND>(a, x, first, slot, x.d);
        const float2* w = cs + x.tok * pairs;
        if constexpr (VEC) {
            const uint4_t in = *reinterpret_cast<const uint4_t*>(src + x.d);
            if (x.copied) { *reinterpret_cast<uint4_t*>(to) = in; continue; }
            float v[8], y[8];
            unpack8<ActT>(in, v);
            if (a.interleaved) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 z = w[x.d / 2 + q];
                    y[2 * q] = v[2 * q] * z.x - v[2 * q + 1] * z.y;
                    y[2 * q + 1] = v[2 * q + 1] * z.x + v[2 * q] * z.y;
                }
            } else {
                float v2[8], y2[8];
                unpack8<ActT>(*reinterpret_cast<const uint4_t*>(src + x.d2), v2);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float2 z = w[x.d + q];
                    y[q] = v[q] * z.x - v2[q] * z.y;
                    y2[q] = v2[q] * z.x + v[q] * z.y;
                }
                *reinterpret_cast<uint4_t*>(rope_dst<APPEND>(a, x, first, slot, x.d2)) = pack8<ActT>(y2);
            }
            *reinterpret_cast<uint4_t*>(to) = pack8<ActT>(y);
        } else {
            if (x.copied) { *to = src[x.d]; continue; }
            const float x0 = ActT::widen(src[x.d]), x1 = ActT::widen(src[x.d2]);
            const float2 z = w[a.interleaved ? x.d / 2 : x.d];
            *to = ActT::narrow(x0 * z.x - x1 * z.y);
            *rope_dst<APPEND>(a, x, first, slot, x.d2) = ActT::narrow(x1 * z.x + x0 * z.y);
        }
    }
}

}  // namespace smelt

#define SMELT_SERVING_KERNEL(THREADS) extern "C" __global__ __launch_bounds__(THREADS)

#define SMELT_ROPE_KERNELS(T, ACT)                                                                                            \
    SMELT_SERVING_KERNEL(256) void smelt_rope_vec_##T(smelt_serving::RopeArgs a) { smelt::rope_body<ACT, true, false>(a); }       \
    SMELT_SERVING_KERNEL(256) void smelt_rope_any_##T(smelt_serving::RopeArgs a) { smelt::rope_body<ACT, false, false>(a); }      \
    SMELT_SERVING_KERNEL(256) void smelt_paged_append_vec_##T(smelt_serving::RopeArgs a) { smelt::rope_body<ACT, true, true>(a); } \
    SMELT_SERVING_KERNEL(256) void smelt_paged_append_any_##T(smelt_serving::RopeArgs a) { smelt::rope_body<ACT, false, true>(a); }
