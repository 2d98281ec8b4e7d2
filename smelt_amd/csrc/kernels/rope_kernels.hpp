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
// workgroup (LDS) and used by all of its heads.
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

// one unit of a rotated head: a pair of 16-byte pieces (half), one piece (interleaved), or a copied piece;
// without VEC one pair of values, or one copied value
template <class ActT, bool VEC, int TARGET>
__device__ __forceinline__ void rope_unit(const RopeArgs& a, const RopeRows& r, const float2* cs, uint32_t token, int32_t slot, uint32_t head, uint32_t unit) {
    const uint16_t* src = r.src + (size_t)token * r.src_stride + (size_t)head * a.dim;
    auto at = [&](uint32_t d) { return r.dst + rope_at<TARGET>(a, r, token, slot, head, d); };
    if (VEC) {
        const uint32_t rotated = a.interleaved ? a.rot / 8 : a.rot / 16;
        if (TARGET == kToValues || unit >= rotated) {
            const uint32_t d = TARGET == kToValues ? unit * 8 : a.rot + (unit - rotated) * 8;
            *reinterpret_cast<uint4_t*>(at(d)) = *reinterpret_cast<const uint4_t*>(src + d);
            return;
        }
        const uint32_t d = unit * 8;
        float x[8], y[8];
        unpack8<ActT>(*reinterpret_cast<const uint4_t*>(src + d), x);
        if (a.interleaved) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 w = cs[d / 2 + k];
                y[2 * k] = x[2 * k] * w.x - x[2 * k + 1] * w.y;
                y[2 * k + 1] = x[2 * k + 1] * w.x + x[2 * k] * w.y;
            }
            *reinterpret_cast<uint4_t*>(at(d)) = pack8<ActT>(y);
        } else {
            const uint32_t d2 = d + a.rot / 2;
            float x2[8], y2[8];
            unpack8<ActT>(*reinterpret_cast<const uint4_t*>(src + d2), x2);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float2 w = cs[d + k];
                y[k] = x[k] * w.x - x2[k] * w.y;
                y2[k] = x2[k] * w.x + x[k] * w.y;
            }
            *reinterpret_cast<uint4_t*>(at(d)) = pack8<ActT>(y);
            *reinterpret_cast<uint4_t*>(at(d2)) = pack8<ActT>(y2);
        }
    } else {
        const uint32_t pairs = a.rot / 2;
        if (TARGET == kToValues || unit >= pairs) {
            const uint32_t d = TARGET == kToValues ? unit : a.rot + (unit - pairs);
            *at(d) = src[d];
            return;
        }
        const uint32_t d0 = a.interleaved ? 2 * unit : unit, d1 = a.interleaved ? 2 * unit + 1 : unit + pairs;
        const float x0 = ActT::widen(src[d0]), x1 = ActT::widen(src[d1]);
        const float2 w = cs[unit];
        *at(d0) = ActT::narrow(x0 * w.x - x1 * w.y);
        *at(d1) = ActT::narrow(x1 * w.x + x0 * w.y);
    }
}

// One workgroup per `tokens_per_group` tokens; its threads walk the tokens' units.
template <class ActT, bool VEC, bool APPEND>
__device__ __forceinline__ void rope_body(const RopeArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    float2* cs = reinterpret_cast<float2*>(smem);
    const uint32_t first = blockIdx.x * a.tokens_per_group;
    const uint32_t count = a.tokens - first < a.tokens_per_group ? a.tokens - first : a.tokens_per_group;
    rope_angles(a, first, count, cs);
    __syncthreads();
    const uint32_t pairs = a.rot / 2;
    for (uint32_t i = threadIdx.x; i < count * a.per_token; i += blockDim.x) {
        const uint32_t tok = fast_div(i, a.per_token, a.per_token_inv);
        uint32_t u = i - tok * a.per_token;
        const uint32_t token = first + tok;
        const float2* w = cs + tok * pairs;
        if (!APPEND || u < a.q.units) {
            const uint32_t head = fast_div(u, a.per_head, a.per_head_inv);
            rope_unit<ActT, VEC, kToRows>(a, a.q, w, token, 0, head, u - head * a.per_head);
            continue;
        }
        if (APPEND) {
            u -= a.q.units;
            const int32_t slot = a.slots[token];
            if (slot < 0 || ((uint32_t)slot >> a.page_shift) >= a.pages) continue;   // nowhere to go
            if (u < a.k.units) {
                const uint32_t head = fast_div(u, a.per_head, a.per_head_inv);
                rope_unit<ActT, VEC, kToKeys>(a, a.k, w, token, slot, head, u - head * a.per_head);
            } else {
                u -= a.k.units;
                const uint32_t head = fast_div(u, a.per_copy, a.per_copy_inv);
                rope_unit<ActT, VEC, kToValues>(a, a.v, w, token, slot, head, u - head * a.per_copy);
            }
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
