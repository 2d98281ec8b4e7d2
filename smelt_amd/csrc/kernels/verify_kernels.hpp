// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   p = softmax(target / t), q = softmax(draft / t) (or all of it on the drafted token);
//   draft x of row i is taken while u_i q(x) < p(x); the first one refused is replaced by a token drawn from
//   max(p - q, 0), and when all are taken one more is drawn from the last row's p: the lowest index whose running
//   sum passes u * total.  t <= 0: the largest logit instead, lowest index first.
//
// Bound by the logits' bytes.  Four launches: (1) every row's runs of logits to (top, its index, sum of exponentials);
// (2) each sequence's accepted count from those, and the chosen row's exponentials once more in 64 bits; (3) the leftover
// weights of a refused draft; (4) the place of u in the running sum.  Sums that decide which token is drawn are 64-bit: with a
// 248320-entry vocabulary neighbouring tokens' places in the running sum are 4e-6 apart and closer, and a 32-bit exponential is already
// off by 6e-8 of each weight.  The first launch's 32-bit exponentials only meet the accept test, whose sides are apart by more unless u falls
// within about 1e-7 of the ratio.  Sums are added in a fixed order: the same inputs give the same tokens.
#pragma once
#include "common.hpp"
#include "serving_args.hpp"

namespace smelt {

using smelt_serving::VerifyArgs;
using smelt_serving::VerifyStat;

// not-a-number counts as -inf, +inf as the largest finite value
__device__ __forceinline__ float verify_logit(float v) { return v == v ? __builtin_fminf(v, 3.3895314e38f) : -__builtin_inff(); }

struct VerifySequence {
    uint32_t first, rows;       // token rows of the sequence
    float t;
    bool greedy;
};
__device__ __forceinline__ VerifySequence verify_sequence(const VerifyArgs& a, uint32_t s) {
    VerifySequence q;
    q.first = smelt_serving::clamp_count(a.offsets[s], a.rows);
    const uint32_t end = smelt_serving::clamp_count(a.offsets[s + 1], a.rows);
    q.rows = end > q.first ? end - q.first : 0u;
    q.t = a.temperature[s];
    q.greedy = !(q.t > 0.0f);
    return q;
}

__device__ __forceinline__ uint32_t verify_sequence_of(const VerifyArgs& a, uint32_t row) {
    uint32_t lo = 0, hi = a.sequences;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (smelt_serving::clamp_count(a.offsets[mid], a.rows) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// calls use(index, logit) for eight neighbouring logits at a time, of the thread's share of [first, last)
template <class ActT, class F>
__device__ __forceinline__ void verify_walk(const uint16_t* row, uint32_t first, uint32_t last, bool vector, F use) {
    for (uint32_t i = first + threadIdx.x * 8; i < last; i += blockDim.x * 8) {
        float x[8];
        if (vector && i + 8 <= last) {
            const uint4_t v = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(row + i));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[2 * k] = verify_logit(ActT::widen((uint16_t)(w[k] & 0xFFFFu)));
                x[2 * k + 1] = verify_logit(ActT::widen((uint16_t)(w[k] >> 16)));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = i + k < last ? verify_logit(ActT::widen(row[i + k])) : -__builtin_inff();
        }
        use(i, x);
    }
}

template <class T, class F>
__device__ __forceinline__ T verify_reduce(T v, T* scratch, F join) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = join(v, __shfl_xor(v, off));
    const uint32_t wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == 0) scratch[wave] = v;
    __syncthreads();
    v = scratch[0];
    for (uint32_t w = 1; w < waves; ++w) v = join(v, scratch[w]);
    return v;
}

__device__ __forceinline__ double verify_weight(float logit, float top, double t) {
    return logit == -__builtin_inff() ? 0.0 : exp(((double)logit - (double)top) / t);
}

// (1) grid: runs x rows x {target, draft}
template <class ActT>
__device__ __forceinline__ void verify_stats(const VerifyArgs& a) {
    __shared__ float tops[16];
    __shared__ uint32_t wheres[16];
    __shared__ double sums[16];
    const uint32_t chunk = blockIdx.x, row = blockIdx.y, which = blockIdx.z;
    if (row >= smelt_serving::clamp_count(a.offsets[a.sequences], a.rows)) return;
    const VerifySequence q = verify_sequence(a, verify_sequence_of(a, row));
    if (which == 1 && (q.greedy || row + 1 >= q.first + q.rows)) return;    // no draft is asked about here
    const uint16_t* src = (which ? a.draft : a.target) + (size_t)row * a.stride;
    const uint32_t first = chunk * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
    float top = -__builtin_inff();
    uint32_t where = ~0u;
    float run = 0.0f;
    const float c = q.greedy ? 0.0f : __builtin_fminf(1.4426950408889634f / q.t, 3.0e38f);
    verify_walk<ActT>(src, first, last, a.vector, [&](uint32_t i, const float* x) {
        float m = x[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) m = __builtin_fmaxf(m, x[k]);
        if (m > top) {
            run *= top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - m) * c);
            top = m;
#pragma unroll
            for (int k = 7; k >= 0; --k) where = x[k] == m ? i + k : where;
        }
        if (!q.greedy && top != -__builtin_inff()) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += x[k] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((x[k] - top) * c);
            run += s;
        }
    });
    const float all = verify_reduce(top, tops, [](float x, float y) { return __builtin_fmaxf(x, y); });
    const uint32_t lowest = verify_reduce(top == all ? where : ~0u, wheres, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
    const double mine = top == -__builtin_inff() ? 0.0 : (double)run * (double)__builtin_amdgcn_exp2f((top - all) * c);
    const double sum = verify_reduce(mine, sums, [](double x, double y) { return x + y; });
    if (threadIdx.x == 0) {
        VerifyStat& st = a.stats[((size_t)which * a.rows + row) * a.chunks + chunk];
        st.top = all;
        st.where = lowest;
        st.sum = sum;
    }
}

// a row's runs put together by one wave
struct VerifyRow { float top; uint32_t where; double sum; };
__device__ __forceinline__ VerifyRow verify_row(const VerifyArgs& a, uint32_t which, uint32_t row, float t, bool greedy) {
    const VerifyStat* st = a.stats + ((size_t)which * a.rows + row) * a.chunks;
    const uint32_t lane = threadIdx.x % kWave;
    VerifyRow r{-__builtin_inff(), ~0u, 0.0};
    for (uint32_t c = lane; c < a.chunks; c += kWave)
        if (st[c].top > r.top) { r.top = st[c].top; r.where = st[c].where; }
    float top = r.top;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off));
    uint32_t where = r.top == top && top != -__builtin_inff() ? r.where : ~0u;
    double sum = 0.0;
    if (!greedy)
        for (uint32_t c = lane; c < a.chunks; c += kWave) sum += st[c].sum * verify_weight(st[c].top, top, (double)t);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = __shfl_xor(where, off);
        where = o < where ? o : where;
        sum += __shfl_xor(sum, off);
    }
    return VerifyRow{top, where, sum};
}

// accepted drafts of the sequence, by the whole workgroup; the waves take a draft each
template <class ActT>
__device__ __forceinline__ uint32_t verify_accepted(const VerifyArgs& a, const VerifySequence& q, uint32_t* refused) {
    const uint32_t wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    if (threadIdx.x == 0) *refused = q.rows ? q.rows - 1 : 0u;
    __syncthreads();
    for (uint32_t base = 0; base + 1 < q.rows; base += waves) {
        const uint32_t i = base + wave;
        bool ok = true;
        if (i + 1 < q.rows) {
            const uint32_t row = q.first + i;
            const int32_t x = a.draft_tokens[row];
            const VerifyRow p = verify_row(a, 0, row, q.t, q.greedy);
            if (q.greedy) ok = p.where != ~0u && x == (int32_t)p.where;
            else {
                ok = x >= 0 && (uint32_t)x < a.vocab && p.sum > 0.0;
                if (ok) {
                    const double t = (double)q.t;
                    const double px = verify_weight(verify_logit(ActT::widen(a.target[(size_t)row * a.stride + x])), p.top, t) / p.sum;
                    double qx = 1.0;
                    if (a.draft) {
                        const VerifyRow d = verify_row(a, 1, row, q.t, false);
                        qx = d.sum > 0.0 ? verify_weight(verify_logit(ActT::widen(a.draft[(size_t)row * a.stride + x])), d.top, t) / d.sum : 0.0;
                    }
                    ok = (double)a.u_accept[row] * qx < px;
                }
            }
        }
        if (!ok && threadIdx.x % kWave == 0) atomicMin(refused, i);
        __syncthreads();
        if (*refused < base + waves) break;    // (the same for every wave: the barrier is behind the last write)
    }
    __syncthreads();
    return *refused;
}

// (2) grid: runs x sequences
template <class ActT>
__device__ __forceinline__ void verify_choose(const VerifyArgs& a) {
    __shared__ uint32_t refused;
    __shared__ double scratch[16];
    __shared__ float tops[2];
    const uint32_t chunk = blockIdx.x, s = blockIdx.y;
    const VerifySequence q = verify_sequence(a, s);
    const uint32_t taken = verify_accepted<ActT>(a, q, &refused);
    if (chunk == 0 && threadIdx.x == 0) a.choice[s] = (int32_t)taken;
    if (q.rows == 0 || q.greedy) return;
    const uint32_t row = q.first + taken;
    const bool leftover = taken + 1 < q.rows;
    const uint32_t first = chunk * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
    if (threadIdx.x < kWave) {
        const VerifyRow p = verify_row(a, 0, row, q.t, false);
        VerifyRow d{0.0f, 0u, 0.0};
        if (a.draft && leftover) d = verify_row(a, 1, row, q.t, false);
        if (threadIdx.x == 0) { tops[0] = p.top; tops[1] = d.top; }
    }
    __syncthreads();
    const double t = (double)q.t;
    const int32_t without = !a.draft && leftover ? a.draft_tokens[row] : -1;
    double sum = 0.0, rest = 0.0;
    verify_walk<ActT>(a.target + (size_t)row * a.stride, first, last, a.vector, [&](uint32_t i, const float* x) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double w = verify_weight(x[k], tops[0], t);
            sum += w;
            if ((int32_t)(i + k) != without) rest += w;
        }
    });
    double* out = a.sums + (size_t)s * 3 * a.chunks + chunk;
    auto add = [](double x, double y) { return x + y; };
    sum = verify_reduce(sum, scratch, add);
    rest = verify_reduce(rest, scratch, add);
    if (threadIdx.x == 0) { out[0] = sum; out[2 * a.chunks] = rest; }
    if (a.draft && leftover) {
        double dsum = 0.0;
        verify_walk<ActT>(a.draft + (size_t)row * a.stride, first, last, a.vector, [&](uint32_t, const float* x) {
#pragma unroll
            for (int k = 0; k < 8; ++k) dsum += verify_weight(x[k], tops[1], t);
        });
        dsum = verify_reduce(dsum, scratch, add);
        if (threadIdx.x == 0) out[a.chunks] = dsum;
    }
}

// what launches 3 and 4 need of the chosen row
struct VerifyChosen {
    uint32_t row, taken;
    bool leftover;              // a draft was refused
    float p_top, d_top;
    double p_inv, d_inv;        // 1 / sum of all runs (0: the row has no weight)
};
__device__ __forceinline__ VerifyChosen verify_chosen(const VerifyArgs& a, uint32_t s, const VerifySequence& q, double* scratch) {
    VerifyChosen c;
    c.taken = (uint32_t)a.choice[s];
    c.row = q.first + c.taken;
    c.leftover = c.taken + 1 < q.rows;
    if (threadIdx.x < kWave) {
        const bool two = a.draft && c.leftover;
        const VerifyRow p = verify_row(a, 0, c.row, q.t, true);
        VerifyRow d{0.0f, 0u, 0.0};
        if (two) d = verify_row(a, 1, c.row, q.t, true);
        const double* sums = a.sums + (size_t)s * 3 * a.chunks;
        double ps = 0.0, ds = 0.0;
        for (uint32_t k = threadIdx.x; k < a.chunks; k += kWave) { ps += sums[k]; if (two) ds += sums[a.chunks + k]; }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) { ps += __shfl_xor(ps, off); ds += __shfl_xor(ds, off); }
        if (threadIdx.x == 0) { scratch[0] = p.top; scratch[1] = d.top; scratch[2] = ps; scratch[3] = ds; }
    }
    __syncthreads();
    c.p_top = (float)scratch[0]; c.d_top = (float)scratch[1];
    c.p_inv = scratch[2] > 0.0 ? 1.0 / scratch[2] : 0.0;
    c.d_inv = scratch[3] > 0.0 ? 1.0 / scratch[3] : 0.0;
    __syncthreads();
    return c;
}

// (3) grid: runs x sequences; only for refused drafts of a draft model
template <class ActT>
__device__ __forceinline__ void verify_leftover(const VerifyArgs& a) {
    __shared__ double scratch[16];
    const uint32_t chunk = blockIdx.x, s = blockIdx.y;
    const VerifySequence q = verify_sequence(a, s);
    if (q.rows == 0 || q.greedy || (uint32_t)a.choice[s] + 1 >= q.rows) return;
    const VerifyChosen c = verify_chosen(a, s, q, scratch);
    const uint32_t first = chunk * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
    const uint16_t* draft = a.draft + (size_t)c.row * a.stride;
    const double t = (double)q.t;
    double sum = 0.0;
    verify_walk<ActT>(a.target + (size_t)c.row * a.stride, first, last, a.vector, [&](uint32_t i, const float* x) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (i + k >= last) continue;
            const double w = verify_weight(x[k], c.p_top, t) * c.p_inv - verify_weight(verify_logit(ActT::widen(draft[i + k])), c.d_top, t) * c.d_inv;
            sum += w > 0.0 ? w : 0.0;
        }
    });
    sum = verify_reduce(sum, scratch, [](double x, double y) { return x + y; });
    if (threadIdx.x == 0) a.sums[((size_t)s * 3 + 2) * a.chunks + chunk] = sum;
}

// (4) grid: sequences
template <class ActT>
__device__ __forceinline__ void verify_draw(const VerifyArgs& a) {
    __shared__ double scratch[16];
    __shared__ double start;
    __shared__ uint32_t found, last_weight, wanted_chunk, use_rest;
    const uint32_t s = blockIdx.x;
    const VerifySequence q = verify_sequence(a, s);
    if (threadIdx.x == 0) a.counts[s] = a.choice[s];
    if (q.rows == 0) return;
    const uint32_t taken = (uint32_t)a.choice[s];
    int32_t token = -1;
    if (q.greedy) {
        if (threadIdx.x < kWave) {
            const VerifyRow p = verify_row(a, 0, q.first + taken, q.t, true);
            if (threadIdx.x == 0) found = p.where;
        }
        __syncthreads();
        token = found == ~0u ? -1 : (int32_t)found;
    } else {
        const VerifyChosen c = verify_chosen(a, s, q, scratch);
        const double* sums = a.sums + (size_t)s * 3 * a.chunks;
        const double t = (double)q.t;
        bool rest = c.leftover;
        if (threadIdx.x == 0) {
            double total = 0.0;
            if (rest) for (uint32_t k = 0; k < a.chunks; ++k) total += sums[2 * a.chunks + k];
            if (!(total > 0.0)) { rest = false; total = 0.0; for (uint32_t k = 0; k < a.chunks; ++k) total += sums[k]; }
            const double* from = sums + (rest ? 2 * a.chunks : 0);
            const double want = (double)a.u_sample[s] * total;
            double run = 0.0;
            uint32_t at = ~0u, heavy = ~0u;
            double at_run = 0.0, heavy_run = 0.0;
            for (uint32_t k = 0; k < a.chunks; ++k) {
                const double next = run + from[k];
                if (from[k] > 0.0) { heavy = k; heavy_run = run; }
                if (at == ~0u && next > want) { at = k; at_run = run; }
                run = next;
            }
            if (at == ~0u) { at = heavy; at_run = heavy_run; }     // u rounded up to the total: the last token with a weight
            wanted_chunk = at;
            start = want - at_run;
            found = ~0u;
            last_weight = 0u;
            use_rest = rest ? 1u : 0u;
        }
        __syncthreads();
        rest = use_rest != 0u;
        if (wanted_chunk != ~0u) {
            const uint32_t first = wanted_chunk * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
            const uint16_t* target = a.target + (size_t)c.row * a.stride;
            const uint16_t* draft = a.draft ? a.draft + (size_t)c.row * a.stride : nullptr;
            const int32_t without = !a.draft && rest ? a.draft_tokens[c.row] : -1;
            const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
            double before = 0.0;
            for (uint32_t base = first; base < last; base += blockDim.x) {
                const uint32_t i = base + threadIdx.x;
                double w = 0.0;
                if (i < last && (int32_t)i != without) {
                    w = verify_weight(verify_logit(ActT::widen(target[i])), c.p_top, t);
                    if (draft && rest) {
                        w = w * c.p_inv - verify_weight(verify_logit(ActT::widen(draft[i])), c.d_top, t) * c.d_inv;
                        w = w > 0.0 ? w : 0.0;
                    }
                }
                double run = w;
#pragma unroll
                for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
                    const double up = __shfl_up(run, d);
                    if (lane >= d) run += up;
                }
                if (lane == kWave - 1) scratch[wave] = run;
                __syncthreads();
                double mine = before;
                for (uint32_t k = 0; k < waves; ++k) {
                    if (k < wave) mine += scratch[k];
                    before += scratch[k];
                }
                if (w > 0.0) {
                    if (mine + run > start) atomicMin(&found, i);
                    atomicMax(&last_weight, i);
                }
                __syncthreads();
                if (found != ~0u) break;
            }
            token = (int32_t)(found != ~0u ? found : last_weight);
        }
    }
    for (uint32_t i = threadIdx.x; i < q.rows; i += blockDim.x) {
        const uint32_t row = q.first + i;
        a.tokens[row] = i < taken ? a.draft_tokens[row] : (i == taken ? token : -1);
    }
}

}  // namespace smelt

#define SMELT_VERIFY_KERNELS(T, ACT)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void smelt_verify_stats_##T(smelt_serving::VerifyArgs a) { smelt::verify_stats<ACT>(a); }       \
    extern "C" __global__ __launch_bounds__(256) void smelt_verify_choose_##T(smelt_serving::VerifyArgs a) { smelt::verify_choose<ACT>(a); }     \
    extern "C" __global__ __launch_bounds__(256) void smelt_verify_leftover_##T(smelt_serving::VerifyArgs a) { smelt::verify_leftover<ACT>(a); } \
    extern "C" __global__ __launch_bounds__(1024) void smelt_verify_draw_##T(smelt_serving::VerifyArgs a) { smelt::verify_draw<ACT>(a); }
