// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
//   p = softmax(target / t), q = softmax(draft / t) (or all of it on the drafted token);
//   draft x of row i is taken while u_i q(x) < p(x); the first one refused is replaced by a token drawn from
//   max(p - q, 0), and when all are taken one more is drawn from the last row's p: the lowest index whose running
//   sum passes u * total.  t <= 0: the largest logit instead, lowest index first.
//
// Bound by the logits' bytes.  Four launches: (1) every row's runs of logits to (top, sum of exponentials), a wave a run; (2) each
// sequence's accepted count from those, and the chosen row's exponentials once more in 64 bits; (3) the leftover weights of a
// refused draft; (4) the place of u in the running sum.  Sums that decide which token is drawn are 64-bit, from 64-bit
// exponentials: with a 248320-entry vocabulary neighbouring places in the running sum are 4e-6 apart and closer, and a 32-bit
// exponential is already off by 6e-8 of each weight.  The first launch's 32-bit exponentials only meet the accept test, which they can
// turn when u falls within a few 1e-7 of the ratio.  Sums are added in a fixed order: the same inputs give the same tokens.
// 64 sequences of 1 to 8 rows, 248320 logits: 105 us (254 MB, 50 us at a copy's rate): launch 1 takes 44 us (5.8 TB/s), 2 and 3 30 and
// 23 us (the chosen rows' 64-bit exponentials: twenty 64-bit instructions a logit, about 14 us each), 4 takes 12.  One sequence: 25 us, four
// launches of two or three dependent loads each.  Rows that do not lie at whole 16 bytes (a stride that is no multiple of 8) are read two
// bytes at a time: the 64 sequences with a vocabulary of 248319 216 us, one of 151935 31.
#pragma once
#include "common.hpp"
#include "serving_args.hpp"

namespace smelt {

using smelt_serving::VerifyArgs;
using smelt_serving::VerifyChoice;
using smelt_serving::VerifyStat;

// Not-a-number counts as -inf: the hardware's median of three takes the smallest operand when one of them is not a number.  (Written
// as an instruction: the compiler reads a median with -inf as a minimum, which would take the other operand.)  +inf counts as
// the largest finite value.
__device__ __forceinline__ float verify_logit(float v) {
    float r;
    asm("v_med3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(v), "s"(-__builtin_inff()), "v"(3.3895314e38f));
    return r;
}

struct VerifySequence {
    uint32_t first, rows;       // token rows of the sequence
    float t;
    bool greedy;
    float rate;                 // log2(e) / t, kept finite
    double rate64;
};
__device__ __forceinline__ VerifySequence verify_sequence(const VerifyArgs& a, uint32_t s) {
    VerifySequence q;
    q.first = smelt_serving::clamp_count(a.offsets[s], a.rows);
    const uint32_t end = smelt_serving::clamp_count(a.offsets[s + 1], a.rows);
    q.rows = end > q.first ? end - q.first : 0u;
    q.t = a.temperature[s];
    q.greedy = !(q.t > 0.0f);
    q.rate64 = q.greedy ? 0.0 : 1.4426950408889634074 / (double)q.t;
    q.rate = q.greedy ? 0.0f : __builtin_fminf((float)q.rate64, 3.0e38f);
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

// exp((logit - top) / t) in 32 bits; the larger of a number and not-a-number is the number, so that -inf at t = inf weighs nothing
__device__ __forceinline__ float verify_weight32(float logit, float top, float rate) {
    return __builtin_amdgcn_exp2f(__builtin_fmaxf((logit - top) * rate, -200.0f));
}

// ... in 64 bits: 2^a by its nearest whole power n and the Taylor series of 2^f, |f| <= 1/2, up to f^10 (the next term is at most 2.2e-13: a weight is off by
// at most 3.0e-13 of itself, and neighbouring places of the running sum are about 4e-6 apart).
// n is the low word of the sum with 1.5 * 2^52.  The coefficients sit in scalar registers, opaque to the compiler: it would otherwise
// accumulate into a copy of each that it makes first, two instructions a term.
struct VerifyExp {
    double c[10];
    __device__ __forceinline__ VerifyExp() : c{7.054911620801121e-09, 1.0178086009239696e-07, 1.3215486790144305e-06, 1.5252733804059838e-05, 1.5403530393381606e-04,
                                               1.3333558146428441e-03, 9.618129107628477e-03, 5.5504108664821576e-02, 2.402265069591007e-01, 6.931471805599453e-01} {
#pragma unroll
        for (int k = 0; k < 10; ++k) asm("" : "+s"(c[k]));      // ln(2)^(10 - k) / (10 - k)!
    }
    __device__ __forceinline__ double weight(float logit, float top, double rate) const {
        const double a = __builtin_fmax(((double)logit - (double)top) * rate, -1100.0);
        const double shifted = a + 6755399441055744.0, f = a - (shifted - 6755399441055744.0);
        double p = c[0];
#pragma unroll
        for (int k = 1; k < 10; ++k) p = __builtin_fma(p, f, c[k]);
        p = __builtin_fma(p, f, 1.0);
        return __builtin_amdgcn_ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, shifted));
    }
};

template <class ActT>
__device__ __forceinline__ void verify_unpack(uint4_t v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[2 * k] = verify_logit(ActT::widen((uint16_t)(w[k] & 0xFFFFu)));
        x[2 * k + 1] = verify_logit(ActT::widen((uint16_t)(w[k] >> 16)));
    }
}

// eight neighbouring logits from i on, -inf from `last` on
template <class ActT>
__device__ __forceinline__ void verify_load8(const uint16_t* row, uint32_t i, uint32_t last, bool vector, float* x) {
    if (vector && i + 8 <= last) {
        verify_unpack<ActT>(*reinterpret_cast<const uint4_t*>(row + i), x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = i + k < last ? verify_logit(ActT::widen(row[i + k])) : -__builtin_inff();
    }
}

// calls use(index, target logits, draft logits) for eight neighbouring logits at a time of a wave's run; four loads of a lane
// (and row) are in flight
template <class ActT, bool TWO, class F>
__device__ __forceinline__ void verify_walk(const uint16_t* target, const uint16_t* draft, uint32_t first, uint32_t last, bool vector, F use) {
    constexpr uint32_t U = 4, step = kWave * 8;
    const uint32_t lane = threadIdx.x % kWave;
    for (uint32_t base = first; base < last; base += U * step) {
        float x[8], y[8];
        if (vector && base + U * step <= last) {
            uint4_t tx[U], ty[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                tx[u] = *reinterpret_cast<const uint4_t*>(target + base + u * step + lane * 8);
                if (TWO) ty[u] = *reinterpret_cast<const uint4_t*>(draft + base + u * step + lane * 8);
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                verify_unpack<ActT>(tx[u], x);
                if (TWO) verify_unpack<ActT>(ty[u], y);
                use(base + u * step + lane * 8, x, y);
            }
        } else {
            for (uint32_t i = base + lane * 8; i < last && i < base + U * step; i += step) {
                verify_load8<ActT>(target, i, last, vector, x);
                if (TWO) verify_load8<ActT>(draft, i, last, vector, y);
                use(i, x, y);
            }
        }
    }
}

template <class T>
__device__ __forceinline__ T wave_total(T v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ float wave_top(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, off));
    return v;
}
__device__ __forceinline__ uint32_t wave_lowest(uint32_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { const uint32_t o = __shfl_xor(v, off); v = o < v ? o : v; }
    return v;
}

// (1) grid: ceil(runs / 4) x rows x {target, draft}
template <class ActT>
__device__ __forceinline__ void verify_stats(const VerifyArgs& a) {
    const uint32_t lane = threadIdx.x % kWave, run = blockIdx.x * 4 + threadIdx.x / kWave, row = blockIdx.y, which = blockIdx.z;
    if (run >= a.runs || row >= smelt_serving::clamp_count(a.offsets[a.sequences], a.rows)) return;
    const VerifySequence q = verify_sequence(a, verify_sequence_of(a, row));
    if (which == 1 && (q.greedy || row + 1 >= q.first + q.rows)) return;    // no draft is asked about here
    const uint16_t* src = (which ? a.draft : a.target) + (size_t)row * a.stride;
    const uint32_t first = run * a.span, last = first + a.span < a.vocab ? first + a.span : a.vocab;
    float top = -__builtin_inff(), sum = 0.0f;
    uint32_t where = ~0u;
    verify_walk<ActT, false>(src, nullptr, first, last, a.vector, [&](uint32_t i, const float* x, const float*) {
        float m = x[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) m = __builtin_fmaxf(m, x[k]);
        if (m > top) {
            sum *= verify_weight32(top, m, q.rate);
            top = m;
            if (q.greedy) {
#pragma unroll
                for (int k = 7; k >= 0; --k) where = x[k] == m ? i + k : where;
            }
        }
        if (!q.greedy) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += verify_weight32(x[k], top, q.rate);
            sum += s;
        }
    });
    const float all = wave_top(top);
    const float total = wave_total(sum * verify_weight32(top, all, q.rate));
    if (lane == 0) a.stats[((size_t)which * a.rows + row) * a.runs + run] = VerifyStat{all, all == -__builtin_inff() ? 0.0f : total};
    if (q.greedy) {
        const uint32_t lowest = wave_lowest(top == all ? where : ~0u);
        if (lane == 0) a.where[(size_t)row * a.runs + run] = lowest;
    }
}

// a row's runs put together by one wave, four loads of a lane in flight
struct VerifyRow { float top, sum; };
__device__ __forceinline__ VerifyRow verify_row(const VerifyArgs& a, uint32_t which, uint32_t row, float rate) {
    const VerifyStat* st = a.stats + ((size_t)which * a.rows + row) * a.runs;
    VerifyRow r{-__builtin_inff(), 0.0f};
    for (uint32_t c = threadIdx.x % kWave; c < a.runs; c += 4 * kWave) {
        VerifyStat x[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) x[k] = c + k * kWave < a.runs ? st[c + k * kWave] : VerifyStat{-__builtin_inff(), 0.0f};
        const float m = __builtin_fmaxf(__builtin_fmaxf(x[0].top, x[1].top), __builtin_fmaxf(x[2].top, x[3].top));
        const float top = __builtin_fmaxf(r.top, m);
        r.sum *= verify_weight32(r.top, top, rate);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) r.sum += x[k].sum * verify_weight32(x[k].top, top, rate);
        r.top = top;
    }
    const float top = wave_top(r.top);
    r.sum = wave_total(r.sum * verify_weight32(r.top, top, rate));
    r.top = top;
    return r;
}
__device__ __forceinline__ uint32_t verify_best(const VerifyArgs& a, uint32_t row) {
    const VerifyStat* st = a.stats + (size_t)row * a.runs;
    float top = -__builtin_inff();
    uint32_t where = ~0u;
    for (uint32_t c = threadIdx.x % kWave; c < a.runs; c += kWave)
        if (st[c].top > top) { top = st[c].top; where = a.where[(size_t)row * a.runs + c]; }
    const float all = wave_top(top);
    return wave_lowest(top == all && all != -__builtin_inff() ? where : ~0u);
}

// accepted drafts of the sequence, by the whole workgroup; the waves take a row each, the last one's for its largest logit
constexpr uint32_t kVerifyTops = 64;
template <class ActT>
__device__ __forceinline__ uint32_t verify_accepted(const VerifyArgs& a, const VerifySequence& q, uint32_t* refused, float2* tops) {
    const uint32_t wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    if (threadIdx.x == 0) *refused = q.rows ? q.rows - 1 : 0u;
    __syncthreads();
    for (uint32_t base = 0; base < q.rows; base += waves) {
        const uint32_t i = base + wave;
        bool ok = true;
        if (i < q.rows) {
            const uint32_t row = q.first + i;
            const bool last = i + 1 == q.rows;
            const int32_t x = last ? 0 : a.draft_tokens[row];
            if (q.greedy) {
                const uint32_t best = verify_best(a, row);
                ok = last || (best != ~0u && x == (int32_t)best);
            } else {
                const VerifyExp e;
                const bool known = x >= 0 && (uint32_t)x < a.vocab, drafted = a.draft && !last;
                const size_t at = (size_t)row * a.stride + (known ? (uint32_t)x : 0u);
                const float px = verify_logit(ActT::widen(a.target[at])), dx = drafted ? verify_logit(ActT::widen(a.draft[at])) : 0.0f;
                double left = (double)a.u_accept[row];
                const VerifyRow p = verify_row(a, 0, row, q.rate);
                VerifyRow d{0.0f, 0.0f};
                if (drafted) {
                    d = verify_row(a, 1, row, q.rate);
                    left = d.sum > 0.0f ? left * e.weight(dx, d.top, q.rate64) / (double)d.sum : 0.0;
                }
                ok = last || (known && p.sum > 0.0f && left < e.weight(px, p.top, q.rate64) / (double)p.sum);
                if (threadIdx.x % kWave == 0) tops[i % kVerifyTops] = float2{p.top, d.top};
            }
        }
        if (!ok && threadIdx.x % kWave == 0) atomicMin(refused, i);
        __syncthreads();
        if (*refused < base + waves) break;    // (the same for every wave: later writes are larger, and so are the rows that overwrite tops)
    }
    __syncthreads();
    return *refused;
}

// (2) grid: ceil(runs / 4) x sequences
template <class ActT>
__device__ __forceinline__ void verify_choose(const VerifyArgs& a) {
    __shared__ uint32_t refused;
    __shared__ float2 tops[kVerifyTops];
    const uint32_t lane = threadIdx.x % kWave, run = blockIdx.x * 4 + threadIdx.x / kWave, s = blockIdx.y;
    const VerifySequence q = verify_sequence(a, s);
    const uint32_t taken = verify_accepted<ActT>(a, q, &refused, tops);
    const uint32_t row = q.first + taken;
    const bool leftover = taken + 1 < q.rows, first_wave = blockIdx.x == 0 && threadIdx.x < kWave;
    if (q.rows == 0 || q.greedy) {
        if (first_wave) {
            const uint32_t where = q.rows ? verify_best(a, row) : ~0u;
            if (lane == 0) a.choice[s] = VerifyChoice{taken, where, 0.0f, 0.0f};
        }
        return;
    }
    const bool two = a.draft && leftover;
    const float top = tops[taken % kVerifyTops].x, draft_top = two ? tops[taken % kVerifyTops].y : 0.0f;
    if (first_wave && lane == 0) a.choice[s] = VerifyChoice{taken, ~0u, top, draft_top};
    if (run >= a.runs) return;
    const uint32_t first = run * a.span, last = first + a.span < a.vocab ? first + a.span : a.vocab;
    const int32_t without = !a.draft && leftover ? a.draft_tokens[row] : -1;
    double* out = a.sums + (size_t)s * 3 * a.runs + run;
    double sum = 0.0, dsum = 0.0;
    const uint16_t* target = a.target + (size_t)row * a.stride;
    const uint16_t* draft = two ? a.draft + (size_t)row * a.stride : nullptr;
    const VerifyExp e;
    // (a refused draft that was given is left out of the sum: taking it away afterwards would take the small weights beside it along)
    auto add = [&](uint32_t i, const float* x) {
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += e.weight((int32_t)(i + k) == without ? -__builtin_inff() : x[k], top, q.rate64);
    };
    if (two)
        verify_walk<ActT, true>(target, draft, first, last, a.vector, [&](uint32_t i, const float* x, const float* y) {
            add(i, x);
#pragma unroll
            for (int k = 0; k < 8; ++k) dsum += e.weight(y[k], draft_top, q.rate64);
        });
    else
        verify_walk<ActT, false>(target, nullptr, first, last, a.vector, [&](uint32_t i, const float* x, const float*) { add(i, x); });
    // (a row without any weight: its top is -inf and the differences above are not numbers, which weigh nothing)
    sum = wave_total(sum);
    if (two) dsum = wave_total(dsum);
    if (lane == 0) {
        const bool here = without >= 0 && (uint32_t)without >= first && (uint32_t)without < last;
        out[0] = here ? sum + e.weight(verify_logit(ActT::widen(target[(uint32_t)without])), top, q.rate64) : sum;
        if (two) out[a.runs] = dsum;
        out[2 * a.runs] = sum;
    }
}

// what launches 3 and 4 need of the chosen row: 1 / sum of all runs (0: the row has no weight), by one wave
struct VerifyInverse { double p, d; };
__device__ __forceinline__ VerifyInverse verify_inverse(const VerifyArgs& a, uint32_t s, bool two) {
    const double* sums = a.sums + (size_t)s * 3 * a.runs;
    double ps = 0.0, ds = 0.0;
    for (uint32_t k = threadIdx.x % kWave; k < a.runs; k += kWave) { ps += sums[k]; if (two) ds += sums[a.runs + k]; }
    ps = wave_total(ps);
    ds = wave_total(ds);
    return VerifyInverse{ps > 0.0 ? 1.0 / ps : 0.0, ds > 0.0 ? 1.0 / ds : 0.0};
}

// The leftover weight max(p - q, 0) of a token.  Both products are rounded before the difference, so that equal rows leave exactly nothing
// over (a fused multiply-add would leave the rounding of one of them, and a token would be drawn from that).
__device__ __forceinline__ double verify_rest(const VerifyExp& e, float x, float y, const VerifyChoice& c, const VerifyInverse& inv, double rate) {
#pragma clang fp contract(off)
    return __builtin_fmax(e.weight(x, c.top, rate) * inv.p - e.weight(y, c.draft_top, rate) * inv.d, 0.0);
}

// (3) grid: ceil(runs / 4) x sequences; only for refused drafts of a draft model
template <class ActT>
__device__ __forceinline__ void verify_leftover(const VerifyArgs& a) {
    const uint32_t lane = threadIdx.x % kWave, run = blockIdx.x * 4 + threadIdx.x / kWave, s = blockIdx.y;
    const VerifySequence q = verify_sequence(a, s);
    if (run >= a.runs || q.rows == 0 || q.greedy) return;
    const VerifyChoice c = a.choice[s];
    if (c.taken + 1 >= q.rows) return;
    const VerifyInverse inv = verify_inverse(a, s, true);
    const uint32_t first = run * a.span, last = first + a.span < a.vocab ? first + a.span : a.vocab;
    const uint16_t* target = a.target + (size_t)(q.first + c.taken) * a.stride;
    const uint16_t* draft = a.draft + (size_t)(q.first + c.taken) * a.stride;
    double sum = 0.0;
    const VerifyExp e;
    verify_walk<ActT, true>(target, draft, first, last, a.vector, [&](uint32_t, const float* x, const float* y) {
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += verify_rest(e, x[k], y[k], c, inv, q.rate64);
    });
    sum = wave_total(sum);
    if (lane == 0) a.sums[((size_t)s * 3 + 2) * a.runs + run] = sum;
}

// sum over the workgroup's threads before this one, and over all of them
__device__ __forceinline__ double block_prefix(double v, double* wave_sums, double* total) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    double run = v;
#pragma unroll
    for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
        const double up = __shfl_up(run, d);
        if (lane >= d) run += up;
    }
    __syncthreads();
    if (lane == kWave - 1) wave_sums[wave] = run;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll 4
    for (uint32_t w = 0; w < waves; ++w) {
        if (w == wave) before = all;
        all += wave_sums[w];
    }
    *total = all;
    return before + run - v;
}

// (4) grid: sequences, 1024 threads.  One workgroup runs this once, so its time is latency: of its loads and of fetching its instructions
// (with its loops unrolled sixteen times over it took 14 and 18 us at 151936 and 248320 logits, so 10 and 12).
template <class ActT>
__device__ __forceinline__ void verify_draw(const VerifyArgs& a) {
    __shared__ double wave_sums[16];
    __shared__ double start, heavy_start;
    __shared__ uint32_t found, heavy, token_found, last_weight;
    const uint32_t s = blockIdx.x;
    const VerifySequence q = verify_sequence(a, s);
    const VerifyChoice c = a.choice[s];
    if (threadIdx.x == 0) { a.counts[s] = (int32_t)c.taken; found = token_found = ~0u; heavy = last_weight = 0u; }
    if (q.rows == 0) return;
    const uint32_t row = q.first + c.taken;
    int32_t token = q.greedy && c.where != ~0u ? (int32_t)c.where : -1;
    if (!q.greedy) {
        const double* sums = a.sums + (size_t)s * 3 * a.runs;
        bool rest = c.taken + 1 < q.rows;
        const bool two = a.draft && rest;
        const VerifyInverse inv = verify_inverse(a, s, two);
        // the run that holds u's place: the first whose running sum passes it; should rounding leave none, the last with a weight
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {
            const double* from = sums + (rest ? 2 * a.runs : 0);
            double total = 0.0, mine = 0.0, before = 0.0;
#pragma unroll 1
            for (uint32_t base = 0; base < a.runs; base += blockDim.x) {
                double part;
                mine = base + threadIdx.x < a.runs ? from[base + threadIdx.x] : 0.0;
                before = total + block_prefix(mine, wave_sums, &part);
                total += part;
            }
            if (!(total > 0.0) && rest) { rest = false; continue; }      // nothing left over: the target's own weights
            const double want = (double)a.u_sample[s] * total;
            double run = 0.0;
#pragma unroll 1
            for (uint32_t base = 0; base < a.runs; base += blockDim.x) {
                const uint32_t k = base + threadIdx.x;
                if (a.runs > blockDim.x) {       // what the first loop kept is its last round's
                    double part;
                    mine = k < a.runs ? from[k] : 0.0;
                    before = run + block_prefix(mine, wave_sums, &part);
                    run += part;
                }
                if (mine > 0.0 && before + mine > want) atomicMin(&found, k);
                const unsigned long long weights = __ballot(mine > 0.0);
                if (weights && (threadIdx.x % kWave) == 63u - (uint32_t)__builtin_clzll(weights)) atomicMax(&heavy, k + 1);
                __syncthreads();
                if (k == found) start = want - before;
                if (k + 1 == heavy) heavy_start = want - before;
            }
            break;
        }
        __syncthreads();
        const uint32_t at = found != ~0u ? found : heavy - 1;      // (~0: no token has a weight)
        if (at != ~0u) {
            const double begin = found != ~0u ? start : heavy_start;
            const uint32_t first = at * a.span, last = first + a.span < a.vocab ? first + a.span : a.vocab;
            const uint16_t* target = a.target + (size_t)row * a.stride;
            const uint16_t* draft = two && rest ? a.draft + (size_t)row * a.stride : target;
            const int32_t without = !a.draft && rest ? a.draft_tokens[row] : -1;
            // neighbouring logits of a thread (the span is 512 times a power of two); loads first, from places inside the run
            constexpr uint32_t E = smelt_serving::kVerifyMaxSpan / 1024;
            const uint32_t each = a.span > blockDim.x ? a.span / blockDim.x : 1u, i0 = first + threadIdx.x * each;
            const uint32_t end = i0 + each < last ? i0 + each : last;
            float x[E], y[E];
#pragma unroll
            for (uint32_t k = 0; k < E; ++k) {
                const uint32_t i = i0 + k < end ? i0 + k : first;
                x[k] = ActT::widen(target[i]);
                y[k] = ActT::widen(draft[i]);
            }
            const VerifyExp e;
            double w[E], sum = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < E; ++k) {
                w[k] = 0.0;
                if (k < each) {
                    const float logit = verify_logit(x[k]);
                    const double v = two && rest ? verify_rest(e, logit, verify_logit(y[k]), c, inv, q.rate64) : e.weight(logit, c.top, q.rate64);
                    w[k] = i0 + k < end && (int32_t)(i0 + k) != without ? v : 0.0;
                }
                sum += w[k];
            }
            double all, run = block_prefix(sum, wave_sums, &all);
            uint32_t mine = ~0u, heaviest = 0u;
#pragma unroll
            for (uint32_t k = 0; k < E; ++k) {
                run += w[k];
                if (w[k] > 0.0) { if (run > begin && mine == ~0u) mine = i0 + k; heaviest = i0 + k; }
            }
            // one lane of a wave speaks for it
            mine = wave_lowest(mine);
            heaviest = ~wave_lowest(~heaviest);
            if (threadIdx.x % kWave == 0) {
                if (mine != ~0u) atomicMin(&token_found, mine);
                atomicMax(&last_weight, heaviest);
            }
            __syncthreads();
            token = (int32_t)(token_found != ~0u ? token_found : last_weight);
        }
    }
    for (uint32_t i = threadIdx.x; i < q.rows; i += blockDim.x)
        a.tokens[q.first + i] = i < c.taken ? a.draft_tokens[q.first + i] : (i == c.taken ? token : -1);
}

}  // namespace smelt

#define SMELT_VERIFY_KERNELS(T, ACT)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void smelt_verify_stats_##T(smelt_serving::VerifyArgs a) { smelt::verify_stats<ACT>(a); }       \
    extern "C" __global__ __launch_bounds__(256) void smelt_verify_choose_##T(smelt_serving::VerifyArgs a) { smelt::verify_choose<ACT>(a); }     \
    extern "C" __global__ __launch_bounds__(256) void smelt_verify_leftover_##T(smelt_serving::VerifyArgs a) { smelt::verify_leftover<ACT>(a); } \
    extern "C" __global__ __launch_bounds__(1024) void smelt_verify_draw_##T(smelt_serving::VerifyArgs a) { smelt::verify_draw<ACT>(a); }
