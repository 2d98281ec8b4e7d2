"""Plain 64-bit definitions of the serving operators, and helpers that lay their operands out in slots."""
from __future__ import annotations

import numpy as np

import fixtures as fx

EPS = {fx.F16: 2.0 ** -10, fx.BF16: 2.0 ** -7}          # a rounding is off by half of this, relative
TINY = {fx.F16: 2.0 ** -25, fx.BF16: 2.0 ** -134}       # ... or by half of the smallest subnormal


def values(rng, shape, dtype, scale=1.0):
    """(bits, float64 values) of normal data in the 16-bit type."""
    b = fx.to_bits(rng.normal(0, scale, shape).astype(np.float32), dtype)
    return b, fx.from_bits(b, dtype).astype(np.float64)


def wide(bits, dtype):
    return fx.from_bits(bits, dtype).astype(np.float64)


# ---- rotary positions ----------------------------------------------------------------------------------------------------
def rope(x, positions, table, amplitude, rot, interleaved):
    """x [tokens, heads, dim] float64 -> (rotated, bound on the arithmetic before rounding)."""
    y, reach = x.copy(), np.zeros_like(x)
    half = rot // 2
    i = 2 * np.arange(half) if interleaved else np.arange(half)
    j = i + 1 if interleaved else i + half
    angle = positions.astype(np.float64)[:, None] * table[None, :half]
    c, s = amplitude * np.cos(angle)[:, None], amplitude * np.sin(angle)[:, None]
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    reach[..., i] = reach[..., j] = abs(amplitude) * (np.abs(x[..., i]) + np.abs(x[..., j]))
    return y, reach


def check_rope(got_bits, want, reach, dtype, what):
    """Half a step of the type, and 2^-20 of what went in: the turn's fraction in 32 bits (2^-25 turns are 2^-22 radians), cos and
    sin to 2 ulp, three products and a sum."""
    tol = EPS[dtype] / 2 * np.abs(want) + reach * 2.0 ** -20 + TINY[dtype]
    off = np.abs(wide(got_bits, dtype).reshape(want.shape) - want)
    assert np.all(off <= tol), f"{what}: {(off / tol).max():.3f} of the tolerance at {np.unravel_index((off / tol).argmax(), off.shape)}"


# ---- paged cache ---------------------------------------------------------------------------------------------------------
def keys_to_pages(k, page):
    """[pages, kv_heads, page, dim] -> the cache's [pages, kv_heads, dim / 8, page, 8]."""
    p, h, n, d = k.shape
    return np.ascontiguousarray(k.reshape(p, h, n, d // 8, 8).transpose(0, 1, 3, 2, 4))


def keys_from_pages(k):
    p, h, c, n, e = k.shape
    return k.transpose(0, 1, 3, 2, 4).reshape(p, h, n, c * e)


# ---- attention -----------------------------------------------------------------------------------------------------------
def attention(q, k, v, pages, table, lens, offsets, scale, window, prefix_pages, prefix_len):
    """q [tokens, heads, dim], k / v [pages, kv_heads, page, dim] float64.  Returns (y, mean |v| under the weights, largest sum of
    |q k| scale) with y NaN where no sequence owns the row."""
    tokens, heads, dim = q.shape
    kv_heads, page = k.shape[1], k.shape[2]
    group = heads // kv_heads
    y = np.full(q.shape, np.nan)
    reach = np.zeros(q.shape)
    sharp = np.zeros((tokens, heads))
    count = np.zeros(tokens, int)
    for s in range(len(lens)):
        lo, hi = offsets[s], offsets[s + 1]
        n, own = hi - lo, lens[s]
        ids = [prefix_pages[j // page] for j in range(prefix_len)] + [table[s][j // page] for j in range(own)]
        offs = [j % page for j in range(prefix_len)] + [j % page for j in range(own)]
        ids, offs = np.array(ids, int), np.array(offs, int)
        known = (ids >= 0) & (ids < pages)
        safe = np.where(known, ids, 0)
        for i in range(n):
            p = prefix_len + own - n + i
            j = np.arange(len(ids))
            seen = known & (j <= p)
            if window:
                seen &= j > p - window
            count[lo + i] = seen.sum()
            for h in range(heads):
                kk, vv = k[safe[seen], h // group, offs[seen]], v[safe[seen], h // group, offs[seen]]
                if not len(kk):
                    y[lo + i, h] = 0.0
                    continue
                t = kk @ q[lo + i, h] * scale
                with np.errstate(all="ignore"):
                    top = t.max()
                    w = np.exp(t - (0.0 if np.isneginf(top) else top))
                total = w.sum()
                if total == 0.0:
                    y[lo + i, h] = 0.0
                    continue
                y[lo + i, h] = (w @ vv) / total
                reach[lo + i, h] = (w @ np.abs(vv)) / total
                sharp[lo + i, h] = abs(scale) * (np.abs(kk) @ np.abs(q[lo + i, h])).max()
    return y, reach, sharp, count


def attention_tolerance(y, reach, sharp, count, dim, dtype):
    """Probabilities rounded to the type (half a step), the result rounded once more, 32-bit dot products of `dim` terms (both
    roundings of a product and sum: (2 dim + 8) 2^-24 of the sum of magnitudes, in p twice: numerator and sum), 32-bit sums over the keys."""
    shift = (2 * dim + 8) * 2.0 ** -24 * np.maximum(sharp, 1.0)[..., None]
    return (EPS[dtype] / 2 + 2 * shift + (2 * count[:, None, None] + 64) * 2.0 ** -24) * reach + EPS[dtype] / 2 * np.abs(y) + TINY[dtype]


# ---- draft verification --------------------------------------------------------------------------------------------------
def _softmax(x, t):
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.float64(3.3895314e38)))
    top = x.max()
    if np.isneginf(top):
        return np.zeros_like(x)
    with np.errstate(all="ignore"):
        w = np.where(np.isneginf(x), 0.0, np.exp((x - top) / t))
    return w / w.sum()


def verify(target, draft, draft_tokens, offsets, u_accept, u_sample, temperature, tokens):
    """Float64 logits; returns (tokens, counts)."""
    tokens, counts = tokens.copy(), []
    vocab = target.shape[1]
    for s in range(len(offsets) - 1):
        lo, n, taken = offsets[s], offsets[s + 1] - offsets[s], 0
        for i in range(n):
            r, x = lo + i, int(draft_tokens[lo + i])
            last = i == n - 1
            t = float(temperature[s])
            if not t > 0:
                row = np.where(np.isnan(target[r]), -np.inf, target[r])
                best = -1 if np.isneginf(row.max()) else int(row.argmax())
                ok, choice = best >= 0 and x == best, best
            else:
                p = _softmax(target[r], t)
                if draft is not None:
                    q = _softmax(draft[r], t)
                else:
                    q = np.zeros(vocab)
                    if 0 <= x < vocab:
                        q[x] = 1.0
                ok = 0 <= x < vocab and float(u_accept[r]) * q[x] < p[x]
                w = p if last else np.maximum(p - q, 0.0)
                if w.sum() == 0:
                    w = p
                run = np.cumsum(w)
                over = np.flatnonzero(run > float(u_sample[s]) * run[-1])
                nz = np.flatnonzero(w)
                choice = int(over[0]) if len(over) else (int(nz[-1]) if len(nz) else -1)
            if ok and not last:
                tokens[r] = x
                taken += 1
                continue
            tokens[r] = choice
            tokens[r + 1:lo + n] = -1
            break
        counts.append(taken)
    return tokens, np.array(counts, np.int32)
