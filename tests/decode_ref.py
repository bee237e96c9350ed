"""Plain 64-bit implementations of the decode-step calls (rope, sdpa_prefix, logits_adjust), with the
error that the arithmetic they are computed in allows, and the calls themselves on device buffers."""
from __future__ import annotations

import numpy as np

import kurumi_amd as K
from hipmem import DevBuf, synchronize
from kurumi_amd import DType
from kutest import bf16_bits_to_f32, f32_to_bf16_bits

FLOATS = [DType.F32, DType.BF16, DType.F16]
# a rounding is off by at most half a step
HALF_STEP = {DType.F32: 2.0 ** -24, DType.BF16: 2.0 ** -8, DType.F16: 2.0 ** -11}
# below the smallest normal value the steps are of one size: f16 values under 2^-14 lie 2^-24 apart, so a
# rounding there is off by up to 2^-25 whatever the value (bf16 and f32 have theirs at 2^-134 and 2^-150)
LEAST = {DType.F32: 0.0, DType.BF16: 2.0 ** -134, DType.F16: 2.0 ** -25}
U = 2.0 ** -24  # of f32, which everything is computed in


def narrow(x: np.ndarray, dt: DType) -> np.ndarray:
    """Values in the storage of `dt`."""
    with np.errstate(over="ignore"):
        x = np.asarray(x, np.float32)
        return f32_to_bf16_bits(x) if dt == DType.BF16 else x.astype(np.float16).view(np.uint16) if dt == DType.F16 else x.copy()


def widen(bits: np.ndarray, dt: DType) -> np.ndarray:
    x = bf16_bits_to_f32(bits) if dt == DType.BF16 else bits.view(np.float16) if dt == DType.F16 else bits
    return x.astype(np.float64)


def rounding(want: np.ndarray, dt: DType) -> np.ndarray:
    """What rounding a value once to `dt` may be off by (0 for f32, whose rounding the formulas count)."""
    return 0.0 if dt == DType.F32 else np.maximum(HALF_STEP[dt] * np.abs(want), LEAST[dt])


def dev(a: np.ndarray | None) -> DevBuf | None:
    return None if a is None else DevBuf.from_numpy(a)


def ptr(b: DevBuf | None, elements: int = 0, dt: DType = DType.F32):
    return None if b is None else b.ptr + elements * dt.width


def assert_within(got: np.ndarray, want: np.ndarray, tol: np.ndarray, what: str) -> None:
    """Each element within its own tolerance; infinities and NaN in the same places."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} and {want.shape}"
    fine = np.isfinite(want)
    same = np.where(np.isnan(want), np.isnan(got), got == want)
    assert same[~fine].all(), f"{what}: {int((~same[~fine]).sum())} values that are not finite differ"
    tol = np.broadcast_to(tol, want.shape)
    with np.errstate(invalid="ignore"):
        off = np.where(fine, np.abs(got - want) - tol, -1.0)
    bad = ~(off <= 0)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off)), want.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} out of tolerance; worst at {i}: got {got[i]!r}, "
                             f"want {want[i]!r}, tolerance {tol[i]!r}")


# ---- rope ----


def rope(x, positions, freqs, rot, layout, scale=1.0, inverse=False):
    """[tokens, heads, d] in f64, and the error allowed before the output's own rounding.

    The fraction of a turn is rounded to f32 (2^-25 of a turn is 2^-22.3 of a radian), sine and cosine
    are good to 2 steps of f32 (2^-23 each), scaled (2^-24), and two products are added (2^-23 of their
    sizes): below 2^-20 of |x_lo| + |x_hi|. Positions of 2^20 and more lose 2^-53 of their turns in f64."""
    x = np.asarray(x, np.float64)
    a = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    c, s = scale * np.cos(a), scale * np.sin(a) * (-1 if inverse else 1)
    y, tol = x.copy(), np.zeros_like(x)
    lo, hi = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == K.ROPE_HALF else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    far = 8 * np.abs(a) * 2.0 ** -53
    tol[..., lo] = tol[..., hi] = (np.abs(x[..., lo]) + np.abs(x[..., hi])) * (2.0 ** -20 + far) * abs(scale)
    return y, tol


# ---- sdpa_prefix ----


def own_rows(b, n, seq_rows, pages, page):
    """Rows of a sequence's first n own keys; -1 where its page is none."""
    j = np.arange(n)
    if pages is None:
        return b * seq_rows + j
    p = pages[b][j // page].astype(np.int64)
    return np.where(p < 0, -1, p * page + j % page)


def sdpa_prefix(q, pk, pv, k, v, lens, scale, *, seq_rows=0, pages=None, page=0, npages=1 << 40, dt=DType.F32):
    """out, lse in f64 and their tolerances. q [b, t, h, d]; pk, pv [p, kv, d]; k, v [rows, kv, d].

    A score is a dot product of d terms in f32, then scaled: off by at most (d + 2) u sum |q k| scale,
    which moves a probability by as much of itself; exp2 and its argument's rounding, |score| log2 e u,
    add a few u. The sums over n keys round n times at most. The probabilities that meet 16-bit values
    round to half a step (f16 ones to 2^-25 of the largest at least), their sum does not. The output
    rounds once more."""
    nb, nt, nh, d = q.shape
    kv = pk.shape[1] if pk is not None else k.shape[1]
    g = nh // kv
    out, lse = np.zeros(q.shape), np.full(q.shape[:3], -np.inf)
    tol, ltol = np.zeros(q.shape), np.zeros(q.shape[:3])
    with np.errstate(all="ignore"):
        for b in range(nb):
            rows = own_rows(b, max(0, int(lens[b])) if lens is not None else 0, seq_rows, pages, page)
            for t in range(nt):
                r = rows[: max(0, len(rows) - (nt - 1 - t))]
                if pages is not None:
                    r = r[(r >= 0) & (r < npages * page)]
                keys = np.concatenate([x for x in (pk, k[r] if len(r) else None) if x is not None]) if pk is not None or len(r) else None
                vals = np.concatenate([x for x in (pv, v[r] if len(r) else None) if x is not None]) if pk is not None or len(r) else None
                if keys is None or not len(keys):
                    continue
                for h in range(nh):
                    s = keys[:, h // g] @ q[b, t, h] * scale
                    m = s.max()
                    p = np.exp(s - m)
                    vv = vals[:, h // g]
                    l = p.sum()
                    out[b, t, h] = p @ vv / l
                    lse[b, t, h] = np.nan if np.isnan(s).any() else m + np.log(l) if np.isfinite(m) else m
                    ds = ((d + 2) * U * scale * (np.abs(keys[:, h // g]) @ np.abs(q[b, t, h])) + 4 * U * (np.abs(s) + np.abs(m)) + 8 * U)
                    # a score of -inf weighs nothing, whatever its terms
                    rel = np.where(p > 0, ds + (len(keys) + 16) * U, 0.0)
                    half = HALF_STEP[dt] if dt != DType.F32 else 0.0
                    # numerator and denominator are off by the same kind of error
                    le = (p * rel).sum() / l
                    e = (p * (rel + half)) @ np.abs(vv) / l + le * np.abs(out[b, t, h])
                    if dt == DType.F16:
                        e = e + len(keys) * 2.0 ** -25 * np.abs(vv).max(0) / l
                    tol[b, t, h] = e + (rounding(out[b, t, h], dt) if dt != DType.F32 else U * np.abs(out[b, t, h]))
                    ltol[b, t, h] = le + 4 * U * (np.abs(lse[b, t, h]) + 1)
    return out, lse, np.nan_to_num(tol), np.nan_to_num(ltol)


# ---- logits_adjust ----


def logits_adjust(x, *, tokens=None, lens=None, prompts=None, rep=None, pres=None, freq=None, bias=None, mask=None, mask_index=None, out=DType.F32):
    """[rows, vocab] in f64 and the tolerance. bias: per row a list of (id, value); mask: boolean [mask rows, vocab].

    A division or product, a product and sum, a difference and each bias round once in f32, each by u of
    what it adds up to; then the output rounds."""
    rows, vocab = x.shape
    y, size = np.array(x, np.float64), np.abs(np.asarray(x, np.float64))
    for r in range(rows):
        if tokens is not None:
            n = tokens.shape[1] if lens is None else min(max(int(lens[r]), 0), tokens.shape[1])
            m = 0 if prompts is None else min(max(int(prompts[r]), 0), n)
            t = tokens[r].astype(np.int64)
            ok = (t >= 0) & (t < vocab)
            inside = np.arange(len(t)) < n
            seen = np.bincount(t[ok & inside], minlength=vocab) > 0
            made = np.bincount(t[ok & inside & (np.arange(len(t)) >= m)], minlength=vocab).astype(np.float64)
            if rep is not None:
                w = np.float64(rep[r])
                y[r] = np.where(seen, np.where(y[r] > 0, y[r] / w, y[r] * w), y[r])
            size[r] = np.abs(y[r])
            take = (0 if freq is None else np.float64(freq[r])) * made + (0 if pres is None else np.float64(pres[r])) * (made > 0)
            y[r], size[r] = np.where(made > 0, y[r] - take, y[r]), size[r] + np.abs(take)
        for i, w in (bias[r] if bias is not None else ()):
            if 0 <= i < vocab:
                y[r, i] += np.float64(w)
                size[r, i] += abs(float(w))
        if mask is not None:
            at = r if mask_index is None else int(mask_index[r])
            if 0 <= at < len(mask):
                y[r, ~mask[at]] = -np.inf
    n = 4 + (max((len(b) for b in bias), default=0) if bias is not None else 0)
    return y, n * U * size + rounding(np.where(np.isfinite(y), y, 0), out)


def packed(mask: np.ndarray) -> np.ndarray:
    """Boolean rows as 32-bit words, bit v % 32 of word v / 32; the bits past the vocabulary set."""
    rows, vocab = mask.shape
    words = -(-vocab // 32)
    bits = np.ones((rows, words * 32), np.uint8)
    bits[:, :vocab] = mask
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32)


def csr(bias):
    """Per-row lists of (id, value) as ids, values and offsets."""
    ids = np.array([i for b in bias for i, _ in b], np.int32)
    vals = np.array([w for b in bias for _, w in b], np.float32)
    return ids, vals, np.cumsum([0] + [len(b) for b in bias]).astype(np.int32)
