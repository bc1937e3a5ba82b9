"""The 8-bit cache's operators restated in 64 bits (numpy / torch on the CPU):
what tests/test_q8.py and tests/test_gpu_q8.py compare with."""
import numpy as np
import torch

BLOCK = 32


def scale_word(e, bad):
    return (0x7FC00000 | (e + 127)) if bad else (e + 127) << 23


def quantise_block(x):
    """(codes int8, scale word) of a block's values (float64, not finite allowed), any shape."""
    fin = np.isfinite(x)
    top = float(np.abs(x[fin]).max()) if fin.any() else 0.0
    e = -24
    while e < 9 and round(top / 2.0 ** e) > 127:   # (Python rounds halves to even)
        e += 1
    c = np.clip(np.rint(np.where(fin, x, 0.0) / 2.0 ** e), -127, 127)
    return np.where(fin, c, -128).astype(np.int8), scale_word(e, not fin.all())


def word_exp(w):
    w = np.asarray(w, np.uint32)
    nan = (w & 0x7F800000) == 0x7F800000
    return np.where(nan, w & 0xFF, w >> 23).astype(np.int64) - 127


def row_values(codes, words):
    """Each row's values at its block's exponent, -128 as NaN: codes [rows][D], words [rows / 32]."""
    e = np.repeat(word_exp(words), BLOCK)[:codes.shape[0]]
    return np.where(codes == -128, np.nan, codes.astype(np.float64) * 2.0 ** e[:, None])


def store(codes, words, row0, new):
    """codes int8 [H][rows][D], words uint32 [H][rows/32] in place; new float [n][H][D]."""
    with np.errstate(over="ignore"):
        new = new.astype(np.float16).astype(np.float64)
    end = row0 + new.shape[0]
    for h in range(codes.shape[0]):
        for b in range(row0 // BLOCK, -(-end // BLOCK)):
            lo, hi = b * BLOCK, min(end, (b + 1) * BLOCK)
            x = row_values(codes[h, lo:lo + BLOCK], words[h, b:b + 1])[:hi - lo]
            for i in range(max(lo, row0), hi):
                x[i - lo] = new[i - row0, h]
            codes[h, lo:hi], words[h, b] = quantise_block(x)


def evict(w, n, keep, recent):
    """The kept rows of one head: w float [rows]."""
    key = [(np.inf, 1) if np.isnan(x) else (float(x), 0) for x in w[:n - recent]]
    heavy = sorted(range(n - recent), key=lambda i: key[i], reverse=True)[:keep - recent]
    return sorted(heavy) + list(range(n - recent, n))


def attend(k, v, vs, q, n_past, mask=None, flash=False):
    """One head group in 64 bits.  k, v float64 [n_kv][D] (NaN rows allowed), vs [n_kv] V's scales, q float64 [T][r][D], mask float32
    [T][>= n_kv] or None.  Returns out [T][r][D], the rows' weights summed over tokens and heads [n_kv], and what the
    tolerances go by: sum p |v| [T][r][D], the error of a score [T][r] and max p vs [T][r]."""
    T, r, D = q.shape
    n_kv = k.shape[0]
    scale = float(np.float32(1.0) / np.sqrt(np.float32(D)))
    s = torch.einsum("trd,nd->trn", q, k) * scale
    if mask is None:
        hidden = torch.arange(n_kv)[None, :] > n_past + torch.arange(T)[:, None]
        t = s
    else:
        m = mask[:, :n_kv]
        hidden = m == float("-inf")
        t = (s.float() + m[:, None, :]).double()   # (the sum is one in 32 bits: a mask of the type's lowest value absorbs the score)
    hidden = hidden[:, None, :].expand(T, r, n_kv)
    t = torch.where(hidden, torch.full_like(t, float("-inf")), t)
    top = t.amax(-1, keepdim=True)
    top = torch.where(torch.isnan(t).any(-1, keepdim=True), torch.full_like(top, float("nan")), top)
    p = torch.where(hidden, torch.zeros_like(t), torch.exp(t - torch.where(top == float("-inf"), torch.zeros_like(top), top)))
    z = p.sum(-1, keepdim=True)
    empty = hidden.all(-1, keepdim=True)
    p = torch.where(empty, torch.zeros_like(p), p / z)
    # a hidden key's values do not enter, whatever they are
    vv = torch.nan_to_num(v, nan=0.0)
    out, mag = p @ vv, p @ vv.abs()
    seen_nan = ((~hidden) & torch.isnan(v).any(-1)[None, None, :]).any(-1, keepdim=True)
    out = torch.where(seen_nan.expand_as(out), torch.full_like(out, float("nan")), out)
    if not flash:
        out = torch.where(empty.expand_as(out), torch.full_like(out, float("nan")), out)
    fine = torch.isfinite(z) & ~empty   # (the values do not enter a softmax)
    weight = torch.where(fine, p, torch.zeros_like(p)).sum((0, 1))
    # a score: D products summed in 32 bits, and the sum with the mask rounded once more
    dot = torch.nan_to_num(torch.einsum("trd,nd->trn", q.abs(), torch.nan_to_num(k).abs()) * scale)
    big = torch.where(hidden | ~torch.isfinite(t), torch.zeros_like(t), t.abs()).clamp(max=1e6).amax(-1)
    err = (D + 4) * 2.0 ** -24 * torch.where(hidden, torch.zeros_like(dot), dot).amax(-1) + 2.0 ** -22 * big
    return out, weight, mag, err, (torch.nan_to_num(p) * vs).amax(-1)
