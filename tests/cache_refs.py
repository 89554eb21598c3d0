"""Plain definitions of the paged cache's operators (numpy, 64 bits where they compute numbers), and their error bounds."""

import numpy as np
import torch

from request_refs import HALF_STEP_BF16, HALF_STEP_F32, f64

DEV = "cuda:0"


def ceil(a, b):
    return -(-a // b)


def tables(lengths, table, free, count, rows, total, page, base=None, keep=None, max_rows=None):
    """step_tables_ on lists and an int array, in place: (slots, positions, request, free count)."""
    base = list(lengths) if base is None else base
    capacity, back = table.shape[1], []
    for r, n in enumerate(lengths):
        b = max(0, min(base[r], n))
        for c in range(ceil(b, page), ceil(n, page)):
            back.append(int(table[r, c]))
            table[r, c] = -1
        lengths[r] = b
    free[count:count + len(back)] = back[::-1]
    count += len(back)
    out = [[-1] * total for _ in range(3)]
    row, short = 0, False
    for r, n in enumerate(rows):
        n = max(0, min(n, total if max_rows is None else max_rows, total - row))
        mine = [m for m in range(row, row + n) if keep is None or keep[m]]
        row += n
        have, want = ceil(lengths[r], page), ceil(lengths[r] + len(mine), page)
        if want > capacity:
            continue
        short = short or want - have > count
        if want > have and short:
            continue
        for c in range(have, want):
            count -= 1
            table[r, c] = free[count]
        for i, m in enumerate(mine):
            at = lengths[r] + i
            out[0][m], out[1][m], out[2][m] = int(table[r, at // page]) * page + at % page, at, r
        lengths[r] += len(mine)
    return *out, count


def codes(x):
    """(scale, exact code before rounding) of rows x [..., D]."""
    scale = (np.abs(x).max(-1) / 127).astype(np.float32)
    return scale, x / np.where(scale > 0, scale, 1).astype(np.float64)[..., None]


def token_rows(cache):
    """(K, V) of every slot, float64 [pages * page, Hk, D], of a cache's tensors."""
    keys, values = f64(cache.keys), f64(cache.values)
    pages, heads, _, page, e = keys.shape
    k = keys.transpose(0, 3, 1, 2, 4).reshape(pages * page, heads, -1)
    v = values.transpose(0, 2, 4, 1, 3).reshape(pages * page, heads, -1)
    if cache.key_scales is not None:
        k = k * f64(cache.key_scales).transpose(0, 2, 1).reshape(pages * page, heads, 1)
        v = v * f64(cache.value_scales).transpose(0, 2, 1).reshape(pages * page, heads, 1)
    return k, v


def attention(q, k, v, scale, sees):
    """(out, mag, delta): softmax attention of q [n, Hq, D] over k, v [L, Hk, D], sees [n, L]; the sum of the magnitudes of its
    terms, and how far fp32 may move a logit: (D + 4) half steps of its terms' magnitudes, and the exponential's own
    argument, at most 2^10 in powers of two, by two half steps."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, mag, delta = np.zeros((n, hq, d)), np.zeros((n, hq, d)), np.zeros((n, hq, 1))
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        for i in range(n):
            at = sees[i]
            if not at.any():
                continue
            s = scale * (kh[at] @ q[i, h])
            terms = abs(scale) * (np.abs(kh[at]) @ np.abs(q[i, h]))
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], mag[i, h] = w @ vh[at], w @ np.abs(vh[at])
            delta[i, h] = (d + 4) * HALF_STEP_F32 * terms.max() + 2 * HALF_STEP_F32 * min(np.ptp(s) * 1.5 + 16, 1024)
    return out, mag, delta


def attention_bound(out, mag, delta, length):
    """One rounding of each probability to bf16 and one of the result; in fp32 the sums over `length` tokens (numerator and
    denominator), a logit's error in both, and 16 half steps for exponentials, quotient and gate."""
    return (HALF_STEP_BF16 * 1.01 * np.abs(out)
            + mag * (HALF_STEP_BF16 * 1.01 + 2.1 * delta + (2 * length + 16) * HALF_STEP_F32) + 1e-37)


def visible(cached, n, ancestors=None):
    sees = np.ones((n, cached + n), bool)
    for i in range(n):
        for j in range(n):
            sees[i, cached + j] = j <= i if ancestors is None else j < 64 and bool(int(ancestors[i]) >> j & 1)
    return sees


def tree_masks(rng, n):
    """A random tree's masks, as int64."""
    masks = []
    for i in range(n):
        masks.append((masks[rng.randrange(i)] if i else 0) | 1 << i)
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)
