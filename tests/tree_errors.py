"""How far tree attention is off as a whole, next to the bounds of single values in drafts.py: the root of the mean square over a row's values, relative to the row's own, and what the documented roundings leave of it."""
import numpy as np


def seen_by(s, i, j, window, page):
    """Positions that row j of sequence i sees."""
    a, n = int(s["start"][i]), int(s["start"][i + 1] - s["start"][i])
    done = int(s["lens"][i]) - n
    least = int(s["pos"][a + j]) - window + 1 if window else -1
    sees = list(range(max(0, least), done)) + [done + x for x in range(n) if int(s["mask"][a + j]) >> x & 1 and s["pos"][a + x] >= least]
    return np.array(sees, np.int64)


def relative_rms(got, want):
    """Over the rows and heads whose values are not all zeros: each one's own, and of those again the root of the mean square."""
    off, size = np.sqrt(((got - want) ** 2).mean(-1)), np.sqrt((want ** 2).mean(-1))
    return float(np.sqrt(((off[size > 0] / size[size > 0]) ** 2).mean()))


def rms_tolerance(spread, hd, keys):
    """Roundings are off by half a step at most and either way, so n of them together by sqrt(n) half steps.  `spread`: the root of the sum of squares of a score's products, around which its partial sums lie and its value
    does too.  A score: its query's two binary16 parts (2^-22 of each product), 2 hd products added in f32, the factor and the product with it (4 roundings), all of which move its probability.  That is off by 2^-21 for the
    exponential and its argument, 2^-22 for its two parts; numerator and denominator add 2 `keys` terms; 16 joins and the division.  A value is a mean over keys whose errors are their own, so it moves by as much as one of
    them relative to its size.  All added up instead of their squares, and twice that."""
    score = spread * (2.0 ** -22 + ((2 * hd) ** 0.5 + 4) * 2.0 ** -24)
    return 2 * (score + 2.0 ** -21 + 2.0 ** -22 + 2 * (2 * keys) ** 0.5 * 2.0 ** -24 + 16 * 2.0 ** -24)


def emulate(s, kv, window, query_parts, probability_parts):
    """The kernels' arithmetic in numpy: parts of binary16, products added in f32."""
    q, page = s["q"], s["k"].shape[1]
    rows, H, hd = q.shape
    out = np.zeros((rows, H, hd), np.float32)

    def parts(x, n):
        got = []
        for _ in range(n):
            h = x.astype(np.float16)
            got.append(h.astype(np.float32))
            x = x - got[-1]
        return got
    for i in range(len(s["lens"])):
        for j in range(int(s["start"][i + 1] - s["start"][i])):
            sees, r = seen_by(s, i, j, window, page), int(s["start"][i]) + j
            if not sees.size:
                continue
            at = (s["table"][i, sees // page], sees % page)
            for h in range(H):
                k, v = (s[n][at][:, h // (H // kv)].astype(np.float32) for n in ("k", "v"))
                up = np.float32(2.0 ** (14 - np.floor(np.log2(np.abs(q[r, h]).max()))))
                x = sum(k @ p for p in parts(q[r, h] * up, query_parts)) * np.float32(1.44269504 / up)
                p = np.exp2(x - np.ceil(x.max()) + np.float32(8))
                out[r, h] = sum(y @ v for y in parts(p, probability_parts)) / p.sum(dtype=np.float32)
    return out
