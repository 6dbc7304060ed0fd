"""Plain 64-bit forms of a step's operators, and the error bounds their tests use."""
import math

import numpy as np


def quantize(x):
    """f16 [n, width] -> Q8_0 rows uint8 [n, width / 32 * 34] (d = amax / 127, code = round half
    away(x * (1 / d)) in f32, scale f16(d)) and the values code * f16(d) rounded to f16."""
    b = x.astype(np.float32).reshape(x.shape[0], -1, 32)
    d = np.abs(b).max(-1, keepdims=True) / np.float32(127)
    inv = np.where(d != 0, np.float32(1) / np.where(d != 0, d, np.float32(1)), np.float32(0)).astype(np.float32)
    y = b * inv
    t = np.trunc(y)
    code = np.clip(t + np.where(np.abs(y - t) >= 0.5, np.sign(y), 0), -128, 127)
    rows = np.concatenate([d.astype(np.float16).view(np.uint8), code.astype(np.int8).view(np.uint8)], -1)
    values = (code * d.astype(np.float16).astype(np.float32)).astype(np.float16)
    return rows.reshape(x.shape[0], -1), values.reshape(x.shape)


def dequantize(rows):
    """Values code * scale of Q8_0 rows, f64 [n, width]."""
    b = rows.reshape(rows.shape[0], -1, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    return (np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64) * d).reshape(rows.shape[0], -1)


def slots(table_row, page, first, end):
    p = np.arange(first, end)
    return np.asarray(table_row, np.int64)[p // page] * page + p % page


def attention(q, k, v, start, window):
    """q f16 [n, H, hd] at positions start .., k and v f64 [start + n, Hk, hd]: (out f64, bound).

    Bound of what a kernel with f32 sums and f16 operands may be off by. e = 2^-11 is half a
    step of f16. Rounding K by e moves a score by at most e s, s = sum |q k| / sqrt(hd); weights
    move by a factor exp(+-e s) above and below the line: 2 e s of A = sum w |v|. Rounding each
    weight by e counts above and below the line (the sum may be taken of rounded weights or
    not): 2 e A; V: e A; the result: e |out|; 2^-14 (s + 1) A for f32 sums, exp2 and 1 / sqrt(hd);
    weights below 2^-14 round by 2^-25 of the largest: 2^-25 sum |v|."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    out, bound = np.zeros((n, H, hd)), np.zeros((n, H, hd))
    e = 2.0 ** -11
    for t in range(n):
        P = start + t
        lo = max(0, P - window + 1) if window else 0
        for h in range(H):
            kk, vv = k[lo:P + 1, h // G], v[lo:P + 1, h // G]
            qq = q[t, h].astype(np.float64)
            x = kk @ qq / math.sqrt(hd)
            w = np.exp(x - x.max())
            w /= w.sum()
            out[t, h] = w @ vv
            A = w @ np.abs(vv)
            s = (np.abs(kk) @ np.abs(qq)).max() / math.sqrt(hd)
            bound[t, h] = (A * (np.expm1(2 * e * s) + 3 * e + 2.0 ** -14 * (s + 1)) + e * np.abs(out[t, h])
                           + 2.0 ** -25 * np.abs(vv).sum(0) + 2.0 ** -24)
    return out, bound


def verify(logits, tokens, probs, u, n_new, temperature):
    """(accepted [seqs], answer [rows]) by the definition, in f64."""
    accepted, answer, off = [], [], 0
    V = logits.shape[1]
    for s, n in enumerate(n_new):
        got = []
        for i in range(n):
            x = logits[off + i].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            if x.max() == -np.inf:
                got.append(-1)
                break
            d = int(tokens[off + i + 1]) if i < n - 1 else -1
            if temperature == 0:
                best = int(np.flatnonzero(x == x.max())[-1])
                got.append(best)
                if i < n - 1 and d == best:
                    continue
                break
            with np.errstate(invalid="ignore"):
                p = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / float(np.float32(temperature))))
            p /= p.sum()
            if i < n - 1:
                ui = float(u[off + i])
                ui = ui if ui >= 0 else 0.0
                q = None
                if probs is not None:
                    q = probs[off - s + i].astype(np.float64)
                    q = np.where(q > 0, q, 0.0)
                qd = 1.0 if q is None else (q[d] if 0 <= d < V else 0.0)
                if 0 <= d < V and ui * qd < p[d]:
                    got.append(d)
                    continue
                rest = p.copy()
                if q is not None:
                    rest = np.maximum(p - q, 0)
                elif 0 <= d < V:
                    rest[d] = 0
                p = rest if rest.sum() > 0 else p
            ui = float(u[off + n - 1])  # not the refused draft's, which is known to be great
            ui = ui if ui >= 0 else 0.0
            c = np.cumsum(p)
            over = np.flatnonzero(c > ui * c[-1])
            got.append(int(over[0]) if over.size else int(np.flatnonzero(p > 0)[-1]))
            break
        # the last entry is the token chosen behind the accepted drafts
        accepted.append(len(got) - 1)
        answer += got + [-1] * (n - len(got))
        off += n
    return np.array(accepted, np.int32), np.array(answer, np.int32)
