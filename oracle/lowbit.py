"""Plain float64 forms of the 8-bit block-scaled product and of distillation from a teacher's top logits (NumPy).  The
reference has neither: the definitions are those documented in include/ocrhip.h, written row by row."""
import numpy as np

E4M3_MAX = 448.0
BLOCK = 128


def e4m3_table():
    """float64 value of every e4m3 byte (bias 7, three mantissa bits, no infinities, 0x7F / 0xFF NaN)."""
    out = np.empty(256)
    for b in range(256):
        s, e, m = b >> 7, b >> 3 & 15, b & 7
        if e == 15 and m == 7:
            v = np.nan
        elif e == 0:
            v = m * 2.0 ** -9
        else:
            v = (8 + m) * 2.0 ** (e - 10)
        out[b] = -v if s else v
    return out


def round_e4m3(x):
    """Nearest e4m3 value of float64 |x| <= 448, halves to the even mantissa; infinities and NaN -> NaN."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid='ignore'):
        _, e = np.frexp(x)
        step = np.exp2(np.maximum(e - 4, -9).astype(np.float64))
        r = np.rint(x / step) * step
    return np.where(np.isfinite(x), r, np.nan)


def scale_exponent(amax):
    """Least integer e >= -127 with amax <= 448 * 2^e; 0 for amax 0."""
    if amax == 0:
        return 0
    e = int(np.ceil(np.log2(amax / E4M3_MAX)))
    while amax > E4M3_MAX * 2.0 ** e:
        e += 1
    while amax <= E4M3_MAX * 2.0 ** (e - 1):
        e -= 1
    return max(e, -127)


def quantize(x, block_rows):
    """(rows, cols) -> (e4m3 values (rows, cols), exponents (row blocks, column blocks))."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    q, e = np.zeros_like(x), np.zeros((rb, cb), dtype=np.int64)
    for i in range(rb):
        for j in range(cb):
            at = np.s_[i * block_rows:(i + 1) * block_rows, j * BLOCK:(j + 1) * BLOCK]
            b = x[at]
            fin = np.abs(b[np.isfinite(b)])
            e[i, j] = scale_exponent(fin.max() if fin.size else 0.0)
            q[at] = round_e4m3(b * 2.0 ** float(-e[i, j]))
    return q, e


def dequantize(q, e, block_rows):
    rows, cols = q.shape
    return q * np.exp2(e[np.arange(rows)[:, None] // block_rows, np.arange(cols)[None, :] // BLOCK].astype(np.float64))


def top_logits(x, k, temperature):
    """-> values, index (rows, k), lse (rows): descending, the lower class first among equals, NaN above every number."""
    x = np.asarray(x, dtype=np.float64)
    rank = np.where(np.isnan(x), 2.0, np.where(x == np.inf, 1.0, 0.0))
    plain = np.where(np.isfinite(x) | (x == -np.inf), x, 0.0)
    index = np.stack([np.lexsort((np.arange(x.shape[1]), -plain[r], -rank[r]))[:k] for r in range(x.shape[0])])
    with np.errstate(invalid='ignore', divide='ignore', over='ignore'):
        m = x.max(axis=1, keepdims=True)
        base = np.where(np.isfinite(m), m, 0.0)
        lse = np.log(np.exp((x - base) / temperature).sum(axis=1)) + base[:, 0] / temperature
    return np.take_along_axis(x, index, 1), index, lse


def distill_row(s, z, idx, lse, t, w):
    """One row: -> (loss, gradient (V,)).  lse None: renormalised over the entries."""
    V = len(s)
    if w == 0:
        return 0.0, np.zeros(V)
    with np.errstate(all='ignore'):
        m = s.max() if not np.isnan(s).any() else np.nan
        e = np.exp((s - m) / t)
        log_q = (s - m) / t - np.log(e.sum())
        q = np.exp(log_q)
        there = [(int(i), float(v)) for i, v in zip(idx, z) if 0 <= i < V and v != -np.inf]
        target = np.zeros(V)
        loss = 0.0
        if lse is None:
            if not there:
                return 0.0, np.zeros(V)
            zt = np.array([v for _, v in there]) / t
            log_p = zt - zt.max() - np.log(np.exp(zt - zt.max()).sum())
        else:
            log_p = np.array([v for _, v in there]) / t - lse
        inside = np.zeros(V, dtype=bool)
        inside[[int(i) for i in idx if 0 <= i < V]] = True
        for (i, _), lp in zip(there, log_p):
            target[i] += np.exp(lp)
        for i in dict.fromkeys(i for i, _ in there):           # entries of one class add up before the logarithm
            own = [lp for (j, _), lp in zip(there, log_p) if j == i]
            if target[i] != 0:
                loss += target[i] * ((own[0] if len(own) == 1 else np.log(target[i])) - log_q[i])
        grad = q - target
        if lse is not None:
            mass = np.exp(log_p).sum()
            rest = max(0.0, 1.0 - mass) if not inside.all() else 0.0
            q = (mass + rest) * q                     # the loss carries (mass + rest) times the log of the student's sum
            grad = q - target
            if not inside.all():
                out = np.where(inside, -np.inf, log_q)
                top = out.max()
                share = np.exp(out - top) / np.exp(out - top).sum()
                log_rest = np.log(np.exp(out - top).sum()) + top if top > -np.inf else top
                if rest > 0:
                    loss += rest * (np.log(rest) - log_rest)
                if log_rest > -np.inf:
                    grad = np.where(inside, grad, q - rest * share)
        return w * t * t * loss, np.where(np.isnan(loss), np.nan, w * t * grad)


def distill(s, z, idx, lse, t, w):
    s, z = np.asarray(s, dtype=np.float64), np.asarray(z, dtype=np.float64)
    out = [distill_row(s[r], z[r], idx[r], None if lse is None else float(lse[r]), t, 1.0 if w is None else float(w[r]))
           for r in range(s.shape[0])]
    return np.array([o[0] for o in out]), np.stack([o[1] for o in out])
