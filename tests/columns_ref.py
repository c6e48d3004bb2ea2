"""The operators over a model's columns in 64 bits, for the tests, and the element types that numpy lacks.

Matrices are numpy arrays of shape (ncols, nrows): one row of the array per column of the matrix, so that its bytes are the
column-major ones. Types are 0 fp32, 1 fp16, 2 bf16, as in the header.
"""
import numpy as np

EPS24 = 2.0 ** -24
HALF_STEP = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}       # of a rounding, relative to the value
TINY = {0: 2.0 ** -149, 1: 2.0 ** -25, 2: 2.0 ** -133}         # of a rounding below the normal numbers, absolute
TYPES = (0, 1, 2)


def encode(x, t):
    """float array -> the array whose bytes the library takes (bf16: uint16, rounded to nearest even)."""
    if t == 0:
        return np.ascontiguousarray(x, dtype=np.float32)
    if t == 1:
        with np.errstate(over="ignore"):
            return np.ascontiguousarray(x).astype(np.float16)
    f = np.ascontiguousarray(x, dtype=np.float32)
    b = f.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7FC0), r)


def decode(a, t):
    """What the library's bytes stand for, in 64 bits."""
    if t == 2:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def np_type(t):
    return (np.float32, np.float16, np.uint16)[t]


def e4m3_table():
    v = np.empty(256)
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if e == 15 and m == 7:
            x = np.nan
        v[c] = -x if s else x
    return v


E4M3 = e4m3_table()


# ---------------------------------------------------------------- normalisation
def rmsnorm(x, r, w, eps, group=None):
    """h, y and, where group is given, scales (ncols, ngroups)."""
    h = x if r is None else x + r
    with np.errstate(all="ignore"):
        y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w
    if group is None:
        return h, y, None
    n = h.shape[1]
    g = group or n
    s = np.stack([np.abs(y[:, a:a + g]).max(1) for a in range(0, n, g)], 1) / 448.0
    return h, y, np.maximum(s, 2.0 ** -126)


def rmsnorm_grad(h, w, eps, dy, dh):
    """dx, dw and the sizes of what was added up in each (for error bounds)."""
    rs = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    g = dy * w
    dx = rs * (g - h * rs ** 2 * (g * h).mean(1, keepdims=True))
    size = rs * (np.abs(g) + np.abs(h) * rs ** 2 * np.abs(g * h).mean(1, keepdims=True))
    if dh is not None:
        dx, size = dx + dh, size + np.abs(dh)
    return dx, (dy * h * rs).sum(0), size, np.abs(dy * h * rs).sum(0)


# ---------------------------------------------------------------- routing
def _p(z, kind):
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == 1:
            return 1 / (1 + np.exp(-z))
        top = z.max()
        if top == -np.inf:
            return np.zeros_like(z)
        e = np.exp(z - top)
        return e / e.sum()


def route(Z, bias, kind, ngroups, topgroups, topk, renorm, scale):
    """ir (ncols, topk), weights, counts."""
    m, E = Z.shape
    size = E // ngroups
    irs, ws, counts = np.zeros((m, topk), np.int64), np.zeros((m, topk)), np.zeros(E, np.int64)
    for c in range(m):
        z = Z[c].astype(np.float64)
        if np.isnan(z).any() or (kind == 0 and (z == np.inf).any()):
            irs[c], ws[c] = np.arange(topk), np.nan
            continue
        p = _p(z, kind)
        key = z.copy() if bias is None and ngroups == 1 else p + (0 if bias is None else bias.astype(np.float64))
        open_ = (z > -np.inf) & (key > -np.inf)
        if ngroups > 1:
            total = []
            for g in range(ngroups):
                k = sorted((key[e] for e in range(g * size, (g + 1) * size) if open_[e]), reverse=True)[:2]
                total.append(sum(k) if k else -np.inf)
            best = sorted(range(ngroups), key=lambda g: (-total[g], g))[:topgroups]
            for e in range(E):
                open_[e] = open_[e] and e // size in best
        order = sorted((e for e in range(E) if open_[e]), key=lambda e: (-key[e], e))[:topk]
        counts[order] += 1
        rest = [e for e in range(E) if e not in order][: topk - len(order)]
        rows = sorted(order + rest)
        w = np.array([p[e] if e in order else 0.0 for e in rows])
        if renorm:
            w = w / w.sum() if w.sum() > 0 else w * 0
        irs[c], ws[c] = rows, scale * w
    return irs, ws, counts


def route_grad(Z, kind, renorm, scale, w, ir, dG):
    """dZ from the formula, entries of weight 0 not taken, and the size of what was added up."""
    m, E = Z.shape
    out, size = np.zeros((m, E)), np.zeros((m, E))
    for c in range(m):
        z = Z[c].astype(np.float64)
        p = _p(z, kind)
        t = ir[c][w[c] != 0]
        g = dG[c][w[c] != 0].astype(np.float64) * scale
        up, mag = np.zeros(E), np.zeros(E)
        if renorm:
            s = p[t].sum()
            if len(t) and s > 0:
                mean = (g * p[t]).sum() / s
                up[t] = (g - mean) / s
                mag[t] = (np.abs(g) + (np.abs(g) * p[t]).sum() / s) / s
        else:
            up[t], mag[t] = g, np.abs(g)
        if kind == 1:
            out[c], size[c] = up * p * (1 - p), mag * p * (1 - p)
        else:
            out[c], size[c] = p * (up - (up * p).sum()), p * (mag + (mag * p).sum())
            if renorm:                         # the parts of the other experts cancel
                keep = np.zeros(E, bool)
                keep[t] = True
                out[c][~keep] = 0
    return out, size


# ---------------------------------------------------------------- distillation
def distill(Z, T, ir, jc, tau, weight, lse=None):
    """loss, lse, dZ, and bounds on what 2^-24 relative errors of the parts can come to in loss and dZ."""
    m, V = Z.shape
    loss, dZ = np.zeros(m), np.zeros((m, V))
    out_lse, eloss, ez = np.zeros(m), np.zeros(m), np.zeros((m, V))
    for c in range(m):
        x = Z[c].astype(np.float64) / tau
        w = 1.0 if weight is None else float(weight[c])
        top = x.max()
        with np.errstate(all="ignore"):
            l = (top + np.log(np.exp(x - top).sum())) if lse is None else float(lse[c])
        out_lse[c] = l
        js = [j for j in range(jc[c], jc[c + 1]) if 0 <= ir[j] < V]
        t = T[js].astype(np.float64) / tau
        if w == 0 or not np.any(t > -np.inf):
            continue
        tt = t.max()
        p = np.exp(t - tt)
        s = p.sum()
        p, logp = p / s, t - tt - np.log(s)
        r = ir[js]
        on = p > 0
        with np.errstate(all="ignore"):
            loss[c] = w * tau * tau * (p[on] * (logp[on] - x[r[on]] + l)).sum()
            q = np.exp(x - l)
        share = np.zeros(V)
        np.add.at(share, r, p)
        dZ[c] = w * tau * (q - share)
        fin = np.where(np.isfinite(x), np.abs(x), 0)
        ptot = np.abs(t[np.isfinite(t)]).max() + abs(tt + np.log(s))
        depth = 160.0 + len(js)
        eloss[c] = abs(w) * tau * tau * EPS24 * (depth * (p[on] * (np.abs(logp[on]) + ptot + np.where(np.isfinite(x[r[on]]), np.abs(x[r[on]]), 0) + abs(l))).sum())
        ez[c] = abs(w) * tau * EPS24 * (q * (8 * (fin + abs(l)) + 160) + share * (8 * ptot + depth))
    return loss, out_lse, dZ, eloss, ez


def q8_product(Q, scales, group, S, ir, jc):
    """A*S and sum of |terms|; Q (ncolsA, k) codes, scales (ncolsA, ngroups)."""
    k = Q.shape[1]
    A = E4M3[Q] * np.repeat(scales.astype(np.float64), group or k, axis=1)[:, :k]
    m = len(jc) - 1
    out, mag = np.zeros((m, k)), np.zeros((m, k))
    for c in range(m):
        v = S[jc[c]:jc[c + 1]].astype(np.float64)[:, None]
        rows = A[ir[jc[c]:jc[c + 1]]]
        out[c], mag[c] = (v * rows).sum(0), np.abs(v * rows).sum(0)
    return out, mag
