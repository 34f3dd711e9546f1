"""Plain 64-bit forms of the 8-bit cache operators (numpy), for the tests."""
import numpy as np

PAGE = 128


def stored(x):
    """What a cache row (last axis) holds: (values f32, scales f32).  The
    integer nearest to 127 x / max|x| (np.rint: ties to even) times the f32
    scale; rows with a NaN or an infinity are NaN."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        a = np.max(np.abs(x), axis=-1, keepdims=True)
        scale = (a * (np.float32(1.0) / np.float32(127.0))).astype(np.float32)
        den = np.where(a > 0, a, 1).astype(np.float64)
        q = np.rint(127.0 * x.astype(np.float64) / den)
        q = np.where(np.isfinite(a), q, 0.0)
        return (q.astype(np.float32) * scale).astype(np.float32), scale[..., 0]


def attention(q, counts, prefix_k, prefix_v, seq_k, seq_v, scale):
    """q [rows, H, d]; prefix_k/v [P, KVH, d]; seq_k/v: per sequence [len,
    KVH, d] (values as stored).  Returns (out, tol): tol bounds the kernel's
    rounding, derived below.

    Errors the kernel may make, eps = 2^-24:
      scores: q as integers of max|q| / 8.3e6 (half a unit each: 2^-23.98 of
        the row's maximum) against |k| <= kmax over d elements, and at most 8
        f32 roundings of the score itself;
      probabilities: exp2 within 2^-22, so relative error e = ln2 * (score
        error in log2 units) + 2^-22 each, on numerator and denominator;
      probability times value scale as integers of 2^-22 times the tile's
        largest value scale or less: at most half a unit per token, times 127:
        n * 2^-23 * vmax, divided by the denominator l >= 1;
      folding tiles and merging parts: f32 sums of at most n / 128 + 64 terms."""
    eps = 2.0 ** -24
    rows, H, d = q.shape
    out = np.zeros((rows, H, d))
    tol = np.zeros((rows, H, 1))
    KVH = prefix_k.shape[1] if prefix_k is not None else seq_k[0].shape[1]
    r = 0
    for i, c in enumerate(counts):
        for t in range(c):
            own = max(0, seq_k[i].shape[0] - c + t + 1)
            for h in range(H):
                g = h * KVH // H
                parts_k, parts_v = [], []
                if prefix_k is not None:
                    parts_k.append(prefix_k[:, g])
                    parts_v.append(prefix_v[:, g])
                parts_k.append(seq_k[i][:own, g])
                parts_v.append(seq_v[i][:own, g])
                k = np.concatenate(parts_k).astype(np.float64)
                v = np.concatenate(parts_v).astype(np.float64)
                n = k.shape[0]
                if n == 0:
                    continue
                qi = q[r, h].astype(np.float64)
                s = (k @ qi) * scale
                e = np.exp(s - s.max())
                l = e.sum()
                out[r, h] = (e / l) @ v
                kmax, vmax, qmax = np.abs(k).max(), np.abs(v).max(), np.abs(qi).max()
                ds = abs(scale) * d * qmax * kmax * eps * 1.02 + 8 * eps * np.abs(s).max()
                rel = ds + 2.0 ** -22
                tol[r, h] = vmax * (2 * rel + n * 2.0 ** -23 / l + (n / 128 + 64) * eps) + 1e-37
            r += 1
    return out, tol


def verify(p, q, drafts, n_draft, u):
    """Accepted tokens and the drawn one, per sequence (list of lists)."""
    res = []
    for i in range(p.shape[0]):
        toks, a = [], 0
        k = int(n_draft[i])
        while a < k:
            x = int(drafts[i, a])
            if x >= p.shape[2] or not float(u[i, a]) * float(q[i, a, x]) < float(p[i, a, x]):
                break
            toks.append(x)
            a += 1
        w = p[i, a].astype(np.float64)
        if a < k:
            with np.errstate(invalid="ignore"):
                d = p[i, a].astype(np.float64) - q[i, a].astype(np.float64)
            d = np.where(np.isfinite(d) & (d > 0), d, 0.0)
            if d.sum() > 0:
                w = d
        w = np.where(np.isfinite(w) & (w > 0), w, 0.0)
        if w.sum() > 0:
            c = np.cumsum(w)
            hit = np.flatnonzero((c > float(u[i, -1]) * c[-1]) & (w > 0))
            toks.append(int(hit[0]) if hit.size else int(np.flatnonzero(w)[-1]))
        res.append(toks)
    return res
