"""64-bit restatement of the sequence operators (sed_amd/sequence.py) from their definitions, with their gradients written out,
and the magnitudes that bound what fp32 arithmetic may lose.  numpy only, one frame after another.

A `walk` function runs one clip in the order of the walk.  Called with absolute values it gives, per output, the sum of the
absolute values of the terms (the scale of the rounding errors); with the decay replaced by one as well, the sum of the terms as
they are before they decay (the scale of the errors in the exponents: S e^-S <= 1/e for a term decayed by e^-S)."""
import numpy as np


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def softplus(v):
    return np.logaddexp(v, 0.0)


def order(n, own, reverse):
    """Rows of a clip in the order of the walk, its own ones only."""
    return np.arange(own)[::-1] if reverse else np.arange(own)


# ---- gated linear recurrence --------------------------------------------------------------------------------------------


def scan_walk(x, delta, decay, A, B, C, skip, h0, gy, glast):
    """One clip: x, delta, gy (n, D), decay (n, D, N) = exp(delta A), B, C (n, D, N).  Returns pre (n, D), the state behind the
    last row, and the gradients by gy (of pre) and glast (of that state)."""
    n, d = x.shape
    h, hs, pre = h0.copy(), [h0.copy()], np.zeros((n, d))
    for t in range(n):
        h = decay[t] * h + (delta[t] * x[t])[:, None] * B[t]
        hs.append(h.copy())
        pre[t] = (h * C[t]).sum(1) + skip * x[t]
    g = glast.copy()
    out = {k: np.zeros_like(x) for k in ("x", "delta")} | {k: np.zeros_like(B) for k in ("B", "C")} | {"A": np.zeros_like(A)}
    for t in range(n - 1, -1, -1):
        g = g + gy[t][:, None] * C[t]
        toB = (g * B[t]).sum(1)
        through = g * decay[t] * hs[t]
        out["C"][t] = gy[t][:, None] * hs[t + 1]
        out["B"][t] = g * (delta[t] * x[t])[:, None]
        out["x"][t] = toB * delta[t] + skip * gy[t]
        out["delta"][t] = toB * x[t] + (through * A).sum(1)
        out["A"] += through * delta[t][:, None]
        g = g * decay[t]
    out["D"] = (gy * x).sum(0)
    out["state"] = g
    return pre, h, out


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, use_softplus=False, frames=None, reverse=False, state=None, dy=None, dlast=None):
    """All outputs and, per output, the two magnitudes: {name: (value, terms, undecayed terms)}, names y, last and d<input>."""
    nb, n, d = x.shape
    ns, g = A.shape[1], B.shape[2]
    group = np.arange(d) // (d // g)
    dy = np.zeros_like(x) if dy is None else dy
    shapes = {"y": x.shape, "last": (nb, d, ns), "dx": x.shape, "ddt": x.shape, "dA": A.shape, "dB": B.shape, "dC": B.shape, "dD": (d,),
              "dz": x.shape, "dbias": (d,), "dstate": (nb, d, ns)}
    out = {k: tuple(np.zeros(s) for _ in range(3)) for k, s in shapes.items()}
    skip = np.zeros(d) if D is None else D
    for b in range(nb):
        rows = order(n, n if frames is None else int(np.clip(frames[b], 0, n)), reverse)
        raw = dt[b, rows] + (0.0 if dt_bias is None else dt_bias)
        delta = softplus(raw) if use_softplus else raw
        slope = sigmoid(raw) if use_softplus else np.ones_like(raw)
        xb, Bb, Cb, gyb = x[b, rows], B[b, rows][:, group], C[b, rows][:, group], dy[b, rows]
        zb = None if z is None else z[b, rows]
        gate = np.ones_like(xb) if z is None else zb * sigmoid(zb)
        h0 = np.zeros((d, ns)) if state is None else state[b]
        gl = np.zeros((d, ns)) if dlast is None else dlast[b]
        decay = np.exp(delta[:, :, None] * A)
        for level in range(3):
            f = (lambda v: v) if level == 0 else np.abs
            dec = decay if level < 2 else np.ones_like(decay)
            pre, last, gr = scan_walk(f(xb), f(delta), dec, f(A), f(Bb), f(Cb), f(skip), f(h0), f(gyb * gate), f(gl))
            out["y"][level][b, rows] = pre * f(gate)
            out["last"][level][b] = last
            out["dx"][level][b, rows] = gr["x"]
            out["ddt"][level][b, rows] = gr["delta"] * slope
            out["dA"][level][...] += gr["A"]
            for k in ("B", "C"):
                for q in range(g):
                    out["d" + k][level][b, rows, q] = gr[k][:, group == q].sum(1)
            out["dD"][level][...] += gr["D"]
            out["dbias"][level][...] += (gr["delta"] * slope).sum(0)
            out["dstate"][level][b] = gr["state"]
            if z is not None:
                s = sigmoid(zb)
                # the slope's terms, not their sum, set the rounding: it has a zero at z = -1.278, where 1 + z (1 - s) cancels
                # (s, 1 - s and the fused step are each rounded, so it is off by u (1 + 3 |z| (1 - s)) there)
                out["dz"][level][b, rows] = f(gyb) * pre * s * (1 + f(zb) * (1 - s))
    return out


# ---- causal convolution -------------------------------------------------------------------------------------------------


def conv(x, weight, bias=None, silu=False, frames=None, reverse=False, state=None, dy=None, dlast=None):
    """{name: (value, terms)}: y, last, dx, dw, db, dstate."""
    nb, n, d = x.shape
    W = weight.shape[1]
    dy = np.zeros_like(x) if dy is None else dy
    shapes = {"y": x.shape, "last": (nb, W - 1, d), "dx": x.shape, "dw": weight.shape, "db": (d,), "dstate": (nb, W - 1, d)}
    out = {k: tuple(np.zeros(s) for _ in range(2)) for k, s in shapes.items()}
    b0 = np.zeros(d) if bias is None else bias
    for b in range(nb):
        rows = order(n, n if frames is None else int(np.clip(frames[b], 0, n)), reverse)
        own = len(rows)
        ext = np.concatenate([np.zeros((W - 1, d)) if state is None else state[b], x[b, rows]])
        u = b0 + sum(weight[:, k] * ext[k:k + own] for k in range(W))
        size = np.abs(b0) + sum(np.abs(weight[:, k] * ext[k:k + own]) for k in range(W))
        s = sigmoid(u)
        du = dy[b, rows] * (s * (1 + u * (1 - s)) if silu else 1.0)
        # |act''| <= 1/2 for silu: an error in u moves the slope by half of it at most
        dsize = np.abs(dy[b, rows]) * ((1.1 + 0.5 * size) if silu else 1.0)
        out["y"][0][b, rows] = u * s if silu else u
        out["y"][1][b, rows] = 1.1 * size if silu else size
        back = np.zeros((own + W - 1, d)), np.zeros((own + W - 1, d))
        for k in range(W):
            for level, (e, w, v) in enumerate(((ext, weight, du), (np.abs(ext), np.abs(weight), dsize))):
                back[level][k:k + own] += w[:, k] * v
                out["dw"][level][:, k] += (v * e[k:k + own]).sum(0)
        out["db"][0][...] += du.sum(0)
        out["db"][1][...] += dsize.sum(0)
        out["last"][0][b] = ext[own:]
        for level, f in enumerate((lambda v: v, np.abs)):
            if dlast is not None:
                back[level][own:] += f(dlast[b])
            out["dx"][level][b, rows] = back[level][W - 1:]
            out["dstate"][level][b] = back[level][:W - 1]
    return out


# ---- group norm ---------------------------------------------------------------------------------------------------------


def _erf(v):
    from scipy.special import erf
    return erf(v)


def activation(u, name):
    """(act(u), act'(u)).  |act'| <= 1.13 and |act''| <= 0.8 for all of them (relu: away from 0)."""
    if name == "silu":
        s = sigmoid(u)
        return u * s, s * (1 + u * (1 - s))
    if name == "relu":
        return np.maximum(u, 0), (u > 0).astype(float)
    if name == "gelu":
        cdf = 0.5 * (1 + _erf(u / np.sqrt(2)))
        return u * cdf, cdf + u * np.exp(-u * u / 2) / np.sqrt(2 * np.pi)
    return u, np.ones_like(u)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, act=None, frames=None, dy=None, adds=100, u32=2.0 ** -24):
    """{name: (value, error bound of fp32 arithmetic)}: y, dx, dw, db; and the smallest |u| over its error, for relu.

    x (B, T, F, C).  adds: additions in a row that form a sum in the code under test.  With m the mean, R the largest distance
    from it and s the spread: the mean is off by adds * u (|m| + R) at most, the variance by 2 adds * u, so the normalised value
    n by En = u (adds (|m| + R) / s + 2 |x| / s + (adds + 4) |n|)."""
    nb, T, F, c = x.shape
    cg = c // groups
    w, b0 = (np.ones(c) if weight is None else weight), (np.zeros(c) if bias is None else bias)
    dy = np.zeros_like(x) if dy is None else dy
    shapes = {"y": x.shape, "dx": x.shape, "dw": (c,), "db": (c,)}
    out = {k: (np.zeros(s), np.zeros(s)) for k, s in shapes.items()}
    clear = np.inf
    for b in range(nb):
        own = T if frames is None else int(np.clip(frames[b], 0, T))
        if own == 0:
            continue
        for g in range(groups):
            ch = slice(g * cg, (g + 1) * cg)
            v, gy = x[b, :own, :, ch], dy[b, :own, :, ch]
            m = v.mean()
            s = np.sqrt(((v - m) ** 2).mean() + eps)
            n = (v - m) / s
            En = u32 * (adds * (abs(m) + np.abs(v - m).max()) / s + 2 * np.abs(v) / s + (adds + 4) * np.abs(n))
            u = n * w[ch] + b0[ch]
            Eu = np.abs(w[ch]) * En + 2 * u32 * (np.abs(n * w[ch]) + np.abs(b0[ch]))
            clear = min(clear, float((np.abs(u) / np.maximum(Eu, 1e-300)).min()))
            f, d = activation(u, act)
            Ed = 0.8 * Eu * (act in ("silu", "gelu")) + 16 * u32 * (1 + np.abs(u)) * (act in ("silu", "gelu"))
            out["y"][0][b, :own, :, ch] = f
            out["y"][1][b, :own, :, ch] = 1.13 * Eu + 16 * u32 * np.abs(f) * (1 + np.abs(u))
            du, Edu = gy * d, np.abs(gy) * (Ed + 2 * u32 * np.abs(d))
            out["db"][0][ch] += du.sum((0, 1))
            out["dw"][0][ch] += (du * n).sum((0, 1))
            out["db"][1][ch] += (Edu + (adds + nb) * u32 * np.abs(du)).sum((0, 1))
            out["dw"][1][ch] += (Edu * np.abs(n) + np.abs(du) * En + (adds + nb) * u32 * np.abs(du * n)).sum((0, 1))
            q, Eq = du * w[ch], np.abs(w[ch]) * (Edu + 2 * u32 * np.abs(du))
            m1, m2 = q.mean(), (q * n).mean()
            E1 = (Eq + adds * u32 * np.abs(q)).mean()
            E2 = (Eq * np.abs(n) + np.abs(q) * En + adds * u32 * np.abs(q * n)).mean()
            out["dx"][0][b, :own, :, ch] = (q - m1 - n * m2) / s
            out["dx"][1][b, :own, :, ch] = (Eq + E1 + np.abs(n) * E2 + En * abs(m2) + (adds + 6) * u32 * (np.abs(q) + abs(m1) + np.abs(n * m2))) / s
    return out, clear
