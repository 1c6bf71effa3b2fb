"""Plain float64 definitions of rotary positions and scored attention (include/om.h), for the tests: one query and one
rule at a time, with gradients by the chain rule."""
import numpy as np


def rope_speeds(rot, scaling="plain", base=10000.0, factor=1.0, trained=0.0, low=0.0, high=1.0):
    """Radians per position of each pair."""
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2.0))
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "bands":
        keep = np.clip((f * trained / (2 * np.pi) - low) / (high - low), 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f


def rope(x, pos, rot, layout, speeds, amp=1.0, back=False):
    """x [rows, heads, d]; the turned values (or the gradient turned back) in float64."""
    x = np.asarray(x, np.float64)
    ang = np.asarray(pos, np.float64)[:, None, None] * speeds
    c, s = amp * np.cos(ang), amp * np.sin(ang) * (-1.0 if back else 1.0)
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def visible(lq, lk, causal=0, window=0, prefix=None, qdoc=None, kdoc=None, b=0):
    see = np.ones((lq, lk), bool)
    for t in range(lq):
        i = t + lk - lq
        for j in range(lk):
            reach = (not causal or j <= i) and (not window or abs(i - j) < window)
            if prefix is not None and j < prefix[b]:
                reach = True
            if qdoc is not None and not (qdoc[b][t] == kdoc[b][j] and kdoc[b][j] >= 0):
                reach = False
            see[t, j] = reach
    return see


def attention(q, k, v, g=None, scale=0.0, cap=0.0, slopes=None, **rule):
    """q, g [B, lq, H, d], k, v [B, lk, Hk, d]; (o, dq, dk, dv) in float64 (gradients only with g). Values that a query
    does not see are never touched."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, lq, H, d = q.shape
    lk, Hk = k.shape[1], k.shape[2]
    scale = 1.0 / np.sqrt(d) if scale == 0.0 else float(np.float32(scale))
    o = np.zeros_like(q)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    dist = np.abs(np.arange(lq)[:, None] + (lk - lq) - np.arange(lk)[None, :])
    with np.errstate(all="ignore"):
        for b in range(B):
            see = visible(lq, lk, b=b, **rule)
            for h in range(H):
                hk = h // (H // Hk)
                kk = np.where(see.any(0)[:, None], k[b, :, hk], 0.0)
                vv = np.where(see.any(0)[:, None], v[b, :, hk], 0.0)
                qq = np.where(see.any(1)[:, None], q[b, :, h], 0.0)
                plain = all(np.isfinite(a).all() for a in (qq, kk, vv))  # sums without the terms of unseen pairs
                x = (qq @ kk.T if plain else (qq[:, None, :] * kk[None, :, :]).sum(2)) * scale
                th = np.zeros_like(x)
                if cap:
                    th = np.tanh(x / np.float64(np.float32(cap)))
                    x = th * np.float64(np.float32(cap))
                if slopes is not None:
                    x = x - np.float64(slopes[h]) * dist
                x = np.where(see, x, -np.inf)
                m = x.max(1, keepdims=True) if lk else np.zeros((lq, 1))
                e = np.where(see, np.exp(x - np.where(m == -np.inf, 0.0, m)), 0.0)
                l = e.sum(1, keepdims=True)
                p = e / np.where(l == 0, 1.0, l)
                o[b, :, h] = p @ vv if plain else np.where(see[:, :, None], p[:, :, None] * vv[None], 0.0).sum(1)
                if g is None:
                    continue
                gg = np.where(see.any(1)[:, None], np.asarray(g[b, :, h], np.float64), 0.0)
                plain = plain and np.isfinite(gg).all() and np.isfinite(o[b, :, h]).all()
                dp = gg @ vv.T if plain else (gg[:, None, :] * vv[None]).sum(2)
                ds = np.where(see, p * (dp - (gg * o[b, :, h]).sum(1, keepdims=True)) * (1.0 - th * th), 0.0) * scale
                if plain:
                    dq[b, :, h], dk[b, :, hk], dv[b, :, hk] = ds @ kk, dk[b, :, hk] + ds.T @ qq, dv[b, :, hk] + p.T @ gg
                    continue
                dq[b, :, h] = np.where(see[:, :, None], ds[:, :, None] * kk[None], 0.0).sum(1)
                dk[b, :, hk] += np.where(see[:, :, None], ds[:, :, None] * qq[:, None, :], 0.0).sum(0)
                dv[b, :, hk] += np.where(see[:, :, None], p[:, :, None] * gg[:, None, :], 0.0).sum(0)
    return (o, dq, dk, dv) if g is not None else o
