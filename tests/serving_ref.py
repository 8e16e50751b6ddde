"""Plain numpy restatements of the 8-bit cache operators and of row sampling,
for their tests: the append's documented f32 steps (codes are compared bit for
bit), attention and sampling in 64 bits."""
import numpy as np

PAGE = 16
F = np.float32




def norm_rotate(x, gamma, cos, sin):
    """x [heads][hd] f32 -> f32, every step rounded in f32 (the mean of squares
    summed in 64 bits)."""
    x = x.astype(F)
    hd = x.shape[-1]
    if gamma is not None:
        mean = ((x.astype(np.float64) ** 2).sum(-1, keepdims=True) / hd).astype(F)
        inv = (F(1) / np.sqrt((mean + F(1e-6)).astype(F))).astype(F)
        x = ((x * inv).astype(F) * gamma.astype(F)).astype(F)
    if cos is not None:
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        x = np.concatenate([((a * cos).astype(F) - (b * sin).astype(F)).astype(F),
                            ((b * cos).astype(F) + (a * sin).astype(F)).astype(F)], -1)
    return x


def quantise(x, inv):
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.rint((x * inv).astype(F))
    y = np.clip(np.where(np.isnan(y), 0, y), -127, 127)
    return y.astype(np.int8)


def append(codes, scales, table, k, v, seq, pos, k_norm=None, cos=None, sin=None, rope_pos=None):
    """Appends in place: codes [page][2][kvh][16][hd] int8, scales [page][2][kvh]."""
    kvh, hd = codes.shape[2], codes.shape[4]
    n = len(seq)
    i = 0
    while i < n:
        s, p = int(seq[i]), int(pos[i])
        if s < 0 or s >= table.shape[0] or p < 0 or p >= table.shape[1] * PAGE:
            i += 1
            continue
        m = 1
        while i + m < n and seq[i + m] == s and pos[i + m] == p + m and (p + m) % PAGE:
            m += 1
        page, slot = int(table[s, p // PAGE]), p % PAGE
        if 0 <= page < codes.shape[0]:
            rows = []
            for j in range(i, i + m):
                rp = int(pos[j] if rope_pos is None else rope_pos[j])
                c, sn = (cos[rp], sin[rp]) if cos is not None and 0 <= rp < len(cos) else (None, None)
                rows.append(np.stack([norm_rotate(k[j].reshape(kvh, hd), k_norm, c, sn),
                                      v[j].reshape(kvh, hd).astype(F)]))
            x = np.stack(rows)  # [m][2][kvh][hd]
            big = np.where(np.isfinite(x), np.abs(x), 0).max(axis=(0, 3)).astype(F)
            need = np.where(big > 0, np.maximum((big * F(1.0 / 127.0)).astype(F), F(2.0 ** -126)), F(0)).astype(F)
            had = scales[page].copy()
            if slot:
                new = np.where(need <= had, had, np.maximum(need, (had * F(1.25)).astype(F))).astype(F)
                ratio = np.where(new > 0, had / np.where(new > 0, new, 1), 0).astype(F)
                codes[page, :, :, :slot] = np.where(
                    (new != had)[:, :, None, None],
                    quantise(codes[page, :, :, :slot].astype(F), ratio[:, :, None, None]), codes[page, :, :, :slot])
            else:
                new = need
            inv = np.where(new > 0, F(1) / np.where(new > 0, new, 1), 0).astype(F)
            codes[page, :, :, slot:slot + m] = quantise(x, inv[None, :, :, None]).transpose(1, 2, 0, 3)
            scales[page] = new
        i += m


def attention(codes, scales, table, q, heads, seq, pos, scale, window, out, lse):
    """64-bit attention into out [n][heads*hd], lse [n][heads] (f64), rows of
    padding left alone.  Returns the largest scale * sum |q_d k_d| and the
    largest |v| that the rows meet."""
    kvh, hd = codes.shape[2], codes.shape[4]
    group = heads // kvh
    most, vmax = 0.0, 0.0
    cap = table.shape[1] * PAGE
    values = {}
    for r in range(len(seq)):
        s = int(seq[r])
        if s < 0 or s >= table.shape[0]:
            continue
        p = min(int(pos[r]), cap - 1)
        out[r] = 0.0
        lse[r] = -np.inf
        lo = max(0, p + 1 - window) if window else 0
        if p < 0:
            continue
        if s not in values:
            pages = table[s]
            ok = (pages >= 0) & (pages < codes.shape[0])
            at = np.where(ok, pages, 0)
            x = codes[at].astype(np.float64) * scales[at].astype(np.float64)[..., None, None]
            values[s] = (x.transpose(1, 2, 0, 3, 4).reshape(2, kvh, cap, hd), np.repeat(ok, PAGE))
        x, ok = values[s]
        see = np.arange(lo, p + 1)
        see = see[ok[see]]
        if not len(see):
            continue
        for h in range(heads):
            kk, vv = x[0, h // group][see], x[1, h // group][see]
            qq = q[r, h * hd:(h + 1) * hd].astype(np.float64)
            a = kk @ qq * scale
            most = max(most, scale * float((np.abs(kk) @ np.abs(qq)).max()))
            vmax = max(vmax, float(np.abs(vv).max()))
            top = a.max()
            w = np.exp(a - top)
            out[r, h * hd:(h + 1) * hd] = w @ vv / w.sum()
            lse[r, h] = top + np.log(w.sum())
    return most, vmax


def sample(logits, temperature, top_k, top_p, min_p, u):
    """One row in 64 bits: (token, kept, logprob, margin); margin is how far u
    lies from the nearest border of the running sum, relative to the total."""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, 0, -np.inf, 1.0
    if not temperature > 0:
        return int(order[0]), 1, 0.0, 1.0
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp(np.where(x[order] == top, 0.0, x[order] - top) / float(temperature)))
    w = np.where(np.isnan(w), 0.0, w)
    n = len(order)
    if top_p < 1:
        n = 1 + int(np.searchsorted(np.cumsum(w)[:-1], float(top_p) * w.sum()))
    if min_p > 0:
        n = min(n, int((w >= min(1.0, float(min_p))).sum()))
    back = np.argsort(order[:n])
    idx, ww = order[:n][back], w[:n][back]
    cum, total = np.cumsum(ww), ww.sum()
    uu = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    i = int(np.searchsorted(cum, uu * total, side="right"))
    if i >= n or ww[i] == 0.0:
        i = int(np.nonzero(ww)[0][-1])
    margin = np.abs(cum / total - uu)
    margin = margin[:-1].min() if n > 1 else 1.0
    return int(idx[i]), n, float(np.log(ww[i] / total)), float(margin)
