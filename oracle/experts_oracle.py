"""64-bit restatement of the general expert router, its gradient and the products with 4-bit weights,
written from their formulas, for the tests."""
import numpy as np


def scores(logits, score):
    x = np.asarray(logits, np.float64)
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return np.where(x >= 0, 1.0 / (1.0 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1.0 + np.exp(-np.abs(x))))
        e = np.exp(x - x.max(axis=1, keepdims=True))
        return e / e.sum(axis=1, keepdims=True)


def picks(logits, score, bias=None, n_group=1, topk_group=1, group_score="max"):
    """(s, pick) [T, E]; pick is -inf for excluded experts and dropped groups."""
    x = np.asarray(logits, np.float64)
    s = scores(x, score)
    pick = s if bias is None else s + np.asarray(bias, np.float64)
    pick = np.where(np.isneginf(x), -np.inf, pick)
    T, E = pick.shape
    if n_group > 1:
        p = pick.reshape(T, n_group, E // n_group)
        best = np.sort(p, axis=2)[:, :, ::-1]
        gs = best[:, :, 0] if group_score == "max" else best[:, :, 0] + best[:, :, 1]
        order = np.argsort(-gs, axis=1, kind="stable")
        keep = np.zeros((T, n_group), bool)
        np.put_along_axis(keep, order[:, :topk_group], True, axis=1)
        pick = np.where(np.repeat(keep, E // n_group, axis=1), pick, -np.inf)
    return s, pick


def route(logits, k, score, bias=None, n_group=1, topk_group=1, group_score="max", renormalize=True, scale=1.0):
    s, pick = picks(logits, score, bias, n_group, topk_group, group_score)
    idx = np.argsort(-pick, axis=1, kind="stable")[:, :k]
    gone = np.isneginf(np.take_along_axis(pick, idx, 1))
    idx = np.where(gone, -1, idx)
    return idx.astype(np.int32), weights(s, idx, renormalize, scale)


def weights(s, idx, renormalize, scale):
    """Weights of given picks (-1: none)."""
    w = np.where(idx < 0, 0.0, np.take_along_axis(s, np.maximum(idx, 0), 1))
    if renormalize:
        w = w / (w.sum(axis=1, keepdims=True) + 1e-20)
    return w * scale


def route_grad(grad_w, logits, idx, score, renormalize, scale):
    """d sum(grad_w * weights) / d logits, row by row from the full Jacobian of the scores."""
    s = scores(logits, score)
    T, E = s.shape
    out = np.zeros((T, E))
    for t in range(T):
        js = [j for j in range(idx.shape[1]) if 0 <= idx[t, j] < E]
        if not js:                                   # constant weights, also where the softmax of the row is NaN
            continue
        ds = np.zeros(E)
        D = sum(s[t, idx[t, j]] for j in js) + 1e-20
        for j in js:
            g = scale * float(grad_w[t, j])
            if renormalize:
                ds[idx[t, j]] += g / D
                for i in js:
                    ds[idx[t, i]] -= g * s[t, idx[t, j]] / D ** 2
            else:
                ds[idx[t, j]] += g
        if score == "sigmoid":
            a = np.exp(-np.abs(np.asarray(logits[t], np.float64)))
            out[t] = ds * (a / (1.0 + a) ** 2)
        else:
            out[t] = s[t] * (ds - (ds * s[t]).sum())
    return out


def unpack_w4(codes, scale, zero, K, group):
    """float64 [..., N, K]: scale * (code - zero)."""
    codes = np.asarray(codes, np.uint8)
    q = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)[..., :K].astype(np.float64)
    z = 8.0 if zero is None else np.repeat(np.asarray(zero, np.float64), group, -1)[..., :K]
    return (q - z) * np.repeat(np.asarray(scale, np.float64), group, -1)[..., :K]


def experts(x, idx, wt, w13, w2, offset=0):
    """(out, size) [T, H] from unpacked weights; size is the same sum over absolute values."""
    x, wt = np.asarray(x, np.float64), np.asarray(wt, np.float64)
    T, H = x.shape
    E, I = w13.shape[0], w13.shape[1] // 2
    out, size = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for j in range(idx.shape[1]):
            e = int(idx[t, j]) - offset
            if not 0 <= e < E:
                continue
            u, ua = w13[e] @ x[t], np.abs(w13[e]) @ np.abs(x[t])
            sg = scores(u[None, I:], "sigmoid")[0]
            h = u[:I] * u[I:] * sg
            # |dh| <= |silu(u2)| du1 + |u1| 1.1 du2: the slope of silu is at most 1.1.
            ha = np.abs(u[I:] * sg) * ua[:I] + np.abs(u[:I]) * 1.1 * ua[I:]
            out[t] += wt[t, j] * (w2[e] @ h)
            size[t] += abs(wt[t, j]) * (np.abs(w2[e]) @ (ha + np.abs(h)))
    return out, size
