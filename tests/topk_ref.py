"""64-bit references of top-k routing, rows to k experts and back, and low-rank adapters, in plain numpy, row by row."""
import numpy as np

LOWEST = {"float32": -3.4028234663852886e38, "float16": -65504.0, "bfloat16": -3.3895313892515355e38}


def select(logits, lowest, k, score, bias=None, groups=1, top_groups=1, group_best=1, renormalise=True, scale=1.0):
    """logits float64 [T, E] -> gate int32 [T, k], weight float64 [T, k]."""
    T, E = logits.shape
    gate, weight = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        l = logits[t]
        ok = l > lowest
        if not ok.any():
            continue
        s = np.zeros(E)
        with np.errstate(over="ignore", invalid="ignore"):
            if score == "softmax":
                e = np.where(l[ok] == l[ok].max(), 1.0, np.exp(l[ok] - l[ok].max()))
                s[ok] = e / e.sum()
            else:
                s[ok] = 1 / (1 + np.exp(-l[ok]))
        key = np.where(ok, l, -np.inf)
        if bias is not None:
            usable = ok & (bias > -np.inf)
            key = np.where(usable, s + np.where(usable, bias, 0), -np.inf)
        if groups > 1:
            size = E // groups
            value = np.full(groups, -np.inf)
            for g in range(groups):
                best = sorted(range(g * size, (g + 1) * size), key=lambda e: -key[e])[:2]
                best = [e for e in best if key[e] > -np.inf]
                if best and group_best == 1:
                    value[g] = key[best[0]]
                elif best:
                    value[g] = sum(key[e] if bias is not None else s[e] for e in best)
            for g in sorted(range(groups), key=lambda g: (-value[g], g))[top_groups:]:
                key[g * size:(g + 1) * size] = -np.inf
        chosen = [e for e in sorted(range(E), key=lambda e: (-key[e], e))[:k] if key[e] > -np.inf]
        gate[t, :len(chosen)] = chosen
        if not chosen:
            continue
        w = s[chosen]
        if renormalise:
            top = l[chosen].max()
            with np.errstate(over="ignore", invalid="ignore"):
                w = np.where(l[chosen] == top, 1.0, np.exp(l[chosen] - top))
                if score == "sigmoid":
                    w = w / (1 + np.exp(l[chosen])) if top <= 0 else 1 / (1 + np.exp(-l[chosen]))
            w = w / w.sum()
        weight[t, :len(chosen)] = w * scale
    return gate, weight


def combine(rows, weight, row_of, residual=None):
    out = np.zeros((weight.shape[0], rows.shape[1]))
    size = np.zeros_like(out)                     # sum of the magnitudes, what rounding errors are relative to
    for t in range(weight.shape[0]):
        rest, used = 1.0, 0.0
        for s in range(weight.shape[1]):
            r = row_of[t, s]
            if 0 <= r < len(rows):
                out[t] += weight[t, s] * rows[r]
                size[t] += abs(weight[t, s] * rows[r])
                rest -= weight[t, s]
                used += abs(weight[t, s])
        if residual is not None:
            out[t] += rest * residual[t]
            size[t] += (1 + used) * abs(residual[t])
    return out, size


def adapters(x, y, a, b, scale, rank, adapter_of_token):
    out = y.copy()
    for t, i in enumerate(adapter_of_token):
        if 0 <= i < len(a):
            r = min(max(int(rank[i]), 0), a.shape[1]) if rank is not None else a.shape[1]
            out[t] += scale[i] * (b[i, :, :r] @ (a[i, :r] @ x[t]))
    return out
