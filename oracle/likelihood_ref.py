"""float64 restatement of the heat map likelihood (log probability of a given pixel, entropy, most likely pixels, and the gradients of the first
two): test infrastructure.  Row by row, from the definition p = softmax(w z) over the allowed pixels (model.py:83-85)."""
import numpy as np


def rows(z, index, w=None, mask=None, topk=0, glogp=None, gentropy=None):
    """z [B, J, V]; index [B, J] or None; w [J] or None; mask [B, J, V] or None (broadcast by the caller).  Returns a dict."""
    B, J, V = z.shape
    z = z.astype(np.float64)
    out = {"logp": np.zeros((B, J)), "entropy": np.zeros((B, J)), "top_logp": np.full((B, J, topk), -np.inf), "top_index": np.full((B, J, topk), -1),
           "gz": np.zeros((B, J, V)), "gw": np.zeros(J), "p": np.zeros((B, J, V)), "logs": np.full((B, J, V), -np.inf)}
    for b in range(B):
        for j in range(J):
            wj = 1.0 if w is None else float(w[j])
            ok = np.ones(V, bool) if mask is None else mask[b, j] != 0
            s = np.where(ok, np.where(ok, z[b, j], 0.0) * wj, -np.inf)
            t = -1 if index is None else int(index[b, j])
            alive = ok & (s != -np.inf)
            if not alive.any():
                if t >= 0:
                    out["logp"][b, j] = -np.inf if t < V else np.nan
                continue
            if np.isnan(s[alive]).any() or np.isposinf(s[alive]).any():
                for k in ("logp", "entropy"):
                    out[k][b, j] = np.nan
                if t < 0:
                    out["logp"][b, j] = 0.0
                out["gz"][b, j] = np.nan
                continue
            M = s[alive].max()
            lp = np.where(alive, (s - M) - np.log(np.exp(s[alive] - M).sum()), -np.inf)     # (M apart: it may be the type's lowest value)
            p = np.exp(lp)
            H = -(p[alive] * lp[alive]).sum()
            out["p"][b, j], out["logs"][b, j], out["entropy"][b, j] = p, lp, H
            if t >= 0:
                out["logp"][b, j] = lp[t] if t < V else np.nan
            order = [i for i in np.lexsort((np.arange(V), -s)) if alive[i]][:topk]
            out["top_logp"][b, j, :len(order)] = lp[order]
            out["top_index"][b, j, :len(order)] = order
            g = 0.0 if glogp is None or t < 0 else float(glogp[b, j])
            h = 0.0 if gentropy is None else float(gentropy[b, j])
            ds = np.zeros(V)
            ds[alive] = -g * p[alive] - h * p[alive] * (lp[alive] + H)
            if 0 <= t < V and alive[t]:
                ds[t] += g
            out["gz"][b, j] = ds * wj
            # sum ds z, with sum ds = 0 (or -g where the given pixel has no probability) taken out: z may be 1e38
            zr = z[b, j][alive][np.argmax(s[alive])]
            out["gw"][j] += (ds[alive] * (z[b, j][alive] - zr)).sum() - (g * zr if 0 <= t < V and not alive[t] else 0.0)
    return out
