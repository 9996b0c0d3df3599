"""Plain 64-bit implementations of the speculative-decoding operators, one sequence and one node at a time (numpy)."""
from __future__ import annotations

import numpy as np


def f64(t):
    return t.detach().double().cpu().numpy()


def tree(parents, T):
    """[ancestor list of node t, itself last] for every node, None for an unused one."""
    out = []
    for t in range(T):
        up = t - 1 if parents is None else int(parents[t])
        out.append(None if up < -1 else (out[up] if up >= 0 else []) + [t])
    return out


def rotate(x, cos, sin, rot, interleaved):
    y = x.copy()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        y[..., a] = x[..., a] * cos[i] - x[..., b] * sin[i]
        y[..., b] = x[..., b] * cos[i] + x[..., a] * sin[i]
    return y


def rope_append(q, k, v, cos, sin, kc, vc, lens, parents, rot, interleaved, positions=None):
    """All arrays float64; kc, vc are updated in place; returns the rotated q."""
    out = np.zeros_like(q)
    for b in range(q.shape[0]):
        nodes = tree(None if parents is None else parents[b], q.shape[1])
        for t, anc in enumerate(nodes):
            if anc is None:
                continue
            pos = int(lens[b]) + len(anc) - 1 if positions is None else int(positions[b, t])
            out[b, t] = rotate(q[b, t], cos[pos], sin[pos], rot, interleaved)
            kc[b, :, int(lens[b]) + t] = rotate(k[b, t], cos[pos], sin[pos], rot, interleaved)
            vc[b, :, int(lens[b]) + t] = v[b, t]
    return out


def attention(q, kc, vc, lens, parents, sinks, window, scale):
    """(out, largest scale * sum |q k| of a visible key, largest |v| of a visible key), float64."""
    B, T, hq, hd = q.shape
    rep = hq // kc.shape[1]
    out, smax, vmax = np.zeros_like(q), 0.0, 0.0
    for b in range(B):
        n = int(lens[b])
        nodes = tree(None if parents is None else parents[b], T)
        for t, anc in enumerate(nodes):
            if anc is None:
                continue
            pos = n + len(anc) - 1
            keys = [j for j in range(max(0, pos - window + 1) if window else 0, n)]
            keys += [n + a for i, a in enumerate(anc) if not window or len(anc) - 1 - i < window]
            if not keys:
                continue
            for h in range(hq):
                K, V = kc[b, h // rep, keys], vc[b, h // rep, keys]
                s = K @ q[b, t, h] * scale
                m = s.max() if sinks is None else max(s.max(), sinks[h])
                e = np.exp(s - m)
                out[b, t, h] = e @ V / (e.sum() + (0.0 if sinks is None else np.exp(sinks[h] - m)))
                smax = max(smax, float((np.abs(K) @ np.abs(q[b, t, h])).max() * scale))
                vmax = max(vmax, float(np.abs(V[np.isfinite(V)]).max(initial=0.0)))
    return out, smax, vmax


def verify(tokens, parents, logits, draft, u, race, temperature):
    """One sequence: (path, next token, smallest relative margin of a decision)."""
    T, V = logits.shape
    par = [t - 1 for t in range(T)] if parents is None else [int(p) for p in parents]
    node, path, margin = 0, [0], np.inf
    while True:
        x = np.where(np.isnan(logits[node]), -np.inf, np.minimum(logits[node], np.finfo(np.float32).max))
        if x.max() == -np.inf:
            return path, -1, margin
        kids = [c for c in range(node + 1, T) if par[c] == node]
        if temperature == 0:
            best = int(x.argmax())
            took = next((c for c in kids if tokens[c] == best), None)
            if took is None:
                return path, best, margin
        else:
            r = np.exp((x - x.max()) / temperature)
            r /= r.sum()
            q = None if draft is None else draft[node].copy()
            took = None
            for c in kids:
                tok = int(tokens[c])
                qc = (1.0 if q is None else q[tok]) if 0 <= tok < V else (1.0 if q is None else 0.0)
                rc = r[tok] if 0 <= tok < V else 0.0
                if max(u[c] * qc, rc) > 0:
                    margin = min(margin, abs(u[c] * qc - rc) / max(u[c] * qc, rc))
                if u[c] * qc < rc:
                    took = c
                    break
                w = r.copy()
                if q is None:
                    if 0 <= tok < V:
                        w[tok] = max(w[tok] - 1.0, 0.0)
                else:
                    w = np.maximum(w - q, 0.0)
                if w.sum() > 0:
                    r = w / w.sum()
                if q is not None and 0 <= tok < V:
                    left = 1.0 - q[tok]
                    q = q / left if left > 0 else 0.0 * q
                    q[tok] = 0.0
            if took is None:
                s = np.where(r > 0, r / race, -np.inf)
                i = int(s.argmax())
                rest = np.delete(s, i)
                if rest.size and rest.max() > 0:
                    margin = min(margin, (s[i] - rest.max()) / s[i])
                return path, i, margin
        node = took
        path.append(node)
