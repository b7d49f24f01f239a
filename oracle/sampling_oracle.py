"""Draws and path probabilities in plain numpy, 64 bits (test infrastructure only; no counterpart in the reference).

The definitions are those of include/snk.h (snk_sample_rows, snk_sample_paths, snk_path_posterior)."""
import numpy as np


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weights of the scores of one row that the truncations keep (0 elsewhere), relative to the largest; None: an empty row."""
    x = np.array(x, dtype=np.float64)
    x[np.isnan(x)] = -np.inf
    m = x.max()
    if m == -np.inf:
        return None
    if temperature == 0.0:
        w = np.zeros(x.size)
        w[int(np.argmax(x))] = 1.0
        return w
    w = np.zeros(x.size)
    for i in range(x.size):
        if x[i] == m:
            w[i] = 1.0
        elif x[i] > -np.inf and m < np.inf:
            w[i] = np.exp((x[i] - m) / temperature)
    order = sorted((i for i in range(x.size) if x[i] > -np.inf), key=lambda i: (-x[i], i))
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1.0:
        total, held, n = sum(w[i] for i in order), 0.0, 0
        while held < top_p * total and n < len(order):
            held += w[order[n]]
            n += 1
        order = order[:n]
    keep = np.zeros(x.size)
    for i in order:
        if w[i] >= min_p:
            keep[i] = w[i]
    return keep


def sample_row(x, u, **rule):
    """(index, log probability) of one draw."""
    keep = kept_weights(x, **rule)
    if keep is None:
        return -1, -np.inf
    total = keep.sum()
    held = 0.0
    pick = -1
    for i in np.flatnonzero(keep):
        held += keep[i]
        pick = int(i)
        if held > u * total:
            break
    return pick, float(np.log(keep[pick]) - np.log(total))


def sample_rows(scores, u, **rules):
    """Rows of scores (R, V), u (R, S); every rule a number or R of them."""
    R, S = u.shape
    index, logp = np.zeros((R, S), dtype=np.int64), np.zeros((R, S))
    for r in range(R):
        rule = {k: (v if np.ndim(v) == 0 else np.asarray(v)[r]) for k, v in rules.items()}
        rule['top_k'] = int(rule.get('top_k', 0))
        for s in range(S):
            index[r, s], logp[r, s] = sample_row(scores[r], u[r, s], **rule)
    return index, logp


def buckets(cand0, cand1, edges):
    apart = np.asarray(cand1)[None, :] - np.asarray(cand0)[:, None]
    return np.searchsorted(np.asarray(edges, dtype=np.int64), apart, side='right')


def trellis(cand, tdist, JC, wj, temperature, bias=None, edges=(), join_class=None):
    """Of one utterance: (-target cost / temperature (T, K), join costs with bias (T - 1, K, K), buckets)."""
    cand = np.asarray(cand)
    T, K = cand.shape
    n = JC.shape[0] - 1
    W = JC.astype(np.float64) * wj
    usable = (cand >= 1) & (cand < n - 1)
    with np.errstate(invalid='ignore'):
        local = np.where(usable & np.isfinite(tdist), -np.asarray(tdist, dtype=np.float64) / temperature, -np.inf)
    C = np.full((max(T - 1, 0), K, K), np.inf)
    B = np.zeros((max(T - 1, 0), K, K), dtype=np.int64)
    for t in range(T - 1):
        a, b = np.where(usable[t], cand[t], 0), np.where(usable[t + 1], cand[t + 1], 0)
        c = np.sqrt(((W[a + 1][:, None, :] - W[b][None, :, :]) ** 2).sum(axis=2))
        B[t] = buckets(cand[t], cand[t + 1], edges)
        if bias is not None:
            k = 0 if join_class is None else int(join_class[t])
            if 0 <= k < bias.shape[0]:
                c = c + bias[k][B[t]]
        c[~usable[t], :] = np.inf
        c[:, ~usable[t + 1]] = np.inf
        C[t] = c
    return local, C, B


def lse(x, axis=None):
    m = np.max(x, axis=axis, keepdims=True)
    m = np.where(np.isinf(m), 0.0, m)
    with np.errstate(divide='ignore'):
        out = m + np.log(np.exp(x - m).sum(axis=axis, keepdims=True))
    return np.squeeze(out, axis=axis) if axis is not None else float(out.ravel()[0])


def forward(local, C, temperature):
    alpha = [local[0]]
    for t in range(C.shape[0]):
        alpha.append(local[t + 1] + lse(alpha[-1][:, None] - C[t] / temperature, 0))
    return np.array(alpha)


def backward(local, C, temperature):
    beta = [np.zeros(local.shape[1])]
    for t in range(C.shape[0] - 1, -1, -1):
        beta.append(lse(-C[t] / temperature + (local[t + 1] + beta[-1])[None, :], 1))
    return np.array(beta[::-1])


def sample_path(cand, tdist, u, temperature, JC, wj, bias=None, edges=(), join_class=None, **rule):
    """One draw: (unit ids (T,) -- -1 throughout without a complete path --, cost, log probability)."""
    tau = temperature if temperature > 0.0 else 1.0
    local, C, _ = trellis(cand, tdist, JC, wj, tau, bias, edges, join_class)
    T = local.shape[0]
    if temperature > 0.0:
        alpha = forward(local, C, tau)
    else:
        alpha = [local[0]]
        for t in range(T - 1):
            alpha.append(local[t + 1] + (alpha[-1][:, None] - C[t]).max(axis=0))
        alpha, rule = np.array(alpha), dict(top_k=1)
    if alpha[-1].max() == -np.inf:
        return np.full(T, -1, dtype=np.int64), np.inf, -np.inf
    slots, logp, x = [0] * T, 0.0, alpha[-1]
    for t in range(T - 1, -1, -1):
        if t + 1 < T:
            x = alpha[t] - C[t][:, slots[t + 1]] / tau
        slots[t], lp = sample_row(x, u[t], **rule)
        logp += lp
    cost = sum(tdist[t][slots[t]] for t in range(T)) + sum(C[t][slots[t], slots[t + 1]] for t in range(T - 1))
    return np.array([cand[t][slots[t]] for t in range(T)], dtype=np.int64), float(cost), logp


def posterior(cand, tdist, temperature, JC, wj, bias=None, edges=(), join_class=None):
    """One utterance: (logZ, posterior (T, K), uses (classes, buckets) or None)."""
    local, C, B = trellis(cand, tdist, JC, wj, temperature, bias, edges, join_class)
    alpha, beta = forward(local, C, temperature), backward(local, C, temperature)
    z = lse(alpha[-1])
    uses = None if bias is None else np.zeros(bias.shape)
    if z == -np.inf:
        return z, np.zeros(local.shape), uses
    for t in range(C.shape[0]):
        k = 0 if join_class is None else int(join_class[t])
        if bias is not None and 0 <= k < bias.shape[0]:
            pair = np.exp(alpha[t][:, None] - C[t] / temperature + (local[t + 1] + beta[t + 1])[None, :] - z)
            np.add.at(uses[k], B[t], pair)
    return z, np.exp(alpha + beta - z), uses
