"""The operators on rows of logits (sample, top_log_probs, distillation_loss)
in 64 bits on the host, from their definitions, and the bounds that their
results on the device are held to."""
import numpy as np
import torch


def rows64(x):
    x = x.detach().to("cpu", torch.float64).numpy()
    return np.where(np.isnan(x), -np.inf, x)


def sample(x, u, temperature, top_k, top_p, min_p):
    """Tokens of the rows x [rows, V]; every setting an array of one float32 value (int for top_k) per row."""
    x = rows64(x)
    out = np.empty(len(x), dtype=np.int64)
    for r, row in enumerate(x):
        m = row.max()
        if not m > -np.inf:
            out[r] = -1
            continue
        order = np.argsort(-row, kind="stable")
        T = min(np.float64(temperature[r]), np.float64(np.finfo(np.float32).max))
        if not T > 0:
            out[r] = order[0]
            continue
        with np.errstate(invalid="ignore", divide="ignore", over="ignore", under="ignore"):
            z = np.where(row == m, 0.0, (row - m) / T)[order]
            w = np.where(z < -708.0, 0.0, np.exp(z))
        k = int(top_k[r])
        if 0 < k < len(row):
            w[k:] = 0.0
        size = k if 0 < k < len(row) else len(row)
        p, q = np.float64(top_p[r]), min(np.float64(min_p[r]), 1.0)
        before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        keep = np.arange(len(row)) < size
        if p < 1.0:
            keep &= before < p * w.sum()
        if q > 0.0:
            keep &= z >= np.log(q)
        keep[0] = True
        kept = np.zeros(len(row))
        kept[order[keep]] = w[keep]
        run = np.cumsum(kept)
        hit = np.flatnonzero((run > np.float64(u[r]) * run[-1]) & (kept > 0))
        out[r] = hit[0] if len(hit) else np.flatnonzero(kept > 0)[-1]
    return out


def top_log_probs(x, n, temperature):
    x = rows64(x)
    values = np.full((len(x), n), -np.inf)
    tokens = np.full((len(x), n), -1, dtype=np.int64)
    for r, row in enumerate(x):
        m = row.max()
        if not m > -np.inf:
            continue
        order = np.argsort(-row, kind="stable")[:n]
        with np.errstate(over="ignore", under="ignore"):
            log_z = np.log(np.exp((row - m) / temperature).sum())
        there = row[order] > -np.inf
        values[r, there] = ((row[order] - m) / temperature - log_z)[there]
        tokens[r, there] = order[there]
    return values, tokens


def distill(x, log_probs, tokens, temperature, tail):
    """Row losses, rows with a teacher, d loss_r / d x [rows, V], and the size of the terms that each gradient value is a sum of."""
    x = x.detach().to("cpu", torch.float64).numpy()
    log_probs = log_probs.detach().to("cpu", torch.float64).numpy()
    tokens = tokens.detach().cpu().numpy()
    N, V = x.shape
    loss, grad, size = np.zeros(N), np.zeros((N, V)), np.zeros((N, V))
    has = np.zeros(N, dtype=bool)
    for r in range(N):
        there = (tokens[r] >= 0) & (tokens[r] < V)
        has[r] = there.any()
        if not has[r]:
            continue
        i, l = tokens[r][there], log_probs[r][there]
        with np.errstate(invalid="ignore", divide="ignore", over="ignore", under="ignore"):
            q = np.exp(l)
            m = x[r].max()
            e = np.exp(np.where(x[r] == m, 0.0, (x[r] - m) / temperature)) if m > -np.inf else np.zeros(V)
            Z = e.sum()
            P = e / Z if Z > 0 else e
            log_P = np.where(x[r] == m, 0.0, (x[r] - m) / temperature) - np.log(Z) if Z > 0 else np.full(V, -np.inf)
            listed = np.zeros(V, dtype=bool)
            listed[i] = True
            P_r = P[~listed].sum()
            q_r = max(0.0, 1.0 - q.sum()) if tail and P_r > 0 else 0.0
            loss[r] = np.where(q > 0, q * (l - log_P[i]), 0.0).sum()
            if q_r > 0:
                loss[r] += q_r * (np.log(q_r) - np.log(P_r))
        Q = np.zeros(V)
        np.add.at(Q, i, q)
        rest = q_r / P_r * P if q_r > 0 else np.zeros(V)
        grad[r] = ((q.sum() + q_r) * P - Q - np.where(listed, 0.0, rest)) / temperature
        size[r] = ((q.sum() + q_r) * P + Q + np.where(listed, 0.0, rest)) / temperature
    return loss, has, grad, size


# log of a row's sum of exponentials, in 32 bits on the device: a thread adds up to 64 terms into one of two sums, five
# and three more additions join them ((64 + 9) 2^-24); an exponential is off by 2^-22; its exponent t is rounded once and its
# factor once (|t| 2^-23 ln 2 each, weighted by the terms' shares: |t| stays below 24 on average). In all below 8e-6.
LOG_Z = 8.0e-6


def top_bound(values):
    return LOG_Z + 2.0 ** -23 * np.abs(np.where(np.isfinite(values), values, 0.0))


def loss_bound(loss, spread):
    """`spread`: how far log P and log q reach in the row; q is rounded to 32 bits (2^-24), the sum of q enters once more with log Z, and
    the tail has a sum of its own."""
    return 3.0 * LOG_Z + 2.0 ** -23 * (np.abs(loss) + spread)


def grad_bound(grad, size, scale, dtype):
    """Each of the terms is off by the sums' error (twice for the tail's) and three roundings, the value by its type's half step."""
    half = torch.finfo(dtype).eps / 2
    smallest = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[dtype]
    return np.abs(scale) * size * (2.0 * LOG_Z + 6.0 * 2.0 ** -24 + 2.0 ** -22) * (1 + half) + half * np.abs(grad) + smallest
