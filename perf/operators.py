"""Cases for the operators on rows of logits: sampling, the best log-probs of a row, and distillation from them.

Each case names the operator (`op`), the rows N, the vocabulary V, the logits' type, and the operator's own arguments. The
sizes are those of the repository's configurations (V = 32000, 50257, 128256, 256000; B*T of its batches as rows).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # one chat request's next token: only latency counts
        dict(name="sample_one", op="sample", N=1, V=32000, dtype="bf16", T=0.7, k=50, p=0.9, q=0.0, mixed=False),
        # a small fp32 batch cut by mass and by ratio alone
        dict(name="sample_nucleus", op="sample", N=64, V=50257, dtype="fp32", T=1.0, k=0, p=0.95, q=0.02, mixed=False),
        # a serving batch in which every request brings its own settings, some of them greedy
        dict(name="sample_mixed", op="sample", N=256, V=128256, dtype="bf16", T=0.8, k=64, p=0.9, q=0.05, mixed=True),
        # roll-outs drawn from the model's own distribution: temperature alone, every token can come
        dict(name="sample_rollout", op="sample", N=512, V=128256, dtype="bf16", T=1.0, k=0, p=1.0, q=0.0, mixed=False),
        # the 20 best log-probs that a server returns beside a few tokens
        dict(name="top_serving", op="top", N=8, V=32000, dtype="fp32", T=1.0, n=20),
        # one row of the largest vocabulary, a long list
        dict(name="top_long", op="top", N=1, V=256000, dtype="fp32", T=1.0, n=128),
        # a teacher's pass over a batch: 64 examples of 32 tokens
        dict(name="top_teacher", op="top", N=2048, V=128256, dtype="bf16", T=2.0, n=64),
        # a small training step in fp16
        dict(name="distill_small", op="distill", N=16, V=32000, dtype="fp16", T=1.0, n=8, tail=True, train=True, mean=True, pad=0.0),
        # the ordinary one: 64 examples of 32 tokens, padded
        dict(name="distill_batch", op="distill", N=2048, V=32000, dtype="bf16", T=2.0, n=64, tail=True, train=True, mean=True, pad=0.2),
        # odd sizes in fp32, without the tail's class, rows added up
        dict(name="distill_odd", op="distill", N=1025, V=50257, dtype="fp32", T=1.0, n=33, tail=False, train=True, mean=False, pad=0.1),
        # an evaluation: each row's loss, no gradient
        dict(name="distill_eval", op="distill", N=257, V=50257, dtype="fp32", T=1.0, n=32, tail=True, train=False, mean=False, pad=0.1),
        # the largest: 4096 tokens of a large vocabulary
        dict(name="distill_large", op="distill", N=4096, V=128256, dtype="bf16", T=1.0, n=64, tail=True, train=True, mean=True, pad=0.1),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("sample", "top", "distill"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    V = _spread(rng, 1000, 256000)
    most = {"sample": 65_000_000, "top": 260_000_000, "distill": 260_000_000}[op]
    N = _spread(rng, 1, max(1, min(4096, most // V)))
    T = rng.choice((0.6, 0.8, 1.0, 1.3, 2.0))
    case = dict(op=op, N=N, V=V, dtype=dtype, T=T)
    if op == "sample":
        case.update(k=rng.choice((0, 0, 1, 20, 50, 400)), p=rng.choice((1.0, 0.5, 0.9, 0.95, 0.99)), q=rng.choice((0.0, 0.0, 0.02, 0.1)),
                    mixed=rng.random() < 0.4)
    elif op == "top":
        case.update(n=_spread(rng, 1, 256))
    else:
        case.update(n=_spread(rng, 1, 256), tail=rng.random() < 0.6, train=rng.random() < 0.75, mean=rng.random() < 0.6,
                    pad=rng.choice((0.0, 0.1, 0.4)))
    return case


def _logits(case, g):
    """Rows as a language model gives them: a Zipf law over the vocabulary in an order of its own, noise, some rows sharp and some flat."""
    N, V = case["N"], case["V"]
    rank = torch.randperm(V, generator=g, device="cuda")
    bias = -1.1 * torch.log(rank.float() + 1.0)
    sharp = torch.rand((N, 1), generator=g, device="cuda") * 1.2 + 0.6
    noise = torch.randn((N, V), generator=g, device="cuda")
    out = noise.mul_(2.0).add_(bias).mul_(sharp).to(_TYPES[case["dtype"]])
    return out, bias


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    N, V = case["N"], case["V"]
    x, bias = _logits(case, g)
    s = dict(case=case, x=x)
    if case["op"] == "sample":
        s["u"] = torch.rand((N,), generator=g, device="cuda")
        s["T"], s["k"], s["p"], s["q"] = case["T"], case["k"], case["p"], case["q"]
        if case["mixed"]:  # each request's own settings; a tenth of them greedy, a fifth without top-k, a third without min-p
            r = torch.rand((4, N), generator=g, device="cuda")
            s["T"] = torch.where(r[0] < 0.1, torch.zeros_like(r[0]), case["T"] * (0.5 + r[0]))
            s["k"] = torch.where(r[1] < 0.2, torch.zeros_like(r[1]), 1.0 + r[1] * max(case["k"], 1)).to(torch.int32)
            s["p"] = (case["p"] + 0.1 * (r[2] - 0.5)).clamp(max=1.0)
            s["q"] = torch.where(r[3] < 0.3, torch.zeros_like(r[3]), case["q"] * r[3])
    elif case["op"] == "distill":
        # a teacher that agrees with the student in part: its best n of its own rows, as it would have kept them
        n = min(case["n"], V)
        lq = torch.empty((N, n), dtype=torch.float32, device="cuda")
        at = torch.empty((N, n), dtype=torch.int32, device="cuda")
        step = max(1, 100_000_000 // V)
        for a in range(0, N, step):
            z = 0.5 * x[a:a + step].float() + 0.6 * bias + torch.randn((min(step, N - a), V), generator=g, device="cuda")
            z = z / case["T"]
            best, i = z.topk(n, dim=1)
            lq[a:a + step] = best - torch.logsumexp(z, dim=1, keepdim=True)
            at[a:a + step] = i.to(torch.int32)
        if case["pad"] > 0:  # padding: rows without a teacher, and lists shorter than n
            none = torch.rand((N, 1), generator=g, device="cuda") < case["pad"]
            short = torch.rand((N, 1), generator=g, device="cuda") < 0.1
            late = torch.arange(n, device="cuda")[None, :] >= (n + 1) // 2
            at[none.expand(N, n) | (short & late)] = -1
        s["lq"], s["at"] = lq, at
        s["x"] = x.requires_grad_(case["train"])
    return s


# --- plain forms: elementary operations, in 32 bits, in 64 where whole numbers hang on a sum ---------------------------------


def _column(v, N, dtype):
    return v.to(dtype).reshape(N, 1) if isinstance(v, torch.Tensor) else torch.full((N, 1), v, dtype=torch.float32, device="cuda").to(dtype)


def _plain_sample(x, u, T, k, p, q):
    N, V = x.shape
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    T, k, p, q = _column(T, N, torch.float64), _column(k, N, torch.int64), _column(p, N, torch.float64), _column(q, N, torch.float64)
    s, order = torch.sort(x, dim=1, descending=True, stable=True)
    best = s[:, :1]
    z = torch.where(s == best, 0.0, (s - best) / torch.where(T > 0, T, 1.0))
    w = torch.where(z < -708.0, 0.0, torch.exp(z))
    keep = (k <= 0) | (torch.arange(V, device=x.device)[None, :] < k)
    w = torch.where(keep, w, 0.0)
    mass = w.cumsum(dim=1)
    before = torch.cat((torch.zeros_like(mass[:, :1]), mass[:, :-1]), dim=1)
    keep = keep & ((p >= 1.0) | (before < p * mass[:, -1:])) & (z >= torch.log(q))
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    w = torch.zeros_like(w).scatter(1, order, w)
    mass = w.cumsum(dim=1)
    over = mass > u.double()[:, None] * mass[:, -1:]
    at = torch.arange(V, device=x.device)[None, :]
    first = torch.where(over, at, V).amin(dim=1)
    last = torch.where(w > 0.0, at, -1).amax(dim=1)
    token = torch.where(first < V, first, last)
    token = torch.where(T[:, 0] > 0, token, order[:, 0])
    return torch.where(best[:, 0] > -math.inf, token, -1).to(torch.int32)


def _plain_top(x, n, T):
    x = x.float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    top = best[:, :1]
    # the sum over a row is a long one: its terms in 32 bits, the sum in 64
    total = torch.exp((x - top) / T).sum(dim=1, keepdim=True, dtype=torch.float64)
    value = ((best[:, :n] - top) / T - torch.log(total)).float()
    return value, torch.where(best[:, :n] > -math.inf, at[:, :n], -1).to(torch.int32)


def _plain_rows(x, lq, at, T, tail):
    """Each row's loss, by operations that torch differentiates."""
    N, V = x.shape
    z = x.float() / T
    there = (at >= 0) & (at < V)
    where = torch.where(there, at, 0).long()
    q64 = torch.where(there, torch.exp(lq.double()), 0.0)  # in 64 bits: 1 - sum is what is left over
    q = q64.float()
    top = z.detach().amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    log_p = torch.gather(z, 1, where) - top - torch.log(total)
    loss = torch.where(q > 0, q * (torch.where(q > 0, lq, 0.0) - torch.where(q > 0, log_p, 0.0)), 0.0).sum(dim=1)
    if tail:
        mark = torch.zeros((N, V + 1), dtype=torch.bool, device=x.device).scatter(1, torch.where(there, where, V), True)
        rest = torch.where(mark[:, :V], 0.0, e).sum(dim=1)
        left = (1.0 - q64.sum(dim=1)).clamp(min=0.0).float()
        on = (left > 0) & (rest > 0) & there.any(dim=1)
        l, r = torch.where(on, left, 1.0), torch.where(on, rest, 1.0)
        loss = loss + torch.where(on, l * (torch.log(l) - torch.log(r) + torch.log(torch.where(on, total[:, 0], 1.0))), 0.0)
    return loss, there.any(dim=1)


def _plain_distill(s):
    c = s["case"]
    with torch.set_grad_enabled(c["train"]):
        loss, there = _plain_rows(s["x"], s["lq"], s["at"], c["T"], c["tail"])
        if not c["train"]:
            return loss
        loss = loss.sum() / there.sum().clamp(min=1) if c["mean"] else loss.sum()
        grad, = torch.autograd.grad(loss, s["x"])
    return loss.detach(), grad


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "differentiable-beam-search-cuda_b200", "python")
    here = os.path.join(os.getcwd(), "differentiable-beam-search-cuda_b200", "python")
    path = here if os.path.isdir(here) else path
    if path not in sys.path:
        sys.path.insert(0, path)
    import torch_dbs_extension
    return torch_dbs_extension


def run(s):
    c = s["case"]
    if own:
        dbs = sys.modules.get("torch_dbs_extension") or _framework()
        if c["op"] == "sample":
            return dbs.sample(s["x"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["q"])
        if c["op"] == "top":
            return dbs.top_log_probs(s["x"], min(c["n"], c["V"]), temperature=c["T"])
        if not c["train"]:
            with torch.no_grad():
                return dbs.distillation_loss(s["x"], s["lq"], s["at"], temperature=c["T"], tail=c["tail"], reduction="none")
        loss = dbs.distillation_loss(s["x"], s["lq"], s["at"], temperature=c["T"], tail=c["tail"], reduction="mean" if c["mean"] else "sum")
        grad, = torch.autograd.grad(loss, s["x"])
        return loss.detach(), grad
    if c["op"] == "sample":
        return _plain_sample(s["x"], s["u"], s["T"], s["k"], s["p"], s["q"])
    if c["op"] == "top":
        return _plain_top(s["x"], min(c["n"], c["V"]), c["T"])
    return _plain_distill(s)


def work(case):
    N, V, es = case["N"], case["V"], _BYTES[case["dtype"]]
    x = N * V * es
    if case["op"] == "sample":  # the row once; an exponential and two sums of what can be kept
        return {"bytes": x + 8 * N + (16 * N if case["mixed"] else 0), "flops": 2.0 * N * V}
    n = min(case["n"], V)
    if case["op"] == "top":  # the row once; maximum, exponential, sum
        return {"bytes": x + 8 * N * n, "flops": 4.0 * N * V}
    if case["train"]:  # the row once, its gradient once
        return {"bytes": 2 * x + 8 * N * n + 4, "flops": 7.0 * N * V}
    return {"bytes": x + 8 * N * n + 4 * N, "flops": 4.0 * N * V}


# --- 64 bits, from the definitions -------------------------------------------------------------------------------------------


def _exact_token(x, u, T, k, p, q):
    """One row on the host: the kept set as a cut in the ordered values, then a walk by index."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if not top > -np.inf:
        return -1
    if not T > 0:
        return int(np.flatnonzero(x == top)[0])
    order = np.argsort(-x, kind="stable")
    if k > 0:
        order = order[:k]
    with np.errstate(invalid="ignore", divide="ignore"):
        z = np.where(x[order] == top, 0.0, (x[order] - top) / T)
        z[z < -708.0] = -np.inf
        weight = np.exp(z)
        size = order.size
        if p < 1.0:
            run_up = np.cumsum(weight)
            size = min(size, 1 + int(np.searchsorted(run_up[:-1], p * run_up[-1], side="left")))
        size = max(1, min(size, int((z >= np.log(q)).sum())))
    by_index = np.argsort(order[:size])
    weight, order = weight[:size][by_index], order[:size][by_index]
    run_up = np.cumsum(weight)
    hit = int(np.searchsorted(run_up, u * run_up[-1], side="right"))
    return int(order[hit]) if hit < size else int(order[np.flatnonzero(weight > 0)[-1]])


def _exact_rows(x, lq, at, T, tail):
    """Losses of some rows, which rows have a teacher, and the gradients' rows before any weight."""
    V = x.shape[1]
    there = (at >= 0) & (at < V)
    has, i = there.any(dim=1), at.clamp(0, V - 1).long()
    log_P = torch.log_softmax(x.double() / T, dim=1)
    P = log_P.exp()
    q = torch.where(there, lq.double().exp(), 0.0)
    Q = torch.zeros_like(P).scatter_add_(1, i, q)
    seen = torch.zeros_like(P).scatter_add_(1, i, there.double()) > 0
    loss = torch.where(q > 0, q * (lq.double() - log_P.gather(1, i)), 0.0).sum(dim=1)
    P_rest = P.masked_fill(seen, 0.0).sum(dim=1)
    q_rest = (1.0 - q.sum(dim=1)).clamp(min=0.0) if tail else torch.zeros_like(loss)
    q_rest = torch.where((P_rest > 0) & has, q_rest, 0.0)
    loss = loss + torch.where(q_rest > 0, q_rest * (q_rest.log() - P_rest.log()), 0.0)
    G = (q.sum(dim=1) + q_rest)[:, None]
    rest = torch.where(q_rest > 0, q_rest / P_rest, 0.0)[:, None]
    return loss, has, (G * P - Q - torch.where(seen, 0.0, rest * P)) / T


def exact(case, seed):
    s = prepare(case, seed)
    x, N, V = s["x"].detach(), case["N"], case["V"]
    if case["op"] == "sample":
        each = [v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(N, np.float64(np.float32(v))) for v in (s["T"], s["k"], s["p"], s["q"])]
        u = s["u"].double().cpu().numpy()
        tokens = []
        for r in range(N):
            tokens.append(_exact_token(x[r].double().cpu().numpy(), u[r], each[0][r], int(each[1][r]), each[2][r], each[3][r]))
        return torch.tensor(tokens, dtype=torch.int32)
    step = max(1, 60_000_000 // V)
    if case["op"] == "top":
        n, values, tokens = min(case["n"], V), [], []
        for r in range(0, N, step):
            row = x[r:r + step].double()
            order = torch.argsort(row, dim=1, descending=True, stable=True)[:, :n]
            values.append(torch.log_softmax(row / case["T"], dim=1).gather(1, order))
            tokens.append(order.to(torch.int32))
        return torch.cat(values), torch.cat(tokens)
    losses, has, grads = [], [], []
    for r in range(0, N, step):
        one, there, grad = _exact_rows(x[r:r + step], s["lq"][r:r + step], s["at"][r:r + step], case["T"], case["tail"])
        losses.append(one)
        has.append(there)
        grads.append(grad if case["train"] else None)
    loss = torch.cat(losses)
    if not case["train"]:
        return loss
    share = 1.0 / max(1, int(torch.cat(has).sum())) if case["mean"] else 1.0
    return loss.sum() * share, torch.cat(grads).mul_(share)
