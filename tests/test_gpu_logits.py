"""The operators on rows of logits on the device against their definitions in
64 bits (logits_reference.py): tokens equal, values within derived bounds."""
import math

import numpy as np
import pytest
import torch

import logits_reference as ref
import torch_dbs_extension as ext

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LOWEST = {t: torch.finfo(t).min for t in DTYPES}


def rows(N, V, dtype, seed, scale=1.0):
    """Rows as a model gives them: a Zipf law over the tokens, noise, sharp and flat rows."""
    g = torch.Generator().manual_seed(seed)
    bias = -1.1 * torch.log(torch.randperm(V, generator=g).float() + 1.0)
    sharp = torch.rand((N, 1), generator=g) * 1.2 + 0.6
    return (scale * sharp * (2.0 * torch.randn((N, V), generator=g) + bias)).to(dtype)


def uniforms(N, seed):
    return torch.rand(N, generator=torch.Generator().manual_seed(seed + 1000))


def check_sample(x, u, T=1.0, k=0, p=1.0, q=0.0, dev=None):
    """x on the host or the device; settings numbers or host tensors."""
    N = x.shape[0]

    def col(v, dtype):
        return (v if isinstance(v, torch.Tensor) else torch.full((N,), v)).to(dtype).numpy()

    def there(v):
        return v.cuda() if isinstance(v, torch.Tensor) else v

    want = ref.sample(x, u.numpy(), col(T, torch.float32), col(k, torch.int32), col(p, torch.float32), col(q, torch.float32))
    got = ext.sample(x.cuda() if dev is None else dev, u.cuda(), temperature=there(T), top_k=there(k), top_p=there(p), min_p=there(q))
    assert got.dtype == torch.int32 and got.shape == (N,)
    assert got.cpu().tolist() == want.tolist()


SETTINGS = [
    dict(), dict(T=0.7), dict(T=0.0), dict(k=1), dict(k=5), dict(k=50, p=0.9, T=0.8), dict(k=600), dict(k=600, p=0.8, q=0.01),
    dict(p=0.5), dict(p=0.95), dict(p=0.9999, T=1.5), dict(q=0.1), dict(q=1.0), dict(p=0.9, q=0.05), dict(k=40, q=0.3, T=2.0),
    dict(k=512, p=0.99),
]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(3, 1), (5, 2), (4, 7), (17, 100), (9, 999), (6, 32000), (3, 50257), (40, 32000), (33, 50257), (35, 8193)])
def test_sample(N, V, dtype, settings):
    seed = N * 31 + V
    check_sample(rows(N, V, dtype, seed), uniforms(N, seed), **settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(40, 4096), (150, 1023), (400, 130), (130, 9001), (300, 32000)])
def test_sample_settings_of_each_row(N, V, dtype):
    g = torch.Generator().manual_seed(N)
    x, u = rows(N, V, dtype, N), uniforms(N, N)
    T = torch.rand(N, generator=g) * 1.5
    T[::7] = 0.0
    k = torch.randint(0, 80, (N,), generator=g, dtype=torch.int32)
    k[::5] = 0
    k[3::11] = 700
    p = torch.rand(N, generator=g) * 1.3
    q = torch.rand(N, generator=g) * 0.2
    q[::3] = 0.0
    T[1], k[2], p[4], q[6] = -1.0, -5, -0.5, 3.0
    check_sample(x, u, T, k, p, q)


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,times", [(5000, 1), (9001, 3)])
def test_sample_ties_and_masks(V, times, dtype, settings):
    g = torch.Generator().manual_seed(5)
    x = torch.round(rows(12, V, torch.float32, 5))            # many equal values
    x[0] = 0.0                                                # all equal
    x[1] = -math.inf                                          # nothing left
    x[2, 10:] = -math.inf
    x[3, 40:] = LOWEST[dtype]
    x[4] = LOWEST[dtype]                                      # all at the lowest value
    x[5, ::3] = math.nan
    x[6] = math.nan
    x[7, [70, 4000]] = math.inf
    x[8] = -math.inf
    x[8, 4321] = -3.0                                         # one left
    x[9] = torch.where(torch.rand(V, generator=g) < 0.5, -math.inf, 4.0)
    x[10] = torch.arange(V, 0, -1) / 100.0                    # in order
    x[11] = torch.where(torch.arange(V) < 300, 2.0, 1.0)
    x = x.to(dtype).repeat(times, 1)
    for u in (0.0, 0.25, 0.5, 1.0 - 2.0 ** -24, 1.0):
        check_sample(x, torch.full((12 * times,), u), **settings)
    check_sample(x, uniforms(12 * times, 3), **settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 30, 50])
def test_sample_more_equal_values_than_a_list_holds(dtype, N):
    x = torch.zeros(N, 32003)
    x[:, 20000:20020] = 1.0
    x[:, ::2] -= 1.0
    for k in (10, 50, 500):
        check_sample(x.to(dtype), uniforms(N, k), k=k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_views(dtype):
    wide = rows(80, 8801, dtype, 8).cuda().view(40, 2, 8801)
    for view in (wide[:, -1], wide[:, 0, 1:], wide[:, 1, 3:-2], wide[1, 1].expand(40, 8801)):
        check_sample(view.cpu(), uniforms(40, 9), k=20, p=0.9, dev=view)
        check_sample(view.cpu(), uniforms(40, 9), dev=view)
    big = rows(6 * 3, 700, dtype, 8).cuda().view(6, 3, 700)
    u = uniforms(6, 8)
    for view in (big[:, -1, :], big[:, 1, 1:], big[:, 0, 5:-3], big[:, 0, :1].expand(6, 1), big[0, 0, :].expand(6, 700),
                 big[:, :, 3].t()[:, :].t()):
        check_sample(view.cpu(), u, k=20, p=0.9, dev=view)
        check_sample(view.cpu(), u, p=0.9, dev=view)
    tokens = ext.sample(big.permute(1, 0, 2), u.cuda().expand(3, 6))
    assert tokens.shape == (3, 6)
    want = ref.sample(big.permute(1, 0, 2).reshape(18, 700), u.repeat(3).numpy(), np.ones(18), np.zeros(18), np.ones(18), np.zeros(18))
    assert tokens.cpu().reshape(-1).tolist() == want.tolist()
    assert ext.sample(big[:0, 0], u[:0].cuda()).shape == (0,)
    one = ext.sample(big[0, 0], u[0].cuda(), top_k=5)         # one row without leading dimensions
    assert one.shape == ()


@pytest.mark.parametrize("V,dtype", [(256000, torch.float32), (256001, torch.bfloat16), (750000, torch.float32), (1_499_999, torch.float16)])
def test_sample_long_rows(V, dtype):
    x, u = rows(2, V, dtype, 9), uniforms(2, 9)
    check_sample(x, u, T=0.9)
    check_sample(x, u, k=100, p=0.95)
    check_sample(x, u, p=0.9)


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 1e3, 3e38])
def test_sample_temperatures(temperature):
    for dtype in DTYPES:
        x, u = rows(5, 3001, dtype, 2), uniforms(5, 2)
        x[0] = 0.5
        check_sample(x, u, T=temperature)
        check_sample(x, u, T=temperature, p=0.9)
        check_sample(x, u, T=temperature, k=30, q=0.5)


def check_top(x, n, temperature=1.0, dev=None):
    want, tokens = ref.top_log_probs(x, n, temperature)
    want = np.where(want < -np.finfo(np.float32).max, -np.inf, want)   # a masked value over 1e-30 is beyond float32
    got, at = ext.top_log_probs(x.cuda() if dev is None else dev, n, temperature=temperature)
    assert got.dtype == torch.float32 and at.dtype == torch.int32
    assert np.array_equal(at.cpu().numpy(), tokens)
    got = got.cpu().double().numpy()
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    fine = np.isfinite(want)
    assert np.all(np.abs(got - want)[fine] <= ref.top_bound(want)[fine])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,n", [(3, 1, 1), (4, 7, 7), (5, 100, 20), (20, 1025, 1024), (2, 32000, 1), (7, 32000, 64), (300, 2000, 33),
                                   (2, 50257, 1000), (1, 128256, 128), (2, 256000, 256),
                                   (40, 32000, 1), (50, 32000, 64), (33, 50257, 256), (34, 128256, 20), (32, 8200, 100)])
def test_top_log_probs(N, V, n, dtype):
    check_top(rows(N, V, dtype, V + n), n)
    check_top(rows(N, V, dtype, V + n), n, temperature=1.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 13, 300])
@pytest.mark.parametrize("V,times", [(6001, 1), (10001, 3)])
def test_top_log_probs_ties_and_masks(V, times, dtype, n):
    x = torch.round(rows(11, V, torch.float32, 6))
    x[0] = 0.0
    x[1] = -math.inf
    x[2, 10:] = -math.inf
    x[3, 40:] = LOWEST[dtype]
    x[4] = LOWEST[dtype]
    x[5, ::3] = math.nan
    x[6] = math.nan
    x[7] = torch.arange(V, 0, -1) / 100.0
    x[8] = torch.arange(V) / 100.0
    x[9] = -50.0
    x[9, 4321] = 60.0
    x[10] = torch.where(torch.arange(V) % 2048 < 5, 3.0, -1.0)   # the best ones in one thread's hands
    check_top(x.to(dtype).repeat(times, 1), n)


def test_top_log_probs_views():
    wide = rows(80, 8801, torch.bfloat16, 4).cuda().view(40, 2, 8801)
    for view in (wide[:, -1], wide[:, 0, 1:], wide[:, 1, 3:-2], wide[1, 1].expand(40, 8801)):
        check_top(view.cpu(), 17, dev=view)
    big = rows(30, 801, torch.bfloat16, 4).cuda().view(5, 6, 801)
    for view in (big[:, -1], big[:, 2, 1:], big[:, 2, 3:-2], big[1, 1].expand(4, 801)):
        check_top(view.cpu(), 17, dev=view)
    values, tokens = ext.top_log_probs(big.transpose(0, 1), 4)
    assert values.shape == tokens.shape == (6, 5, 4)
    values, tokens = ext.top_log_probs(big[:0], 4)
    assert values.shape == (0, 6, 4)


def teacher(N, V, n, seed, pad=0.2, repeat=False):
    g = torch.Generator().manual_seed(seed + 77)
    z = torch.randn((N, V), generator=g) * 3.0
    lq, at = torch.log_softmax(z, dim=1).topk(n, dim=1)
    at = at.clone()
    if pad:
        at[torch.rand((N, 1), generator=g).expand(N, n) < pad] = -1
        at[torch.rand((N, n), generator=g) < 0.1] = V + 5
    if repeat and n > 2:
        at[:, 2] = at[:, 0]
        at[::2, n - 1] = at[::2, 0]
    return lq, at


def check_distill(x, lq, at, T=1.0, tail=True, reduction="mean", scale=1.0, dev=None, token_type=torch.int32, weight=None):
    """Loss and gradient; `weight`: the loss is multiplied by it before the backward."""
    want, has, grad, size = ref.distill(x, lq, at, T, tail)
    count = max(1, has.sum())
    spread = np.maximum(np.abs(np.where(np.isfinite(lq.double().numpy()), lq.double().numpy(), 0)).max(axis=1), 60.0)
    bound = ref.loss_bound(want, spread) * abs(scale)
    leaf = (x.cuda() if dev is None else dev).detach().requires_grad_(True)
    loss = ext.distillation_loss(leaf, lq.cuda(), at.to(token_type).cuda(), temperature=T, tail=tail, reduction=reduction, scale=scale)
    assert loss.dtype == torch.float32
    factor = np.full(len(want), scale / (count if reduction == "mean" else 1.0))
    total = loss
    if weight is not None:
        total = loss * torch.as_tensor(weight, dtype=torch.float32, device="cuda")
        factor = factor * np.asarray(weight, dtype=np.float64)
    got, = torch.autograd.grad(total.sum(), leaf)
    assert got.dtype == x.dtype and got.shape == x.shape
    value = loss.detach().cpu().double().numpy()
    if reduction == "none":
        assert np.array_equal(np.isinf(value), np.isinf(want))
        fine = np.isfinite(want)
        assert np.all(np.abs(value - scale * want)[fine] <= bound[fine])
        assert np.all(value[~has] == 0.0)
    elif np.isfinite(want).all():
        divide = count if reduction == "mean" else 1.0
        assert abs(value - scale * want.sum() / divide) <= bound.sum() / divide + 2.0 ** -23 * abs(value)
    got = got.cpu().double().numpy()
    want_grad = grad * factor[:, None]
    assert np.all(got[~has] == 0.0)
    off = np.abs(got - want_grad) - ref.grad_bound(want_grad, size, np.abs(factor)[:, None], x.dtype)
    assert off.max() <= 0.0, (off.max(), np.unravel_index(off.argmax(), off.shape))
    with torch.no_grad():     # the pass without a gradient gives the same loss
        alone = ext.distillation_loss(leaf, lq.cuda(), at.to(token_type).cuda(), temperature=T, tail=tail, reduction=reduction, scale=scale)
    assert torch.equal(alone, loss.detach()) or not np.isfinite(value).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N,V,n", [(1, 1, 1), (4, 7, 3), (5, 9, 9), (33, 100, 20), (20, 1025, 1), (3, 32000, 64), (400, 257, 33), (2, 50257, 1000)])
def test_distillation(N, V, n, dtype, tail, reduction):
    x = rows(N, V, dtype, V + n)
    lq, at = teacher(N, V, n, V)
    check_distill(x, lq, at, tail=tail, reduction=reduction)
    check_distill(x, lq, at, T=2.0, tail=tail, reduction=reduction, scale=4.0, token_type=torch.int64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_same_token_twice(dtype, tail):
    x = rows(30, 900, dtype, 3)
    lq, at = teacher(30, 900, 40, 3, repeat=True)
    check_distill(x, lq - 1.0, at, tail=tail, reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_masks(dtype, tail):
    N, V, n = 12, 4001, 16
    x = rows(N, V, torch.float32, 4)
    lq, at = teacher(N, V, n, 4, pad=0.0)
    x[0, 2000:] = -math.inf                       # listed ones among them: an infinite loss
    x[1] = -math.inf
    x[2, 3000:] = LOWEST[dtype]
    x[3] = LOWEST[dtype]
    x[4] = math.nan
    at[4] = -1                                    # nothing is asked of a row of NaN
    x[5, 17:] = -math.inf                         # all tokens left are listed: no tail
    at[5] = torch.arange(n)
    lq[6] = -math.inf                             # a teacher without mass
    lq[7, 1:] = -math.inf
    lq[7, 0] = 0.0                                # all mass on one token
    x[8, ::2] = -math.inf
    lq[8] = torch.where(at[8] % 2 == 0, -math.inf, lq[8])   # nothing on the masked ones
    at[9] = V
    x[10] *= 30.0
    x[11, :] = 5.0
    check_distill(x.to(dtype), lq, at, tail=tail, reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction,weight", [("mean", 0.37), ("sum", -2.0), ("mean", 0.0), ("none", "rows"), ("mean", 65536.0)])
def test_distillation_weighted(dtype, reduction, weight):
    x = rows(24, 1234, dtype, 7)
    lq, at = teacher(24, 1234, 20, 7)
    if weight == "rows":
        weight = torch.linspace(-1.0, 3.0, 24)
        weight[::4] = 1.0
        weight = weight.numpy()
    check_distill(x, lq, at, reduction=reduction, weight=weight)


def test_distillation_backward_twice():
    x = rows(24, 1234, torch.bfloat16, 7).cuda().requires_grad_(True)
    lq, at = (t.cuda() for t in teacher(24, 1234, 20, 7))
    loss = ext.distillation_loss(x, lq, at)
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss, x, retain_graph=True)
    assert second.data_ptr() != first.data_ptr()
    assert torch.equal(first, kept) and torch.equal(first, second)
    third, = torch.autograd.grad(3.0 * loss, x)
    assert torch.equal(first, kept)
    assert torch.allclose(third.float(), 3.0 * kept.float(), rtol=2.0 ** -7, atol=0.0)   # two roundings of half a step each
    (loss_b := ext.distillation_loss(x, lq, at)).backward()
    (ext.distillation_loss(x, lq, at)).backward()
    assert torch.equal(x.grad, kept + kept)
    assert torch.equal(loss_b.detach(), loss.detach())


def test_distillation_logits_changed_in_place():
    leaf = rows(4, 100, torch.float32, 7).cuda().requires_grad_(True)
    x = leaf * 1.0
    lq, at = (t.cuda() for t in teacher(4, 100, 5, 7))
    loss = ext.distillation_loss(x, lq, at)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_views(dtype):
    big = rows(40, 803, dtype, 12).cuda().view(8, 5, 803)
    for view in (big[:, -1], big[:, 2, 1:], big[:, 2, 3:-2], big[:, 0, ::2], big[0, 0].expand(6, 803)):
        lq, at = teacher(view.shape[0], view.shape[1], 9, 12)
        x = view.cpu()
        want, has, grad, size = ref.distill(x, lq, at, 1.0, True)
        leaf = view.detach().requires_grad_(True)
        loss = ext.distillation_loss(leaf, lq.cuda(), at.cuda(), reduction="none")
        assert np.all(np.abs(loss.detach().cpu().double().numpy() - want) <= ref.loss_bound(want, 60.0))
        got, = torch.autograd.grad(loss.sum(), leaf)
        got = got.cpu().double().numpy()
        assert np.all(np.abs(got - grad) <= ref.grad_bound(grad, size, 1.0, dtype))
    lq, at = teacher(40, 803, 9, 12)
    leaf = big.transpose(0, 1).detach().requires_grad_(True)      # leading dimensions that do not merge
    loss = ext.distillation_loss(leaf, lq.view(5, 8, 9).cuda(), at.view(5, 8, 9).cuda())
    loss.backward()
    want, has, grad, size = ref.distill(big.transpose(0, 1).reshape(40, 803), lq, at, 1.0, True)
    got = leaf.grad.reshape(40, 803).cpu().double().numpy()
    assert np.all(np.abs(got - grad / has.sum()) <= ref.grad_bound(grad / has.sum(), size, 1.0 / has.sum(), dtype))


def test_distillation_empty_batches():
    x = torch.empty(0, 50, device="cuda", requires_grad=True)
    lq, at = torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda")
    for reduction in ("sum", "mean"):
        loss = ext.distillation_loss(x, lq, at, reduction=reduction)
        assert loss.item() == 0.0
        assert torch.autograd.grad(loss, x)[0].shape == (0, 50)
    assert ext.distillation_loss(x, lq, at, reduction="none").shape == (0,)
    x = torch.full((5, 50), math.nan, device="cuda", requires_grad=True)     # all padding
    loss = ext.distillation_loss(x, torch.zeros(5, 3, device="cuda"), torch.full((5, 3), -1, device="cuda"))
    assert loss.item() == 0.0
    assert torch.count_nonzero(torch.autograd.grad(loss, x)[0]).item() == 0


def test_distillation_gradient_against_differences():
    """The loss along a direction d: (L(x + h d) - L(x - h d)) / 2h differs from <grad, d> by the loss' own bound / h and by the third
    derivative's share, at most h^2 (a softmax's derivatives along |d| <= 1 stay below 6)."""
    x = rows(20, 300, torch.float32, 21).double()
    lq, at = teacher(20, 300, 12, 21)
    g = torch.Generator().manual_seed(2)
    d = torch.rand((20, 300), generator=g, dtype=torch.float64) * 2.0 - 1.0
    for T, tail in ((1.0, True), (2.0, False)):
        leaf = x.float().cuda().requires_grad_(True)
        kw = dict(temperature=T, tail=tail, reduction="none")
        loss = ext.distillation_loss(leaf, lq.cuda(), at.cuda(), **kw)
        grad, = torch.autograd.grad(loss.sum(), leaf)
        h = 0.02
        there = [ext.distillation_loss((x + s * h * d).float().cuda(), lq.cuda(), at.cuda(), **kw).double().cpu() for s in (1, -1)]
        slope = (there[0] - there[1]) / (2.0 * h)
        inner = (grad.double().cpu() * d).sum(dim=1)
        want = ref.distill(x, lq, at, T, tail)[0]
        # the shifted logits are rounded to 32 bits: |x| 2^-24 below 2e-6 each, through a gradient of 1-norm at most 2
        bound = (torch.from_numpy(ref.loss_bound(want, 60.0)) + 4e-6) / h + h * h
        assert torch.all((slope - inner).abs() <= bound)


def test_together():
    """On-policy distillation: tokens drawn by the student, a teacher's top log-probs of the same places, the loss and its gradient;
    then the beams of the same rows through final_scores."""
    B, T, V, n = 3, 4, 1500, 16
    student = rows(B * T, V, torch.bfloat16, 30).cuda().view(B, T, V).requires_grad_(True)
    tutor = rows(B * T, V, torch.bfloat16, 31).cuda().view(B, T, V)
    u = uniforms(B * T, 30).cuda().view(B, T)
    tokens = ext.sample(student, u, temperature=0.8, top_k=40, top_p=0.95)
    assert tokens.shape == (B, T) and int(tokens.min()) >= 0 and int(tokens.max()) < V
    lq, at = ext.top_log_probs(tutor, n, temperature=2.0)
    at[0, -1] = -1                                           # the last place of the first sequence is padding
    loss = ext.distillation_loss(student, lq, at, temperature=2.0, scale=4.0)
    loss.backward()
    want, has, grad, size = ref.distill(student.reshape(-1, V), lq.reshape(-1, n).cpu(), at.reshape(-1, n), 2.0, True)
    factor = 4.0 / has.sum()
    assert has.sum() == B * T - 1
    assert abs(loss.item() - factor * want.sum()) <= factor * ref.loss_bound(want, 60.0).sum() + 2.0 ** -23 * abs(loss.item())
    got = student.grad.reshape(-1, V).cpu().double().numpy()
    assert np.all(np.abs(got - factor * grad) <= ref.grad_bound(factor * grad, size, factor, torch.bfloat16))
    # the best tokens' list and the beam search agree on the best first token
    log_probs = torch.log_softmax(student.detach().float(), dim=-1)[:, :, None, :].expand(B, T, 2, V).contiguous()
    beams, _ = ext.decode(log_probs, ext.DBSOptions(beam_size=2))
    best = ext.top_log_probs(log_probs[:, 0, 0], 2)[1]
    assert torch.equal(beams[:, 0, :].cpu(), best.cpu())


def test_cpu_tensors_come_back_to_the_cpu():
    x = rows(4, 300, torch.float32, 1)
    u = uniforms(4, 1)
    tokens = ext.sample(x, u, top_k=10)
    assert tokens.device.type == "cpu"
    assert torch.equal(tokens, ext.sample(x.cuda(), u.cuda(), top_k=10).cpu())
    values, at = ext.top_log_probs(x, 5)
    assert values.device.type == at.device.type == "cpu"
    leaf = x.clone().requires_grad_(True)
    loss = ext.distillation_loss(leaf, values, at)
    assert loss.device.type == "cpu"
    loss.backward()
    assert leaf.grad.device.type == "cpu" and leaf.grad.abs().max() < 1e-5   # a student that is its own teacher


def test_another_stream_and_two_at_once():
    x = rows(64, 9000, torch.bfloat16, 40).cuda()
    u = uniforms(64, 40).cuda()
    want = ext.sample(x, u, top_k=30), ext.top_log_probs(x, 30), ext.sample(x, u, top_p=0.9)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in side:
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append((ext.sample(x, u, top_k=30), ext.top_log_probs(x, 30), ext.sample(x, u, top_p=0.9)))
    torch.cuda.synchronize()
    for a, (v, t), b in got:
        assert torch.equal(a, want[0]) and torch.equal(v, want[1][0]) and torch.equal(t, want[1][1]) and torch.equal(b, want[2])


def test_captured_and_replayed():
    x = rows(36, 9000, torch.float32, 50).cuda()
    u = uniforms(36, 50).cuda()
    lq, at = (t.cuda() for t in teacher(36, 9000, 10, 50))

    def step():
        leaf = x.detach().requires_grad_(True)
        loss = ext.distillation_loss(leaf, lq, at)
        return (ext.sample(x, u, top_k=20, top_p=0.9), ext.sample(x, u, temperature=1.2), *ext.top_log_probs(x, 7), loss.detach(),
                torch.autograd.grad(loss, leaf)[0], torch.autograd.grad(2.0 * ext.distillation_loss(leaf, lq, at), leaf)[0])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (51, 52):
        x.copy_(rows(36, 9000, torch.float32, seed))
        u.copy_(uniforms(36, seed))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_repeated_calls_give_the_same_bits():
    x = rows(100, 7000, torch.bfloat16, 60).cuda()
    lq, at = (t.cuda() for t in teacher(100, 7000, 50, 60, repeat=True))
    first = None
    for _ in range(5):
        leaf = x.detach().requires_grad_(True)
        loss = ext.distillation_loss(leaf, lq, at)
        now = (loss.detach(), torch.autograd.grad(loss, leaf)[0], *ext.top_log_probs(x, 40))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_rows_behind_the_last_stay_as_they_are():
    import ctypes
    lib = ext._library()
    x = rows(5, 333, torch.float32, 70).cuda()
    tokens = torch.full((8, 4), 7, dtype=torch.int32, device="cuda")
    values = torch.full((8, 4), 7.0, device="cuda")
    grad = torch.full((8, 333), 7.0, device="cuda")
    losses, loss = torch.full((8,), 7.0, device="cuda"), torch.empty((), device="cuda")
    at, lq = torch.zeros(5, 2, dtype=torch.int32, device="cuda"), torch.full((5, 2), -1.0, device="cuda")
    size = ctypes.c_int64()
    assert lib.dbs_device_distill_state_bytes(5, 2, size) == 0
    state = torch.full((size.value + 64,), 7, dtype=torch.uint8, device="cuda")
    s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = ext._vp
    assert lib.dbs_device_top_log_probs(p(x), 0, 5, 333, 333, 4, 1.0, p(values), p(tokens), None, s) == 0
    assert lib.dbs_device_distill(p(x), 0, 5, 333, 333, p(lq), p(at), 4, 2, 1.0, 1, 1, 1.0, p(losses), p(loss), p(state), p(grad), s) == 0
    torch.cuda.synchronize()
    assert torch.all(values[5:] == 7.0) and torch.all(tokens[5:] == 7) and torch.all(grad[5:] == 7.0) and torch.all(losses[5:] == 7.0)
    assert torch.all(tokens[:5] >= 0) and torch.all(state[size.value:] == 7)


@pytest.mark.parametrize("N,V,dtype", [(33, 520_000, torch.float32), (32, 600_000, torch.float32), (33, 1_048_570, torch.bfloat16),
                                       (32, 1_300_001, torch.float16)])
def test_batches_of_long_rows(N, V, dtype):
    """Rows of as many parts as the scan puts together, and of more."""
    x, u = rows(N, V, dtype, V), uniforms(N, V)
    dev = x.cuda()
    check_sample(x, u, T=0.9, dev=dev)
    check_sample(x, u, k=100, p=0.95, dev=dev)
    check_sample(x, u, p=0.5, dev=dev)
    check_top(x, 40, dev=dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [3, 40])
def test_sample_ratio_at_the_ends_of_the_type(N, dtype):
    x = torch.full((N, 9001), LOWEST[dtype], dtype=dtype)
    x[:, 77::100] = torch.finfo(dtype).max
    x[:, 5::1000] = torch.finfo(dtype).max / 2
    u = uniforms(N, 1)
    for T in (1.0, torch.finfo(dtype).max):
        for q in (0.5, 0.7, 0.99):
            check_sample(x, u, T=T, q=q)
            check_sample(x, u, T=T, q=q, p=0.5)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N", [512, 513, 9000])
def test_distillation_of_many_rows(N, reduction):
    lq, at = teacher(N, 130, 5, N)
    check_distill(rows(N, 130, torch.bfloat16, N), lq, at, reduction=reduction)


def test_distillation_has_no_second_derivative():
    x = rows(6, 500, torch.float32, 7).cuda().requires_grad_(True)
    lq, at = (t.cuda() for t in teacher(6, 500, 9, 7))
    plain, = torch.autograd.grad(ext.distillation_loss(x, lq, at), x)
    again, = torch.autograd.grad(ext.distillation_loss(x, lq, at), x, create_graph=True)
    assert torch.equal(plain, again)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        torch.autograd.grad(again.sum(), x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [3, 40])
@pytest.mark.parametrize("temperature", [1e-30, 1e30])
def test_temperatures_at_their_ends(N, dtype, temperature):
    x = rows(N, 9001, torch.float32, 11)
    x[0] = 2.5
    x[1, 3:] = LOWEST[dtype]
    x[2, :40] = torch.finfo(dtype).max
    x = x.to(dtype)
    check_top(x, 20, temperature=temperature)
    lq, at = teacher(N, 9001, 6, 11, pad=0.0)
    x[:3] = 1.5                                   # (losses below stay finite in 32 bits)
    if temperature > 1.0:
        check_distill(x, lq, at, T=temperature, scale=1e30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [12, 48])
def test_rows_far_from_zero(N, dtype):
    """Masks of any size that leave nothing, and logits with a common offset."""
    x = rows(N, 9001, torch.float32, 13)
    for r, size in enumerate((1e4, 1e6, 1e8, 1e9, 1e10, 1e12, 1e15, 1e20, 1e30)):
        x[r] = -size
        x[r, 100 * r:100 * r + 7] = -size * (1.0 - 2.0 ** -6)
    x[9] += 3e5
    x[10] -= 3e5
    x = x.to(dtype)
    check_top(x, 30)
    check_top(x, 30, temperature=0.3)
    for settings in (dict(), dict(k=20), dict(p=0.7), dict(q=0.3)):
        check_sample(x, uniforms(N, 13), **settings)
    lq, at = teacher(N, 9001, 6, 11, pad=0.0)
    at[:9, 0] = 100 * torch.arange(9)            # the best class
    lq[:9, 0], lq[:9, 1:] = 0.0, -math.inf
    check_distill(x, lq, at, reduction="none")


def scanned(dtype, V=40003):
    """Twelve rows (the kinds of the tests above), and as often as a batch is repeated that is scanned."""
    g = torch.Generator().manual_seed(8)
    x = rows(12, V, torch.float32, 8)
    x[0] = torch.round(x[0])
    x[1] = -math.inf
    x[2, 10:] = -math.inf
    x[3, 40:] = LOWEST[dtype]
    x[4] = LOWEST[dtype]
    x[5, ::3] = math.nan
    x[6, [70, 4000]] = math.inf
    x[7] = torch.where(torch.rand(V, generator=g) < 0.5, -math.inf, 4.0)
    x[8] = torch.arange(V, 0, -1) / 100.0
    x[9] = torch.where(torch.arange(V) < 300, 2.0, 1.0)
    x = x.to(dtype)
    return x, -(-21_000_000 // (12 * V * x.element_size()))


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_scanned(dtype, settings):
    x, times = scanned(dtype)
    dev = x.cuda().repeat(times, 1)

    def col(name, default, of):
        return np.full(12, settings.get(name, default), dtype=of)

    for u in (torch.zeros(12), torch.full((12,), 1.0 - 2.0 ** -24), torch.ones(12), uniforms(12, 4)):
        want = ref.sample(x, u.numpy(), col("T", 1.0, np.float32), col("k", 0, np.int32), col("p", 1.0, np.float32), col("q", 0.0, np.float32))
        got = ext.sample(dev, u.cuda().repeat(times), temperature=settings.get("T", 1.0), top_k=settings.get("k", 0),
                         top_p=settings.get("p", 1.0), min_p=settings.get("q", 0.0))
        assert got.cpu().view(times, 12).tolist() == [want.tolist()] * times


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_scanned_with_settings_of_each_row(dtype):
    N = 130 if dtype == torch.float32 else 260
    g = torch.Generator().manual_seed(N)
    T = torch.rand(N, generator=g) * 1.5
    T[::7] = 0.0
    k = torch.randint(0, 80, (N,), generator=g, dtype=torch.int32)
    k[::5] = 0
    k[3::11] = 700
    p = torch.rand(N, generator=g) * 1.3
    q = torch.rand(N, generator=g) * 0.2
    q[::3] = 0.0
    check_sample(rows(N, 40003, dtype, N), uniforms(N, N), T, k, p, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 13, 64, 256])
def test_top_log_probs_scanned(n, dtype):
    x, times = scanned(dtype)
    x[6] = -50.0
    x[6, 4321] = 60.0
    dev = x.cuda().repeat(times, 1)
    check_top(x, n)
    want = ext.top_log_probs(x.cuda(), n)
    got = ext.top_log_probs(dev, n)
    assert torch.equal(got[1].view(times, 12, n), want[1].expand(times, 12, n))
    values = got[0].view(times, 12, n).double().cpu().numpy()
    want, _ = ref.top_log_probs(x, n, 1.0)
    fine = np.broadcast_to(np.isfinite(want), values.shape)
    assert np.array_equal(np.isfinite(values), fine)
    assert np.all(np.abs(values - want)[fine] <= np.broadcast_to(ref.top_bound(want), values.shape)[fine])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(1, 300_001), (3, 555_555)])
def test_few_long_rows(N, V, dtype):
    x, u = rows(N, V, dtype, 6), uniforms(N, 6)
    for settings in (dict(), dict(k=30, p=0.9), dict(p=0.6), dict(q=0.2), dict(p=0.9, q=0.05), dict(T=0.0)):
        check_sample(x, u, **settings)
    for n in (1, 128):
        check_top(x, n)


def test_scanned_on_two_streams_and_captured():
    x = rows(300, 20011, torch.float32, 40).cuda()
    u = uniforms(300, 40).cuda()

    def step():
        return ext.sample(x, u, top_k=30), ext.sample(x, u, top_p=0.9, min_p=0.02), ext.sample(x, u), *ext.top_log_probs(x, 30)

    want = step()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in side:
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append(step())
    torch.cuda.synchronize()
    for many in got:
        assert all(torch.equal(a, b) for a, b in zip(many, want))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(step())
    x.copy_(rows(300, 20011, torch.float32, 41))
    want = step()
    for s, graph in zip(side, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for many in held:
        assert all(torch.equal(a, b) for a, b in zip(many, want))


def test_settings_given_as_tensors_are_read_at_each_call():
    x, u = rows(4, 900, torch.float32, 3).cuda(), uniforms(4, 3).cuda()
    n, T = torch.tensor(3), torch.tensor(0.5)
    k = torch.tensor(2, dtype=torch.int32, device="cuda")
    for i in range(3):
        values, tokens = ext.top_log_probs(x, n, temperature=T)
        want = ext.top_log_probs(x, 3 + i, temperature=0.5 + i)
        assert torch.equal(values, want[0]) and torch.equal(tokens, want[1])
        assert torch.equal(ext.sample(x, u, temperature=T, top_k=k), ext.sample(x, u, temperature=0.5 + i, top_k=2 + i))
        n += 1
        T += 1.0
        k += 1
