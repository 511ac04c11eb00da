"""Rows, settings and lists at the ends of what the operators on rows of logits
accept (sample, top_log_probs, distillation_loss), against their definitions
in 64 bits."""
import math

import numpy as np
import pytest
import torch

import logits_reference as ref
import torch_dbs_extension as ext
from test_gpu_logits import DTYPES, check_distill, check_sample, check_top, rows, teacher, uniforms

pytestmark = pytest.mark.gpu


def below_zero(N, V, dtype, seed):
    """Rows whose maximum is exactly 0 (once, or several times), as logits are after their maximum has been taken off."""
    x = rows(N, V, torch.float32, seed)
    x = (x - x.amax(dim=1, keepdim=True)).to(dtype)
    x[1, 5::1000] = 0.0
    x[2, :] = 0.0
    x[3, 1:] = -math.inf
    x[3, 0] = 0.0
    return x


def check_sample_repeated(x, times, u, T, p=1.0):
    """A batch of `times` copies of the rows x, for rows that only a large batch gives to the scan."""
    N = len(x)
    want = ref.sample(x, u.numpy(), T.numpy(), np.zeros(N, dtype=np.int32), np.full(N, p, dtype=np.float32), np.zeros(N, dtype=np.float32))
    dev, du = x.cuda().repeat(times, 1), u.cuda().repeat(times)
    alike = bool((T == T[0]).all())
    for given in [T.cuda().repeat(times)] + ([float(T[0])] if alike else []):
        got = ext.sample(dev, du, temperature=given, top_p=p)
        assert got.cpu().view(times, N).tolist() == [want.tolist()] * times


@pytest.mark.parametrize("p", [1.0, 0.9])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_scanned_temperatures_at_their_ends(dtype, p):
    """12 rows of 20011, 25 times over: 12 MB and more, which is scanned."""
    x, u = below_zero(12, 20011, dtype, 5), uniforms(12, 5)
    ends = [2.0 ** -149, 1e-38, 1.3e-37, 1.4e-37, 1e-33, 1e-30, 1e-3, 1e3, 1e30, 3e38]
    for T in ends:
        check_sample_repeated(x, 25, u, torch.full((12,), T), p)
    mixed = torch.tensor((ends + [0.0, 1.0]), dtype=torch.float32)
    check_sample_repeated(x, 25, u, mixed, p)


@pytest.mark.parametrize("N,times", [(8, 1), (12, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [3e-39, 1e-38, 1e-37, 2.6e-37, 3e-37, 1e-36])
def test_sample_logits_as_small_as_the_temperature(N, times, dtype, T):
    """Logits of a few T, so that several tokens have a weight whatever T is."""
    g = torch.Generator().manual_seed(3)
    x = (-8.0 * T * torch.rand((N, 20011), generator=g, dtype=torch.float64)).to(dtype)
    x[0] = torch.where(torch.rand(20011, generator=g) < 0.5, -T, 2.0 * T).to(dtype)
    x[1] += 1.0          # what is left of the differences are ties, or steps of many T
    for p in (1.0, 0.7):
        check_sample_repeated(x, times, uniforms(N, 9), torch.full((N,), T), p)
    check_sample(x, uniforms(N, 9), T=T, k=700)


@pytest.mark.parametrize("n", [2, 64, 128, 129, 1024])
def test_distillation_one_token_twice_among_many(n):
    """In each row two slots far from or next to one another have one token; the others have tokens of their own."""
    N, V = 512, 9000
    g = torch.Generator().manual_seed(n)
    at = torch.stack([torch.randperm(V, generator=g)[:n] for _ in range(N)])
    pair = torch.stack([torch.randperm(n, generator=g)[:2] for _ in range(N)])
    at[torch.arange(N), pair[:, 1]] = at[torch.arange(N), pair[:, 0]]
    lq = torch.log_softmax(torch.randn((N, n), generator=g), dim=1) - 0.5
    x = rows(N, V, torch.float32, n)
    check_distill(x, lq, at, reduction="none")
    leaf = x.cuda().requires_grad_(True)
    lq, at = lq.cuda(), at.cuda()
    first = None
    for _ in range(200):     # what the slots' threads see of one another may come in any order
        loss = ext.distillation_loss(leaf, lq, at, reduction="none")
        now = loss.detach(), torch.autograd.grad(loss.sum(), leaf)[0]
        first = first or now
        assert torch.equal(first[0], now[0]) and torch.equal(first[1], now[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("high", [40.0, 62.0, 64.5])
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_rows_that_rise(dtype, high, tail):
    """Each thread's first vectors at 0, the others far above them, and a listed token so far above both that a factor between
    the first vectors' scale and the row's is below 2^-126."""
    V = 16000 if dtype == torch.float32 else 32000
    x = torch.full((80, V), high)
    x[:, :V // 4 + 96] = 0.0
    x += 0.25 * torch.rand((80, V), generator=torch.Generator().manual_seed(1))
    x[:, V - 7] = 90.0
    x[::2, V - 9] = 89.0
    lq = torch.tensor([math.log(0.999), -math.inf]).expand(80, 2).contiguous()
    at = torch.tensor([V - 7, -1]).expand(80, 2).contiguous()
    check_distill(x.to(dtype), lq, at, tail=tail, reduction="none")
    at = torch.tensor([3, V // 2]).expand(80, 2).contiguous()
    check_distill(x.to(dtype), lq, at, tail=tail, reduction="none")


def test_top_log_probs_long_sums():
    """A row of the most elements: a large term, then more small ones than a sum in 32 bits may take (each below half a step of it)."""
    V, S = 1_499_999, 93760          # 16 slices; a thread's first vector is one of a slice's first 256
    i = torch.arange(V)
    x = torch.full((1, V), -16.640625)
    x[0, (i % S < 2048) & (i % 8 < 2)] = 0.0
    check_top(x.to(torch.float16), 3)


def test_sample_top_k_beyond_32_bits():
    x, u = rows(40, 5000, torch.float32, 1), uniforms(40, 1)
    for k in (2 ** 32 + 5, 2 ** 40, 2 ** 63 - 1, -2 ** 32 + 5, -2 ** 63, 2 ** 31, 7):
        every = ext.sample(x.cuda(), u.cuda(), top_k=torch.full((40,), k, dtype=torch.int64, device="cuda"))
        assert torch.equal(every, ext.sample(x.cuda(), u.cuda(), top_k=max(k, 0)))
    for k in (math.inf, 3e9, -math.inf, -3e9, math.nan, 7.0):
        every = ext.sample(x.cuda(), u.cuda(), top_k=torch.full((40,), k, device="cuda"))
        assert torch.equal(every, ext.sample(x.cuda(), u.cuda(), top_k=7 if k == 7.0 else 0))


def test_no_forward_derivative():
    x = rows(6, 500, torch.float32, 7).cuda()
    lq, at = (t.cuda() for t in teacher(6, 500, 9, 7))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                ext.distillation_loss(dual, lq, at)
        assert torch.equal(ext.distillation_loss(x, lq, at), ext.distillation_loss(x.clone(), lq, at))


def distill_by_logarithms(x, lq, listed, T, tail):
    """Row losses and gradients where the first `listed` tokens are listed: from logarithms, as exponentials near 2^-1074 have few bits
    in 64 (exp(-740) is 85 steps of 2^-1074). A rest's class is one whose exponentials by the row's maximum add up to 2^-1075."""
    z = x.double() / T
    log_P = z - torch.logsumexp(z, dim=1, keepdim=True)
    log_rest = torch.logsumexp(log_P[:, listed:], dim=1)
    q = lq.double().exp()
    q_rest = (1.0 - q.sum(dim=1)).clamp(min=0.0) * (tail and 1.0) * (torch.logsumexp(z[:, listed:], dim=1) - z.amax(dim=1) > -1075.0 * math.log(2.0))
    loss = (q * (lq.double() - log_P[:, :listed])).sum(dim=1)
    loss = loss + torch.where(q_rest > 0, q_rest * (q_rest.log() - log_rest), 0.0)
    total = (q.sum(dim=1) + q_rest)[:, None]
    share = torch.where(q_rest[:, None] > 0, q_rest[:, None] * (log_P - log_rest[:, None]).exp(), 0.0)
    share[:, :listed] = q
    return loss.numpy(), ((total * log_P.exp() - share) / T).numpy(), ((total * log_P.exp() + share) / T).numpy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_all_but_masked_tokens_listed(dtype, tail):
    """What no slot lists is masked: by the lowest value or another far below the rest there is no rest's class (its mass is 0 in 64
    bits), and no gradient there; from 745 T below the maximum on (750 for 3300 tokens together) there is one."""
    V, n = 4000, 700
    masks = [torch.finfo(dtype).min, -math.inf, -3e4, -800.0, -750.0, -740.0, -700.0, -100.0, -5.0]
    x = rows(2 * len(masks), V, dtype, 3).clamp(-20.0, 0.0)
    x[:, 17] = 0.0
    for r, mask in enumerate(masks):
        x[2 * r:2 * r + 2, n:] = mask
    at = torch.arange(n).expand(len(x), n).contiguous()
    lq = torch.log_softmax(x[:, :n].float() + torch.randn((1, n), generator=torch.Generator().manual_seed(2)), dim=1) - 0.7
    for T, one_left in ((1.0, False), (2.0, False), (1.0, True)):
        if one_left:
            x[1::2, n + 9] = -30.0                # one token of the rest is not masked
        want, grad, size = distill_by_logarithms(x, lq, n, T, tail)
        leaf = x.cuda().requires_grad_(True)
        loss = ext.distillation_loss(leaf, lq.cuda(), at.cuda(), temperature=T, tail=tail, reduction="none")
        got, = torch.autograd.grad(loss.sum(), leaf)
        off = np.abs(loss.detach().cpu().double().numpy() - want) - ref.loss_bound(want, 745.0)
        assert off.max() <= 0.0, (off.max(), off.argmax())
        assert np.all(np.abs(got.cpu().double().numpy() - grad) <= ref.grad_bound(grad, size, 1.0, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V", [(4, 60), (4, 3000), (3, 60000), (200, 60000)])
def test_sample_top_p_at_a_border_that_small_weights_move(N, V, dtype):
    """`ties` best tokens, and 40 whose mass (from 1.8e-13 on) times p makes a token more than p * ties of the best ones stay: their
    part of the target is 4e-14 and more, 200 steps of a sum in 64 bits."""
    for ties, p in ((2, 0.5), (4, 0.25), (4, 0.75), (8, 0.875)):
        for low in (-33.0, -31.75, -24.0, -20.5):
            x = torch.full((N, V), -math.inf)
            x[:, 3:3 + ties] = 0.0
            x[:, V - 41:V - 1] = low
            x = x.to(dtype)
            dev = x.cuda()
            for u in (0.05, 0.3, 0.6, 0.95):
                for k in (0, V - 30):     # (the rows are the same)
                    want = ref.sample(x[:1], [np.float32(u)], [1.0], [k], [np.float32(p)], [0.0])
                    got = ext.sample(dev, torch.full((N,), u, device="cuda", dtype=torch.float32), top_p=p, top_k=k)
                    assert got.cpu().tolist() == [int(want[0])] * N
