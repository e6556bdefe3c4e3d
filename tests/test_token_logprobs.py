"""Token log-probabilities, entropy and top alternatives from logits against their definition in 64 bits, with the
gradient against the formula and against differences; on the CPU reference and, marked ``gpu``, on the kernels."""

import math

import pytest
import torch

from rl_project_b200.ops.logprob import token_logprobs

F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request):
    yield request.param
    if request.param == "cuda":  # no test leaves an index error behind
        from rl_project_b200.ops._ext import check_bounds

        check_bounds(torch.device("cuda", 0))


def oracle(x, t, k):
    """(lp, entropy, top log-probs, ids) in fp64; differentiable where the logits are finite or -inf."""
    x = x.to(F64)
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp.masked_fill(p == 0, 0.0), torch.zeros_like(p)).sum(-1)
    ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    lp = torch.where(t >= 0, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros_like(ent))
    return lp, ent, logp.gather(1, ids), ids


def logits(N, V, dtype, spread=4.0):
    x = torch.randn(N, V) * spread
    x.scatter_(1, torch.randint(V, (N, 3)), torch.rand(N, 3) * 12)
    return x.to(dtype)


# fp32 throughout: a log-prob is a difference of two numbers below 2^6, each rounded (2^-18), of which the
# log-sum-exp carries the error of a sum of up to 2^17 terms added pairwise or by 2^9 threads (its log is off by
# less than 2^-15); entropy is a sum of the same kind times log-probs below 2^6.
LP_TOL, ENT_TOL = 2 ** -14, 2 ** -13


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (1, 1, 0), (3, 7, 7), (5, 33, 20), (2, 64, 64), (4, 1000, 5),
                                   (33, 4099, 8), (2, 50257, 20), (1, 128256, 5), (200, 512, 1), (0, 10, 2),
                                   (7, 65536, 40)])
def test_values(dev, dtype, N, V, k):
    x = logits(N, V, dtype)
    t = torch.randint(-1, V, (N,))
    r = token_logprobs(x.to(dev), t.to(dev), top=k)
    lp, ent, top, ids = oracle(x, t, k)
    assert r.logprobs.shape == (N,) and r.top_ids.shape == (N, k) and r.top_ids.dtype == torch.int64
    assert r.logprobs.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32
    assert torch.equal(r.top_ids.cpu(), ids)
    assert ((r.logprobs.cpu().to(F64) - lp).abs() <= LP_TOL).all()
    assert ((r.top_logprobs.cpu().to(F64) - top).abs() <= LP_TOL).all()
    assert ((r.entropy.cpu().to(F64) - ent).abs() <= ENT_TOL).all()
    assert not r.logprobs.cpu()[t < 0].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 3000, 40001])
def test_ties(dev, dtype, V):
    """Equal logits rank by their index: few distinct values, all equal, +0 and -0, and rising and falling rows."""
    x = torch.stack([torch.randint(0, 3, (V,)).float(), torch.full((V,), 1.5), torch.zeros(V),
                     torch.arange(V).float().div(V / 40).floor(), torch.arange(V).flip(0).float().div(V / 40).floor()])
    x[2, ::2] = -0.0
    x = x.to(dtype)
    t = torch.zeros(5, dtype=torch.long)
    r = token_logprobs(x.to(dev), t.to(dev), top=32)
    assert torch.equal(r.top_ids.cpu(), oracle(x, t, 32)[3])
    assert r.top_ids[2].tolist() == list(range(32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 5003])
def test_masked_and_unusual_rows(dev, dtype, V):
    low, inf = torch.finfo(dtype).min, math.inf
    x = logits(9, V, dtype)
    x[0, ::3] = -inf  # masked vocabulary
    x[1, ::3] = low  # the same by the type's lowest value
    x[2, :] = -inf  # nothing left
    x[3, :] = low
    x[4, 7] = math.nan
    x[5, 7] = inf
    x[6, :] = -inf
    x[6, 11] = 2.0  # one token left
    x[7] = (x[7].float() + 1000.0).to(dtype)  # a common offset
    x[8, :] = -inf
    x[8, 5:9] = -300.0
    t = torch.tensor([1, 1, 3, 4, 7, 8, 11, 2, 6])
    x = x.to(dev).requires_grad_()
    r = token_logprobs(x, t.to(dev), top=6)
    xc = x.detach().cpu()
    lp, ent, top, ids = oracle(xc, t, 6)
    lp[2], ent[2], top[2] = -inf, 0.0, -inf
    for got, want, tol in ((r.logprobs, lp, LP_TOL), (r.entropy, ent, ENT_TOL), (r.top_logprobs, top, LP_TOL)):
        got = got.detach().cpu().to(F64)
        nan = torch.zeros(9, dtype=torch.bool)
        nan[4:6] = True
        assert torch.isnan(got[nan]).all() and not torch.isnan(got[~nan]).any()
        same = (got == want) | ((got - want).abs() <= tol * want.abs().clamp(min=1).where(want.isfinite(), torch.ones_like(want)))
        assert same[~nan].all(), (got, want)
    assert torch.equal(r.top_ids.cpu()[[0, 1, 2, 3, 6, 7, 8]], ids[[0, 1, 2, 3, 6, 7, 8]])
    assert r.top_ids[4, 0] == 7 and r.top_ids[5, 0] == 7
    keep = torch.tensor([0, 1, 3, 6, 7, 8], device=dev)
    (r.logprobs[keep].sum() + r.entropy[keep].sum() - r.top_logprobs[keep][:, 0].sum()).backward()
    g = x.grad.cpu()
    assert torch.isfinite(g[[0, 1, 3, 6, 7, 8]]).all() and not g[2].any()
    assert not g[0, ::3].any() and not g[1, ::3].any()


def test_targets_and_layouts(dev):
    """Leading dimensions, rows inside wider ones, columns apart, and rows that start on odd addresses."""
    V = 77
    base = torch.randn(2, 6, V + 9)
    for dtype in TYPES:
        b = base.to(dtype)
        for x in (b[..., :V], b[..., 3:V + 3], b[:, ::2, 1:V + 1], b[..., :V].transpose(0, 1),
                  b.transpose(1, 2)[:, :V].transpose(1, 2), torch.randn(2, V, 6).to(dtype).transpose(1, 2)):
            t = torch.randint(-1, V, x.shape[:-1])
            on = x.to(dev) if dev == "cpu" else b.to(dev).as_strided(x.shape, x.stride(), x.storage_offset()) \
                if x.untyped_storage().data_ptr() == b.untyped_storage().data_ptr() else x.to(dev)
            r = token_logprobs(on, t.to(dev), top=3)
            lp, ent, top, ids = oracle(x.reshape(-1, V), t.reshape(-1), 3)
            assert r.logprobs.shape == t.shape and r.top_logprobs.shape == (*t.shape, 3)
            assert torch.equal(r.top_ids.cpu().view(-1, 3), ids)
            assert ((r.logprobs.cpu().view(-1) - lp).abs() <= LP_TOL).all()
            assert ((r.entropy.cpu().view(-1) - ent).abs() <= ENT_TOL).all()


# The gradient is a few terms of at most |g| (1 + 2^5) with p's relative error 2^-18 (its exponent is below 2^6, held
# in fp32), rounded once to the logits' type.
def check_grad(got, want, x, weight):
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert got.dtype == x.dtype
    err = (got.cpu().to(F64) - want).abs()
    bound = half * want.abs() + tiny + 2 ** -17 * weight[:, None]
    assert (err <= bound).all(), ((err - bound).max(), want.abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,k,use", [(4, 33, 0, "lp"), (4, 33, 5, "lp ent top"), (3, 1000, 4, "ent"),
                                       (2, 4099, 20, "top"), (5, 8, 8, "lp ent top"), (1, 1, 1, "lp ent top"),
                                       (2, 50257, 3, "lp top"), (9, 512, 0, "lp ent")])
def test_gradient_formula(dev, dtype, N, V, k, use):
    x = logits(N, V, dtype)
    t = torch.randint(-1, V, (N,))
    if N > 2:
        t[0] = int(x[0].float().argmax())  # the target is the first alternative too
    g_lp, g_ent, g_top = torch.randn(N), torch.randn(N) * 0.3, torch.randn(N, k)
    xd = x.clone().to(dev).requires_grad_()
    r = token_logprobs(xd, t.to(dev), top=k)
    x64 = x.detach().to(F64).requires_grad_()
    lp, ent, top, _ = oracle(x64, t, k)
    loss, want = 0, 0
    if "lp" in use:
        loss, want = loss + (r.logprobs * g_lp.to(dev)).sum(), want + (lp * g_lp).sum()
    if "ent" in use:
        loss, want = loss + (r.entropy * g_ent.to(dev)).sum(), want + (ent * g_ent).sum()
    if "top" in use:
        loss, want = loss + (r.top_logprobs * g_top.to(dev)).sum(), want + (top * g_top).sum()
    loss.backward()
    want.backward()
    weight = 32 * (g_lp.abs() + g_ent.abs() + g_top.abs().sum(1)).to(F64)
    check_grad(xd.grad, x64.grad, x, weight)


def test_gradient_differences(dev):
    """Central differences of the operator itself: fp32, step 2^-5, so the difference of outputs good to 2^-16 is
    good to 2^-11, and the third derivative adds (2^-5)^2 / 6 times a few: together below 2^-9 of the weights' sum."""
    x = (torch.randn(1, 12) * 1.5).to(dev)
    t = torch.tensor([4], device=dev)
    c = torch.randn(5, device=dev)

    def f(y):
        r = token_logprobs(y, t, top=3)
        return c[0] * r.logprobs.sum() + c[1] * r.entropy.sum() + (c[2:] * r.top_logprobs[0]).sum()

    y = x.clone().requires_grad_()
    f(y).backward()
    for j in range(12):
        d = torch.zeros_like(x)
        d[0, j] = 2 ** -5
        diff = (f(x + d) - f(x - d)) / 2 ** -4
        ids = token_logprobs(x, t, top=3).top_ids
        if all(torch.equal(token_logprobs(x + s * d, t, top=3).top_ids, ids) for s in (-1, 1)):
            assert abs(float(diff - y.grad[0, j])) <= 2 ** -9 * float(c.abs().sum())


def test_gradient_through_views_and_twice(dev):
    """Logits used twice, through a slice of a larger tensor that needs the gradient, in rows of odd length."""
    base = torch.randn(6, 55).to(dev).requires_grad_()
    t = torch.randint(0, 50, (4,)).to(dev)
    a, b = token_logprobs(base[1:5, 3:53], t), token_logprobs(base[1:5, 3:53], t.flip(0), top=2)
    (a.logprobs.sum() + b.entropy.sum() + b.top_logprobs.sum()).backward()
    x = base.detach().cpu().to(F64).requires_grad_()
    o, p = oracle(x[1:5, 3:53], t.cpu(), 0), oracle(x[1:5, 3:53], t.cpu().flip(0), 2)
    (o[0].sum() + p[1].sum() + p[2].sum()).backward()
    assert ((base.grad.cpu().to(F64) - x.grad).abs() <= 2 ** -14).all()


def test_bad_target(dev):
    x, t = torch.randn(3, 10).to(dev), torch.tensor([1, 10, 2]).to(dev)
    if dev == "cpu":
        with pytest.raises(IndexError):
            token_logprobs(x, t)
        return
    from rl_project_b200.core.errors import KernelError
    from rl_project_b200.ops._ext import check_bounds

    x.requires_grad_()
    r = token_logprobs(x, t)
    r.logprobs.sum().backward()
    with pytest.raises(KernelError):
        check_bounds(torch.device("cuda", 0))
    assert r.logprobs[1] == 0 and not x.grad[1].any() and x.grad[0].any()
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    token_logprobs(x, t, status=status)
    assert status.item() != 0


def test_vocabulary_of_one(dev):
    """One column, whatever its stride says: transposed rows, columns of wider ones, expanded rows."""
    t = torch.tensor([0, -1, 0], device=dev)
    wide = torch.randn(3, 5, device=dev)
    for x in (torch.randn(1, 3, device=dev).t(), wide[:, 2:3], wide[:1, :1].expand(3, 1)):
        x = x.detach().requires_grad_()
        r = token_logprobs(x, t, top=1)
        assert not r.logprobs.any() and not r.entropy.any() and not r.top_logprobs.any() and not r.top_ids.any()
        grad, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)
        assert grad.shape == (3, 1) and not grad.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [4099, 50257])
def test_one_logit_dominates(dev, dtype, V):
    """No log-prob above 0 and no entropy below it, wherever the largest logit lies and however far above the others:
    the reference that the sums are taken against is one of the row's own logits."""
    N = 48
    for rest in (-6e4, -60.0, -12.0, -math.inf):
        x = torch.full((N, V), rest) + torch.rand(N, V) * 2
        x[:, 3] = 0.0  # early, and what comes behind lies up to 9 above it
        x.scatter_(1, torch.randint(V // 2, V, (N, 1)), torch.rand(N, 1) * 9)
        x = x.to(dtype)
        r = token_logprobs(x.to(dev), x.argmax(-1).to(dev), top=1)
        lp, ent, _, _ = oracle(x, x.argmax(-1), 1)
        assert (r.logprobs <= 0).all() and (r.top_logprobs <= 0).all() and (r.entropy >= 0).all()
        # (two large terms, but with the rest at -12 also up to 2^16 small ones, each of whose additions to a sum above 1
        # rounds by 2^-24 of it: the sum's bound above, which a sum one by one keeps unless all roundings agree)
        assert ((r.logprobs.cpu().to(F64) - lp).abs() <= LP_TOL).all()
        assert ((r.entropy.cpu().to(F64) - ent).abs() <= ENT_TOL).all()


def test_policy_targets_outside_the_vocabulary(dev):
    """Hugging Face scoring: raised where the host can see it, reported in the index-error word where it cannot."""
    from types import SimpleNamespace

    from rl_project_b200.models.hf_policy import HFPolicy

    x = torch.randn(1, 3, 20).to(dev)
    policy = SimpleNamespace(token_logits=lambda ids: x)
    good, bad = torch.tensor([[1, -1, 19]]), torch.tensor([[1, 20, 3]])
    assert HFPolicy.token_logprobs(policy, good, good)[0, 1] == 0
    with pytest.raises(IndexError):
        HFPolicy.token_logprobs(policy, bad, bad)
    if dev == "cuda":
        from rl_project_b200.core.errors import KernelError
        from rl_project_b200.ops._ext import check_bounds

        lp = HFPolicy.token_logprobs(policy, bad, bad.cuda())
        with pytest.raises(KernelError):
            check_bounds(torch.device("cuda", 0))
        assert lp[0, 1] == 0 and lp[0, 0] < 0


def test_derivatives_of_derivatives(dev):
    """Second derivatives, forward-mode AD and torch.func transforms, as through the definition in 64 bits."""
    torch.manual_seed(11)
    N, V, k = 5, 37, 3
    x0, v = torch.randn(N, V) * 2, torch.randn(N, V)
    x0[1, ::4] = -math.inf
    v[1, ::4] = 0
    t = torch.tensor([4, 1, -1, 7, 36])
    c = [torch.randn(N), torch.randn(N), torch.randn(N, k)]
    td = t.to(dev)

    def f(x, targets, c, by=lambda x, t: token_logprobs(x, t, top=k)):
        lp, ent, top = by(x, targets)[:3]
        return (lp * c[0]).sum() + (ent ** 2 * c[1]).sum() + (top * c[2]).sum()

    xd, vd, cd = x0.to(dev).requires_grad_(), v.to(dev), [y.to(dev) for y in c]
    xo, co = x0.to(F64).requires_grad_(), [y.to(F64) for y in c]
    want, = torch.autograd.grad(f(xo, t, co, lambda x, t: oracle(x, t, k)), xo, create_graph=True)
    curve, = torch.autograd.grad((want * v).sum(), xo)
    got, = torch.autograd.grad(f(xd, td, cd), xd, create_graph=True)
    # values up to 2^5 and their products in fp32, sums of 37: 2^5 * 2^-24 * 37 * 4, below 2^-11
    assert ((got.detach().cpu().to(F64) - want.detach()).abs() <= 2 ** -11).all()
    twice, = torch.autograd.grad((got * vd).sum(), xd)
    assert twice.abs().max() > 0.1 and ((twice.cpu().to(F64) - curve).abs() <= 2 ** -11).all()
    slope = (want.detach() * v).sum()
    with torch.autograd.forward_ad.dual_level():
        out = f(torch.autograd.forward_ad.make_dual(xd.detach(), vd), td, cd)
        assert abs(float(torch.autograd.forward_ad.unpack_dual(out).tangent) - float(slope)) <= 2 ** -9
    _, tangent = torch.func.jvp(lambda x: f(x, td, cd), (xd.detach(),), (vd,))
    assert abs(float(tangent) - float(slope)) <= 2 ** -9
    grad = torch.func.grad(lambda x: f(x, td, cd))(xd.detach())
    assert ((grad.cpu().to(F64) - want.detach()).abs() <= 2 ** -11).all()
    lp = torch.func.vmap(lambda x, t: token_logprobs(x[None], t[None]).logprobs[0])(xd.detach(), td)
    assert ((lp.cpu().to(F64) - oracle(x0, t, 0)[0]).abs() <= LP_TOL).all()


def test_refusals(dev):
    x, t = torch.randn(3, 10).to(dev), torch.zeros(3, dtype=torch.long).to(dev)
    for call in (lambda: token_logprobs(x.double(), t), lambda: token_logprobs(x, t[:2]),
                 lambda: token_logprobs(x, t[:, None]), lambda: token_logprobs(x, t, top=11),
                 lambda: token_logprobs(x, t, top=-1), lambda: token_logprobs(x.repeat(1, 10), t, top=65),
                 lambda: token_logprobs(x.long(), t)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_captured_replayed_and_other_stream():
    x = torch.randn(40, 5000, device="cuda").bfloat16()
    t = torch.randint(0, 5000, (40,), device="cuda")
    first = token_logprobs(x, t, top=5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = token_logprobs(x, t, top=5)
    for _ in range(2):
        x.copy_(torch.randn(40, 5000, device="cuda"))
        g.replay()
        want = token_logprobs(x, t, top=5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, want)) and not torch.equal(r.logprobs, first.logprobs)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = token_logprobs(x, t, top=5)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.gpu
def test_captured_training_step():
    """Forward and backward in one graph; replays give the eager gradient of the new logits."""
    x = torch.randn(12, 3001, device="cuda").requires_grad_()
    t = torch.randint(-1, 3001, (12,), device="cuda")

    def step():
        r = token_logprobs(x, t, top=2)
        return torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum(), x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dx = step()
    with torch.no_grad():
        x.copy_(torch.randn(12, 3001, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dx, step())
