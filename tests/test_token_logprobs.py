"""Log probabilities, entropy and best tokens against the formulas in 64 bits."""

import math

import pytest
import torch

from deepspeed_amd.ops.token_logprobs import token_logprobs

TYPES = [torch.bfloat16, torch.float16, torch.float32]
IGNORE = -100


def _inputs(N, V, kind, device, seed=0, spread=3.0, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(N, V, generator=g)).to(kind)
    y = torch.randint(0, V, (N,), generator=g)
    y[torch.rand(N, generator=g) < ignored] = IGNORE
    glp, gent = torch.randn(N, generator=g), torch.randn(N, generator=g)
    return [t.to(device) for t in (x, y, glp, gent)]


def _reference(x, y, glp, gent, top):
    """Values in 64 bits, and how far fp32 may be off: a sum of V exponentials by
    2^-24 (V / 256 + 64) of itself (a thread's share of terms, then a tree), a power
    by 2^-22 times the distance from the maximum."""
    x = x.double().cpu()
    y, glp, gent = y.cpu(), glp.double().cpu(), gent.double().cpu()
    V = x.shape[1]
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    live = y != IGNORE
    at = torch.where(live, y, 0)[:, None]
    far = (x - x.amax(-1, keepdim=True)).abs()
    far = torch.where(far < math.inf, far, 0.0)
    some = torch.where(p > 0, lp, 0.0)
    ent = -(p * some).sum(-1)
    u = 2.0 ** -24 * (V / 256 + 64)
    step = 2.0 ** -22 * (1 + (p * far).sum(-1)) + u
    off_lp = step[:, None] + 2.0 ** -22 * (far + some.abs())
    off_ent = 2 * (step * (1 + (p * some.abs()).sum(-1)) +
                   2.0 ** -22 * (p * far * (1 + some.abs())).sum(-1)) + u * ent
    a, h = glp[:, None] * live[:, None], gent[:, None] * live[:, None]
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    d = a * (hot - p) - h * p * (some + ent[:, None])
    off_d = p * off_lp * (a.abs() + h.abs() * (some.abs() + ent[:, None])) + \
        p * h.abs() * (off_lp + off_ent[:, None]) + 2.0 ** -23 * (d.abs() + p * (
            a.abs() + h.abs() * (some.abs() + ent[:, None])))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    values = [lp.gather(1, at)[:, 0] * live, ent * live, lp.gather(1, order), order, d]
    return values, [off_lp.gather(1, at)[:, 0], off_ent, off_lp.gather(1, order), None,
                    off_d]


def _check(x, y, glp, gent, top=0):
    leaf = x.detach().requires_grad_()
    got = token_logprobs(leaf, y, top=top, ignore_index=IGNORE)
    assert got.logprobs.dtype is torch.float32 and got.top_ids.dtype is torch.int64
    dx, = torch.autograd.grad((got.logprobs, got.entropy), leaf, (glp, gent))
    assert dx.dtype is x.dtype and dx.shape == x.shape
    flat = [t.reshape(-1, t.shape[-1]) if t.dim() > y.dim() else t.reshape(-1)
            for t in (x, y, glp, gent)]
    values, off = _reference(*flat, top)
    live = (flat[1] != IGNORE).cpu()
    for name, a, b, most in zip(("logprobs", "entropy"), got[:2], values, off):
        far = (a.detach().double().cpu().reshape(-1) - b).abs() - most
        assert (far <= 0).all(), (name, float(far.max()))
    best, ids = (t.cpu().reshape(len(live), top) for t in got[2:])
    assert torch.equal(ids[live], values[3][live]) and (ids[~live] == -1).all()
    far = (best.double() - values[2]).abs() - off[2]
    assert (far[live] <= 0).all() and (best[~live] == -math.inf).all()
    info = torch.finfo(dx.dtype)
    far = (dx.double().cpu().reshape(values[4].shape) - values[4]).abs()
    far = far - 1.01 * off[4] - info.eps / 2 * values[4].abs() - info.tiny * info.eps
    assert (far <= 0).all(), ("dlogits", float(far.max()))
    return got, dx


SIZES = [(1, 1), (3, 2), (5, 31), (2, 257), (4, 1000), (3, 8191), (2, 8193), (2, 50257)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", SIZES[:6])
def test_formulas_cpu(size, kind):
    _check(*_inputs(*size, kind, "cpu"), top=min(size[1], 5))


def test_gradcheck_cpu():
    x, y, _, _ = _inputs(4, 7, torch.float64, "cpu")
    assert torch.autograd.gradcheck(
        lambda x: token_logprobs(x, y, ignore_index=IGNORE)[:2],
        x.detach().requires_grad_())


def test_refusals():
    x, y, _, _ = _inputs(4, 7, torch.float32, "cpu")
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(x, y[:3])
    with pytest.raises(ValueError, match="integer tokens"):
        token_logprobs(x, y.float())
    with pytest.raises(ValueError, match="floating logits"):
        token_logprobs(x.long(), y)
    for top in (-1, 8, 33):
        with pytest.raises(ValueError, match="best of"):
            token_logprobs(x, y, top=top)
    with pytest.raises(ValueError, match="best of"):
        token_logprobs(torch.zeros(1, 500_001), y[:1], top=1)


def _odd_values(device):
    """Infinities, NaN, equal logits, tokens that are none, large logits."""
    inf, nan = math.inf, math.nan
    x = torch.tensor([[0.0, -inf, 1.0, -inf, 2.0], [1.0, 1.0, 1.0, 1.0, 1.0],
                      [0.0, -0.0, -1.0, 0.0, -0.0], [nan, 0.0, 1.0, 2.0, 3.0],
                      [-inf] * 5, [inf, 0.0, 0.0, 0.0, 0.0],
                      [-3e4, -1e4, 3e4, 3e4 - 1, 0.0], [5.0, 4.0, 3.0, 2.0, 1.0],
                      [nan] * 5, [-inf, -inf, 7.0, -inf, -inf]], device=device)
    y = torch.tensor([2, 4, 0, 1, 0, 1, 3, 5, IGNORE, 2], device=device)
    leaf = x.clone().requires_grad_()
    got = token_logprobs(leaf, y, top=5, ignore_index=IGNORE)
    ones = torch.ones(10, device=device)
    dx, = torch.autograd.grad((got.logprobs, got.entropy), leaf, (ones, ones))
    sound = torch.tensor([0, 1, 2, 6, 9])
    values, off = _reference(x[sound], y[sound], ones[:5], ones[:5], 5)
    for a, b, most in zip(got[:2], values, off):
        assert ((a.detach().cpu()[sound].double() - b).abs() <= most + 1e-7).all()
    assert torch.equal(got.top_ids.cpu()[sound], values[3])
    assert torch.equal(got.top_logprobs.cpu()[sound] == -inf, values[2] == -inf)
    assert ((dx.cpu()[sound].double() - values[4]).abs() <= off[4] + 1e-7).all()
    # a token behind the last, NaN, nothing but -inf, inf: no number
    sick = [3, 4, 5]
    assert got.logprobs[sick].isnan().all() and got.entropy[sick].isnan().all()
    assert got.logprobs[7].isnan() and torch.isfinite(got.entropy[7])
    assert dx[7].isnan().all()
    assert sorted(got.top_ids[3].tolist()) == [0, 1, 2, 3, 4]
    assert got.logprobs[8] == 0 and got.entropy[8] == 0 and (dx[8] == 0).all()
    assert (got.top_ids[8] == -1).all()


def test_odd_values_cpu():
    _odd_values("cpu")


@pytest.mark.gpu
def test_odd_values_gpu():
    _odd_values("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", SIZES + [(600, 9001), (3, 128256), (1, 500000),
                                          (2100, 77)])
def test_formulas_gpu(size, kind):
    ins = _inputs(*size, kind, "cuda")
    for top in {0, 1, min(32, size[1])}:
        _check(*ins, top=top)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_ties_gpu(kind):
    """Few different logits over many parts: of equal ones the lowest ids."""
    g = torch.Generator().manual_seed(1)
    x = torch.randint(0, 3, (3, 40001), generator=g).to(kind).cuda()
    x[1] = 2
    y = torch.tensor([5, 40000, 0]).cuda()
    ids = token_logprobs(x, y, top=32).top_ids.cpu()
    want = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices
    assert torch.equal(ids, want[:, :32])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_layouts_gpu(kind):
    """Rows of a larger tensor, of odd strides, transposed; more dimensions."""
    x, y, glp, gent = _inputs(12, 1001, kind, "cuda")
    x, y, glp, gent = (t.view(3, 4, *t.shape[1:]) for t in (x, y, glp, gent))
    for top in (0, 3):
        _check(x[:, :-1], y[:, :-1], glp[:, :-1], gent[:, :-1], top)
        _check(x[..., 3:998], y.clamp(max=900), glp, gent, top)
        _check(x.transpose(0, 1), y.t(), glp.t(), gent.t(), top)
        _check(x.transpose(1, 2).contiguous().transpose(1, 2), y, glp, gent, top)
        _check(x.view(3, 2, 2, 1001), y.view(3, 2, 2), glp.view(3, 2, 2),
               gent.view(3, 2, 2), top)
        _check(x[0, 0], y[0, 0], glp[0, 0], gent[0, 0], top)
        _check(x, y.int(), glp[:1, :1].expand(3, 4), gent, top)
        _check(x[:1].expand(3, 4, 1001), y, glp, gent, top)


@pytest.mark.gpu
def test_infinite_logits_in_long_rows_gpu():
    """A masked vocabulary: both ways through a row, and by parts."""
    for rows in (2, 520):
        x, y, glp, gent = _inputs(rows, 20011, torch.bfloat16, "cuda", ignored=0)
        x[:, 7::3] = -math.inf
        x[0, :20000] = -math.inf
        y = y // 3 * 3
        y[0] = 20010
        x.scatter_(1, y[:, None], 1.0)
        for top in (0, 4):
            _check(x, y, glp, gent, top)


@pytest.mark.gpu
def test_parts_and_whole_rows_gpu():
    """Rows of more than four parts, few and many, with masked logits."""
    for rows in (2, 399, 401):
        x, y, glp, gent = _inputs(rows, 40011, torch.bfloat16, "cuda", ignored=1)
        x[:, 7::3] = -math.inf
        live = y != IGNORE
        y = torch.where(live, y // 3 * 3, y)
        x.scatter_(1, y.clamp(min=0)[:, None], 1.0)
        _check(x, y, glp, gent, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_one_best_gpu(kind):
    """The first of equal ones, of a row of the type's lowest value, of minus
    infinity alone, and NaN before all."""
    x = torch.full((6, 20003), torch.finfo(kind).min, dtype=kind, device="cuda")
    x[1, [19999, 77, 20002]] = 3
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 20002] = torch.finfo(kind).min
    x[4, [700, 12345]] = math.nan
    x[5, [0, 20002]] = -0.0
    y = torch.zeros(6, dtype=torch.long, device="cuda")
    ids = token_logprobs(x, y, top=1).top_ids.cpu()
    assert ids.flatten().tolist() == [0, 77, 0, 20002, 700, 0]


@pytest.mark.gpu
def test_peaked_and_large_gpu():
    """Nearly sure rows keep the entropy's digits, large logits theirs."""
    for shift in (0.0, 1e4, -1e4):
        x, y, glp, gent = _inputs(6, 5000, torch.float32, "cuda", ignored=0)
        x = x + shift
        x[:3, 17] += 40
        _check(x, y, glp, gent, 2)


@pytest.mark.gpu
def test_differences_gpu():
    x, y, glp, gent = _inputs(4, 3001, torch.float32, "cuda")
    _, dx = _check(x, y, glp, gent)
    u = torch.randn(x.shape, dtype=torch.float64,
                    generator=torch.Generator().manual_seed(2))
    ends = []
    for step in (1e-5, -1e-5):
        values, _ = _reference(x.double().cpu() + step * u, y, glp, gent, 0)
        ends.append(float((values[0] * glp.cpu().double() +
                           values[1] * gent.cpu().double()).sum()))
    slope = (ends[0] - ends[1]) / 2e-5
    mine = dx.double().cpu() * u
    assert abs(slope - float(mine.sum())) <= 1e-5 * float(mine.abs().sum()) + 1e-5


@pytest.mark.gpu
def test_one_gradient_and_graph_gpu():
    x, y, glp, gent = _inputs(9, 4099, torch.bfloat16, "cuda")
    leaf = x.detach().requires_grad_()
    got = token_logprobs(leaf, y, top=2)
    for out, zero in ((0, 1), (1, 0)):
        dx, = torch.autograd.grad(got[out], leaf, (glp, gent)[out], retain_graph=True)
        full = [glp, gent]
        full[zero] = torch.zeros_like(glp)
        want, = torch.autograd.grad(got[:2], leaf, full, retain_graph=True)
        assert torch.equal(dx, want)
    assert not got.top_logprobs.requires_grad

    def step(x, y):
        leaf = x.detach().requires_grad_()
        got = token_logprobs(leaf, y, top=2)
        return (*(t.detach() for t in got),
                *torch.autograd.grad(got[:2], leaf, (glp, gent)))

    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static, y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, y)
    for seed in range(4):
        fresh = _inputs(9, 4099, torch.bfloat16, "cuda", seed=seed + 3)[0]
        want = step(fresh, y)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_nothing_and_refusals_gpu():
    none = torch.empty(0, 11, device="cuda", requires_grad=True)
    got = token_logprobs(none, torch.empty(0, dtype=torch.long, device="cuda"), top=2)
    assert got.top_ids.shape == (0, 2)
    got.logprobs.sum().backward()
    x, y, _, _ = _inputs(4, 7, torch.float32, "cuda")
    with pytest.raises(ValueError, match="bf16"):
        token_logprobs(x.double(), y)
    with pytest.raises(ValueError, match="device"):
        token_logprobs(x, y.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 4])
def test_far_rows_gpu(top):
    """Rows whose places do not fit 32 bits, of the logits and of their gradient."""
    far = torch.empty(600, 1 << 23, dtype=torch.bfloat16, device="cuda")
    x, y, glp, gent = _inputs(600, 9001, torch.bfloat16, "cuda")
    there = far[:, :9001].copy_(x)
    _check(there, y, glp, gent, top)


@pytest.mark.gpu
def test_wide_gradient_gpu():
    """A gradient of more than 2^31 numbers: its last rows."""
    x = torch.zeros(17000, 128256, dtype=torch.bfloat16, device="cuda")
    y = torch.full((17000,), IGNORE, device="cuda")
    small, t, glp, gent = _inputs(5, 128256, torch.bfloat16, "cuda", ignored=0)
    x[-5:], y[-5:] = small, t
    leaf = x.requires_grad_()
    got = token_logprobs(leaf, y)
    dx, = torch.autograd.grad((got.logprobs[-5:], got.entropy[-5:]), leaf, (glp, gent))
    want, dsmall = _check(small, t, glp, gent)
    assert not dx[:-5].any()
    # by whole rows here, by parts there: sums in other orders, roundings a step apart
    torch.testing.assert_close(dx[-5:].float(), dsmall.float(), rtol=2.0 ** -7,
                               atol=1e-7)
    torch.testing.assert_close(got.logprobs[-5:], want.logprobs, rtol=1e-6, atol=1e-5)


# What programs write over logits that may not be sampled, besides -inf.
MASKS = [-1e30, -1e36, -1.7e38, -2.5e38]


def _masked(kind, mask, rows, V, device):
    """Logits with a stretch of whole parts and single ones masked, tokens that are
    not, and gradients."""
    x, y, glp, gent = _inputs(rows, V, kind, device, seed=3)
    x[:, :V * 2 // 5] = mask
    x[:, V // 2::3] = mask
    y = torch.where(y == IGNORE, y, V // 2 + 1)
    return x, y, glp, gent


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", MASKS)
def test_masked_logits_cpu(mask, kind):
    _check(*_masked(kind, mask, 3, 1003, "cpu"), top=3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", MASKS + ["lowest", "half of it"])
@pytest.mark.parametrize("V", [24003, 40011])
def test_masked_logits_gpu(V, mask, kind):
    """A thread, a part or a chunk that saw masked logits alone adds nothing to the
    entropy of the rest: rows by parts and whole ones."""
    low = torch.finfo(kind).min
    mask = {"lowest": low, "half of it": low / 2}.get(mask, mask)
    for top in (0, 3):
        _check(*_masked(kind, mask, 3, V, "cuda"), top)


def _lowest_rows(kind, rows, V, device):
    """Rows masked from end to end, with the type's lowest value and with others near
    it, and some that are not."""
    x, y, glp, gent = _inputs(rows, V, kind, device, seed=4, ignored=0)
    low = torch.finfo(kind).min
    x[0] = low
    x[1, ::2], x[1, 1::2] = low, low * 0.95
    x[1, 5] = low * 0.9
    x[2] = low / 2
    y[:3] = 5
    return x, y, glp, gent


@pytest.mark.parametrize("kind", TYPES)
def test_lowest_rows_cpu(kind):
    """Every token of a row of one value is as probable, whatever the value."""
    got, _ = _check(*_lowest_rows(kind, 4, 1003, "cpu"))
    assert got.logprobs[0].item() == pytest.approx(-math.log(1003), rel=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [24003, 40011])
def test_lowest_rows_gpu(V, kind):
    for top in (0, 2):
        got, _ = _check(*_lowest_rows(kind, 4, V, "cuda"), top)
        assert got.logprobs[0].item() == pytest.approx(-math.log(V), rel=1e-5)


def _masked_tokens(kind, rows, V, device, top):
    """Tokens of masked logits, and best ones among which are masked ones."""
    for mask in (torch.finfo(kind).min, torch.finfo(kind).min * 0.8):
        x, y, glp, gent = _masked(kind, mask, rows, V, device)
        x[1:] = mask
        x[1:, [3, V - 1]] = 1.0
        y[:2], y[2:] = 7, 3
        got, _ = _check(x, y, glp, gent, top)
        assert torch.isfinite(got.logprobs).all()
        assert torch.isfinite(got.top_logprobs).all()


@pytest.mark.parametrize("kind", TYPES)
def test_masked_tokens_cpu(kind):
    _masked_tokens(kind, 4, 1003, "cpu", 4)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [24003, 40011])
def test_masked_tokens_gpu(V, kind):
    for top in (0, 4):
        _masked_tokens(kind, 4, V, "cuda", top)


def _entropy_alone(device, V):
    """The entropy knows nothing of the token: nor does its gradient, whatever the
    token is, where no log probability has one."""
    x, y, _, gent = _inputs(6, V, torch.float32, device, ignored=0)
    grads = []
    for tokens in (y, torch.tensor([V, -1, -(2 ** 40), 2 ** 40, V + 7, 0]).to(device)):
        leaf = x.detach().requires_grad_()
        got = token_logprobs(leaf, tokens)
        grads += torch.autograd.grad(got.entropy, leaf, gent)
    assert got.logprobs[:5].isnan().all() and torch.isfinite(got.entropy).all()
    assert torch.isfinite(grads[0]).all() and torch.equal(*grads)
    _check(x, y, torch.zeros_like(gent), gent)


def test_entropy_alone_cpu():
    _entropy_alone("cpu", 103)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [103, 40011])
def test_entropy_alone_gpu(V):
    _entropy_alone("cuda", V)


def _nan_above_infinity(device):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[0.0, inf, nan, 1.0, nan, inf], [inf, nan, inf, -inf, 0.0, 1.0]],
                     device=device)
    y = torch.zeros(2, dtype=torch.long, device=device)
    want = [[2, 4, 1, 5, 3, 0], [1, 0, 2, 5, 4, 3]]
    for top in (1, 3, 6):
        ids = token_logprobs(x, y, top=top).top_ids.tolist()
        assert ids == [row[:top] for row in want]


def test_nan_above_infinity_cpu():
    _nan_above_infinity("cpu")


@pytest.mark.gpu
def test_nan_above_infinity_gpu():
    _nan_above_infinity("cuda")


def _no_rows(device):
    """No rows, of any strides and dimensions."""
    for shape in ((0, 11), (2, 0, 11), (0, 3, 4, 11)):
        x = torch.empty(*shape[:-1], 1, device=device, requires_grad=True)
        tokens = torch.empty(shape[:-1], dtype=torch.long, device=device)
        for top in (0, 3):
            got = token_logprobs(x.expand(shape), tokens, top=top)
            assert got.logprobs.shape == got.entropy.shape == tokens.shape
            assert got.top_ids.shape == got.top_logprobs.shape == (*tokens.shape, top)
            dx, = torch.autograd.grad(got.logprobs.sum() + got.entropy.sum(), x)
            assert dx.shape == x.shape


def test_no_rows_cpu():
    _no_rows("cpu")


@pytest.mark.gpu
def test_no_rows_gpu():
    _no_rows("cuda")
