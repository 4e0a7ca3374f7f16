"""Norms and rotation of queries and keys against the formulas in 64 bits."""

import pytest
import torch

from deepspeed_amd.ops.qk_norm import qk_norm_rope
from deepspeed_amd.ops.rope import rope_tables

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(B, S, H, Hk, D, rotated, kind, device, seed=0, table=64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, H + 2 * Hk, D, generator=g).to(kind).to(device)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(kind).to(device) for _ in "qk"]
    dy = [torch.randn(B, S, h, D, generator=g).to(kind).to(device) for h in (H, Hk)]
    cos, sin = rope_tables(rotated, table, theta=100.0)
    pos = torch.randint(0, table, (B, S), generator=g, dtype=torch.int32)
    return (x[:, :, :H], x[:, :, H:H + Hk], *w, cos.to(device), sin.to(device),
            pos.to(device)), dy


def _run(ins, dy, **how):
    leaves = [x.detach().requires_grad_() for x in ins[:4]]
    y = qk_norm_rope(*leaves, *ins[4:], **how)
    return [x.detach() for x in y] + list(torch.autograd.grad(y, leaves, dy))


def _reference(ins, dy, eps=1e-6, layout="half", one_plus=False):
    """Values in 64 bits and how far fp32 arithmetic may be off them, without the
    rounding to the tensors' type: sums of D terms are off by D 2^-24 of the sum of
    their magnitudes, the few operations on a value by 2^-24 each."""
    cos, sin, pos = ins[4:]
    D, n = ins[0].shape[-1], 2 * cos.shape[1]
    B, S = ins[0].shape[:2]
    at = torch.arange(S, device=cos.device).expand(B, S) if pos is None else pos.long()
    c, s = (t.double()[at][:, :, None] for t in (cos, sin))
    i = torch.arange(n, device=cos.device)
    a, b = (i[:n // 2], i[n // 2:]) if layout == "half" else (i[0::2], i[1::2])

    def turn(x, sign, plus=False):
        y = x.clone()
        if plus:      # of magnitudes
            y[..., a] = x[..., a] * c.abs() + x[..., b] * s.abs()
            y[..., b] = x[..., b] * c.abs() + x[..., a] * s.abs()
        else:
            y[..., a] = x[..., a] * c - sign * x[..., b] * s
            y[..., b] = x[..., b] * c + sign * x[..., a] * s
        return y

    u = 2.0 ** -24 * (D + 16)
    values, off = [[] for _ in range(3)], [[] for _ in range(3)]
    for x, w, d in zip(ins[:2], ins[2:4], dy):
        x, w, d = x.double(), w.double() + one_plus, d.double()
        r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        norm = x * r * w
        values[0].append(turn(norm, 1))
        off[0].append(u * turn(norm.abs(), 1, True))
        dn = turn(d, -1)
        size = turn(d.abs(), -1, True)
        values[2].append((dn * x * r).sum((0, 1, 2)))
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        off[2].append((u + 2.0 ** -24 * rows) * (size * (x * r).abs()).sum((0, 1, 2)))
        mix = (dn * w * x * r).mean(-1, keepdim=True)
        values[1].append(r * (dn * w - x * r * mix))
        off[1].append(2 * u * r * (size * w.abs() + (x * r).abs() * (
            size * (w * x * r).abs()).mean(-1, keepdim=True)))
    return sum(values, []), sum(off, [])


def _check(got, values, off):
    for name, x, y, most in zip(("q", "k", "dq", "dk", "dqw", "dkw"), got, values, off):
        info = torch.finfo(x.dtype)
        # half a step of the type, and of its smallest numbers
        far = (x.double() - y).abs() - most * 1.01
        far = far - info.eps / 2 * (y.abs() + most) - info.tiny * info.eps
        assert (far <= 0).all(), (name, float(far.max()))


CASES = [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (2, 7, 5, 1, 128, 64),
         (1, 33, 32, 8, 128, 128), (3, 5, 3, 3, 80, 40), (2, 9, 4, 2, 96, 96),
         (1, 4, 2, 1, 256, 128), (2, 5, 3, 2, 18, 6), (1, 6, 2, 2, 512, 512),
         (1, 3, 2, 1, 510, 254), (1, 700, 2, 1, 32, 16), (2, 1, 7, 7, 66, 66)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", CASES[:8])
def test_formulas_cpu(case, layout):
    for kind in TYPES:
        ins, dy = _inputs(*case, kind, "cpu")
        for plus in (False, True):
            _check(_run(ins, dy, layout=layout, one_plus=plus),
                   *_reference(ins, dy, layout=layout, one_plus=plus))


def test_gradcheck_cpu():
    ins, _ = _inputs(1, 3, 2, 1, 8, 4, torch.float64, "cpu")
    leaves = [x.detach().requires_grad_() for x in ins[:4]]
    for layout in ("half", "interleaved"):
        assert torch.autograd.gradcheck(
            lambda *x: qk_norm_rope(*x, *ins[4:], layout=layout), leaves)


def test_refusals():
    ins, _ = _inputs(2, 3, 4, 2, 8, 8, torch.float32, "cpu")
    q, k, qw, kw, cos, sin, pos = ins
    with pytest.raises(ValueError, match="layout"):
        qk_norm_rope(*ins, layout="pairs")
    with pytest.raises(ValueError, match="D even"):
        qk_norm_rope(q[..., :7], k[..., :7], qw[:7], kw[:7], cos, sin, pos)
    with pytest.raises(ValueError, match="D even"):
        qk_norm_rope(q, k[:1], qw, kw, cos, sin, pos)
    with pytest.raises(ValueError, match="weights"):
        qk_norm_rope(q, k, qw[:4], kw, cos, sin, pos)
    with pytest.raises(ValueError, match="one type"):
        qk_norm_rope(q, k.bfloat16(), qw, kw, cos, sin, pos)
    with pytest.raises(ValueError, match="cos and sin"):
        qk_norm_rope(q, k, qw, kw, cos.double(), sin.double(), pos)
    with pytest.raises(ValueError, match="cos and sin"):
        qk_norm_rope(q[..., :6], k[..., :6], qw[:6], kw[:6], cos, sin, pos)
    with pytest.raises(ValueError, match="int32"):
        qk_norm_rope(q, k, qw, kw, cos, sin, pos.long())
    with pytest.raises(ValueError, match="longer"):
        qk_norm_rope(q, k, qw, kw, cos[:2], sin[:2])


def _constant_angles(device):
    ins, _ = _inputs(2, 3, 4, 2, 64, 64, torch.float32, device)
    for i in (4, 5):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate(ins[:6])]
        with pytest.raises(ValueError, match="no gradient"):
            qk_norm_rope(*leaves, ins[6])


def test_constant_angles_cpu():
    _constant_angles("cpu")


@pytest.mark.gpu
def test_constant_angles_gpu():
    _constant_angles("cuda")


def _bad_positions(device):
    ins, dy = _inputs(2, 5, 4, 2, 64, 32, torch.float32, device)
    for bad in (-1, 64, 2 ** 31 - 1, -2 ** 31):
        pos = ins[6].clone()
        pos[1, 3] = bad
        got = _run((*ins[:6], pos), dy)
        for x in got[:4]:
            assert x[1, 3].isnan().all()
            x[1, 3] = 0
            assert torch.isfinite(x).all()


def test_bad_positions_cpu():
    _bad_positions("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_formulas_gpu(case, kind, layout):
    ins, dy = _inputs(*case, kind, "cuda", table=800)
    for plus in (False, True):
        how = dict(layout=layout, one_plus=plus)
        _check(_run(ins, dy, **how), *_reference(ins, dy, **how))
    ins = (*ins[:6], None)
    _check(_run(ins, dy, layout=layout, eps=0.3),
           *_reference(ins, dy, layout=layout, eps=0.3))


@pytest.mark.gpu
def test_bad_positions_gpu():
    _bad_positions("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_layouts_gpu(kind):
    """Strides and alignment other than a joint projection's; broadcast inputs."""
    ins, dy = _inputs(2, 6, 4, 2, 64, 64, kind, "cuda")
    want = _reference(ins, dy)

    def odd(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
        flat[1:] = x.reshape(-1)
        return flat[1:].view(x.shape)

    def spread(x):
        return x.repeat_interleave(2, -1)[..., ::2]

    def heads_first(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2) if x.dim() == 4 else x

    for change in (odd, spread, heads_first):
        _check(_run((*(change(x) for x in ins[:4]), *ins[4:]),
                    [change(x) for x in dy]), *want)
    one = [x[:1, :, :1].expand_as(x) for x in dy]
    _check(_run(ins, one), *_reference(ins, one))


@pytest.mark.gpu
def test_many_tokens_gpu():
    """More tokens than workgroups of the backward, the same twice."""
    ins, dy = _inputs(3, 2000, 6, 2, 128, 128, torch.float32, "cuda", table=2000)
    got = _run(ins, dy)
    _check(got, *_reference(ins, dy))
    assert all(torch.equal(x, y) for x, y in zip(got, _run(ins, dy)))


@pytest.mark.gpu
def test_differences_gpu():
    """Gradients against differences of the 64-bit formulas along random directions."""
    ins, dy = _inputs(2, 9, 4, 2, 64, 32, torch.float32, "cuda")
    got = _run(ins, dy, layout="interleaved")
    g = torch.Generator(device="cuda").manual_seed(3)
    for i in range(4):
        u = torch.randn(ins[i].shape, generator=g, device="cuda", dtype=torch.float64)
        ends = []
        for step in (1e-5, -1e-5):
            x = [t.double() for t in ins[:4]]
            x[i] = x[i] + step * u
            y, _ = _reference((*x, *ins[4:]), dy, layout="interleaved")
            ends.append(sum(float((a * b.double()).sum()) for a, b in zip(y, dy)))
        slope = (ends[0] - ends[1]) / 2e-5
        size = float((got[2 + i].double() * u).abs().sum())
        assert abs(slope - float((got[2 + i].double() * u).sum())) <= 1e-5 * size + 1e-4


@pytest.mark.gpu
def test_graph_and_one_gradient_gpu():
    ins, dy = _inputs(2, 40, 4, 2, 64, 64, torch.bfloat16, "cuda")
    static = [x.clone() for x in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _run(static, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(static, dy)
    for seed in range(4):
        fresh, _ = _inputs(2, 40, 4, 2, 64, 64, torch.bfloat16, "cuda", seed=seed + 5)
        want = _run(fresh, dy)
        for x, y in zip(static, fresh):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    # a loss of the queries alone
    leaves = [x.detach().requires_grad_() for x in ins[:4]]
    q, _ = qk_norm_rope(*leaves, *ins[4:])
    grads = torch.autograd.grad(q, leaves, dy[0])
    want = _run(ins, [dy[0], torch.zeros_like(dy[1])])[2:]
    assert all(torch.equal(x, y) for x, y in zip(grads, want))
    empty = torch.empty(0, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert qk_norm_rope(empty, empty, *ins[2:6])[0].shape == empty.shape


@pytest.mark.gpu
def test_far_rows_gpu():
    """Rows whose places do not fit 32 bits."""
    far = torch.empty(1, 300, 1 << 23, dtype=torch.bfloat16, device="cuda")
    ins, dy = _inputs(1, 300, 4, 2, 128, 128, torch.bfloat16, "cuda", table=300)
    want = _run(ins, dy)
    there = []
    for i, x in enumerate((*ins[:2], *dy)):
        y = far[:, :, i * 4096:i * 4096 + x.shape[2] * 128].unflatten(-1, (-1, 128))
        there.append(y.copy_(x))
    got = _run((*there[:2], *ins[2:]), there[2:])
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def _no_tokens(device):
    """Rows of no tokens: the weights' gradients are there, and 0."""
    cos, sin = rope_tables(64, 8, device=device)
    for shape in ((2, 0, 3, 64), (0, 5, 3, 64)):
        w = [torch.ones(64, device=device, requires_grad=True) for _ in "qk"]
        q, k = (torch.empty(shape, device=device, requires_grad=True) for _ in "qk")
        out = qk_norm_rope(q, k, *w, cos, sin)
        assert [x.shape for x in out] == [q.shape, k.shape]
        grads = torch.autograd.grad(out[0].sum() + out[1].sum(), (q, k, *w))
        assert [x.shape for x in grads] == [x.shape for x in (q, k, *w)]
        assert not grads[2].any() and not grads[3].any()


def test_no_tokens_cpu():
    _no_tokens("cpu")


@pytest.mark.gpu
def test_no_tokens_gpu():
    _no_tokens("cuda")
