"""The operators for packed rows together, as a model's layer and a policy's loss use
them: normed and turned heads, attention over documents, log probabilities; and the
same layer's next token over the paged pool."""

import math

import pytest
import torch

from deepspeed_amd.ops import (masked_attention, packed_rows, qk_norm_rope,
                               rope_tables, token_logprobs)
from deepspeed_amd.ops.paged_attention import paged_decode_attention

H, HK, D, WIDTH, VOCAB, CAP = 4, 2, 128, 64, 333, 20.0


class Layer(torch.nn.Module):
    """One decoder layer's attention and a head, in the type of its weights."""

    def __init__(self, device, dtype):
        super().__init__()
        g = torch.Generator().manual_seed(0)

        def weight(*shape):
            w = torch.randn(*shape, generator=g) / math.sqrt(shape[-1])
            return torch.nn.Parameter(w.to(device, dtype))

        self.table = weight(VOCAB, WIDTH)
        self.qkv = weight((H + 2 * HK) * D, WIDTH)
        self.out = weight(WIDTH, H * D)
        self.head = weight(VOCAB, WIDTH)
        self.qn = torch.nn.Parameter(torch.ones(D, device=device, dtype=dtype))
        self.kn = torch.nn.Parameter(torch.ones(D, device=device, dtype=dtype))
        cos, sin = rope_tables(D, 512, device=device)
        self.tables = cos, sin
        self.slopes = torch.exp2(-torch.arange(1, H + 1.0)).to(device)

    def heads(self, ids, positions):
        x = torch.nn.functional.embedding(ids, self.table) * 8
        y = (x @ self.qkv.t()).view(*ids.shape, H + 2 * HK, D)
        q, k = qk_norm_rope(y[:, :, :H], y[:, :, H:H + HK], self.qn, self.kn,
                            *self.tables, positions)
        return x, q, k, y[:, :, H + HK:]

    def logits(self, x, o):
        return (x + o.flatten(2) @ self.out.t()) @ self.head.t()

    def forward(self, ids, positions, rows):
        x, q, k, v = self.heads(ids, positions)
        o = masked_attention(q, k, v, rows, softcap=CAP, alibi_slopes=self.slopes)
        return self.logits(x, o)


def _batch(lens, device):
    g = torch.Generator().manual_seed(1)
    total = sum(map(abs, lens))
    ids = torch.randint(0, VOCAB, (1, total), generator=g)
    doc, pos, at = [], [], 0
    for i, n in enumerate(lens):
        doc += [i if n > 0 else -1] * abs(n)
        pos += range(abs(n))
    target = ids.roll(-1, 1)
    for n in lens:                       # the last of a document has no next token
        at += abs(n)
        target[0, at - 1] = -100
        if n < 0:
            target[0, at + n:at] = -100
    return [t.to(device) for t in (ids, torch.tensor([pos], dtype=torch.int32),
                                   torch.tensor([doc], dtype=torch.int32), target)]


def _loss(got, advantage):
    return -(got.logprobs * advantage).sum() - 0.01 * got.entropy.sum()


def _packed_equals_apart(device, dtype, tight):
    """A packed row is what its documents are by themselves, gradients among it."""
    lens = [37, 90, 1, -6, 25]
    model = Layer(device, dtype)
    ids, pos, doc, target = _batch(lens, device)
    advantage = torch.randn(target.shape, generator=torch.Generator().manual_seed(2))
    advantage = advantage.to(device)
    got = token_logprobs(model(ids, pos, packed_rows(doc)), target, top=3)
    _loss(got, advantage).backward()
    packed = [p.grad.clone() for p in model.parameters()]
    assert (got.logprobs[target == -100] == 0).all()
    model.zero_grad()
    total, at = 0.0, 0
    for n in lens:
        part = slice(at, at + abs(n))
        at += abs(n)
        if n < 0:
            continue
        alone = token_logprobs(model(ids[:, part], pos[:, part], None),
                               target[:, part], top=3)
        total = total + _loss(alone, advantage[:, part])
        torch.testing.assert_close(alone.logprobs, got.logprobs[:, part], rtol=tight,
                                   atol=tight)
        torch.testing.assert_close(alone.entropy, got.entropy[:, part], rtol=tight,
                                   atol=tight)
    total.backward()
    for x, p in zip(packed, model.parameters()):
        off = (x.double() - p.grad.double()).norm() / p.grad.double().norm()
        assert off <= tight, float(off)


def _next_token(device, dtype, tight):
    """The answer to a prompt's next token: the pool's form of the same layer."""
    model = Layer(device, dtype)
    n, bs = 70, 16
    ids, pos, _, _ = _batch([n], device)
    with torch.no_grad():
        whole = token_logprobs(model(ids, pos, None)[:, -1], ids[:, 0], top=5)
        _, _, k, v = model.heads(ids, pos)
        x, q, _, _ = model.heads(ids[:, -1:], pos[:, -1:])
        blocks = -(-n // bs)
        order = torch.randperm(blocks + 2, generator=torch.Generator().manual_seed(3))
        pools = [torch.full((blocks + 2, HK, bs, D), float("nan"), device=device,
                            dtype=dtype) for _ in "kv"]
        for pool, rows in zip(pools, (k, v)):
            for t in range(n):
                pool[order[t // bs], :, t % bs] = rows[0, t]
        table = order[:blocks].int()[None].to(device)
        o = paged_decode_attention(q[:, 0].contiguous(), *pools, table,
                                   torch.tensor([n], device=device), softcap=CAP,
                                   alibi_slopes=model.slopes)
        one = token_logprobs(model.logits(x, o[:, None])[:, 0], ids[:, 0], top=5)
    torch.testing.assert_close(one.logprobs, whole.logprobs, rtol=tight, atol=tight)
    torch.testing.assert_close(one.top_logprobs, whole.top_logprobs, rtol=tight,
                               atol=tight)
    torch.testing.assert_close(one.entropy, whole.entropy, rtol=tight, atol=tight)


def test_packed_equals_apart_cpu():
    _packed_equals_apart("cpu", torch.float32, 2e-5)


def test_next_token_cpu():
    _next_token("cpu", torch.float32, 2e-5)


# bf16, half a step 2^-8 relative: the logits, up to 4, are rounded once each way, 2 x 4
# half steps, and the stream, the attention's output and its projection they are made of,
# each of the size of 1, twice each way: 16 in all.
BF16_STEPS = 16 * 2.0 ** -8


@pytest.mark.gpu
def test_packed_equals_apart_gpu():
    _packed_equals_apart("cuda", torch.bfloat16, BF16_STEPS)


@pytest.mark.gpu
def test_next_token_gpu():
    _next_token("cuda", torch.bfloat16, BF16_STEPS)


@pytest.mark.gpu
def test_inference_mode_and_autocast_gpu():
    model = Layer("cuda", torch.bfloat16)
    ids, pos, doc, target = _batch([40, 24], "cuda")
    want = token_logprobs(model(ids, pos, packed_rows(doc)), target, top=2)
    with torch.inference_mode():
        got = token_logprobs(model(ids, pos, packed_rows(doc)), target, top=2)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = token_logprobs(model(ids, pos, packed_rows(doc)), target, top=2)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    _loss(got, torch.ones_like(got.logprobs)).backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_gpu():
    """Refused while an eager graph of the same leaves lives; sound after its end."""
    def leaf(*shape):
        return torch.randn(*shape, device="cuda").bfloat16().requires_grad_()

    q, k, v = leaf(1, 70, 4, 64), leaf(1, 70, 2, 64), leaf(1, 70, 2, 64)
    qw, kw = leaf(64), leaf(64)
    cos, sin = rope_tables(64, 70, device="cuda")
    x, y = leaf(5, 999), torch.arange(5, device="cuda")
    calls = [(lambda: masked_attention(q, k, v), (q, k, v)),
             (lambda: qk_norm_rope(q, k, qw, kw, cos, sin)[0], (q, k, qw, kw)),
             (lambda: token_logprobs(x, y).logprobs, (x,))]
    for call, leaves in calls:
        out = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = torch.zeros(3, device="cuda")
            with pytest.raises(RuntimeError, match="eager graph"):
                call()
            with torch.no_grad():
                there = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(there, out) and not held.any()
        ones = torch.ones_like(out)
        want = torch.autograd.grad(out, leaves, ones)
        del out, graph, there
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call(), leaves, ones)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call(), leaves, ones)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_capture_beside_a_graph_of_the_same_weights_gpu():
    """The same where the inputs come from weights, however far behind: refused while
    an eager graph of these lives, sound after its end."""
    w = torch.randn(1, 9, 4, 64, device="cuda").bfloat16().requires_grad_()
    heads = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    cos, sin = rope_tables(64, 9, device="cuda")
    one = torch.zeros(1, 9, 4, dtype=torch.long, device="cuda")
    calls = [lambda x: masked_attention(x, x.detach(), x.detach()),
             lambda x: qk_norm_rope(x.detach(), x, heads, heads, cos, sin)[1],
             lambda x: token_logprobs(x, one).logprobs]
    for call in calls:
        eager = call((w * 2).exp())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = torch.zeros(3, device="cuda")
            with pytest.raises(RuntimeError, match="eager graph"):
                call((w * 2).exp())
            with torch.no_grad():
                there = call((w * 2).exp())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(there, eager) and not held.any()
        del eager, graph, there

    def step():
        q, k = qk_norm_rope(w * 2, w.exp(), heads, heads, cos, sin)
        got = token_logprobs(masked_attention(q, k, w.sin()), one)
        ones = torch.ones_like(got.logprobs)
        return torch.autograd.grad((got.logprobs, got.entropy), w, (ones, ones))[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(step(), want)


@pytest.mark.gpu
def test_gradients_in_batches_are_refused_gpu():
    w = torch.randn(1, 9, 4, 64, device="cuda").bfloat16().requires_grad_()
    heads = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    cos, sin = rope_tables(64, 9, device="cuda")
    one = torch.zeros(1, 9, 4, dtype=torch.long, device="cuda")
    for name, out in (("masked_attention", masked_attention(w, w, w)),
                      ("qk_norm_rope", qk_norm_rope(w, w, heads, heads, cos, sin)[0]),
                      ("token_logprobs", token_logprobs(w, one).logprobs)):
        many = torch.stack([torch.ones_like(out)] * 2)
        with pytest.raises(RuntimeError, match=name + ".*not in batches"):
            torch.autograd.grad(out, w, many, is_grads_batched=True, retain_graph=True)
        torch.autograd.grad(out, w, many[0])
