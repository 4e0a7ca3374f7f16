"""Attention over packed rows and its single-token form over the paged pool, against
the formulas in 64 bits, and what both refuse."""

import math

import pytest
import torch

from deepspeed_amd.ops.masked_attention import (PackedRows, _torch_spans,
                                                masked_attention, packed_rows)
from deepspeed_amd.ops.paged_attention import paged_decode_attention

BF16 = 2.0 ** -8        # a rounding to bf16, relative
# fp32 scores of up to 128 products and their exponentials, and a tanh of 1 - 2 / (e +
# 1): less than 2^-14 of a weight for caps and scores up to 100
FP32 = 2.0 ** -13


def _ids(rows, pad=None):
    """Document ids [B, S] of rows of lengths; negative lengths are padding."""
    out = []
    for lens in rows:
        row, at = [], 0
        for n in lens:
            row += [at if n > 0 else -1] * abs(n)
            at += n > 0
        out.append(row)
    return torch.tensor(out, dtype=torch.int32)


def _seen(ids, prefix, causal):
    """[B, S, S] truth values, pair by pair."""
    B, S = ids.shape
    seen = torch.zeros(B, S, S, dtype=torch.bool)
    for b in range(B):
        row = ids[b].tolist()
        s = 0
        while s < S:
            e = s
            while e < S and row[e] == row[s]:
                e += 1
            if row[s] >= 0:
                seen[b, s:e, s:e] = True
                if causal:
                    seen[b, s:e, s:e] = torch.ones(e - s, e - s).tril().bool()
                    if prefix is not None and row[s] < prefix.shape[1]:
                        n = min(e - s, max(0, int(prefix[b, row[s]])))
                        seen[b, s:e, s:s + n] = True
            s = e
    return seen


def _reference(q, k, v, do, seen, scale, cap, slopes):
    """(values, how far off bf16 kernels may be) of o, dq, dk, dv in 64 bits. Hidden
    pairs are left out of every sum."""
    B, S, H, D = q.shape
    Hk = k.shape[2]
    G = H // Hk
    q, k, v, do = (x.double().transpose(1, 2) for x in (q, k, v, do))
    # a hidden row's infinities are nobody's
    some = seen.any(1)[:, None, :, None]
    k, v = (torch.where(some, x, 0.0).repeat_interleave(G, 1) for x in (k, v))
    have = seen.any(2)[:, None, :, None]
    q, do = (torch.where(have, x, 0.0) for x in (q, do))
    kt, vt = (x.transpose(2, 3).contiguous() for x in (k, v))
    seen = seen[:, None]
    t = (q @ kt) * scale
    bend = torch.ones_like(t)
    if cap:
        bend = 1 - torch.tanh(t / cap) ** 2
        t = torch.tanh(t / cap) * cap
    at = torch.arange(S, device=q.device)
    if slopes is not None:
        t = t - slopes.double().view(H, 1, 1) * (at[:, None] - at).abs()
    t = t.masked_fill(~seen, -math.inf)
    p = torch.where(seen, torch.softmax(t, -1), 0.0)
    o = p @ v
    dp = do @ vt
    delta = (do * o).sum(-1, keepdim=True)
    ds = torch.where(seen, p * (dp - delta) * bend, 0.0)

    def group(x):
        return x.view(B, Hk, G, S, D).sum(2)

    pt, dst = p.transpose(2, 3).contiguous(), ds.transpose(2, 3).contiguous()
    dq, dk, dv = ds @ k * scale, group(dst @ q) * scale, group(pt @ do)
    # o: weights rounded to bf16, then o itself (kept to 2^-16 for the backward)
    off_o = (BF16 + FP32) * (p @ v.abs())
    off_delta = (do.abs() * (off_o + 2.0 ** -15 * o.abs())).sum(-1, keepdim=True)
    # dS: its own rounding, the sum it is less by, and the weights' fp32
    off_ds = BF16 * ds.abs() + bend * p * (
        off_delta + FP32 * (dp.abs() + delta.abs()
                            + do.abs() @ vt.abs()))
    if cap:
        # 1 - tanh^2 = 4 r (1 - r) of an r = 1 / (e^2x + 1) up to 1 in fp32: r is off by
        # 2^-23 (its sum and its reciprocal by 2^-24 each), 1 - r is exact from 1/2 on,
        # so four times their product by up to 4 x 2^-23, be it ever so small
        off_ds = off_ds + 2.0 ** -21 * p * (dp.abs() + delta.abs())
    off_ds = torch.where(seen, off_ds, 0.0)
    off = [off_o, off_ds @ k.abs() * abs(scale),
           group(off_ds.transpose(2, 3).contiguous() @ q.abs()) * abs(scale),
           group((BF16 + FP32) * (pt @ do.abs()))]
    values = [x.transpose(1, 2) for x in (o, dq, dk, dv)]
    # their own rounding; below it bf16's smallest numbers
    return values, [x.transpose(1, 2) * 1.01 + BF16 * y.abs() + 1e-30
                    for x, y in zip(off, values)]


def _check(got, values, off, names=("o", "dq", "dk", "dv")):
    for name, x, y, most in zip(names, got, values, off):
        far = (x.double() - y).abs()
        assert torch.isfinite(x).all(), name
        bad = far > most
        assert not bad.any(), (name, int(bad.sum()), float((far - most).max()),
                               bad.nonzero()[:4].tolist())


def _inputs(B, S, H, Hk, D, device, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, H + 2 * Hk, D, generator=g).bfloat16()
    x[:, :, :H] *= spread
    do = torch.randn(B, S, H, D, generator=g).bfloat16()
    x, do = x.to(device), do.to(device)
    return x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:], do


def _grads(q, k, v, do, rows, **how):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    o = masked_attention(q, k, v, rows, **how)
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))


DOCUMENTS = [[[1]], [[2], [1, -1]], [[40, 24], [-64]], [[33, 1, 31], [-5, 50, -10]],
             [[100, 157], [1, 255, -1]], [[64, 64, 128, 65], [321]],
             [[300, 20, 193], [256, 256, 1]], [[700, -40, 300]]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows", DOCUMENTS)
def test_spans(rows, causal):
    """What the spans say is what pair by pair is seen, both ways round, and they
    grow along a row."""
    ids = _ids(rows)
    g = torch.Generator().manual_seed(1)
    for prefix in [None] + [torch.randint(-2, 90, (len(rows), n), generator=g,
                                          dtype=torch.int32) for n in (0, 2, 7)]:
        if prefix is not None and not causal:
            continue
        lo, hi, klo, khi = _torch_spans(ids, prefix, causal).long()
        at = torch.arange(ids.shape[1])
        seen = _seen(ids, prefix, causal)
        assert torch.equal((at >= lo[..., None]) & (at < hi[..., None]), seen)
        assert torch.equal(((at >= klo[..., None]) & (at < khi[..., None]))
                           .transpose(1, 2), seen)
        for x in (lo, hi, klo, khi):
            assert (x[:, 1:] >= x[:, :-1]).all()


@pytest.mark.parametrize("cap,bias", [(0.0, False), (2.0, True)])
@pytest.mark.parametrize("causal", [True, False])
def test_formulas_cpu(causal, cap, bias):
    """The plain path on the CPU: values against pair by pair, gradients against
    differences in 64 bits."""
    ids = _ids([[5, 3, -2], [1, 6, 3]])
    prefix = torch.tensor([[2, 9], [0, 3]], dtype=torch.int32) if causal else None
    rows = packed_rows(ids, prefix, causal)
    g = torch.Generator().manual_seed(2)
    q, k, v, do = (torch.randn(2, 10, h, 4, generator=g, dtype=torch.float64)
                   for h in (4, 2, 2, 4))
    slopes = torch.tensor([0.5, 0.25, 0.1, 1.0]) if bias else None
    how = dict(scale=0.7, softcap=cap, alibi_slopes=slopes)
    values, _ = _reference(q, k, v, do, _seen(ids, prefix, causal), 0.7, cap, slopes)
    for x, y in zip(_grads(q, k, v, do, rows, **how), values):
        torch.testing.assert_close(x, y, rtol=1e-9, atol=1e-12)
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    assert torch.autograd.gradcheck(
        lambda *x: masked_attention(*x, rows, **how), (q, k, v))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (10.0, True)])
def test_hidden_infinities_cpu(value, cap, bias):
    """What a query does not see is not in its row nor in its gradients: padding,
    another document's keys, values and queries, a later token."""
    ids = _ids([[7, 6, -3], [-3, 5, 8]])
    seen = _seen(ids, None, True)
    slopes = torch.tensor([0.5, 0.1, 0.0, 2.0]) if bias else None
    how = dict(scale=0.3, softcap=cap, alibi_slopes=slopes)
    g = torch.Generator().manual_seed(7)
    q, k, v, do = (torch.randn(2, 16, h, 4, generator=g, dtype=torch.float64)
                   for h in (4, 2, 2, 4))
    pad = ids < 0
    for x in (q, k, v, do):
        x[pad] = value
    rows = packed_rows(ids)
    want, _ = _reference(q, k, v, do, seen, 0.3, cap, slopes)
    for x, y in zip(_grads(q, k, v, do, rows, **how), want):
        torch.testing.assert_close(x, y, rtol=1e-9, atol=1e-12)
        assert (x[pad] == 0).all()
    # one of the first document, seen by its last 2 tokens only
    other = torch.ones(2, 16, dtype=torch.bool)
    other[0, :7] = False
    well = other.clone()
    well[0, :5] = True
    for i in range(3):
        sick = [x.clone() for x in (q, k, v)]
        sick[i][0, 5] = value
        got = _grads(*sick, do, rows, **how)
        for x, y, part in zip(got, want, (well, other, other, other)):
            torch.testing.assert_close(x[part], y[part], rtol=1e-9, atol=1e-12)
        if i == 2:
            assert not torch.isfinite(got[0][0, 5:7]).any()
    # without documents: later tokens are as hidden
    q, k, v, do = (torch.where(pad[..., None, None], 0.0, x) for x in (q, k, v, do))
    want = _grads(q, k, v, do, None, **how)
    for x in (k, v):
        x[:, 12] = value
    for i, (x, y) in enumerate(zip(_grads(q, k, v, do, None, **how), want)):
        if i < 2:
            torch.testing.assert_close(x[:, :12], y[:, :12], rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("causal", [True, False])
def test_no_tokens_cpu(causal):
    for B, S in ((2, 0), (0, 5), (0, 0)):
        q, k, v = (torch.empty(B, S, h, 4, requires_grad=True) for h in (4, 2, 2))
        ids = torch.empty(B, S, dtype=torch.int64)
        for rows in (None, packed_rows(ids, causal=causal)):
            o = masked_attention(q, k, v, rows, causal=causal, softcap=1.0)
            assert o.shape == q.shape
            grads = torch.autograd.grad(o.sum(), (q, k, v))
            assert [x.shape for x in grads] == [x.shape for x in (q, k, v)]


def test_refusals():
    q, k, v, _ = _inputs(2, 6, 4, 2, 64, "cpu")
    ids = _ids([[6], [2, 4]])
    rows = packed_rows(ids)
    with pytest.raises(ValueError, match="rows of another batch"):
        masked_attention(q[:1], k[:1], v[:1], rows)
    with pytest.raises(ValueError, match="multiple of Hkv"):
        masked_attention(q[:, :, :3], k, v)
    with pytest.raises(ValueError, match="multiple of Hkv"):
        masked_attention(q, k, v[:, :5])
    with pytest.raises(ValueError, match="one type"):
        masked_attention(q, k.float(), v.float())
    for cap in (-1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="softcap"):
            masked_attention(q, k, v, softcap=cap)
    with pytest.raises(ValueError, match="one number a query head"):
        masked_attention(q, k, v, alibi_slopes=torch.ones(2))
    with pytest.raises(ValueError, match="no gradient"):
        masked_attention(q, k, v, alibi_slopes=torch.ones(4, requires_grad=True))
    with pytest.raises(ValueError, match="int32 or int64"):
        packed_rows(ids.float())
    with pytest.raises(ValueError, match="without causal"):
        packed_rows(ids, torch.ones(2, 2, dtype=torch.int32), causal=False)
    with pytest.raises(ValueError, match="prefix_lens"):
        packed_rows(ids, torch.ones(3, 2, dtype=torch.int32))


def _decode_inputs(lens, H, Hk, bs, device, seed=0, spread=1.0, spare=3):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).int()
    table = torch.full((len(lens), max(max(need), 1)), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    pools = [torch.randn(sum(need) + spare, Hk, bs, 128, generator=g).bfloat16()
             for _ in range(2)]
    q = torch.randn(len(lens), H, 128, generator=g).bfloat16() * spread
    return [x.to(device) for x in (q, *pools, table,
                                   torch.tensor(lens, dtype=torch.int32))]


def _decode_reference(q, kpool, vpool, table, lens, scale, cap, slopes):
    n, H, D = q.shape
    Hk = kpool.shape[1]
    out, off = torch.zeros(n, H, D).double(), torch.zeros(n, H, D).double()
    for i, length in enumerate(lens.tolist()):
        if not length:
            continue
        blocks = table[i, :-(-length // kpool.shape[2])].long()
        k, v = (x[blocks].double().cpu().transpose(1, 2).reshape(-1, Hk, D)[:length]
                for x in (kpool, vpool))
        far = torch.arange(length - 1, -1, -1).double()
        for h in range(H):
            t = (k[:, h * Hk // H] @ q[i, h].double().cpu()) * scale
            if cap:
                t = torch.tanh(t / cap) * cap
            if slopes is not None:
                t = t - float(slopes[h]) * far
            p = torch.softmax(t, 0)
            out[i, h] = p @ v[:, h * Hk // H]
            off[i, h] = FP32 * (p @ v[:, h * Hk // H].abs())
    return out, off + BF16 * out.abs() + 1e-30


@pytest.mark.parametrize("cap,bias", [(0.0, True), (5.0, False), (5.0, True)])
def test_decode_cpu(cap, bias):
    """The plain path: as a last row of masked_attention would have it, a bad block
    NaN for its own request alone, no request 0."""
    q, kp, vp, table, lens = _decode_inputs([1, 0, 16, 37], 4, 2, 16, "cpu")
    slopes = torch.tensor([0.5, 0.25, 0.1, 1.0]) if bias else None
    how = dict(softcap=cap, alibi_slopes=slopes)
    o = paged_decode_attention(q, kp, vp, table, lens, **how)
    want, off = _decode_reference(q, kp, vp, table, lens, 128 ** -0.5, cap, slopes)
    assert ((o.double() - want).abs() <= off).all()
    assert (o[1] == 0).all()
    k, v = (x[table[3, :3].long()].transpose(1, 2).reshape(1, -1, 2, 128)[:, :37]
            for x in (kp, vp))
    rows = torch.zeros(1, 37, 4, 128).bfloat16()
    rows[:, -1] = q[3]
    whole = masked_attention(rows, k, v, **how)[0, -1]
    torch.testing.assert_close(whole.float(), o[3].float(), rtol=2 * BF16, atol=1e-4)
    for bad in (-1, kp.shape[0], 2 ** 31 - 1):
        table[3, 1] = bad
        again = paged_decode_attention(q, kp, vp, table, lens, **how)
        assert torch.equal(again[:3], o[:3]) and again[3].isnan().all()


def test_decode_refusals():
    q, kp, vp, table, lens = _decode_inputs([5, 9], 4, 2, 16, "cpu")
    with pytest.raises(ValueError, match="softcap"):
        paged_decode_attention(q, kp, vp, table, lens, softcap=-1.0)
    with pytest.raises(ValueError, match="one number a query head"):
        paged_decode_attention(q, kp, vp, table, lens, alibi_slopes=torch.ones(3))
    with pytest.raises(ValueError, match="multiple of Hkv"):
        paged_decode_attention(q[:, :3], kp, vp, table, lens, softcap=1.0)
    with pytest.raises(ValueError, match="block_table"):
        paged_decode_attention(q, kp, vp, table[:1], lens, softcap=1.0)


# ------------------------------------------------------------------------- GPU


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows", DOCUMENTS + [[[5000, 1, 7000, 3000]], [[20000]],
                                              [[4095, 4097, -1], [1, 8191, 1]],
                                              [[1] * 1500]])
def test_spans_gpu(rows, causal):
    ids = _ids(rows)
    g = torch.Generator().manual_seed(1)
    for prefix in [None] + [torch.randint(-2, 90, (len(rows), n), generator=g,
                                          dtype=torch.int32) for n in (0, 2, 7)]:
        if prefix is not None and not causal:
            continue
        want = _torch_spans(ids, prefix, causal)
        for kind in (torch.int32, torch.int64):
            got = packed_rows(ids.to("cuda", kind),
                              None if prefix is None else prefix.to("cuda", kind),
                              causal)
            assert got.spans.dtype is torch.int32
            assert torch.equal(got.spans.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("cap,bias,spread", [(0.0, False, 1), (0.0, True, 1),
                                             (20.0, False, 4), (5.0, True, 2)])
@pytest.mark.parametrize("heads", [(2, 2, 64), (4, 2, 96), (6, 1, 128), (8, 8, 64)])
@pytest.mark.parametrize("rows", DOCUMENTS)
def test_documents_gpu(rows, heads, cap, bias, spread):
    H, Hk, D = heads
    ids = _ids(rows)
    B, S = ids.shape
    q, k, v, do = _inputs(B, S, H, Hk, D, "cuda", spread=spread)
    slopes = torch.exp2(-torch.arange(1, H + 1).float()).cuda() if bias else None
    g = torch.Generator().manual_seed(3)
    prefix = torch.randint(0, 60, (B, 3), generator=g, dtype=torch.int32)
    for causal, pre in ((True, None), (True, prefix), (False, None)):
        packed = packed_rows(ids.cuda(), None if pre is None else pre.cuda(), causal)
        got = _grads(q, k, v, do, packed, softcap=cap, alibi_slopes=slopes)
        seen = _seen(ids, pre, causal).cuda()
        _check(got, *_reference(q, k, v, do, seen, D ** -0.5, cap, slopes))
        empty = ~seen.any(2)
        for x in got[:2]:
            assert (x[empty] == 0).all()
        for x in got[2:]:
            assert (x[~seen.any(1)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S", [1, 3, 64, 129, 511])
@pytest.mark.parametrize("scale", [None, -0.2, 0.0])
def test_without_rows_gpu(S, causal, scale):
    q, k, v, do = _inputs(2, S, 4, 2, 128, "cuda", seed=S)
    at = torch.arange(S)
    seen = (at <= at[:, None] if causal else at == at).expand(2, S, S).cuda()
    slopes = torch.tensor([0.5, 0.1, 0.0, 2.0]).cuda()
    for cap, sl in ((0.0, None), (10.0, None), (3.0, slopes)):
        got = _grads(q, k, v, do, None, causal=causal, scale=scale, softcap=cap,
                     alibi_slopes=sl)
        _check(got, *_reference(q, k, v, do, seen,
                                128 ** -0.5 if scale is None else scale, cap, sl))


@pytest.mark.gpu
def test_long_rows_gpu():
    """Splits of the gradients of shared heads, many tiles, uneven documents."""
    ids = _ids([[1500, 30, 2, 400, 1068, -96]])
    q, k, v, do = _inputs(1, ids.shape[1], 8, 2, 128, "cuda", seed=5, spread=3)
    prefix = torch.tensor([[700, 30, 5, 0, 1]], dtype=torch.int32)
    rows = packed_rows(ids.cuda(), prefix.cuda())
    got = _grads(q, k, v, do, rows, softcap=30.0)
    seen = _seen(ids, prefix, True).cuda()
    _check(got, *_reference(q, k, v, do, seen, 128 ** -0.5, 30.0, None))
    again = _grads(q, k, v, do, rows, softcap=30.0)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (10.0, True)])
def test_hidden_infinities_gpu(value, cap, bias):
    """What a query does not see is not in its row, whatever it holds: padding,
    another document, a later token."""
    ids = _ids([[70, 60, -30], [-3, 50, 107]])
    H, Hk, D = 4, 2, 64
    slopes = torch.tensor([0.5, 0.1, 0.0, 2.0]).cuda() if bias else None
    how = dict(softcap=cap, alibi_slopes=slopes)
    rows = packed_rows(ids.cuda())
    seen = _seen(ids, None, True).cuda()
    q, k, v, do = _inputs(2, 160, H, Hk, D, "cuda", seed=7)
    pad = (ids < 0).cuda()
    for x in (q, k, v, do):
        x[pad] = value
    got = _grads(q, k, v, do, rows, **how)
    want = _reference(q, k, v, do, seen, D ** -0.5, cap, slopes)
    _check(got, *want)
    for x in (got[0], got[1], got[2], got[3]):
        assert (x[pad] == 0).all()
    # one key and value of the first document, seen by its last 5 tokens only
    sick_k, sick_v = k.clone(), v.clone()
    sick_v[0, 65] = value
    o = masked_attention(q, sick_k, sick_v, rows, **how)
    well = torch.ones(2, 160, dtype=torch.bool)
    well[0, 65:70] = False
    assert torch.equal(torch.isfinite(o).all(-1).all(-1).cpu(), well)
    far = (o.double() - want[0][0]).abs() <= want[1][0]
    assert far[well].all()
    # and its gradients: rows of the other documents are as they were
    got = _grads(q, sick_k, sick_v, do, rows, **how)
    other = (ids != ids[0, 0]).cuda()
    other[1] = True
    for x, y, off in zip(got[1:], want[0][1:], want[1][1:]):
        assert ((x.double() - y).abs() <= off)[other].all()


@pytest.mark.gpu
def test_layouts_gpu():
    """Strides, alignment and broadcast inputs other than a joint projection's."""
    ids = _ids([[90, 40], [20, 110]])
    rows = packed_rows(ids.cuda())
    seen = _seen(ids, None, True).cuda()
    q, k, v, do = _inputs(2, 130, 4, 2, 64, "cuda", seed=9)
    want = _reference(q, k, v, do, seen, 0.125, 0.0, None)

    def heads_first(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    def odd(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
        flat[1:] = x.reshape(-1)
        return flat[1:].view(x.shape)

    def spread(x):
        wide = torch.empty(*x.shape[:3], 2 * x.shape[3], dtype=x.dtype, device=x.device)
        wide[..., ::2] = x
        return wide[..., ::2]

    for change in (heads_first, odd, spread):
        _check(_grads(*(change(x) for x in (q, k, v, do)), rows), *want)
    # one batch row's key for both rows; an expanded gradient
    k1 = k[:1].expand(2, -1, -1, -1)
    one = do[:, :1, :1].expand(2, 130, 4, 64)
    want = _reference(q, k1, v, one, seen, 0.125, 0.0, None)
    _check(_grads(q, k1, v, one, rows), *want)
    leaf = k[:1].detach().requires_grad_()
    o = masked_attention(q, leaf.expand(2, -1, -1, -1), v, rows)
    dk, = torch.autograd.grad(o, leaf, one)
    # of a sum in bf16 of two rows: each term's and the sum's rounding
    y, off = want[0][2], want[1][2]
    assert ((dk.double() - y.sum(0)).abs() <= off.sum(0) + 2 * BF16 * y.abs().sum(0)
            ).all()


@pytest.mark.gpu
def test_differences_gpu():
    """The kernels' gradients against differences of the formulas in 64 bits."""
    ids = _ids([[100, 41]])
    prefix = torch.tensor([[30, 0]], dtype=torch.int32)
    seen = _seen(ids, prefix, True).cuda()
    slopes = torch.tensor([0.3, 0.05]).cuda()
    q, k, v, do = _inputs(1, 141, 2, 1, 96, "cuda", seed=11, spread=2)
    rows = packed_rows(ids.cuda(), prefix.cuda())
    got = _grads(q, k, v, do, rows, softcap=8.0, alibi_slopes=slopes)

    def loss(*x):
        o = _reference(*x, do, seen, 96 ** -0.5, 8.0, slopes)[0][0]
        return float((o * do.double()).sum())

    _, off = _reference(q, k, v, do, seen, 96 ** -0.5, 8.0, slopes)
    g = torch.Generator(device="cuda").manual_seed(4)
    for i in range(3):
        x = [t.double() for t in (q, k, v)]
        u = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        ends = []
        for step in (1e-5, -1e-5):
            y = list(x)
            y[i] = x[i] + step * u
            ends.append(loss(*y))
        slope = (ends[0] - ends[1]) / 2e-5
        most = float((off[i + 1] * u.abs()).sum()) + 1e-4
        assert abs(slope - float((got[i + 1].double() * u).sum())) <= most


@pytest.mark.gpu
def test_graph_and_streams_gpu():
    """Captured with its backward and replayed over changing inputs beside eager
    calls; and on another stream than the current one's."""
    ids = _ids([[150, 90], [60, 160, -20]]).cuda()
    static = [x.clone() for x in _inputs(2, 240, 4, 2, 64, "cuda")]

    def step(q, k, v, do):
        return _grads(q, k, v, do, packed_rows(ids), softcap=10.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in range(4):
        fresh = _inputs(2, 240, 4, 2, 64, "cuda", seed=20 + seed)
        want = step(*fresh)
        for x, y in zip(static, fresh):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            there = step(*fresh)
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(there, want))


@pytest.mark.gpu
def test_refusals_gpu():
    q, k, v, _ = _inputs(1, 8, 2, 2, 64, "cuda")
    with pytest.raises(ValueError, match="bf16"):
        masked_attention(q.half(), k.half(), v.half())
    with pytest.raises(ValueError, match="heads of 64"):
        masked_attention(q[..., :32], k[..., :32], v[..., :32])
    with pytest.raises(ValueError, match="device"):
        masked_attention(q, k, v, packed_rows(torch.zeros(1, 8, dtype=torch.int32)))
    empty = torch.empty(0, 8, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert masked_attention(empty, empty, empty).shape == empty.shape
    none = torch.empty(2, 0, 2, 64, dtype=torch.bfloat16, device="cuda",
                       requires_grad=True)
    ids = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    masked_attention(none, none, none, packed_rows(ids)).sum().backward()
    # spans that say more than there is read nothing outside of the rows
    wild = torch.full((4, 1, 8), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    wild[::2] = -2 ** 31
    full = masked_attention(q, k, v, causal=False)
    assert torch.equal(masked_attention(q, k, v, PackedRows(wild, False)), full)


@pytest.mark.gpu
@pytest.mark.parametrize("cap,bias,spread", [(0.0, True, 1), (30.0, False, 4),
                                             (5.0, True, 2)])
@pytest.mark.parametrize("lens,heads,bs", [
    ([1], (8, 8), 64), ([33, 0, 1, 64], (32, 8), 64), ([31, 32, 500], (28, 4), 16),
    ([130, 129], (16, 1), 32), ([7, 300], (5, 5), 5), ([3000, 10, 700], (32, 8), 128)])
@pytest.mark.parametrize("splits", [None, 1, 7])
def test_decode_gpu(lens, heads, bs, splits, cap, bias, spread):
    H, Hk = heads
    q, kp, vp, table, n = _decode_inputs(lens, H, Hk, bs, "cuda", spread=spread)
    slopes = torch.exp2(-torch.arange(1, H + 1).float() / 4).cuda() if bias else None
    for scale in (None, -0.1):
        o = paged_decode_attention(q, kp, vp, table, n, splits=splits, scale=scale,
                                   softcap=cap, alibi_slopes=slopes)
        want, off = _decode_reference(q, kp, vp, table, n,
                                      128 ** -0.5 if scale is None else scale, cap,
                                      slopes)
        assert ((o.double().cpu() - want).abs() <= off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64])
def test_decode_bad_pages_gpu(bs):
    """A block that is not in the pool, and a length past the table's end."""
    q, kp, vp, table, n = _decode_inputs([100, 200, 40], 8, 2, bs, "cuda")
    slopes = torch.full((8,), 0.1).cuda()
    o = paged_decode_attention(q, kp, vp, table, n, softcap=10.0, alibi_slopes=slopes)
    for bad in (-1, kp.shape[0], 2 ** 31 - 1, -2 ** 31):
        sick = table.clone()
        sick[1, 2] = bad
        for splits in (None, 1, 3):
            got = paged_decode_attention(q, kp, vp, sick, n, splits=splits,
                                         softcap=10.0, alibi_slopes=slopes)
            assert got[1].isnan().all() and torch.isfinite(got[[0, 2]]).all()
    # what lies behind a request's last key does not count
    vp2, kp2 = vp.clone(), kp.clone()
    last = int(table[0, 100 // bs])
    kp2[last, :, 100 % bs:] = float("nan")
    vp2[last, :, 100 % bs:] = float("nan")
    again = paged_decode_attention(q, kp2, vp2, table, n, softcap=10.0,
                                   alibi_slopes=slopes)
    assert torch.equal(again, o)
    long = n.clone()
    long[1] = 2 ** 31 - 1
    table[1] = table[1].clamp(min=0)
    most = n.clone()
    most[1] = table.shape[1] * bs
    assert torch.equal(paged_decode_attention(q, kp, vp, table, long, softcap=10.0),
                       paged_decode_attention(q, kp, vp, table, most, softcap=10.0))
    with pytest.raises(ValueError, match="up to 16 a key head"):
        paged_decode_attention(q.float(), kp, vp, table, n, softcap=1.0)


@pytest.mark.gpu
def test_second_derivatives_raise_gpu():
    """Gradients that a graph is asked for say so when they are differentiated, and
    are the same until then."""
    q, k, v, do = _inputs(1, 9, 2, 1, 64, "cuda")
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    plain = torch.autograd.grad(masked_attention(*leaves), leaves, do)
    o = masked_attention(*leaves)
    graph = torch.autograd.grad(o, leaves, do, create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(plain, graph))
    with pytest.raises(RuntimeError, match="differentiable once"):
        graph[0].float().sum().backward()
    # only the gradient that is asked for, by other types of a call
    dv, = torch.autograd.grad(masked_attention(q, k, leaves[2]), leaves[2], do)
    assert torch.equal(dv, plain[2])
    with torch.no_grad():
        assert not masked_attention(*leaves).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-3, 0.5, 200.0, 201.0, 1e3, 1e5, 1e20])
def test_caps_gpu(cap):
    """Caps far below and far above the scores: what is left of them is as exact."""
    ids = _ids([[90, 40]])
    seen = _seen(ids, None, True).cuda()
    q, k, v, do = _inputs(1, 130, 4, 2, 64, "cuda", seed=13, spread=4)
    got = _grads(q, k, v, do, packed_rows(ids.cuda()), softcap=cap)
    _check(got, *_reference(q, k, v, do, seen, 0.125, cap, None))
    q, kp, vp, table, n = _decode_inputs([130, 75], 8, 2, 16, "cuda", spread=4)
    o = paged_decode_attention(q, kp, vp, table, n, softcap=cap)
    want, off = _decode_reference(q, kp, vp, table, n, 128 ** -0.5, cap, None)
    assert ((o.double().cpu() - want).abs() <= off).all()


@pytest.mark.gpu
def test_far_rows_gpu():
    """Rows and blocks whose places do not fit 32 bits."""
    far = torch.empty(1, 300, 1 << 23, dtype=torch.bfloat16, device="cuda")
    q, k, v, do = _inputs(1, 300, 2, 1, 128, "cuda", seed=15)
    want = _grads(q, k, v, do, None, softcap=20.0)
    there = []
    for i, x in enumerate((q, k, v, do)):
        y = far[:, :, i * 4096:i * 4096 + x.shape[2] * 128].unflatten(-1, (-1, 128))
        there.append(y.copy_(x))
    got = _grads(*there, None, softcap=20.0)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    del far, there, got
    q, kp, vp, table, n = _decode_inputs([130, 75], 8, 2, 64, "cuda")
    want = paged_decode_attention(q, kp, vp, table, n, softcap=20.0)
    first = (1 << 31) // (2 * 64 * 128) + 1
    pools = [torch.empty(first + len(kp), 2, 64, 128, dtype=torch.bfloat16,
                         device="cuda") for _ in "kv"]
    for pool, x in zip(pools, (kp, vp)):
        pool[first:] = x
    table = torch.where(table < 0, table, table + first)
    assert torch.equal(want, paged_decode_attention(q, *pools, table, n, softcap=20.0))


@pytest.mark.gpu
def test_seen_infinities_gpu():
    """What a query does see stays what it is: rows behind a value that is not finite,
    gradients that are not, and the rows and keys apart from them."""
    q, k, v, do = _inputs(1, 300, 2, 1, 64, "cuda", seed=17)
    ids = _ids([[200, 100]])
    rows = packed_rows(ids.cuda())
    want = _reference(q, k, v, do, _seen(ids, None, True).cuda(), 0.125, 0.0, None)

    def near(name, x, part):
        i = ("o", "dq", "dk", "dv").index(name)
        assert ((x.double() - want[0][i]).abs() <= want[1][i])[0, part].all(), name

    sick = v.clone()
    sick[0, 40] = float("inf")
    got = _grads(q, k, sick, do, rows)
    assert (got[0][0, 40:200] == float("inf")).all()
    near("o", got[0], slice(200, None))
    near("o", got[0], slice(40))
    for name, x in zip(("dq", "dk", "dv"), got[1:]):
        near(name, x, slice(200, None))
    near("dq", got[1], slice(40))
    do = do.clone()
    do[0, 250] = float("nan")
    got = _grads(q, k, v, do, rows)
    for name, x in zip(("dq", "dk", "dv"), got[1:]):
        near(name, x, slice(200))
        near(name, x, slice(251, None))
    near("dq", got[1], slice(250))
    assert got[1][0, 250].isnan().all() and got[2][0, 200:251].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [True, False])
def test_wild_spans_gpu(queries):
    """Spans whose ends lie anywhere are those inside of the row: forward and both
    passes of the backward read and write nothing else."""
    ends = [-2 ** 31, -1, 0, 3, 69, 70, 2 ** 31 - 2, 2 ** 31 - 1]
    S = 70
    q, k, v, do = _inputs(1, S, 2, 1, 64, "cuda", seed=19)
    for lo in ends:
        for hi in ends:
            spans = torch.tensor([0, S, 0, S], dtype=torch.int32).repeat(S, 1).t()
            spans[0 if queries else 2], spans[1 if queries else 3] = lo, hi
            spans = spans.contiguous().view(4, 1, S)
            got = _grads(q, k, v, do, PackedRows(spans.cuda(), False))
            want = _grads(q, k, v, do, PackedRows(spans.clamp(0, S).cuda(), False))
            # (keys seen by queries that see nothing have no gradient that is a number)
            for x, y in zip(got, want):
                torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)
            if queries and max(lo, 0) >= min(hi, S):
                assert not got[0].any() and not got[1].any()


def _long_prefixes(device):
    """Lengths past 32 bits mean all of the document, or nothing below 0."""
    ids = _ids([[5, 4, 3], [6, 6]]).to(device)
    lens = torch.tensor([[2 ** 31, 2 ** 32 + 1, -2 ** 32 + 2], [2 ** 63 - 1, -2 ** 63, 2]])
    got = packed_rows(ids, lens.to(device))
    want = packed_rows(ids, lens.clamp(0, 12).int().to(device))
    assert torch.equal(got.spans, want.spans)


def test_long_prefixes_cpu():
    _long_prefixes("cpu")


@pytest.mark.gpu
def test_long_prefixes_gpu():
    _long_prefixes("cuda")


def _long_pages(device):
    """Blocks and lengths past 32 bits are not others that they would wrap to."""
    q, kp, vp, table, lens = _decode_inputs([20, 32, 9], 4, 2, 16, device)
    table, lens = table.clamp(min=0).long(), lens.long()
    o = paged_decode_attention(q, kp, vp, table, lens, softcap=5.0)
    for far in (2 ** 32, -2 ** 32, 2 ** 62):
        sick = table.clone()
        sick[1, 1] += far
        got = paged_decode_attention(q, kp, vp, sick, lens, softcap=5.0)
        assert got[1].isnan().all() and torch.equal(got[::2], o[::2])
    most = lens.clone()
    most[0] = table.shape[1] * 16
    long = lens.clone()
    long[0] += 2 ** 32
    assert torch.equal(paged_decode_attention(q, kp, vp, table, long, softcap=5.0),
                       paged_decode_attention(q, kp, vp, table, most, softcap=5.0))
    long[0] = 5 - 2 ** 32
    assert not paged_decode_attention(q, kp, vp, table, long, softcap=5.0)[0].any()


def test_long_pages_cpu():
    _long_pages("cpu")


@pytest.mark.gpu
def test_long_pages_gpu():
    _long_pages("cuda")


@pytest.mark.gpu
def test_wide_tables_gpu():
    """Tables wider than any request, and one of more keys than are counted."""
    q, kp, vp, table, lens = _decode_inputs([20, 32], 4, 2, 16, "cuda")
    want = paged_decode_attention(q, kp, vp, table, lens, splits=1, softcap=5.0)
    wide = torch.full((2, 1 << 20), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    for splits in (None, 1):
        o = paged_decode_attention(q, kp, vp, wide, lens, splits=splits, softcap=5.0)
        torch.testing.assert_close(o.float(), want.float(), rtol=2 * BF16, atol=1e-4)
    far = table[:, :1].expand(2, (1 << 26) + 1)
    with pytest.raises(ValueError, match="2\\^30 keys"):
        paged_decode_attention(q, kp, vp, far, lens, softcap=5.0)
    many = 1 << 12
    with pytest.raises(ValueError, match="2\\^31 blocks"):
        paged_decode_attention(q[:1].expand(many, -1, -1), kp, vp,
                               table[:1, :1].expand(many, 1 << 19),
                               lens[:1].expand(many), softcap=5.0)


def _low_scores(device, kind, D):
    """Rows whose scores are all far below 0: their softmax is that of the differences,
    in both forms."""
    S, H, Hk = 40, 4, 2
    g = torch.Generator().manual_seed(21)
    q = torch.full((1, S, H, D), 1e15).to(device, kind)
    k = torch.full((1, S, Hk, D), -1e15).to(device, kind)
    v = torch.randn(1, S, Hk, D, generator=g).to(device, kind)
    n = torch.arange(1, S + 1, device=device).double()[:, None, None]
    want = (v[0].double().cumsum(0) / n).repeat_interleave(H // Hk, 1)
    off = v[0].double().abs().cumsum(0).repeat_interleave(H // Hk, 1) / n
    off = (BF16 + FP32) * off + BF16 * want.abs()
    flat = torch.zeros(H, device=device)
    pools = [x.view(1, S // 8, 8, Hk, D)[0].transpose(1, 2).contiguous() for x in (k, v)]
    table = torch.arange(S // 8, device=device, dtype=torch.int32)[None]
    for how in (dict(alibi_slopes=flat), dict(softcap=9e29),
                dict(softcap=9e29, alibi_slopes=flat)):
        o = masked_attention(q, k, v, scale=1.0, **how)
        assert ((o[0].double() - want).abs() <= off).all(), how
        for length in (1, 33, S):
            o = paged_decode_attention(q[:, 0], *pools, table, torch.tensor(
                [length], dtype=torch.int32, device=device), scale=1.0, **how)
            near = (o[0].double() - want[length - 1]).abs() <= off[length - 1]
            assert near.all(), (how, length)


def test_low_scores_cpu():
    _low_scores("cpu", torch.float32, 128)


@pytest.mark.gpu
def test_low_scores_gpu():
    _low_scores("cuda", torch.bfloat16, 128)


def _decode_transforms(device, kind):
    """A tangent, a transform's gradient and a transform's batch."""
    q, kp, vp, table, lens = _decode_inputs([20, 32], 4, 2, 16, device)
    q, kp, vp = (x.to(kind) for x in (q, kp, vp))
    table = table.clamp(min=0)
    how = dict(softcap=5.0, alibi_slopes=torch.full((4,), 0.1, device=device))

    def answer(q):
        return paged_decode_attention(q, kp, vp, table, lens, **how)

    o, slope = torch.func.jvp(answer, (q,), (q,))
    grads = torch.func.grad(lambda q: answer(q).sum())(q)
    many = torch.func.vmap(answer)(torch.stack([q, -q]))
    return answer, q, [x.double().cpu() for x in (o, slope, grads, many)]


def test_decode_transforms_cpu():
    """Against differences in 64 bits."""
    answer, q, (o, slope, grads, many) = _decode_transforms("cpu", torch.float64)
    h = 1e-5
    ends = [answer(q * (1 + s * h)) for s in (1, -1)]
    torch.testing.assert_close((ends[0] - ends[1]) / (2 * h), slope, rtol=1e-6, atol=1e-8)
    torch.testing.assert_close((grads * q).sum(), slope.sum(), rtol=1e-9, atol=1e-9)
    assert torch.equal(o, answer(q)) and torch.equal(many[1], answer(-q))


@pytest.mark.gpu
def test_decode_transforms_gpu():
    """They see the formulas, which a kernel called directly would pass by."""
    _, _, got = _decode_transforms("cuda", torch.bfloat16)
    _, _, want = _decode_transforms("cpu", torch.float64)
    for x, y in zip(got, want):
        # bf16's rounding at the end; the tangent is of sums of fp32 beside it
        assert ((x - y).abs() <= BF16 * y.abs() + FP32 * y.abs().max()).all()


@pytest.mark.gpu
def test_decode_without_gradient_gpu():
    """Queries or pools that need a gradient: the same answer, and a word when the
    gradient is asked for."""
    q, kp, vp, table, lens = _decode_inputs([20, 0, 32], 4, 2, 16, "cuda")
    want = paged_decode_attention(q, kp, vp, table, lens, softcap=5.0)
    assert not want.requires_grad
    for i in range(3):
        ins = [x.detach().requires_grad_(i == j) for j, x in enumerate((q, kp, vp))]
        o = paged_decode_attention(*ins, table, lens, softcap=5.0)
        assert torch.equal(o, want) and o.requires_grad
        with pytest.raises(RuntimeError, match="no gradient on a GPU"):
            o.float().sum().backward()
        none = paged_decode_attention(ins[0][:0], *ins[1:], table[:0], lens[:0],
                                      softcap=5.0)
        assert none.shape == (0, 4, 128)
        with torch.no_grad():
            o = paged_decode_attention(*ins, table, lens, softcap=5.0)
        assert torch.equal(o, want) and not o.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-37, 1e-39, 1e-46, -1e-37, -1e-39, -1e-300])
def test_tiny_scales_gpu(scale):
    """Scales that fp32 does not hold, or hardly, leave the mean of what is seen."""
    q, k, v, do = _inputs(1, 70, 2, 1, 64, "cuda", seed=23)
    at = torch.arange(70)
    seen = (at <= at[:, None])[None].cuda()
    for cap in (0.0, 5.0):
        got = _grads(q, k, v, do, None, scale=scale, softcap=cap)
        _check(got, *_reference(q, k, v, do, seen, scale, cap, None))


@pytest.mark.gpu
def test_size_refusals_gpu():
    """Sizes that the kernels do not count are refused under the call's own name."""
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    for shape in ((1, 1 << 30, 1, 64), (1 << 15, 1 << 16, 1, 64)):
        with pytest.raises(RuntimeError, match="masked_attention: size"):
            masked_attention(*(q.expand(shape) for _ in "qkv"))


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [150.0, 201.0, 1e4])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 2, 96), (6, 1, 128)])
def test_wide_caps_gpu(heads, bias, cap):
    """Caps on either side of those that take a series near 0, with the distance bias
    and without, heads of every size; the single token's form as well."""
    H, Hk, D = heads
    ids = _ids([[90, 40], [33, -7, 90]])
    seen = _seen(ids, None, True).cuda()
    slopes = torch.exp2(-torch.arange(1, H + 1).float()).cuda() if bias else None
    q, k, v, do = _inputs(2, 130, H, Hk, D, "cuda", seed=25, spread=4)
    got = _grads(q, k, v, do, packed_rows(ids.cuda()), softcap=cap, alibi_slopes=slopes)
    _check(got, *_reference(q, k, v, do, seen, D ** -0.5, cap, slopes))
    q, kp, vp, table, n = _decode_inputs([130, 75, 0, 700], H, Hk, 16, "cuda", spread=4)
    for splits in (None, 1):
        o = paged_decode_attention(q, kp, vp, table, n, splits=splits, softcap=cap,
                                   alibi_slopes=slopes)
        want, off = _decode_reference(q, kp, vp, table, n, 128 ** -0.5, cap, slopes)
        assert ((o.double().cpu() - want).abs() <= off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("spread", [1, 4, 8])
@pytest.mark.parametrize("heads", [(4, 1, 128), (4, 4, 64), (4, 2, 96)])
def test_gradients_digits_gpu(heads, spread, cap):
    """Gradients of queries and keys are off 64 bits by little more than their own
    rounding, scores close together or far apart: scores' gradients keep 16 bits, and
    what is left is the weights' rounding in sum(do o), which is half of a score's
    gradient at most, sqrt(1 + 1 / 4) of the own rounding in all. A rounding of the
    scores' gradients to bf16 would be sqrt(2) and more."""
    H, Hk, D = heads
    q, k, v, do = _inputs(1, 1024, H, Hk, D, "cuda", seed=3, spread=spread)
    at = torch.arange(1024)
    seen = (at <= at[:, None])[None].cuda()
    got = _grads(q, k, v, do, None, softcap=cap)
    values, _ = _reference(q, k, v, do, seen, D ** -0.5, cap, None)
    for name, x, y in zip(("dq", "dk"), got[1:3], values[1:3]):
        own = (y.bfloat16().double() - y).norm()
        assert (x.double() - y).norm() <= 1.25 ** 0.5 * 1.05 * own, name
