"""Operators of training and answering on packed documents, one call at a time:

  attention   causal or full attention, forward and backward, over rows that hold
              several documents, with prefixes that see themselves both ways, scores
              capped by a tanh and a bias that falls with the distance
  decode      one new token a request over the paged key/value pool, with the same
              cap and bias
  heads       RMS norms of the queries' and keys' heads and the position rotation,
              forward and backward
  logprobs    log probabilities of given tokens with the entropy and the best
              alternatives, forward and backward

``listed`` names the cases, ``draw`` gives more of the same ranges. Where ``own`` is
false ``run`` computes the formulas by elementary operations in 32 bits, else by the
framework's operators. ``exact`` computes them in 64 bits.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
IGNORE = -100


def listed():
    return [
        # a short fine-tuning batch: two rows of a few questions and answers
        dict(name="attention short prefixes", op="attention", batch=2, seq=333,
             heads=8, kv_heads=8, dim=64, documents=3, pad=21, causal=True,
             prefix=True, cap=0.0, bias=False),
        # an encoder with a distance bias over packed sentences, every key seen
        dict(name="attention encoder distance", op="attention", batch=8, seq=1999,
             heads=12, kv_heads=12, dim=64, documents=11, pad=0, causal=False,
             prefix=False, cap=0.0, bias=True),
        # prompts and answers under capped scores, heads of 96
        dict(name="attention capped prefixes", op="attention", batch=2, seq=4096,
             heads=32, kv_heads=32, dim=96, documents=4, pad=100, causal=True,
             prefix=True, cap=50.0, bias=False),
        # pre-training on packed documents, grouped key heads
        dict(name="attention documents", op="attention", batch=4, seq=4096,
             heads=32, kv_heads=8, dim=128, documents=9, pad=0, causal=True,
             prefix=False, cap=0.0, bias=False),
        # one long document of a long context, capped
        dict(name="attention capped 8192", op="attention", batch=1, seq=8192,
             heads=32, kv_heads=8, dim=128, documents=1, pad=0, causal=True,
             prefix=False, cap=30.0, bias=False),
        # a single chat, one token at a time
        dict(name="decode chat", op="decode", requests=1, context=700, heads=32,
             kv_heads=8, block=64, cap=50.0, bias=False),
        # a serving batch of uneven requests under a distance bias
        dict(name="decode batch", op="decode", requests=48, context=4000, heads=32,
             kv_heads=8, block=64, cap=0.0, bias=True),
        # the queries and keys of one decoding step
        dict(name="heads decode", op="heads", type="bf16", batch=16, seq=1, heads=32,
             kv_heads=8, dim=128, rotated=128, layout="half", train=False),
        # a training step's, out of the joint projection
        dict(name="heads train", op="heads", type="bf16", batch=2, seq=4096, heads=32,
             kv_heads=8, dim=128, rotated=128, layout="half", train=True),
        # half of smaller heads turned, neighbours in pairs, odd length
        dict(name="heads train interleaved", op="heads", type="fp16", batch=3, seq=1777,
             heads=28, kv_heads=4, dim=64, rotated=32, layout="interleaved",
             train=True),
        # the answer of a decoding step: the sampled tokens and five others
        dict(name="logprobs decode", op="logprobs", type="bf16", rows=24, vocab=128256,
             top=5, train=False),
        # a policy's update: log probabilities and entropy of a batch's answers
        dict(name="logprobs train", op="logprobs", type="bf16", rows=4096, vocab=128256,
             top=0, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    op = rng.choice(["attention", "attention", "decode", "heads", "logprobs"])
    if op == "attention":
        kv, group = rng.choice([(8, 4), (8, 1), (4, 7), (12, 1), (2, 16), (32, 1)])
        causal = rng.random() < 0.75
        seq = _log(rng, 64, 8192)
        return dict(op=op, batch=_log(rng, 1, 8), seq=seq, heads=kv * group,
                    kv_heads=kv, dim=rng.choice([64, 96, 128]),
                    documents=rng.randint(1, max(1, min(12, seq // 16))),
                    pad=rng.choice([0, rng.randint(1, seq // 8)]), causal=causal,
                    prefix=causal and rng.random() < 0.5,
                    cap=rng.choice([0.0, 20.0, 30.0, 50.0]),
                    bias=rng.random() < 0.4)
    if op == "decode":
        kv, group = rng.choice([(8, 4), (32, 1), (4, 7), (1, 16)])
        cap = rng.choice([0.0, 30.0, 50.0])
        return dict(op=op, requests=_log(rng, 1, 64), context=_log(rng, 100, 16000),
                    heads=kv * group, kv_heads=kv, block=rng.choice([16, 32, 64, 128]),
                    cap=cap, bias=not cap or rng.random() < 0.5)
    if op == "heads":
        kv, group = rng.choice([(8, 4), (32, 1), (4, 7), (2, 8)])
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        train = rng.random() < 0.6
        return dict(op=op, type=rng.choice(["bf16", "fp16", "fp32"]),
                    batch=_log(rng, 1, 4 if train else 64),
                    seq=_log(rng, 16, 4096) if train else 1, heads=kv * group,
                    kv_heads=kv, dim=dim, rotated=rng.choice([dim, dim // 2]),
                    layout=rng.choice(["half", "interleaved"]), train=train)
    train = rng.random() < 0.5
    return dict(op=op, type=rng.choice(["bf16", "fp16", "fp32"]),
                rows=_log(rng, 1, 4096 if train else 128),
                vocab=_log(rng, 1000, 200000), top=0 if train else rng.randint(0, 20),
                train=train)


def _scores(case):
    """Scores that the plain form makes."""
    return case["batch"] * case["heads"] * case["seq"] ** 2 \
        if case["op"] == "attention" else 0


def draw(rng):
    """No more work than in a listed case, for the plain form either."""
    most = [(work(c), _scores(c)) for c in listed()]
    while True:
        case = _drawn(rng)
        w, n = work(case), _scores(case)
        if any(w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"] and n <= top
               for m, top in most):
            return case


# ------------------------------------------------------------------------ inputs


def _lengths(case):
    """The documents' lengths of each row: uneven, by the sizes alone, so that the
    work is the same for every seed (which changes their order)."""
    rng = random.Random("%(seq)d %(documents)d %(pad)d %(batch)d" % case)
    rows = []
    for _ in range(case["batch"]):
        left, n = case["seq"] - case["pad"], case["documents"]
        shares = [rng.uniform(0.1, 1.0) ** 2 for _ in range(n)]
        lens = [max(1, int(left * s / sum(shares))) for s in shares]
        lens[lens.index(max(lens))] += left - sum(lens)
        rows.append(lens)
    return rows


def _prefix_of(length):
    return length // 3


def _pairs(case):
    """Pairs of a query and a key that it sees."""
    total = 0
    for lens in _lengths(case):
        for n in lens:
            p = _prefix_of(n) if case["prefix"] else 0
            total += n * n if not case["causal"] else \
                n * (n + 1) // 2 + max(0, p * (p - 1) // 2)
    return total


def _attention_inputs(case, seed, g):
    B, S, H, Hk, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    rng = random.Random(seed)
    ids = torch.full((B, S), -1, dtype=torch.int32)
    prefix = torch.zeros(B, case["documents"], dtype=torch.int32)
    for b, lens in enumerate(_lengths(case)):
        rng.shuffle(lens)
        at = 0
        for d, n in enumerate(lens):
            ids[b, at:at + n] = d
            prefix[b, d] = _prefix_of(n)
            at += n
    # queries, keys and values as the joint projection leaves them
    x = torch.randn(B, S, H + 2 * Hk, D, generator=g, device=DEVICE,
                    dtype=torch.bfloat16)
    if case["cap"]:      # scores that reach into the cap's bend
        x[:, :, :H] *= 4
    dout = torch.randn(B, S, H, D, generator=g, device=DEVICE, dtype=torch.bfloat16)
    return dict(q=x[:, :, :H], k=x[:, :, H:H + Hk], v=x[:, :, H + Hk:], dout=dout,
                ids=ids.to(DEVICE),
                prefix=prefix.to(DEVICE) if case["prefix"] else None,
                slopes=_slopes(H) if case["bias"] else None)


def _slopes(heads):
    h = torch.arange(1, heads + 1, device=DEVICE, dtype=torch.float32)
    return torch.exp2(-8.0 * h / heads)


def _contexts(case):
    """Lengths of the requests, by the sizes alone: from a quarter of the longest."""
    rng = random.Random("%(requests)d %(context)d" % case)
    top = case["context"]
    return [top] + [rng.randint(max(1, top // 4), top)
                    for _ in range(case["requests"] - 1)]


def _decode_inputs(case, seed, g):
    H, Hk, bs, D = case["heads"], case["kv_heads"], case["block"], 128
    lens = _contexts(case)
    random.Random(seed).shuffle(lens)
    need = [-(-n // bs) for n in lens]
    order = torch.randperm(sum(need), generator=g, device=DEVICE).cpu().int()
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    pools = [torch.randn(sum(need), Hk, bs, D, generator=g, device=DEVICE,
                         dtype=torch.bfloat16) for _ in range(2)]
    q = torch.randn(len(lens), H, D, generator=g, device=DEVICE, dtype=torch.bfloat16)
    if case["cap"]:
        q *= 4
    return dict(q=q, kpool=pools[0], vpool=pools[1], table=table.to(DEVICE),
                lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE),
                slopes=_slopes(H) if case["bias"] else None)


def _heads_inputs(case, seed, g):
    B, S, H, Hk, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    t = TYPES[case["type"]]
    x = torch.randn(B, S, H + 2 * Hk, D, generator=g, device=DEVICE, dtype=t)
    # a decoding step's tokens each have a position of their own, a packed batch's
    # begin again with every document
    places = torch.randint(0, 4096, (B, 1), generator=g, device=DEVICE)
    pos = (places + torch.arange(S, device=DEVICE)) % 4096
    freq = 10000.0 ** (-torch.arange(0, case["rotated"], 2, dtype=torch.float64,
                                     device=DEVICE) / case["rotated"])
    angle = torch.arange(4096, dtype=torch.float64, device=DEVICE)[:, None] * freq

    def weight():
        return (1 + 0.2 * torch.randn(D, generator=g, device=DEVICE)).to(t)

    s = dict(q=x[:, :, :H], k=x[:, :, H:H + Hk], qw=weight(), kw=weight(),
             cos=angle.cos().float(), sin=angle.sin().float(), pos=pos.int())
    if case["train"]:
        s["dq"] = torch.randn(B, S, H, D, generator=g, device=DEVICE, dtype=t)
        s["dk"] = torch.randn(B, S, Hk, D, generator=g, device=DEVICE, dtype=t)
    return s


def _logprobs_inputs(case, seed, g):
    N, V = case["rows"], case["vocab"]
    x = torch.empty(N, V, device=DEVICE, dtype=TYPES[case["type"]])
    x.normal_(0.0, 2.5, generator=g)
    tokens = torch.randint(0, V, (N,), generator=g, device=DEVICE)
    s = dict(logits=x, tokens=tokens)
    if case["train"]:
        # the prompts' tokens do not count
        tokens[torch.rand(N, generator=g, device=DEVICE) < 0.2] = IGNORE
        s["glp"] = torch.randn(N, generator=g, device=DEVICE)
        s["gent"] = 0.1 * torch.randn(N, generator=g, device=DEVICE)
    return s


_INPUTS = dict(attention=_attention_inputs, decode=_decode_inputs, heads=_heads_inputs,
               logprobs=_logprobs_inputs)


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    return dict(case=case, **_INPUTS[case["op"]](case, seed, g))


def work(case):
    if case["op"] == "attention":
        B, S, H, Hk, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
        # q, out and their gradients, k, v and theirs; two products and five
        return dict(bytes=2 * B * S * D * (4 * H + 4 * Hk) + 4 * B * S,
                    flops=2 * 7 * D * H * _pairs(case))
    if case["op"] == "decode":
        keys = sum(_contexts(case))
        H, Hk, n = case["heads"], case["kv_heads"], case["requests"]
        return dict(bytes=2 * 128 * (2 * keys * Hk + 2 * n * H) + 4 * n
                    + 4 * keys // case["block"], flops=4 * 128 * H * keys)
    if case["op"] == "heads":
        rows = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"])
        n = rows * case["dim"] * SIZE[case["type"]]
        # in and out; backward the gradients in, x again, the gradients out
        return dict(bytes=n * (4 if case["train"] else 2) +
                    case["batch"] * case["seq"] * 4, flops=0)
    N, V = case["rows"], case["vocab"]
    return dict(bytes=N * V * SIZE[case["type"]] * (2 if case["train"] else 1) + 16 * N,
                flops=0)


# ------------------------------------------------------------------- plain forms


def _visible(ids, prefix, causal):
    """[B, S, S]: which keys a query sees."""
    S = ids.shape[1]
    at = torch.arange(S, device=ids.device)
    seen = (ids[:, :, None] == ids[:, None, :]) & (ids >= 0)[:, :, None]
    if not causal:
        return seen
    early = at[None, :] <= at[:, None]
    if prefix is None:
        return seen & early
    begins = torch.ones_like(ids, dtype=torch.bool)
    begins[:, 1:] = ids[:, 1:] != ids[:, :-1]
    first = torch.where(begins, at, 0).cummax(1).values
    inside = at - first < prefix.gather(1, ids.clamp(min=0).long())
    return seen & (early | inside[:, None, :])


def _attention(s):
    case = s["case"]
    B, S, H, D = s["q"].shape
    Hk, cap = case["kv_heads"], case["cap"]
    G, scale = H // Hk, 1.0 / math.sqrt(D)

    def rows(x):          # [B, Hk, heads of a group, S, D]
        return x.float().reshape(B, S, Hk, -1, D).permute(0, 2, 3, 1, 4)

    q, do = rows(s["q"]), rows(s["dout"])
    k, v = rows(s["k"])[:, :, 0], rows(s["v"])[:, :, 0]
    q, do = q.reshape(B, Hk, G * S, D), do.reshape(B, Hk, G * S, D)
    t = (q @ k.transpose(2, 3)) * scale
    bend = None
    if cap:
        bend = torch.tanh(t / cap)
        t = bend * cap
        bend = 1 - bend * bend
    t = t.view(B, Hk, G, S, S)
    if s["slopes"] is not None:
        at = torch.arange(S, device=t.device, dtype=torch.float32)
        t = t - s["slopes"].view(Hk, G, 1, 1) * (at[:, None] - at[None, :]).abs()
    seen = _visible(s["ids"], s["prefix"], case["causal"])[:, None, None]
    t = t.masked_fill(~seen, -math.inf)
    top = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(top > -math.inf, top, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    p = p.view(B, Hk, G * S, S)
    del t, seen
    o = p @ v
    dv = p.transpose(2, 3) @ do
    dt = p * (do @ v.transpose(2, 3) - (do * o).sum(-1, keepdim=True))
    if bend is not None:
        dt = dt * bend
    dq = (dt @ k) * scale
    dk = (dt.transpose(2, 3) @ q) * scale

    def back(x, heads):
        x = x.view(B, Hk, heads, S, D).permute(0, 3, 1, 2, 4)
        return x.reshape(B, S, Hk * heads, D).to(torch.bfloat16)

    return dict(out=back(o, G), dq=back(dq, G), dk=back(dk, 1), dv=back(dv, 1))


def _decode(s):
    case = s["case"]
    n, H, D = s["q"].shape
    Hk = case["kv_heads"]
    table = s["table"].long()

    def rows(pool):       # [n, Hk, keys, D]
        return pool[table].float().permute(0, 2, 1, 3, 4).reshape(n, Hk, -1, D)

    k, v = rows(s["kpool"]), rows(s["vpool"])
    q = s["q"].float().view(n, Hk, H // Hk, D)
    t = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    if case["cap"]:
        t = torch.tanh(t / case["cap"]) * case["cap"]
    at = torch.arange(k.shape[2], device=t.device)
    back = s["lens"].long()[:, None] - 1 - at
    if s["slopes"] is not None:
        t = t - s["slopes"].view(1, Hk, H // Hk, 1) * back[:, None, None].abs()
    t = t.masked_fill((back < 0)[:, None, None], -math.inf)
    p = torch.exp(t - t.amax(-1, keepdim=True))
    o = (p / p.sum(-1, keepdim=True)) @ v
    return o.reshape(n, H, D).to(torch.bfloat16)


def _split(x, rotated, layout):
    """The two coordinates of each turned pair."""
    if layout == "half":
        return x[..., :rotated // 2], x[..., rotated // 2:rotated]
    return x[..., 0:rotated:2], x[..., 1:rotated:2]


def _joined(a, b, rest, layout):
    turned = torch.cat([a, b], -1) if layout == "half" else \
        torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _turned(x, c, s, rotated, layout):
    a, b = _split(x, rotated, layout)
    return _joined(a * c - b * s, b * c + a * s, x[..., rotated:], layout)


def _heads(s):
    case = s["case"]
    rotated, layout = case["rotated"], case["layout"]
    at = s["pos"].long()
    c, sn = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    out = {}
    for name, x, w in (("q", s["q"], s["qw"]), ("k", s["k"], s["kw"])):
        xf, wf = x.float(), w.float()
        r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
        unit = xf * r
        out[name] = _turned(unit * wf, c, sn, rotated, layout).to(x.dtype)
        if not case["train"]:
            continue
        dn = _turned(s["d" + name].float(), c, -sn, rotated, layout)
        out["d" + name + "_weight"] = (dn * unit).sum((0, 1, 2)).to(x.dtype)
        dn = dn * wf
        dx = r * (dn - unit * (dn * unit).mean(-1, keepdim=True))
        out["d" + name] = dx.to(x.dtype)
    return out


def _logprobs(s):
    case = s["case"]
    x, tokens = s["logits"].float(), s["tokens"]
    live = tokens != IGNORE
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = e / total
    entropy = torch.where(live, -(p * (x - lse)).sum(-1), 0.0)
    own_ids = torch.where(live, tokens, 0)[:, None]
    lp = torch.where(live, (x.gather(1, own_ids) - lse)[:, 0], 0.0)
    out = dict(logprobs=lp, entropy=entropy)
    if case["top"]:
        best, order = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_logprobs"] = (best - lse)[:, :case["top"]].contiguous()
        out["top_ids"] = order[:, :case["top"]].contiguous()
    if case["train"]:
        glp = torch.where(live, s["glp"], 0.0)[:, None]
        gent = torch.where(live, s["gent"], 0.0)[:, None]
        d = -p * (glp + gent * (x - lse + entropy[:, None]))
        d.scatter_add_(1, own_ids, glp)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


_PLAIN = dict(attention=_attention, decode=_decode, heads=_heads, logprobs=_logprobs)


# ------------------------------------------------------------ the framework's own


def _own_attention(s):
    from deepspeed_amd.ops.masked_attention import masked_attention, packed_rows
    case = s["case"]
    q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
    rows = packed_rows(s["ids"], s["prefix"], causal=case["causal"])
    out = masked_attention(q, k, v, rows, softcap=case["cap"],
                           alibi_slopes=s["slopes"])
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"])
    return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)


def _own_decode(s):
    from deepspeed_amd.ops.paged_attention import paged_decode_attention
    return paged_decode_attention(s["q"], s["kpool"], s["vpool"], s["table"],
                                  s["lens"], softcap=s["case"]["cap"],
                                  alibi_slopes=s["slopes"])


def _own_heads(s):
    from deepspeed_amd.ops.qk_norm import qk_norm_rope
    case = s["case"]
    ins = [s[n] for n in ("q", "k", "qw", "kw")]
    if case["train"]:
        ins = [x.detach().requires_grad_() for x in ins]
    q, k = qk_norm_rope(*ins, s["cos"], s["sin"], s["pos"], eps=EPS,
                        layout=case["layout"])
    out = dict(q=q.detach(), k=k.detach())
    if case["train"]:
        grads = torch.autograd.grad((q, k), ins, (s["dq"], s["dk"]))
        out.update(zip(("dq", "dk", "dq_weight", "dk_weight"), grads))
    return out


def _own_logprobs(s):
    from deepspeed_amd.ops.token_logprobs import token_logprobs
    case = s["case"]
    x = s["logits"].detach().requires_grad_() if case["train"] else s["logits"]
    got = token_logprobs(x, s["tokens"], top=case["top"], ignore_index=IGNORE)
    out = dict(logprobs=got.logprobs.detach(), entropy=got.entropy.detach())
    if case["top"]:
        out.update(top_logprobs=got.top_logprobs, top_ids=got.top_ids)
    if case["train"]:
        out["dlogits"], = torch.autograd.grad((got.logprobs, got.entropy), (x,),
                                              (s["glp"], s["gent"]))
    return out


_OWN = dict(attention=_own_attention, decode=_own_decode, heads=_own_heads,
            logprobs=_own_logprobs)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------- in 64 bits


def _exact_attention(s, case):
    B, S, H, D = s["q"].shape
    G = H // case["kv_heads"]
    out = {n: torch.zeros(s[m].shape, dtype=torch.float64, device=DEVICE)
           for n, m in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    at = torch.arange(S, device=DEVICE)
    for b in range(B):
        # a document at a time: nothing is seen outside one's own
        ids = s["ids"][b].tolist()
        ends = [i + 1 for i in range(S) if i + 1 == S or ids[i + 1] != ids[i]]
        for lo, hi in zip([0] + ends[:-1], ends):
            if ids[lo] < 0:
                continue
            n = hi - lo
            i, j = at[:n, None], at[None, :n]
            hidden = torch.zeros(n, n, dtype=torch.bool, device=DEVICE)
            if case["causal"]:
                p = int(s["prefix"][b, ids[lo]]) if case["prefix"] else 0
                hidden = (j > i) & (j >= p)
            for h in range(H):
                q, do = (s[m][b, lo:hi, h].double() for m in ("q", "dout"))
                k, v = (s[m][b, lo:hi, h // G].double() for m in ("k", "v"))
                z = torch.mm(q, k.t()) / math.sqrt(D)
                slope = torch.ones_like(z)
                if case["cap"]:
                    z = z / case["cap"]
                    slope = torch.cosh(z) ** -2
                    z = torch.tanh(z) * case["cap"]
                if case["bias"]:
                    z = z - float(s["slopes"][h]) * (i - j).abs().double()
                w = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
                o = torch.mm(w, v)
                dw = torch.mm(do, v.t())
                dz = w * (dw - (dw * w).sum(-1, keepdim=True)) * slope / math.sqrt(D)
                out["out"][b, lo:hi, h] = o
                out["dq"][b, lo:hi, h] = torch.mm(dz, k)
                out["dk"][b, lo:hi, h // G] += torch.mm(dz.t(), q)
                out["dv"][b, lo:hi, h // G] += torch.mm(w.t(), do)
    return out


def _exact_decode(s, case):
    n, H, D = s["q"].shape
    G, bs = H // case["kv_heads"], case["block"]
    out = torch.empty(n, H, D, dtype=torch.float64, device=DEVICE)
    for r, length in enumerate(s["lens"].tolist()):
        blocks = s["table"][r, :-(-length // bs)].long()
        k, v = (s[m][blocks].double().transpose(1, 2).reshape(-1, case["kv_heads"], D)
                [:length] for m in ("kpool", "vpool"))
        far = torch.arange(length - 1, -1, -1, device=DEVICE, dtype=torch.float64)
        for h in range(H):
            z = torch.mv(k[:, h // G], s["q"][r, h].double()) / math.sqrt(D)
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if case["bias"]:
                z = z - float(s["slopes"][h]) * far
            out[r, h] = torch.mv(v[:, h // G].t(), torch.softmax(z, 0))
    return out


def _exact_heads(s, case):
    """The rotation as a complex product, the gradients by automatic differentiation."""
    rotated, half = case["rotated"], case["layout"] == "half"
    at = s["pos"].long()
    phase = torch.complex(s["cos"].double(), s["sin"].double())[at][:, :, None]
    out = {}
    for name in "qk":
        x = s[name].double().detach().requires_grad_()
        w = s[name + "w"].double().detach().requires_grad_()
        norm = x / (x.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w
        z = norm[..., :rotated]
        z = z.unflatten(-1, (2, -1)).transpose(-1, -2) if half else \
            z.unflatten(-1, (-1, 2))
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * phase)
        z = (z.transpose(-1, -2) if half else z).flatten(-2)
        y = torch.cat([z, norm[..., rotated:]], -1)
        out[name] = y.detach()
        if case["train"]:
            out["d" + name], out["d" + name + "_weight"] = torch.autograd.grad(
                y, (x, w), s["d" + name].double())
    return out


def _exact_logprobs(s, case):
    N, V = s["logits"].shape
    kept = {}
    for lo in range(0, N, 512):
        x = s["logits"][lo:lo + 512].double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        token = s["tokens"][lo:lo + 512]
        live = token != IGNORE
        at = token.clamp(min=0)[:, None]
        ent = -(p * lp).sum(-1)
        part = dict(logprobs=lp.gather(1, at)[:, 0] * live, entropy=ent * live)
        if case["top"]:
            order = torch.argsort(x, dim=-1, descending=True, stable=True)
            part["top_ids"] = order[:, :case["top"]]
            part["top_logprobs"] = lp.gather(1, part["top_ids"])
        if case["train"]:
            a, e = (s[n][lo:lo + 512].double() * live for n in ("glp", "gent"))
            hot = torch.zeros_like(p).scatter_(1, at, 1.0)
            part["dlogits"] = a[:, None] * (hot - p) \
                - e[:, None] * p * (lp + ent[:, None])
        for n, y in part.items():
            kept.setdefault(n, []).append(y)
    return {n: torch.cat(y) for n, y in kept.items()}


_EXACT = dict(attention=_exact_attention, decode=_exact_decode, heads=_exact_heads,
              logprobs=_exact_logprobs)


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed), case)
