"""Cases for timing and checking the block-sparse attention and relative bias operators.

Each case is a call (or the short run of calls) that a program makes of `ias.attention`; with `own`
false the same result comes from elementary torch operations.

q is (batch, q_len, q_heads, dim), k and v are (batch, k_len, k_heads, dim).  The queries of a sequence
are its last tokens: query i stands at position i + k_length - q_length.  A pattern is int32 (batch,
k_heads, q_len, keep): the blocks of keys that a query reads, -1 where there are fewer.
"""
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SEGMENT = 32  # tokens that speak of one thing, in the inputs


def _attention():
    folder = os.path.join(os.getcwd(), "ia-spgemm_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from ias import attention
    return attention


# ---------------------------------------------------------------- cases
def _case(name, op, **kw):
    c = dict(name=name, op=op, dtype="bf16", b=1, sq=1, sk=1, hq=1, hkv=1, d=64, keep=1, block=64, causal=True,
             buckets=0, ragged=False)
    c.update(kw)
    return c


def listed():
    return [
        # the pattern of a prompt, before its attention
        _case("select_prompt_4k", "select", sq=4096, sk=4096, hq=32, hkv=8, d=128, keep=16),
        # a padded batch of prompts in fp16, odd lengths, one group of heads for each key head
        _case("select_ragged_fp16", "select", dtype="fp16", b=3, sq=1501, sk=1501, hq=8, hkv=2, d=64, keep=6, ragged=True),
        # one user's next token: latency
        _case("step_one", "step", sk=4097, hq=32, hkv=8, d=128, keep=16),
        # a full server's next tokens over long caches
        _case("step_many", "step", b=16, sk=32768, hq=32, hkv=8, d=128, keep=32, ragged=True),
        # single tokens with a relative bias, fp16, one key head
        _case("step_bias_fp16", "step", dtype="fp16", b=5, sk=9001, hq=16, hkv=1, d=64, keep=12, buckets=32),
        # a prompt's attention
        _case("attend_prompt_8k", "attend", sq=8192, sk=8192, hq=32, hkv=8, d=128, keep=16),
        # both directions, as many key heads as query heads, odd lengths
        _case("attend_both_ways", "attend", dtype="fp16", b=2, sq=1999, sk=2111, hq=8, hkv=8, d=64, keep=8, causal=False,
              buckets=32),
        # a training step's attention with a learned bias over a padded batch
        _case("train_bias_2k", "train", b=2, sq=2048, sk=2048, hq=16, hkv=4, d=64, keep=8, buckets=32, ragged=True),
        # a training step's attention on a long sequence
        _case("train_8k", "train", sq=8192, sk=8192, hq=16, hkv=2, d=128, keep=16),
        # the dense bias of an encoder layer, and of a short odd one
        _case("bias_2k", "bias", sq=2048, sk=2048, hq=16, buckets=32, causal=False),
        # the gradient of the bias from the gradient of dense scores
        _case("bias_grad_2k", "bias_grad", b=2, sq=2048, sk=2048, hq=16, buckets=32, causal=False),
        _case("bias_grad_odd_fp32", "bias_grad", dtype="fp32", b=3, sq=317, sk=1033, hq=5, buckets=48, causal=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "step", "attend", "train", "bias", "bias_grad"])
    dtype = rng.choice(["bf16", "fp16"])
    if op in ("bias", "bias_grad"):
        kw = dict(dtype=rng.choice(["bf16", "fp16", "fp32"]), b=rng.randint(1, 2) if op == "bias_grad" else 1,
                  sq=_spread(rng, 1, 2048), sk=_spread(rng, 1, 2048), hq=rng.randint(1, 16),
                  buckets=rng.randint(2, 64), causal=rng.random() < 0.5)
        return {k: v for k, v in _case("", op, **kw).items() if k != "name"}
    hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8, 16]) if hkv <= 2 else rng.choice([1, 2, 4])
    kw = dict(dtype=dtype, hq=hkv * group, hkv=hkv, d=rng.choice([64, 128, 80, 64, 128]), block=rng.choice([64, 64, 128]),
              ragged=rng.random() < 0.4, buckets=rng.choice([0, 0, 16, 32, 50]))
    if op == "step":
        kw.update(b=_spread(rng, 1, 16), sk=_spread(rng, 64, 32768), keep=rng.randint(2, 32))
    else:
        top = 4096 if hkv * group <= 16 else 2048
        n = _spread(rng, 64, top)
        kw.update(b=rng.randint(1, 2), sq=n, sk=n, keep=rng.randint(2, 24), causal=rng.random() < 0.8)
        if op == "attend" and rng.random() < 0.3:
            kw.update(sq=_spread(rng, 2, n))  # the rest of a prompt after a kept prefix
    if op == "select":
        kw.update(buckets=0)
    return {k: v for k, v in _case("", op, **kw).items() if k != "name"}


# ---------------------------------------------------------------- inputs
def _edges(buckets, causal):
    """Edges of log-spaced buckets: `buckets` - 1 ascending distances; both sides of 0 unless causal."""
    side = (buckets - 1) if causal else (buckets - 1) // 2
    exact = max(1, side // 2)
    far = [exact + int(round((max(256, 2 * side) - exact) * (i + 1) ** 2 / (side - exact) ** 2)) for i in range(side - exact)]
    for i in range(len(far)):
        far[i] = max(far[i], (far[i - 1] if i else exact) + 1)
    back = sorted(-x + 1 for x in (list(range(1, exact + 1)) + far))
    if causal:
        return back[: buckets - 1]
    fore = [x for x in list(range(1, exact + 1)) + far]
    e = sorted(set(back + fore))
    while len(e) < buckets - 1:
        e.append(e[-1] + 7)
    return e[: buckets - 1]


def _speech(gen, c, n, heads):
    """(batch, n, heads, dim) of noise, and the directions that its segments of tokens will share."""
    segments = -(-n // SEGMENT)
    topic = torch.randn(c["b"], segments, heads, c["d"], generator=gen, device="cuda", dtype=torch.float32) * 0.5
    x = torch.randn(c["b"], n, heads, c["d"], generator=gen, device="cuda", dtype=torch.float32)
    return topic, x


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DT[c["dtype"]]
    s = {"case": c}
    if c["buckets"]:
        s["edges"] = torch.tensor(_edges(c["buckets"], c["causal"]), dtype=torch.int32, device="cuda")
        s["table"] = torch.randn(c["buckets"], c["hq"], generator=gen, device="cuda").to(dt)
    if c["op"] == "bias":
        return s
    if c["op"] == "bias_grad":
        s["grad"] = torch.randn(c["b"], c["hq"], c["sq"], c["sk"], generator=gen, device="cuda").to(dt)
        return s
    topic, x = _speech(gen, c, c["sk"], c["hkv"])
    s["k"] = (x * 0.87 + topic.repeat_interleave(SEGMENT, 1)[:, : c["sk"]]).to(dt)
    s["v"] = torch.randn(c["b"], c["sk"], c["hkv"], c["d"], generator=gen, device="cuda").to(dt)
    # a segment of queries asks for what a random segment of keys holds
    segments = -(-c["sq"] // SEGMENT)
    pick = torch.randint(0, topic.shape[1], (segments,), generator=gen, device="cuda")
    ask = topic[:, pick].repeat_interleave(SEGMENT, 1)[:, : c["sq"]].repeat_interleave(c["hq"] // c["hkv"], 2)
    s["q"] = (torch.randn(c["b"], c["sq"], c["hq"], c["d"], generator=gen, device="cuda") * 0.87 + ask).to(dt)
    del topic, x, ask
    s["q_lens"] = s["k_lens"] = None
    if c["ragged"]:
        cut = torch.randint(0, max(1, c["sk"] // 2), (c["b"],), generator=gen, device="cuda")
        cut[0] = 0
        s["k_lens"] = (c["sk"] - cut).to(torch.int32)
        if c["sq"] == c["sk"]:
            s["q_lens"] = s["k_lens"].clone()
        else:
            s["q_lens"] = torch.full((c["b"],), c["sq"], dtype=torch.int32, device="cuda")
    if c["op"] == "step":
        # the summaries are kept with the cache; the newest token's block is still to be brought up to date
        s["summary"] = _summary(s["k"], c["block"], s["k_lens"])
        last = (_lens(s["k_lens"], c["b"], c["sk"]) - 1).clamp(min=0)
        s["summary"][torch.arange(c["b"], device="cuda"), :, last // c["block"]] = 0
    if c["op"] in ("attend", "train"):
        s["blocks"] = _select(s["q"], _summary(s["k"], c["block"], s["k_lens"], torch.float32), c, s["q_lens"], s["k_lens"],
                              torch.float32)
    if c["op"] == "train":
        s["dout"] = torch.randn(c["b"], c["sq"], c["hq"], c["d"], generator=gen, device="cuda").to(dt)
        if c["ragged"]:
            s["dout"] *= (torch.arange(c["sq"], device="cuda") < s["q_lens"][:, None])[:, :, None, None]
    return s


# ---------------------------------------------------------------- plain forms
def _lens(lens, b, n):
    return lens.long() if lens is not None else torch.full((b,), n, dtype=torch.int64, device="cuda")


def _positions(c, q_lens, k_lens):
    """(batch, q_len) position of each query, and whether the query is there."""
    ql, kl = _lens(q_lens, c["b"], c["sq"]), _lens(k_lens, c["b"], c["sk"])
    i = torch.arange(c["sq"], device="cuda")
    return i + (kl - ql)[:, None], i < ql[:, None]


def _summary(k, block, k_lens, t=torch.float64):
    """Means of the blocks of keys, (batch, heads, blocks, dim)."""
    b, n, h, d = k.shape
    m = -(-n // block)
    kl = _lens(k_lens, b, n)
    there = torch.arange(n, device=k.device) < kl[:, None]
    x = torch.where(there[:, :, None, None], k, 0).to(t)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, m * block - n)).view(b, m, block, h, d).sum(2)
    count = (kl[:, None] - torch.arange(m, device=k.device) * block).clamp(0, block)
    return (x / count.clamp(min=1)[:, :, None, None]).to(k.dtype).transpose(1, 2).contiguous()


def _summary_last(k, summary, block, k_lens):
    """The means of the blocks that hold the newest token, put in their places."""
    b, n, h, d = k.shape
    kl = _lens(k_lens, b, n)
    c = (kl - 1).clamp(min=0) // block
    j = c[:, None] * block + torch.arange(block, device=k.device)
    there = j < kl[:, None]
    rows = torch.arange(b, device=k.device)
    x = torch.where(there[:, :, None, None], k[rows[:, None], j.clamp(max=n - 1)], 0).double().sum(1)
    summary[rows, :, c] = (x / there.sum(1).clamp(min=1)[:, None, None]).to(k.dtype)
    return summary


def _select(q, summary, c, q_lens, k_lens, t=torch.float64):
    """The pattern: first block, own block (causal), then the highest scores; ascending, -1 behind."""
    b, n, hq, d = q.shape
    hkv, m = summary.shape[1:3]
    keep = c["keep"]
    p, there = _positions(c, q_lens, k_lens)
    qg = q.view(b, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d).to(t)
    s = (qg @ summary.to(t).transpose(2, 3).contiguous()).view(b, hkv, n, hq // hkv, m)
    s = torch.where(s.isnan(), -math.inf, s).amax(3) + 0.0
    if c["causal"]:
        seen = torch.where(p >= 0, p // c["block"] + 1, 0)
    else:
        seen = (-(-_lens(k_lens, b, c["sk"]) // c["block"]))[:, None].expand(b, n)
    seen = torch.where(there, seen, 0)[:, None, :, None]
    col = torch.arange(m, device=q.device)
    must = (col < 1) | ((col == seen - 1) if c["causal"] else False)
    # by (whether it has to be there, the score), stable: the lower block first among equals
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices
    rank = torch.where(must, 0, torch.where(col < seen, 1, 2)).expand(s.shape).gather(-1, order)
    order = order.gather(-1, torch.sort(rank, dim=-1, stable=True).indices)
    w = min(keep, m)
    best = order[..., :w]
    best = torch.where(torch.arange(w, device=q.device) < seen.clamp(max=w), best, m)
    best = torch.sort(best, dim=-1).values
    best = torch.where(best == m, -1, best)
    return torch.nn.functional.pad(best, (0, keep - w), value=-1).to(torch.int32).contiguous()


def _bucket(d, edges):
    return torch.searchsorted(edges.long(), d.contiguous(), right=True)


def _allowed(blocks, c, q_lens, k_lens):
    """(batch, k_heads, q_len, k_len): the pairs that take part."""
    b, hkv, n, keep = blocks.shape
    m = -(-c["sk"] // c["block"])
    p, there = _positions(c, q_lens, k_lens)
    at = torch.where((blocks >= 0) & (blocks < m), blocks, m).long()
    on = torch.zeros(b, hkv, n, m + 1, dtype=torch.bool, device=blocks.device).scatter_(3, at, True)[..., :m]
    on = on.repeat_interleave(c["block"], 3)[..., : c["sk"]]
    j = torch.arange(c["sk"], device=blocks.device)
    ok = there[:, :, None] & (j < _lens(k_lens, b, c["sk"])[:, None, None])
    if c["causal"]:
        ok = ok & (j <= p[:, :, None])
    return on & ok[:, None]


def _bias(table, edges, c, p):
    """(batch, q_heads, q_len, k_len) of the bias in 32 bits."""
    d = torch.arange(c["sk"], device="cuda") - p[:, :, None]
    return table.float()[_bucket(d, edges)].permute(0, 3, 1, 2)


def _heads(x, hq):
    """(batch, n, heads, dim) as (batch, q_heads, n, dim) in 32 bits."""
    return x.transpose(1, 2).float().repeat_interleave(hq // x.shape[2], 1)


def _dense(s, c):
    """Probabilities and log-sums over the pattern: dense scores, masked."""
    hq, g = c["hq"], c["hq"] // c["hkv"]
    x = (_heads(s["q"], hq) * c["d"] ** -0.5) @ _heads(s["k"], hq).transpose(2, 3).contiguous()
    if c["buckets"]:
        x += _bias(s["table"], s["edges"], c, _positions(c, s["q_lens"], s["k_lens"])[0])
    ok = _allowed(s["blocks"], c, s["q_lens"], s["k_lens"]).repeat_interleave(g, 1)
    x = x.masked_fill_(~ok, -math.inf)
    top = x.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    x = x.sub_(top).exp_()
    total = x.sum(3, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf)
    return x.div_(torch.where(total > 0, total, 1)), lse.squeeze(3)


def _gathered(s, c, blocks):
    """The form for few queries: the keys of the pattern, gathered."""
    b, hkv, n, keep = blocks.shape
    g, d = c["hq"] // hkv, c["d"]
    p, there = _positions(c, s["q_lens"], s["k_lens"])
    j = (blocks.long()[..., None] * c["block"] + torch.arange(c["block"], device="cuda")).flatten(3)
    ok = (blocks >= 0).repeat_interleave(c["block"], 3) & there[:, None, :, None]
    ok &= j < _lens(s["k_lens"], b, c["sk"])[:, None, None, None]
    if c["causal"]:
        ok &= j <= p[:, None, :, None]
    at = (torch.arange(b, device="cuda")[:, None, None, None], j.clamp(0, c["sk"] - 1),
          torch.arange(hkv, device="cuda")[None, :, None, None])
    kk, vv = s["k"][at].float(), s["v"][at].float()
    q = s["q"].view(b, n, hkv, g, d).transpose(1, 2).float() * d ** -0.5
    x = q @ kk.transpose(3, 4).contiguous()
    if c["buckets"]:
        bias = s["table"].float()[_bucket(j - p[:, None, :, None], s["edges"])]
        x = x + bias.view(*j.shape, hkv, g).diagonal(0, 1, 4).permute(0, 4, 1, 3, 2)
    x = x.masked_fill(~ok[:, :, :, None], -math.inf)
    top = x.amax(4, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    x = (x - top).exp()
    total = x.sum(4, keepdim=True)
    out = (x / torch.where(total > 0, total, 1)) @ vv
    return out.transpose(1, 2).reshape(b, n, c["hq"], d).to(s["q"].dtype)


def _plain(s):
    c = s["case"]
    dt, g = DT[c["dtype"]], c["hq"] // c["hkv"]
    if c["op"] == "select":
        m = _summary(s["k"], c["block"], s["k_lens"])
        return {"summary": m, "blocks": _select(s["q"], m, c, s["q_lens"], s["k_lens"])}
    if c["op"] == "step":
        m = _summary_last(s["k"], s["summary"], c["block"], s["k_lens"])
        blocks = _select(s["q"], m, c, s["q_lens"], s["k_lens"])
        return {"summary": m, "blocks": blocks, "out": _gathered(s, c, blocks)}
    if c["op"] == "attend":
        p, lse = _dense(s, c)
        return {"out": (p @ _heads(s["v"], c["hq"])).transpose(1, 2).to(dt).contiguous(), "lse": lse}
    if c["op"] == "train":
        p, lse = _dense(s, c)
        q, k, v, do = (_heads(s[n], c["hq"]) for n in ("q", "k", "v", "dout"))
        o = p @ v
        dv = p.transpose(2, 3).contiguous() @ do
        ds = do @ v.transpose(2, 3).contiguous()
        ds = ds.sub_((do * o).sum(3, keepdim=True)).mul_(p)
        got = {"out": o.transpose(1, 2).to(dt).contiguous()}
        got["dq"] = (ds @ k * c["d"] ** -0.5).transpose(1, 2).to(dt).contiguous()
        dk = ds.transpose(2, 3).contiguous() @ q * c["d"] ** -0.5
        for name, x in (("dk", dk), ("dv", dv)):
            got[name] = x.view(c["b"], c["hkv"], g, c["sk"], c["d"]).sum(2).transpose(1, 2).to(dt).contiguous()
        if c["buckets"]:
            where = _bucket(torch.arange(c["sk"], device="cuda") - _positions(c, s["q_lens"], s["k_lens"])[0][:, :, None], s["edges"])
            sums = torch.zeros(c["hq"], c["buckets"], device="cuda")
            sums.scatter_add_(1, where.reshape(1, -1).expand(c["hq"], -1), ds.transpose(0, 1).reshape(c["hq"], -1))
            got["dtable"] = sums.t().to(dt).contiguous()
        return got
    d = torch.arange(c["sk"], device="cuda") - (torch.arange(c["sq"], device="cuda") + c["sk"] - c["sq"])[:, None]
    where = _bucket(d, s["edges"])
    if c["op"] == "bias":
        return s["table"].t()[:, where].contiguous()
    sums = torch.zeros(c["hq"], c["buckets"], device="cuda")
    return sums.scatter_add_(1, where.reshape(1, -1).expand(c["hq"], -1), s["grad"].float().sum(0).view(c["hq"], -1)).t().to(dt).contiguous()


def run(state):
    if not own:
        return _plain(state)
    A, s, c = _attention(), state, state["case"]
    if c["op"] == "bias":
        return A.rel_bias(s["table"], s["edges"], c["sq"], c["sk"])
    if c["op"] == "bias_grad":
        return A.rel_bias_grad(s["grad"], s["edges"])
    lens = dict(q_lens=s["q_lens"], k_lens=s["k_lens"])
    pick = dict(k_len=c["sk"], block=c["block"], causal=c["causal"], first=1, local=1 if c["causal"] else 0, **lens)
    kw = dict(block=c["block"], causal=c["causal"], table=s.get("table"), edges=s.get("edges"), **lens)
    if c["op"] == "select":
        m = A.block_summary(s["k"], block=c["block"], k_lens=s["k_lens"])
        return {"summary": m, "blocks": A.block_select(s["q"], m, c["keep"], **pick)}
    if c["op"] == "step":
        m = A.block_summary(s["k"], block=c["block"], k_lens=s["k_lens"], fresh=1, out=s["summary"])
        blocks = A.block_select(s["q"], m, c["keep"], **pick)
        return {"summary": m, "blocks": blocks, "out": A.block_attention(s["q"], s["k"], s["v"], blocks, **kw)[0]}
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw)
    if c["op"] == "attend":
        return {"out": out, "lse": lse}
    dq, dk, dv, dtable = A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], **kw)
    got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if dtable is not None:
        got["dtable"] = dtable
    return got


# ---------------------------------------------------------------- work
def _pairs(c):
    """About how many (query, key) pairs of one head take part."""
    n, most = c["sq"], c["keep"] * c["block"]
    first = c["sk"] - c["sq"] + 1 if c["causal"] else c["sk"]
    if not c["causal"]:
        return n * min(most, c["sk"])
    ramp = max(0, min(n, most - first))
    return ramp * first + ramp * (ramp - 1) // 2 + (n - ramp) * min(most, c["sk"])


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    cells = c["hq"] * c["sq"] * c["sk"]
    if c["op"] == "bias":
        return {"bytes": cells * e, "flops": 0}
    if c["op"] == "bias_grad":
        return {"bytes": c["b"] * cells * e, "flops": c["b"] * cells}
    m = -(-c["sk"] // c["block"])
    q = c["b"] * c["sq"] * c["hq"] * c["d"] * e
    k = c["b"] * c["sk"] * c["hkv"] * c["d"] * e
    read = min(k, c["b"] * c["hkv"] * c["sq"] * c["keep"] * c["block"] * c["d"] * e)
    pattern = c["b"] * c["hkv"] * c["sq"] * c["keep"] * 4
    seen = 0.5 if c["causal"] and c["sq"] > 1 else 1.0
    score = 2.0 * c["b"] * c["hq"] * c["sq"] * m * c["d"] * seen
    pairs = float(c["b"] * c["hq"] * _pairs(c))
    if c["op"] == "select":
        return {"bytes": q + k + k // c["block"] + pattern, "flops": score}
    if c["op"] == "step":
        return {"bytes": 2 * q + 2 * read + k // c["block"] + pattern, "flops": score + 4 * c["d"] * pairs}
    if c["op"] == "attend":
        return {"bytes": 2 * q + 2 * read + pattern, "flops": 4 * c["d"] * pairs}
    return {"bytes": 4 * q + 4 * read + pattern, "flops": 14 * c["d"] * pairs}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, one batch element and key head at a time; gradients by differentiation."""
    c, s = case, prepare(case, seed)
    f8 = torch.float64
    if c["op"] in ("bias", "bias_grad"):
        dist = torch.arange(c["sk"], device="cuda")[None] - torch.arange(c["sq"], device="cuda")[:, None] - (c["sk"] - c["sq"])
        where = (s["edges"].long()[:, None, None] <= dist).sum(0)
        if c["op"] == "bias":
            return torch.stack([s["table"][:, h].to(f8)[where] for h in range(c["hq"])])
        g = s["grad"].to(f8).sum(0)
        return torch.stack([torch.where(where == n, g, 0.0).sum((1, 2)) for n in range(c["buckets"])])
    kl = s["k_lens"].tolist() if s["k_lens"] is not None else [c["sk"]] * c["b"]
    ql = s["q_lens"].tolist() if s["q_lens"] is not None else [c["sq"]] * c["b"]
    g, m, size = c["hq"] // c["hkv"], -(-c["sk"] // c["block"]), c["block"]
    got = {}
    if c["op"] == "select" or c["op"] == "step":
        means = torch.zeros(c["b"], c["hkv"], m, c["d"], dtype=f8, device="cuda")
        for b in range(c["b"]):
            for n in range(-(-kl[b] // size)):
                means[b, :, n] = s["k"][b, n * size: min(kl[b], (n + 1) * size)].to(f8).mean(0)
        if c["op"] == "select":
            return {"summary": means, "blocks": None}
        held = means.to(s["k"].dtype)
        blocks = torch.full((c["b"], c["hkv"], 1, c["keep"]), -1, dtype=torch.int64, device="cuda")
        for b in range(c["b"]):
            top = -(-kl[b] // size)
            for h in range(c["hkv"]):
                score = (held[b, h, :top].to(f8) @ s["q"][b, 0, h * g: (h + 1) * g].to(f8).t()).amax(1).tolist()
                want = [0, top - 1] if c["causal"] else [0]
                for n in sorted(range(top), key=lambda n: (-score[n], n)):
                    if n not in want and len(want) < c["keep"]:
                        want.append(n)
                want = sorted(set(want))[: c["keep"]]
                blocks[b, h, 0, : len(want)] = torch.tensor(want, device="cuda")
        got.update({"summary": means, "blocks": None})
    else:
        blocks = s["blocks"].long()
    names = [n for n in ("q", "k", "v", "table") if n in s]
    leaf = {n: s[n].to(f8).requires_grad_(c["op"] == "train") for n in names}
    out = torch.zeros(c["b"], c["sq"], c["hq"], c["d"], dtype=f8, device="cuda")
    lse = torch.full((c["b"], c["hq"], c["sq"]), -math.inf, dtype=f8, device="cuda")
    for b in range(c["b"]):
        for h in range(c["hkv"]):
            n, t = ql[b], kl[b]
            pos = torch.arange(n, device="cuda") + t - n
            if c["op"] == "step":  # the keys of the pattern alone
                keys = torch.cat([torch.arange(x * size, min(t, (x + 1) * size), device="cuda") for x in blocks[b, h, 0].tolist() if x >= 0])
                ok = torch.ones(1, len(keys), dtype=torch.bool, device="cuda")
            else:
                keys = torch.arange(t, device="cuda")
                ok = (blocks[b, h, :n, :, None] == torch.arange(m, device="cuda")).any(1)[:, keys // size]
            if c["causal"]:
                ok = ok & (keys <= pos[:, None])
            q = leaf["q"][b, :n, h * g: (h + 1) * g].transpose(0, 1)
            x = q @ leaf["k"][b, keys, h].t() / math.sqrt(c["d"])
            if c["buckets"]:
                where = torch.bucketize(keys - pos[:, None], s["edges"].long(), right=True)
                x = x + torch.stack([leaf["table"][:, h * g + i][where] for i in range(g)])
            x = torch.where(ok, x, -math.inf)
            some = ok.any(1)
            x = torch.where(some[:, None], x, 0.0)
            o = torch.where(some[:, None], torch.softmax(x, -1) @ leaf["v"][b, keys, h], 0.0)
            if c["op"] == "train":
                (o * s["dout"][b, :n, h * g: (h + 1) * g].to(f8).transpose(0, 1)).sum().backward()
            out[b, :n, h * g: (h + 1) * g] = o.detach().transpose(0, 1)
            lse[b, h * g: (h + 1) * g, :n] = torch.where(some, torch.logsumexp(x.detach(), -1), -math.inf)
    got["out"] = out
    if c["op"] == "attend":
        got["lse"] = lse
    if c["op"] == "train":
        got.update({"dq": leaf["q"].grad, "dk": leaf["k"].grad, "dv": leaf["v"].grad})
        if c["buckets"]:
            got["dtable"] = leaf["table"].grad
    return got
