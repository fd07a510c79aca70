"""Block-sparse attention and the relative position bias (ias.attention):
results against 64 bits at the sizes and masks where they can go wrong."""
import math

import pytest
import torch

import attention_ref as ref

gpu = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def A():
    from ias import attention
    return attention


def make(c, seed=0, layout="bshd"):
    """Inputs of a case on the GPU; what lies behind a sequence's end is NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    B, n, nk, hq, hkv, d = c["b"], c["sq"], c["sk"], c["hq"], c["hkv"], c["d"]
    dt = DT[c["dtype"]]
    if layout == "packed":     # q, k, v side by side in one tensor
        w = rnd(B, max(n, nk), hq + 2 * hkv, d).to(dt)
        q, k, v = w[:, :n, :hq], w[:, :nk, hq:hq + hkv], w[:, :nk, hq + hkv:]
    elif layout == "bhsd":     # heads before tokens
        q, k, v = (rnd(B, h, m, d).to(dt).transpose(1, 2) for h, m in ((hq, n), (hkv, nk), (hkv, nk)))
    else:
        q, k, v = (rnd(B, m, h, d).to(dt) for h, m in ((hq, n), (hkv, nk), (hkv, nk)))
    s = dict(q=q, k=k, v=v, dout=rnd(B, n, hq, d).to(dt), q_lens=None, k_lens=None, table=None, edges=None)
    if c.get("q_lens"):
        s["q_lens"] = torch.tensor(c["q_lens"], dtype=torch.int32, device="cuda")
        s["k_lens"] = torch.tensor(c["k_lens"], dtype=torch.int32, device="cuda")
        for b in range(B):
            for x, m in ((q, c["q_lens"][b]), (s["dout"], c["q_lens"][b]), (k, c["k_lens"][b]), (v, c["k_lens"][b])):
                x[b, m:] = math.nan
    nb = c.get("nb", 0)
    if nb:
        s["table"] = rnd(nb, hq).to(dt)
        e = torch.unique(torch.randint(-nk, nk // 4 + 2, (4 * nb,), generator=gen, device="cuda"))[: nb - 1]
        while e.numel() < nb - 1:
            e = torch.cat([e, e[-1:] + 1 if e.numel() else torch.zeros(1, dtype=torch.int64, device="cuda")])
        s["edges"] = e.to(torch.int32).contiguous()
    blocks = -(-nk // c["block"])
    # unordered sets with repeats, entries outside the range, and rows that read nothing
    s["blocks"] = torch.randint(-1, blocks + 1, (B, hkv, n, c["keep"]), generator=gen, device="cuda", dtype=torch.int32)
    if c["sq"] > 3:
        s["blocks"][:, :, 2] = -1
    if c.get("all"):
        s["blocks"] = torch.arange(c["keep"], device="cuda", dtype=torch.int32).expand(B, hkv, n, -1).contiguous()
    return s


def case(dtype="bf16", b=1, sq=70, sk=200, hq=4, hkv=2, d=64, block=64, keep=3, causal=True, **kw):
    return dict(dtype=dtype, b=b, sq=sq, sk=sk, hq=hq, hkv=hkv, d=d, block=block, keep=keep, causal=causal, **kw)


CASES = [
    case(),
    case("fp16", b=2, sq=1, sk=1, keep=1),
    case(sq=1, sk=1000, hq=8, hkv=1, d=128, keep=9),
    case("fp16", sq=1, sk=3000, hq=16, hkv=1, d=128, keep=60, nb=20, all=True),
    case(b=3, sq=5, sk=333, hq=6, hkv=6, d=128, keep=4, nb=9),
    case("fp16", b=2, sq=129, sk=129, hq=5, hkv=1, d=80, keep=2, causal=False),
    case(b=2, sq=100, sk=300, hq=8, hkv=2, d=128, keep=5, causal=False, nb=64),
    case(b=4, sq=65, sk=65, hq=4, hkv=2, d=128, keep=2, nb=17, q_lens=[65, 0, 1, 40], k_lens=[65, 0, 1, 64]),
    case("fp16", b=3, sq=64, sk=256, hq=2, hkv=2, d=8, keep=4, q_lens=[64, 10, 33], k_lens=[20, 256, 65]),
    case(b=2, sq=33, sk=520, hq=16, hkv=1, d=120, block=128, keep=4, nb=2),
    case("fp16", sq=40, sk=900, hq=20, hkv=1, d=64, block=192, keep=3),
    case(sq=17, sk=1500, hq=64, hkv=1, d=64, keep=7, nb=33),
    case("fp16", sq=300, sk=700, hq=3, hkv=3, d=128, keep=11, all=True, nb=32),
    case(sq=257, sk=257, hq=2, hkv=1, d=64, keep=5, all=True, nb=1),
]


def names(c):
    return "-".join(str(c[k]) for k in ("dtype", "b", "sq", "sk", "hq", "hkv", "d", "block", "keep")) + ("" if c["causal"] else "-full")


def kw(c, s):
    return dict(block=c["block"], causal=c["causal"], q_lens=s["q_lens"], k_lens=s["k_lens"], table=s["table"], edges=s["edges"])


def near(got, want, bound, what):
    got = got.double()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    off = torch.where(inf, 0.0, (got - torch.where(inf, 0.0, want)).abs() - bound)
    assert not got[~inf].isnan().any(), f"{what}: NaN"
    assert off.max() <= 0 if off.numel() else True, f"{what}: {float(off.max()):.3g} over its bound at {int(off.argmax())}"


def check(A, c, s, scale=None):
    k = kw(c, s)
    want, bound = ref.attention(s["q"], s["k"], s["v"], s["blocks"], c["block"], c["causal"],
                                c["d"] ** -0.5 if scale is None else scale, s["q_lens"], s["k_lens"], s["table"],
                                s["edges"], s["dout"])
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], scale=scale, **k)
    near(out, want["out"], bound["out"], "out")
    near(lse, want["lse"], bound["lse"], "lse")
    dq, dk, dv, dt = A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], scale=scale, **k)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv), ("dtable", dt)):
        if x is not None:
            near(x, want[name], bound[name], name)
    return out, lse, dq, dk, dv, dt


@gpu
@pytest.mark.parametrize("c", CASES, ids=names)
def test_forward_and_gradients(A, c):
    check(A, c, make(c))


@gpu
@pytest.mark.parametrize("c", [
    # the longest lists and tables that a workgroup holds
    case(sq=40, sk=19200, hq=1, hkv=1, d=128, keep=256, nb=32),
    case("fp16", sq=9, sk=16390, hq=64, hkv=1, d=128, keep=256, nb=64),
    # many short walks (one wave each), and a few (two)
    case(b=2, sq=2100, sk=130, hq=8, hkv=4, d=64, keep=2, nb=8),
    case("fp16", b=3, sq=500, sk=500, hq=8, hkv=8, d=128, keep=6, q_lens=[500, 499, 3], k_lens=[400, 499, 500]),
], ids=names)
def test_limits_and_shares(A, c):
    check(A, c, make(c, 14))


@gpu
@pytest.mark.parametrize("layout", ["packed", "bhsd"])
def test_strides(A, layout):
    c = case(b=2, sq=90, sk=200, hq=4, hkv=2, d=64, nb=8)
    check(A, c, make(c, 3, layout))


@gpu
def test_same_bits_twice_and_on_another_stream(A):
    c = case(b=2, sq=300, sk=600, hq=8, hkv=2, d=128, keep=5, nb=16)
    s = make(c, 4)
    first = check(A, c, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
        again = (out, lse) + A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], **kw(c, s))
    torch.cuda.synchronize()
    for x, y in zip(first, again):
        assert torch.equal(x, y)


@gpu
def test_scale_and_lowest_bias(A):
    c = case(b=1, sq=66, sk=130, hq=2, hkv=1, d=64, nb=3, keep=3, all=True)
    s = make(c, 5)
    check(A, c, s, scale=-0.2)
    # a bucket at the type's lowest value: nothing of it is left beside the others, and a row of it alone is a row of equals
    s["edges"] = torch.tensor([-40, 0], dtype=torch.int32, device="cuda")
    s["table"][0] = torch.finfo(torch.bfloat16).min
    check(A, c, s)
    s["table"][:] = torch.finfo(torch.bfloat16).min
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
    v = s["v"].double()
    for i in (0, 5, 65):
        # scores of that size differ by no bit of the product
        mean = v[0, : i + 65, 0].mean(0)
        bound = 2 ** -8 * mean.abs() + (2 ** -8 + ref.C) * v[0, : i + 65, 0].abs().mean(0)
        assert ((out[0, i, 0].double() - mean).abs() <= bound).all()
    s["table"][:] = -math.inf
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv, dt = A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], **kw(c, s))
    assert all((x == 0).all() for x in (dq, dk, dv, dt))


@gpu
def test_masked_infinities_reach_nobody(A):
    """NaN and infinities in a key, value, query or gradient change only the results that read them."""
    c = case(b=1, sq=150, sk=256, hq=4, hkv=2, d=64, keep=2, nb=5)
    s = make(c, 6)
    s["blocks"][..., 0] = 0
    s["blocks"][..., 1] = torch.arange(150, device="cuda") % 3    # every third query reads block 2
    check(A, c, s)
    want, bound = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, True, 0.125, None, None, s["table"], s["edges"], s["dout"])
    k, v = s["k"].clone(), s["v"].clone()
    k[0, 140, 0], v[0, 141, 0], v[0, 255, 1] = math.inf, math.nan, math.inf    # block 2, and one that nobody reads
    out, lse = A.block_attention(s["q"], k, v, s["blocks"], **kw(c, s))
    dq = A.block_attention_grad(s["dout"], s["q"], k, v, out, lse, s["blocks"], **kw(c, s))[0]
    i = torch.arange(150, device="cuda")
    reads = (i % 3 == 2) & (i + 106 >= 140)      # through key head 0
    for got, name in ((out, "out"), (dq, "dq")):
        near(got[0, ~reads, :2], want[name][0, ~reads, :2], bound[name][0, ~reads, :2], name)
        near(got[0, :, 2:], want[name][0, :, 2:], bound[name][0, :, 2:], name)
    near(lse[0, :2][:, ~reads], want["lse"][0, :2][:, ~reads], bound["lse"][0, :2][:, ~reads], "lse")
    assert out[0, (i % 3 == 2) & (i + 106 >= 141), :2].isnan().any(2).all()
    # a query and a gradient row that are not finite reach the keys they read, and no others
    q, do = s["q"].clone(), s["dout"].clone()
    q[0, 50, 0] = math.nan       # reads block 0 and block 2 up to key 156
    do[0, 53, 1] = math.inf      # reads block 0 and block 2 up to key 159
    out, lse = A.block_attention(q, s["k"], s["v"], s["blocks"], **kw(c, s))
    dq, dk, dv, dt = A.block_attention_grad(do, q, s["k"], s["v"], out, lse, s["blocks"], **kw(c, s))
    j = torch.arange(256, device="cuda")
    free = ((j >= 64) & (j < 128)) | (j >= 160)
    for got, name in ((dk, "dk"), (dv, "dv")):
        near(got[0, free], want[name][0, free], bound[name][0, free], name)
        near(got[0, :, 1], want[name][0, :, 1], bound[name][0, :, 1], name)
    kept = (i != 50) & (i != 53)
    near(dq[0, kept], want["dq"][0, kept], bound["dq"][0, kept], "dq")
    near(dt[:, 2:], want["dtable"][:, 2:], bound["dtable"][:, 2:], "dtable")


@gpu
def test_rows_behind_the_end_are_left(A):
    c = case(b=2, sq=40, sk=100, hq=2, hkv=1, d=64, q_lens=[40, 7], k_lens=[100, 30])
    s = make(c, 7)
    out = torch.full((2, 40, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    A.block_attention(s["q"], s["k"], s["v"], s["blocks"], out=out, **kw(c, s))
    assert (out[1, 7:] == 7).all() and not (out[1, :7] == 7).all() and not (out[0] == 7).all()
    blocks = torch.full((2, 1, 40, 3), 9, dtype=torch.int32, device="cuda")
    A.block_select(s["q"].nan_to_num(), A.block_summary(s["k"], k_lens=s["k_lens"]), 3, k_len=100, q_lens=s["q_lens"],
                   k_lens=s["k_lens"], out=blocks)
    assert (blocks[1, :, 7:] == 9).all() and (blocks[1, :, :7] < 2).all()


@gpu
@pytest.mark.parametrize("dtype,b,n,h,d,block,lens", [
    ("bf16", 1, 1, 1, 8, 64, None), ("fp16", 2, 200, 3, 64, 64, [200, 65]), ("bf16", 3, 500, 2, 128, 128, [0, 1, 500]),
    ("bf16", 1, 1029, 2, 104, 1024, None)])
def test_summary(A, dtype, b, n, h, d, block, lens):
    k = torch.randn(b, n, h, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(DT[dtype])
    kl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = torch.zeros(b, h, -(-n // block), d, dtype=torch.float64, device="cuda")
    for x in range(b):
        m = n if lens is None else lens[x]
        k[x, m:] = math.nan
        for c in range(-(-m // block)):
            want[x, :, c] = k[x, c * block:min(m, (c + 1) * block)].double().mean(0)
    got = A.block_summary(k, block=block, k_lens=kl)
    assert torch.equal(got, want.float().to(DT[dtype]))
    # a cache that grew: only the blocks of the new tokens are written
    for fresh in (1, 63, 64, 65, n, 10 * n):
        part = torch.full_like(got, 5.0)
        A.block_summary(k, block=block, k_lens=kl, fresh=fresh, out=part)
        for x in range(b):
            m = n if lens is None else lens[x]
            lo, hi = max(0, m - fresh) // block, -(-m // block)
            assert torch.equal(part[x, :, lo:hi], got[x, :, lo:hi])
            assert (part[x, :, :lo] == 5).all() and (part[x, :, hi:] == 5).all()


SELECT = [
    ("bf16", 1, 1, 64, 1, 1, 64, 64, 1, True, 0, 1, None, None),
    ("bf16", 2, 100, 1000, 8, 2, 128, 64, 6, True, 1, 1, None, None),
    ("fp16", 1, 37, 4000, 3, 3, 80, 64, 9, False, 2, 0, None, None),
    ("bf16", 3, 70, 500, 16, 1, 64, 128, 3, True, 1, 2, [70, 0, 20], [500, 40, 10]),
    ("fp16", 2, 1, 20000, 16, 2, 128, 64, 40, True, 1, 3, None, [20000, 12345]),
    ("bf16", 1, 5, 3000, 40, 1, 64, 64, 100, True, 0, 0, None, None),
]


@gpu
@pytest.mark.parametrize("dtype,b,n,nk,hq,hkv,d,block,keep,causal,first,local,ql,kl", SELECT)
def test_select(A, dtype, b, n, nk, hq, hkv, d, block, keep, causal, first, local, ql, kl):
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(b, n, hq, d, device="cuda", generator=gen).to(DT[dtype])
    m = (torch.randn(b, hkv, -(-nk // block), d, device="cuda", generator=gen) / 8).to(DT[dtype])
    m[:, :, 1::3] = m[:, :, :1]            # equal scores: the lower block wins
    if m.shape[2] > 5:
        m[:, :, 4] = math.nan
        m[:, :, 5] = math.inf
    ql, kl = (None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ql, kl))
    if kl is not None and ql is None:
        ql = torch.full((b,), n, dtype=torch.int32, device="cuda")
    got = A.block_select(q, m, keep, k_len=nk, block=block, causal=causal, first=first, local=local, q_lens=ql, k_lens=kl)
    want = ref.select(q, m, keep, nk, block, causal, first, local, ql, kl)
    assert torch.equal(got.cpu(), want)


@gpu
def test_captured_and_replayed(A):
    """Summary, selection, attention and gradients in one graph, beside eager work."""
    c = case(b=2, sq=200, sk=500, hq=4, hkv=2, d=64, keep=4, nb=6)
    s, t = make(c, 8), make(c, 9)

    def step(x):
        m = A.block_summary(x["k"])
        blocks = A.block_select(x["q"], m, 4, k_len=500)
        out, lse = A.block_attention(x["q"], x["k"], x["v"], blocks, **kw(c, x))
        return (m, blocks, out, lse) + A.block_attention_grad(x["dout"], x["q"], x["k"], x["v"], out, lse, blocks, **kw(c, x))

    step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(s)
    for turn in range(3):
        fresh = make(c, 20 + turn)
        for n in ("q", "k", "v", "dout", "table", "edges"):
            s[n].copy_(fresh[n])
        want = step(s)
        step(t)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y)


@gpu
def test_gradients_against_differences(A):
    """The formulas' gradients: a small step of an input moves the loss by them (64-bit reference)."""
    c = case("fp16", b=1, sq=12, sk=70, hq=2, hkv=1, d=16, keep=2, nb=5)
    s = make(c, 10)
    want, _ = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, True, 0.25, None, None, s["table"], s["edges"], s["dout"])

    def loss(**new):
        x = {n: new.get(n, s[n].double()) for n in ("q", "k", "v", "table")}
        r, _ = ref.attention(x["q"], x["k"], x["v"], s["blocks"], 64, True, 0.25, None, None, x["table"], s["edges"])
        return float((r["out"] * s["dout"].double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(11)
    for n, g in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("table", "dtable")):
        step = torch.randn(s[n].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        slope = (loss(**{n: s[n].double() + h * step}) - loss(**{n: s[n].double() - h * step})) / (2 * h)
        assert abs(slope - float((want[g] * step).sum())) <= 1e-6 * (1 + abs(slope))


# ------------------------------------------------------------------ dense bias
@gpu
@pytest.mark.parametrize("dtype,b,h,n,nk,nb", [
    ("fp32", 1, 1, 1, 1, 1), ("bf16", 2, 3, 17, 65, 7), ("fp16", 1, 16, 130, 259, 32), ("fp32", 3, 5, 317, 1033, 48),
    ("bf16", 2, 2, 1, 3000, 64), ("fp16", 1, 4, 700, 1, 9), ("bf16", 2, 4, 64, 512, 33)])
def test_rel_bias(A, dtype, b, h, n, nk, nb):
    gen = torch.Generator(device="cuda").manual_seed(12)
    table = torch.randn(nb, h, generator=gen, device="cuda").to(DT[dtype])
    edges = torch.sort(torch.randint(-nk - 5, n + 5, (nb - 1,), generator=gen, device="cuda")).values.to(torch.int32)
    d = torch.arange(nk, device="cuda") - torch.arange(n, device="cuda")[:, None] - (nk - n)
    bucket = (edges.long()[:, None, None] <= d).sum(0)
    got = A.rel_bias(table, edges, n, nk)
    assert torch.equal(got, table.t()[:, bucket])
    grad = torch.randn(b, h, n, nk + 3, generator=gen, device="cuda").to(DT[dtype])[..., 1:nk + 1]   # odd strides
    for g in (grad, grad.contiguous(), grad[:1, :1].expand(b, h, n, nk)):
        x = g.double()
        want = torch.stack([torch.where(bucket == t, x, 0.0).sum((0, 2, 3)) for t in range(nb)])
        size = torch.stack([torch.where(bucket == t, x.abs(), 0.0).sum((0, 2, 3)) for t in range(nb)])
        # fp32 sums of up to 2^12 terms in a row, then their results: below 2^-12 of the magnitudes' sum
        bound = 2.0 ** -12 * size + torch.finfo(DT[dtype]).eps / 2 * want.abs() + 1e-30
        got = A.rel_bias_grad(g, edges)
        assert got.shape == (nb, h) and got.dtype == DT[dtype]
        assert ((got.double() - want).abs() <= bound).all()
        assert torch.equal(got, A.rel_bias_grad(g, edges))


@gpu
def test_dense_bias_is_the_bias_of_the_scores(A):
    """Attention over every block with a table = dense attention with rel_bias added, and so their gradients."""
    n, nk, h, d, nb = 75, 150, 3, 64, 12
    c = case("fp16", b=2, sq=n, sk=nk, hq=h, hkv=h, d=d, keep=3, causal=False, nb=nb, all=True)
    s = make(c, 13)
    out, lse, dq, dk, dv, dt = check(A, c, s)
    bias = A.rel_bias(s["table"], s["edges"], n, nk)
    q, k, v, do = (s[x].double().transpose(1, 2) for x in ("q", "k", "v", "dout"))
    P = torch.softmax(q @ k.transpose(2, 3).contiguous() * d ** -0.5 + bias.double(), -1)
    o = P @ v
    assert (out.double().transpose(1, 2) - o).abs().max() <= 2 ** -10 * v.abs().max()
    dS = P * (do @ v.transpose(2, 3).contiguous() - (do * o).sum(3, keepdim=True))
    dense = A.rel_bias_grad(dS.float().contiguous(), s["edges"])
    size = A.rel_bias_grad(dS.abs().float().contiguous(), s["edges"])
    assert ((dense - dt.float()).abs() <= 2 ** -6 * size + 1e-3).all()


# ------------------------------------------------------------------ refusals (no GPU)
def _call(name, **change):
    """The status of a C call on made-up device addresses with one thing changed; nothing is launched."""
    import ctypes as C

    import ias
    f = dict(dtype=1, device=0, stream=None, batch=1, q_len=4, k_len=128, q_heads=4, k_heads=2, head_dim=64, block=64,
             keep=2, causal=1, scale=0.125, num_buckets=0, q_lens=None, k_lens=None, table=None, edges=None)
    f.update({k: v for k, v in change.items() if k in f})
    a = ias.Attention(**f)
    h = {n: ias.Heads(1 << 20, 4 * 4 * 64, 4 * 64, 64) for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")}
    for n, x in change.get("heads", {}).items():
        h[n] = x
    p = {n: None if x is None else C.byref(x) for n, x in h.items()}
    some, ws, nws = 1 << 20, change.get("ws", 1 << 20), change.get("nws", 1 << 40)
    if name == "summary":
        return ias.lib.ias_block_summary(C.byref(a), p["k"], change.get("fresh", 0), change.get("summary", some))
    if name == "select":
        return ias.lib.ias_block_select(C.byref(a), p["q"], change.get("summary", some), change.get("first", 1),
                                        change.get("local", 1), change.get("blocks", some))
    if name == "attend":
        return ias.lib.ias_block_attention(C.byref(a), p["q"], p["k"], p["v"], change.get("blocks", some), p["out"],
                                           some, ws, nws)
    return ias.lib.ias_block_attention_grad(C.byref(a), p["dout"], p["q"], p["k"], p["v"], p["out"],
                                            change.get("lse", some), change.get("blocks", some), p["dq"], p["dk"], p["dv"],
                                            change.get("dtable"), ws, nws)


INVALID, MISMATCH, UNSUPPORTED, OVERFLOW, CAPACITY = 1, 2, 7, 9, 11


@pytest.mark.parametrize("name", ["summary", "select", "attend", "grad"])
@pytest.mark.parametrize("change,status", [
    (dict(dtype=0), UNSUPPORTED), (dict(dtype=5), UNSUPPORTED), (dict(device=-1), INVALID), (dict(batch=-1), INVALID),
    (dict(q_len=-1), INVALID), (dict(k_len=-2), INVALID), (dict(q_heads=3), MISMATCH), (dict(k_heads=0), MISMATCH),
    (dict(q_heads=130), UNSUPPORTED), (dict(head_dim=60), UNSUPPORTED), (dict(head_dim=136), UNSUPPORTED),
    (dict(head_dim=0), UNSUPPORTED), (dict(block=32), UNSUPPORTED), (dict(block=96), UNSUPPORTED),
    (dict(block=2048), UNSUPPORTED), (dict(k_len=64 * 16384 + 1), UNSUPPORTED), (dict(scale=math.inf), INVALID),
    (dict(scale=math.nan), INVALID), (dict(batch=1 << 30, q_len=1 << 20), OVERFLOW),
    (dict(table=1 << 20, num_buckets=65, edges=1 << 20), UNSUPPORTED), (dict(table=1 << 20, num_buckets=2), INVALID),
])
def test_shapes_are_refused(name, change, status):
    assert _call(name, **change) == status


@pytest.mark.parametrize("name,change,status", [
    ("select", dict(keep=0), UNSUPPORTED), ("attend", dict(keep=257), UNSUPPORTED), ("grad", dict(keep=0), UNSUPPORTED),
    ("select", dict(first=2, local=1), INVALID), ("select", dict(first=-1), INVALID), ("select", dict(causal=0), INVALID),
    ("select", dict(summary=None), INVALID), ("select", dict(blocks=None), INVALID), ("summary", dict(summary=None), INVALID),
    ("summary", dict(fresh=-1), INVALID), ("attend", dict(blocks=None), INVALID), ("grad", dict(lse=None), INVALID),
    ("grad", dict(dtable=1 << 20), INVALID),
    ("attend", dict(table=1 << 20, num_buckets=3, edges=1 << 20, ws=None), CAPACITY),
    ("attend", dict(table=1 << 20, num_buckets=3, edges=1 << 20, nws=64), CAPACITY),
    ("attend", dict(table=1 << 20, num_buckets=3, edges=1 << 20, ws=(1 << 20) + 16), INVALID),
    ("grad", dict(nws=8), CAPACITY),
])
def test_arguments_are_refused(name, change, status):
    assert _call(name, **change) == status


def test_addresses_and_strides_are_refused():
    import ias
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        for bad, status in ((None, INVALID), (ias.Heads(None, 1024, 256, 64), INVALID),
                            (ias.Heads((1 << 20) + 8, 1024, 256, 64), UNSUPPORTED),
                            (ias.Heads(1 << 20, 1024, 258, 64), UNSUPPORTED),
                            (ias.Heads(1 << 20, 1024, 256, 60), UNSUPPORTED),
                            (ias.Heads(1 << 20, 1 << 30, (1 << 24) + 8, 64), UNSUPPORTED),
                            (ias.Heads(1 << 20, 1 << 30, -256, 64), UNSUPPORTED)):
            assert _call("grad", heads={n: bad}) == status, n
    # nothing to do is done without an address
    assert _call("attend", q_len=0, blocks=None, heads={n: ias.Heads(None, 0, 0, 0) for n in ("q", "out")}) == 0
    assert _call("select", batch=0, blocks=None) == 0


def test_bias_arguments_are_refused():
    import ctypes as C

    import ias
    f, x = ias.lib.ias_rel_bias, 1 << 20
    assert f(3, 4, 5, 6, 7, x, x, x, 0, None) == UNSUPPORTED
    assert f(0, 4, 5, 6, 0, x, x, x, 0, None) == UNSUPPORTED
    assert f(0, 4, 5, 6, 65, x, x, x, 0, None) == UNSUPPORTED
    assert f(0, -4, 5, 6, 7, x, x, x, 0, None) == INVALID
    assert f(0, 4, 5, 6, 7, None, x, x, 0, None) == INVALID
    assert f(0, 4, 5, 6, 7, x, None, x, 0, None) == INVALID
    assert f(0, 4, 1 << 31, 6, 7, x, x, x, 0, None) == OVERFLOW
    assert f(0, 4, 1 << 18, 1 << 18, 7, x, x, x, 0, None) == OVERFLOW
    assert f(0, 4, 0, 6, 7, None, None, None, 0, None) == 0
    n = C.c_int64(0)
    assert ias.lib.ias_rel_bias_grad_workspace(1, 1 << 16, 1, 1 << 24, 7, C.byref(n)) == OVERFLOW
    assert ias.lib.ias_rel_bias_grad_workspace(1, 1, 1 << 17, 1 << 17, 7, C.byref(n)) == 0
    assert ias.lib.ias_rel_bias_grad_workspace(2, 4, 5, 6, 7, C.byref(n)) == 0 and n.value > 0
    g = ias.lib.ias_rel_bias_grad
    assert g(0, 2, 4, 5, 6, 7, x, 120, 30, 6, x, x, x, n.value - 4, 0, None) == CAPACITY
    assert g(0, 2, 4, 5, 6, 7, None, 120, 30, 6, x, x, x, n.value, 0, None) == INVALID
    assert g(0, 2, 4, 5, 6, 7, x, 120, 30, 6, x, None, x, n.value, 0, None) == INVALID


def test_struct_layouts_match_header(tmp_path):
    import ctypes as C
    import os
    import subprocess

    import ias
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ias.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu\\n", sizeof(ias_heads), sizeof(ias_attention), '
                   'offsetof(ias_attention, scale), offsetof(ias_attention, clear));return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(ias.Heads), C.sizeof(ias.Attention), ias.Attention.scale.offset, ias.Attention.clear.offset]


def test_tensors_of_the_host_are_refused():
    from ias import attention
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention.block_summary(q)
    with pytest.raises(ValueError):
        attention.rel_bias(torch.zeros(3, 2), torch.zeros(2, dtype=torch.int32), 4, 4)


@gpu
@pytest.mark.parametrize("kind", ["near", "same", "zero", "huge", "tiny"])
@pytest.mark.parametrize("m", [70, 600])
def test_select_where_scores_are_close(A, kind, m):
    """Order by 64 bits where fp32 sums do not tell the scores apart, overflow or vanish."""
    gen = torch.Generator(device="cuda").manual_seed(15)
    b, n, hq, hkv, d, keep = 2, 9, 6, 2, 64, 20
    q = torch.randn(b, n, hq, d, device="cuda", generator=gen).to(torch.bfloat16)
    base = torch.randn(1, 1, 1, d, device="cuda", generator=gen).to(torch.bfloat16)
    s = base.expand(b, hkv, m, d).clone()
    if kind == "near":    # one channel differs by its last place: scores a few 2^-16 of the sum apart
        at = torch.randint(0, d, (b, hkv, m), device="cuda", generator=gen)
        step = torch.randint(-1, 2, (b, hkv, m), device="cuda", generator=gen).to(torch.int16)
        s.view(torch.int16).scatter_add_(3, at[..., None], step[..., None])
    elif kind == "zero":
        q[:, ::2] = 0
        s = torch.randn(b, hkv, m, d, device="cuda", generator=gen).to(torch.bfloat16)
    elif kind in ("huge", "tiny"):
        s = torch.randn(b, hkv, m, d, device="cuda", generator=gen).to(torch.bfloat16)
        s, q = (x * (2.0 ** (100 if kind == "huge" else -100)) for x in (s, q))
    got = A.block_select(q, s, keep, k_len=m * 64, first=1, local=1)
    assert torch.equal(got.cpu(), ref.select(q, s, keep, m * 64, 64, True, 1, 1, None, None))


@gpu
def test_offsets_beyond_32_bits(A):
    """A cache of 2^20 tokens inside a wider tensor of over 2^32 bytes."""
    n = 1 << 20
    c = case(b=1, sq=2, sk=n, hq=2, hkv=1, d=128, keep=5, nb=6)
    s = make(dict(c, sk=64))
    wide = torch.zeros(1, n, 20, 128, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(16)
    s["k"], s["v"] = wide[:, :, 18:19], wide[:, :, 19:20]
    for x in (s["k"], s["v"]):
        x.copy_(torch.randn(1, n, 1, 128, device="cuda", generator=gen))
    s["blocks"] = torch.tensor([[0, 16383, 5000, 16382, 12345], [16383, 1, 9, -1, -1]], dtype=torch.int32,
                               device="cuda").view(1, 1, 2, 5)
    s["edges"] = torch.tensor([-(1 << 19), -5000, -64, -3, 0], dtype=torch.int32, device="cuda")
    check(A, c, s)
    m = A.block_summary(s["k"])
    got = A.block_select(s["q"], m, 5, k_len=n)
    assert torch.equal(got.cpu(), ref.select(s["q"], m, 5, n, 64, True, 1, 1, None, None))


@gpu
def test_nothing_to_read_and_nobody_to_ask(A):
    """No keys: zeros.  No queries: gradients of the keys are zeros."""
    z = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)  # noqa: E731
    blocks = torch.zeros(2, 1, 3, 4, dtype=torch.int32, device="cuda")
    q, k = z(2, 3, 4, 64), z(2, 0, 1, 64)
    table, edges = z(5, 4), torch.arange(-3, 1, dtype=torch.int32, device="cuda")
    for bias in ({}, dict(table=table, edges=edges)):
        out, lse = A.block_attention(q, k, k, blocks, **bias)
        assert (out == 0).all() and (lse == -math.inf).all()
        dq, dk, dv, dt = A.block_attention_grad(q, q, k, k, out, lse, blocks, **bias)
        assert (dq == 0).all() and dk.shape == k.shape and (dt is None or (dt == 0).all())
    m = A.block_summary(k)
    assert m.shape == (2, 1, 0, 64) and (A.block_select(q, m, 4, k_len=0) == -1).all()
    q, k = z(2, 0, 4, 64), z(2, 70, 1, 64)
    out, lse = A.block_attention(q, k, k, blocks[:, :, :0].contiguous(), table=table, edges=edges)
    assert out.shape == q.shape
    dq, dk, dv, dt = A.block_attention_grad(q, q, k, k, out, lse, blocks[:, :, :0].contiguous(), table=table, edges=edges)
    assert (dk == 0).all() and (dv == 0).all() and (dt == 0).all()
    assert A.block_select(q, A.block_summary(k), 4, k_len=70).shape == (2, 1, 0, 4)
    assert A.rel_bias(table, edges, 0, 7).shape == (4, 0, 7)
    assert (A.rel_bias_grad(z(1, 4, 0, 7), edges) == 0).all()


@gpu
def test_first_call_is_captured(A):
    """A graph whose capture is the first call of its shapes, and two graphs replayed in turn."""
    c = case("fp16", b=1, sq=90, sk=190, hq=2, hkv=2, d=120, block=128, keep=2, nb=40)
    s, t = make(c, 17), make(c, 18)
    graphs, held = [], []
    for x in (s, t):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = A.block_attention(x["q"], x["k"], x["v"], x["blocks"], **kw(c, x))
            held.append((out, lse) + A.block_attention_grad(x["dout"], x["q"], x["k"], x["v"], out, lse, x["blocks"], **kw(c, x)))
        graphs.append(g)
    for turn in range(3):
        for g, x, h in zip(graphs, (s, t), held):
            g.replay()
            for a, b in zip(h, check(A, c, x)):
                assert torch.equal(a, b)


@gpu
def test_launches_beyond_32_bits_are_refused(A):
    """2^24 + 8 workgroups of 256 threads."""
    b = (1 << 24) + 8
    q = torch.zeros(b, 1, 1, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(Exception, match="threads in a launch"):
        A.block_select(q, torch.empty(b, 1, 0, 8, dtype=torch.bfloat16, device="cuda"), 1, k_len=0, first=0)
    with pytest.raises(Exception, match="threads in a launch"):
        A.block_summary(q)
    one = torch.zeros(1, 1, 3, 1, device="cuda").transpose(2, 3).contiguous().transpose(2, 3)   # one column, of any stride
    assert (A.rel_bias_grad(one, torch.zeros(0, dtype=torch.int32, device="cuda")) == 0).all()
