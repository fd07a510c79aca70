"""Block-sparse attention and the relative bias at the ends of their types' and sizes' ranges."""
import math

import pytest
import torch

import attention_ref as ref
from test_attention import A, CAPACITY, DT, INVALID, OVERFLOW, UNSUPPORTED, _call, case, check, kw, make, near  # noqa: F401

gpu = pytest.mark.gpu


# ------------------------------------------------------------------ dense bias
@gpu
@pytest.mark.parametrize("dtype,n,nk,h", [
    ("bf16", 1 << 24, 1, 16), ("fp32", 1 << 24, 3, 16), ("fp16", 12_000_000, 1, 32), ("bf16", 1 << 23, 1, 64)])
def test_gradient_of_a_tall_bias(A, dtype, n, nk, h):
    """q_len x spans x heads beyond 2^43.  A constant gradient, of stride 0: sums are counts, exact in fp32 up to 2^24."""
    grad = torch.full((1, 1, 1, nk), 2.0 ** -10, device="cuda").to(DT[dtype]).expand(1, h, n, nk)
    edges = torch.tensor([-(n // 2), -1000, 0], dtype=torch.int32, device="cuda")
    got = A.rel_bias_grad(grad, edges).double()
    want = torch.zeros(4, dtype=torch.float64, device="cuda")
    for j in range(nk):    # distances j - i - (nk - n), i < n: the n values that end at j - (nk - n)
        lo, hi = j - nk + 1, j - nk + n
        cut = [lo] + [min(max(e, lo), hi + 1) for e in (-(n // 2), -1000, 0)] + [hi + 1]
        for t in range(4):
            want[t] += (cut[t + 1] - cut[t]) * 2.0 ** -10
    bound = (2.0 ** -12 + torch.finfo(DT[dtype]).eps / 2) * want
    assert ((got - want[:, None]).abs() <= bound[:, None]).all()


# ------------------------------------------------------------------ biases of the type's lowest value
@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("sq,sk,hq,hkv,d", [(300, 300, 4, 4, 128), (1, 6000, 4, 2, 64), (40, 2000, 2, 1, 64)])
def test_log_sums_of_the_lowest_bias(A, dtype, sq, sk, hq, hkv, d):
    """Walks shared by workgroups: the log of the sum is the lowest value too, not -infinity."""
    c = case(dtype, sq=sq, sk=sk, hq=hq, hkv=hkv, d=d, keep=-(-sk // 64), nb=3, all=True)
    s = make(c, 35)
    s["q"] *= 0        # beside 65504 fp32 does not hold a score to fp16's half step
    s["table"][:] = torch.finfo(DT[dtype]).min
    want, bound = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, True, d ** -0.5, None, None, s["table"], s["edges"])
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
    near(out, want["out"], bound["out"], "out")
    near(lse, want["lse"], bound["lse"], "lse")

@gpu
@pytest.mark.parametrize("sq,hq,hkv,d", [(80, 2, 1, 64), (300, 4, 4, 128), (3, 4, 2, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_of_rows_of_the_lowest_bias(A, dtype, sq, hq, hkv, d):
    """Rows that see nothing but a bucket at the type's lowest value are rows of equals, beside ordinary ones."""
    c = case(dtype, b=2, sq=sq, sk=sq + 7, hq=hq, hkv=hkv, d=d, keep=6, nb=3, all=True, q_lens=[sq, sq - 1], k_lens=[sq, sq + 3])
    s = make(c, 34)
    s["edges"] = torch.tensor([-30, -20], dtype=torch.int32, device="cuda")
    if dtype == "fp16":
        s["q"] = torch.where(s["q"].isnan(), s["q"], 0.0).half()    # scores of 65504 differ by what fp32 holds there
    for low in (torch.finfo(DT[dtype]).min, -3e4):
        if low == -3e4:
            s["q"] = torch.where(s["q"].isnan(), s["q"], 0.0).to(DT[dtype])
        s["table"][2] = low         # the keys at distances of -20 and more: all that the first rows see
        check(A, c, s)
        check(A, c, s, scale=-0.3)
        s["table"][:] = low
        check(A, c, s)


@gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("b,n,nk", [(4096, 16, 64), (1, 60_000, 60_000), (300, 700, 900)])
def test_bias_gradient_of_many_terms(A, dtype, b, n, nk):
    """A constant gradient, of stride 0: the roundings of a long sum go the same way."""
    grad = torch.full((nk,), 0.1, device="cuda").to(DT[dtype]).expand(b, 1, n, nk)
    edges = torch.tensor([-(n // 2), 0, 3], dtype=torch.int32, device="cuda")
    got = A.rel_bias_grad(grad, edges).double()[:, 0]
    i = torch.arange(n, device="cuda").double() + (nk - n)      # position of each query: keys j with j - i in a bucket
    cut = [torch.zeros_like(i)] + [(i + e).clamp(0, nk) for e in edges.tolist()] + [torch.full_like(i, nk)]
    want = torch.stack([(cut[t + 1] - cut[t]).sum() for t in range(4)]) * b * float(grad[0, 0, 0, 0])
    # chains of at most 3443 / 8 sums of eight (or 2048 values singly, where rows are fewer than eight), 32 such
    # chains, 8 + 6 of a workgroup, 66 + 6 of all: below 2^10 roundings of 2^-24 here
    assert ((got - want).abs() <= (2.0 ** -14 + torch.finfo(DT[dtype]).eps / 2) * want).all()


# ------------------------------------------------------------------ fp16
def two_keys(value, dout, key):
    """Head 8, two keys of equal score: dS = +-8 value dout / 2, dq = dS key 2 / sqrt(8)."""
    t = lambda x: torch.tensor(x, device="cuda").to(torch.float16)  # noqa: E731
    sign = torch.tensor([1.0, -1.0], device="cuda")[None, :, None, None].expand(1, 2, 1, 8)
    return dict(q=t([0.0]).expand(1, 1, 1, 8).contiguous(), k=(sign * key).to(torch.float16), v=(sign * value).to(torch.float16),
                dout=t([dout]).expand(1, 1, 1, 8).contiguous(), q_lens=None, k_lens=None, table=None, edges=None,
                blocks=torch.zeros(1, 1, 1, 1, dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("nb", [0, 3])
def test_score_gradients_beyond_fp16(A, nb):
    """dS = 160000, dq = 1131: an ordinary number from one that the type does not hold."""
    c = case("fp16", sq=1, sk=2, hq=1, hkv=1, d=8, keep=1, causal=False)
    s = two_keys(200.0, 200.0, 0.01)
    if nb:
        s["table"] = torch.zeros(nb, 1, dtype=torch.float16, device="cuda")
        s["edges"] = torch.tensor([-1, 0], dtype=torch.int32, device="cuda")
        want = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, False, 8 ** -0.5, None, None, s["table"], s["edges"], s["dout"])
        out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
        got = A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], **kw(c, s))
        for name, x in zip(("dq", "dk", "dv"), got):
            near(x, want[0][name], want[1][name], name)
        return
    dq = check(A, c, s)[2]
    assert 1100 < float(dq.abs().max()) < 1160


@gpu
@pytest.mark.parametrize("nb", [0, 9])
@pytest.mark.parametrize("sq,sk,hq,hkv,d", [(70, 70, 4, 2, 64), (1, 130, 6, 1, 128), (33, 200, 2, 1, 128)])
def test_large_score_gradients_fp16(A, sq, sk, hq, hkv, d, nb):
    """Gradients of 1000 (a scaled loss) and values of 30."""
    c = case("fp16", sq=sq, sk=sk, hq=hq, hkv=hkv, d=d, keep=-(-sk // 64), all=True, nb=nb)
    s = make(c, 31)
    s["dout"] *= 1000
    s["v"] *= 30
    s["q"] *= 0.02
    s["k"] *= 0.02
    s["table"] = None if nb == 0 else s["table"] * 0.125
    want, bound = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, True, d ** -0.5, None, None, s["table"], s["edges"], s["dout"])
    assert all(want[n].abs().max() < 60000 for n in ("dq", "dk", "dv"))
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
    got = A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], **kw(c, s))
    for name, x in zip(("dq", "dk", "dv"), got):
        near(x, want[name], bound[name], name)


@gpu
@pytest.mark.parametrize("sq,keys", [(1024, 4096), (1, 4096), (300, 2048)])
def test_small_score_gradients_fp16(A, sq, keys):
    """dS of some 2^-22, all alike, whose sums are ordinary numbers; every step of fp16 there is 2^-24."""
    c = case("fp16", sq=sq, sk=keys, hq=1, hkv=1, d=64, keep=keys // 64, causal=False, all=True)
    s = make(c, 32)
    sign = torch.where(torch.arange(keys, device="cuda") % 2 == 0, 1.0, -1.0)[None, :, None, None]
    s["k"] = (4 * sign).expand(1, keys, 1, 64).half().contiguous()
    s["v"] = (0.25 * keys / 4096 * sign).expand(1, keys, 1, 64).half().contiguous()
    s["q"] = (4 * (1 - 2 * (torch.arange(64, device="cuda") % 2))).expand(1, sq, 1, 64).half().contiguous()   # q.k = 0
    s["dout"] = torch.full((1, sq, 1, 64), 1e-4, device="cuda").half()
    check(A, c, s)


@gpu
@pytest.mark.parametrize("nb", [0, 4])
def test_probabilities_of_many_keys_in_the_gradient_fp16(A, nb):
    """200,000 keys: probabilities of 2^-17.6, below what fp16 holds to its 11 bits."""
    c = case("fp16", sq=2, sk=200_000, hq=2, hkv=1, d=64, block=1024, keep=196, causal=False, all=True, nb=nb)
    s = make(c, 33)
    s["q"] *= 0.05
    s["dout"] *= 200
    if nb:
        s["table"] = s["table"] * 0.1
        s["edges"] = torch.tensor([-150_000, -77_777, -5], dtype=torch.int32, device="cuda")
    check(A, c, s)


# ------------------------------------------------------------------ long walks
@gpu
@pytest.mark.parametrize("nb", [0, 2])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_log_sums_of_long_walks(A, dtype, nb):
    """One key e^16.5 times as likely as each of 2^17 others of its wave: singly they vanish beside it in fp32."""
    n, sq, d = 1 << 18, 16384, 64
    q = torch.full((1, sq, 1, d), 0.5, device="cuda").to(DT[dtype])
    k, v = torch.zeros(1, n, 1, d, device="cuda").to(DT[dtype]), torch.ones(1, n, 1, d, device="cuda").to(DT[dtype])
    for first in (0, 32):          # pieces of 32 keys go to two waves in turn
        k[0, first] = 4.21875      # a score of 16.875, exact in both types
    blocks = torch.arange(256, device="cuda", dtype=torch.int32).expand(1, 1, sq, 256).contiguous()
    table = torch.zeros(nb, 1, device="cuda").to(DT[dtype]) if nb else None
    edges = torch.tensor([0], dtype=torch.int32, device="cuda") if nb else None
    lse = A.block_attention(q, k, v, blocks, block=1024, causal=False, table=table, edges=edges)[1]
    score = (q[0, 0, 0].double() @ k[0, :, 0].double().t()) * 0.125
    # 4096 pieces a wave, each sum rounded by at most 2^-24 of what it has by then
    assert (lse.double() - torch.logsumexp(score, 0)).abs().max() <= 4096 * 2.0 ** -24 + ref.C / 8


@gpu
@pytest.mark.parametrize("nb", [0, 2])
def test_small_probabilities_beside_a_large_one_fp16(A, nb):
    """One key e^16.8 times as likely as each of 2^18 others, which make 1 % of the result together."""
    n, sq, d, x = 1 << 18, 16384, 64, 16.8
    c = case("fp16", sq=sq, sk=n, hq=1, hkv=1, d=d, block=1024, keep=256, causal=False, all=True, nb=nb)
    q = torch.full((1, sq, 1, d), 0.5, device="cuda").half()
    k, v = torch.zeros(1, n, 1, d, device="cuda").half(), torch.ones(1, n, 1, d, device="cuda").half()
    k[0, ::131072] = x * 0.25       # 0.125 * 64 * 0.5 * 4.2 = 16.8; the first key of each of two waves
    k[0, 32::131072] = x * 0.25
    v[0, ::131072] = 0
    v[0, 32::131072] = 0
    blocks = torch.arange(256, device="cuda", dtype=torch.int32).expand(1, 1, sq, 256).contiguous()
    table = edges = None
    if nb:
        table = torch.zeros(nb, 1, dtype=torch.float16, device="cuda")
        edges = torch.tensor([0], dtype=torch.int32, device="cuda")
    out, lse = A.block_attention(q, k, v, blocks, block=1024, causal=False, table=table, edges=edges)
    score = (q[0, 0, 0].double() @ k[0, :, 0].double().t()) * 0.125
    p = torch.softmax(score, 0)
    want = float(p @ v[0, :, 0, 0].double())
    assert 0.002 < want < 0.1
    # half a step of the result, and of each probability; fp32 elsewhere
    assert (out.double() - want).abs().max() <= (2.0 ** -11 * 2 + ref.C) * want
    assert (lse.double() - torch.logsumexp(score, 0)).abs().max() <= ref.C / 8 * 18


# ------------------------------------------------------------------ torch's graph
@pytest.mark.parametrize("name", ["q", "k", "v", "table", "dout", "out", "lse"])
def test_tensors_that_require_gradients_are_refused(name):
    """Results without a graph would lose a gradient in silence; refused before anything else is looked at."""
    from ias import attention
    t = {n: torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16) for n in ("q", "k", "v", "dout", "out")}
    t.update(table=torch.zeros(3, 2, dtype=torch.bfloat16), lse=torch.zeros(1, 2, 4))
    edges, blocks = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 2, 4, 1, dtype=torch.int32)
    t[name].requires_grad_()
    forward = lambda: attention.block_attention(t["q"], t["k"], t["v"], blocks, table=t["table"], edges=edges, out=t["out"])  # noqa: E731
    grad = lambda: attention.block_attention_grad(  # noqa: E731
        t["dout"], t["q"], t["k"], t["v"], t["out"], t["lse"], blocks, table=t["table"], edges=edges)
    calls = [grad] + ([forward] if name not in ("dout", "lse") else [])
    calls += {"k": [lambda: attention.block_summary(t["k"])], "table": [lambda: attention.rel_bias(t["table"], edges, 4, 4)],
              "dout": [lambda: attention.rel_bias_grad(t["dout"], edges)]}.get(name, [])
    for call in calls:
        with pytest.raises(ValueError, match=f"{name if call is not calls[-1] or name != 'dout' else 'grad'} requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="HIP device"):    # goes on to the next check
            call()


@gpu
def test_leaves_without_recording_and_given_outputs(A):
    """Under no_grad leaves are taken; a given output counts as written."""
    c = case(b=1, sq=70, sk=130, hq=4, hkv=2, d=64, keep=2)
    s = make(c, 36)
    plain = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
    for n in ("q", "k", "v"):
        s[n] = s[n].clone().requires_grad_()
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(plain, A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))))
        m = A.block_summary(s["k"])
        out, blocks = torch.empty_like(s["q"]), torch.empty_like(s["blocks"])
        before = [x._version for x in (out, blocks, m)]
        A.block_summary(s["k"], fresh=1, out=m)
        A.block_select(s["q"], m, 2, k_len=130, out=blocks)
        A.block_attention(s["q"], s["k"], s["v"], s["blocks"], out=out, **kw(c, s))
        assert all(x._version > v for x, v in zip((out, blocks, m), before))
    assert A.block_select(s["q"], m, 2, k_len=130).shape == blocks.shape
    with torch.inference_mode():
        out = torch.empty_like(s["q"])
        A.block_attention(s["q"], s["k"], s["v"], s["blocks"], out=out, **kw(c, s))
    x = torch.ones_like(plain[0], requires_grad=True)
    held = torch.zeros_like(plain[0])
    y = (x * held).sum()
    A.block_attention(s["q"].detach(), s["k"].detach(), s["v"].detach(), s["blocks"], out=held, **kw(c, s))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ------------------------------------------------------------------ refusals (no GPU)
@pytest.mark.parametrize("name,change", [
    # k_grad_q has few workgroups, the join 2^22 x 4 of 256 threads; the transpose and the items' kernel
    ("grad", dict(batch=1 << 13, q_len=1, k_len=1 << 15, q_heads=1, k_heads=1)),
    ("grad", dict(batch=1 << 24, q_len=1, k_len=64, q_heads=1, k_heads=1)),
    ("grad", dict(batch=1 << 10, q_len=1, k_len=1 << 18, q_heads=1, k_heads=1, block=1024)),
    ("attend", dict(batch=1 << 24, q_len=1, k_len=64, q_heads=1, k_heads=1)),
])
def test_a_call_is_refused_before_its_first_launch(name, change):
    """Shapes of which some launch has 2^32 threads: known before any is made (here: before a device is looked for)."""
    assert _call(name, nws=1 << 62, **change) == OVERFLOW


@pytest.mark.parametrize("name", ["summary", "select", "attend", "grad"])
@pytest.mark.parametrize("batch", [0, 1])
def test_the_largest_length_is_refused(name, batch):
    """The number of blocks of 2^63 - 1 keys is not one of 64-bit arithmetic."""
    assert _call(name, batch=batch, k_len=(1 << 63) - 1) == UNSUPPORTED
    assert _call(name, batch=batch, k_len=(1 << 63) - 40, block=1024) == UNSUPPORTED


def test_outputs_whose_rows_lie_over_each_other_are_refused():
    """4 queries and 128 keys of 4 and 2 heads of 64: strides (batch, token, head)."""
    import ias
    for name, heads, n in (("out", 4, 4), ("dq", 4, 4), ("dk", 2, 128), ("dv", 2, 128)):
        call = "attend" if name == "out" else "grad"
        for strides in ((0, 0, 64), (heads * n * 64, heads * 64, 0), (heads * n * 64, 0, 64), (heads * n * 64, 64 * heads, 56),
                        (heads * n * 64, 64 * heads - 8, 64), (0, 64, 64 * n - 64)):
            assert _call(call, heads={name: ias.Heads(1 << 20, *strides)}) == INVALID, (name, strides)
        assert _call(call, batch=2, heads={name: ias.Heads(1 << 20, 64 * heads * n - 64, 64 * heads, 64)}) == INVALID
        # heads before tokens, wider rows, an axis of one element, and inputs that repeat rows: on to the next check
        bias = dict(table=1 << 20, num_buckets=3, edges=1 << 20, nws=64)
        for strides in ((0, 64, 64 * n), (heads * n * 64, 64 * heads + 8, 64), (heads * n * 64, heads * 64, 64), (0, heads * 64, 64)):
            assert _call(call, heads={name: ias.Heads(1 << 20, *strides)}, **bias) == CAPACITY, (name, strides)
        assert _call(call, heads={"q": ias.Heads(1 << 20, 0, 0, 0), "k": ias.Heads(1 << 20, 0, 256, 0)}, **bias) == CAPACITY
