"""Block-sparse attention: paths of the kernels that ordinary inputs take, and larger plans."""
import pytest
import torch

import attention_ref as ref
from test_attention import A, DT, case, check, kw, make, near  # noqa: F401

gpu = pytest.mark.gpu

# queries x blocks where something has to be chosen by score: dtype, b, n, nk, hq, hkv, d, block, keep, causal, first, local, ql, kl
FINITE = [
    ("bf16", 1, 130, 4096, 32, 8, 128, 64, 16, True, 1, 1, None, None),        # four heads a key head, 64 blocks
    ("fp16", 1, 70, 4000, 16, 2, 80, 64, 9, True, 1, 1, None, None),           # eight
    ("fp16", 2, 33, 64 * 129, 4, 4, 128, 64, 20, False, 2, 0, None, None),     # one, 129 blocks
    ("bf16", 1, 40, 64 * 512, 8, 2, 64, 64, 7, True, 0, 2, None, None),        # 512 blocks
    ("fp16", 1, 9, 64 * 600, 6, 2, 64, 64, 12, True, 1, 1, None, None),        # beyond those held in registers
    ("bf16", 1, 21, 64 * 70, 40, 1, 64, 64, 6, True, 1, 0, None, None),        # 64 rows a workgroup
    ("fp16", 1, 12, 64 * 200, 64, 1, 128, 64, 30, True, 1, 1, None, None),
    ("bf16", 1, 17, 64 * 100, 33, 1, 120, 64, 8, False, 0, 0, None, None),
    ("bf16", 5, 1, 64 * 300, 32, 8, 128, 64, 16, True, 1, 1, None, [19200, 64, 1, 7777, 64 * 17]),   # single tokens
    ("fp16", 2, 1, 64 * 90, 4, 1, 64, 64, 5, True, 1, 1, None, None),
    ("bf16", 3, 70, 128 * 40, 16, 4, 64, 128, 3, True, 1, 1, [70, 0, 20], [5120, 40, 1000]),
    ("fp16", 1, 50, 64 * 128, 3, 3, 8, 64, 10, True, 1, 1, None, None),        # three queries' heads in a row of four
]


@gpu
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("dtype,b,n,nk,hq,hkv,d,block,keep,causal,first,local,ql,kl", FINITE)
def test_select_by_finite_scores(A, dtype, b, n, nk, hq, hkv, d, block, keep, causal, first, local, ql, kl, far):
    """Scores from the matrix instructions, their bound, and the few computed again; far: blocks of very different sizes."""
    gen = torch.Generator(device="cuda").manual_seed(41)
    q = torch.randn(b, n, hq, d, device="cuda", generator=gen).to(DT[dtype])
    m = torch.randn(b, hkv, -(-nk // block), d, device="cuda", generator=gen) / 8
    if far:
        m *= torch.exp2(-8 * torch.rand(m.shape[:3], device="cuda", generator=gen))[..., None]
    m = m.to(DT[dtype])
    ql, kl = (None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ql, kl))
    if kl is not None and ql is None:
        ql = torch.full((b,), n, dtype=torch.int32, device="cuda")
    got = A.block_select(q, m, keep, k_len=nk, block=block, causal=causal, first=first, local=local, q_lens=ql, k_lens=kl)
    want = ref.select(q, m, keep, nk, block, causal, first, local, ql, kl)
    assert torch.equal(got.cpu(), want)


@gpu
@pytest.mark.parametrize("nb", [0, 5])
@pytest.mark.parametrize("dtype,sq", [("bf16", 70), ("fp16", 3)])
def test_scale_of_zero(A, dtype, sq, nb):
    """Scores are the bias alone; queries and keys get no gradient."""
    c = case(dtype, sq=sq, sk=200, hq=4, hkv=2, d=64, nb=nb)
    s = make(c, 42)
    _, _, dq, dk, dv, _ = check(A, c, s, scale=0.0)
    assert (dq == 0).all() and (dk == 0).all() and not (dv == 0).all()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("c", [case(sq=12, sk=70, hq=2, hkv=1, d=16, keep=2, nb=5), case(sq=90, sk=90, hq=4, hkv=2, d=128, keep=2, nb=3)])
def test_kernels_gradients_against_differences(A, dtype, c):
    """A step of an input moves the loss (64 bits) as the kernels' gradient says, within its bound along the step."""
    c = dict(c, dtype=dtype)
    s = make(c, 43)
    scale = c["d"] ** -0.5
    _, bound = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, True, scale, None, None, s["table"], s["edges"], s["dout"])
    out, lse = A.block_attention(s["q"], s["k"], s["v"], s["blocks"], **kw(c, s))
    got = dict(zip(("q", "k", "v", "table"), A.block_attention_grad(s["dout"], s["q"], s["k"], s["v"], out, lse, s["blocks"], **kw(c, s))))

    def loss(**new):
        x = {n: new.get(n, s[n].double()) for n in ("q", "k", "v", "table")}
        r, _ = ref.attention(x["q"], x["k"], x["v"], s["blocks"], 64, True, scale, None, None, x["table"], s["edges"])
        return float((r["out"] * s["dout"].double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(44)
    for n in ("q", "k", "v", "table"):
        step = torch.randn(s[n].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        slope = (loss(**{n: s[n].double() + h * step}) - loss(**{n: s[n].double() - h * step})) / (2 * h)
        off = float((bound["d" + n] * step.abs()).sum())
        assert abs(slope - float((got[n].double() * step).sum())) <= off + 1e-6 * (1 + abs(slope)), n


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_where_items_are_longer(A, dtype):
    """Every query of 4096 reads 140 blocks: 2^19 entries and more, where an item takes more than 1024 rows."""
    c = case(dtype, sq=4096, sk=140 * 64, hq=16, hkv=1, d=128, keep=140, all=True)
    check(A, c, make(c, 45))


@gpu
@pytest.mark.parametrize("c", [
    # a padded batch, a bias and heads of 80, 120 in fp16 training; a continued prompt; blocks of 128
    case("fp16", b=3, sq=300, sk=300, hq=6, hkv=2, d=80, keep=3, nb=20, q_lens=[300, 177, 1], k_lens=[300, 177, 1]),
    case("fp16", b=2, sq=100, sk=1000, hq=4, hkv=4, d=120, block=128, keep=5, q_lens=[100, 33], k_lens=[1000, 900]),
    case("bf16", b=2, sq=100, sk=1000, hq=8, hkv=1, d=128, block=128, keep=5, nb=30),
    case("fp16", b=2, sq=4, sk=1000, hq=4, hkv=1, d=128, keep=6, nb=12),
], ids=lambda c: "-".join(str(c[k]) for k in ("dtype", "b", "sq", "sk", "hq", "hkv", "d", "block", "keep")))
@pytest.mark.parametrize("size", [1.0, 2.0 ** -12, 64.0])
def test_gradients_of_other_sizes(A, c, size):
    """dout of another size than 1."""
    s = make(c, 46)
    s["dout"] = (s["dout"].float() * size).to(s["dout"].dtype)
    check(A, c, s)


@gpu
def test_select_by_the_smallest_numbers_fp16(A):
    """Queries or summaries below fp16's normal numbers: their bits count."""
    gen = torch.Generator(device="cuda").manual_seed(47)
    q = torch.randn(1, 40, 8, 64, device="cuda", generator=gen)
    m = torch.randn(1, 2, 100, 64, device="cuda", generator=gen)
    for a, b in ((2.0 ** -18, 1.0), (1.0, 2.0 ** -18), (2.0 ** -16, 2.0 ** -17)):
        x, y = (q * a).half(), (m * b).half()
        got = A.block_select(x, y, 9, k_len=6400)
        assert torch.equal(got.cpu(), ref.select(x, y, 9, 6400, 64, True, 1, 1, None, None))


@gpu
@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
def test_inputs_of_the_smallest_numbers_fp16(A, name):
    c = case("fp16", b=2, sq=90, sk=200, hq=4, hkv=2, d=64, nb=8)
    s = make(c, 48)
    s[name] = (s[name].float() * 2.0 ** -17).half()
    if name in ("q", "k"):
        other = "k" if name == "q" else "q"
        s[other] = (s[other].float() * 256).half()      # so that scores come of it
        s["dout"] = (s["dout"].float() / 64).half()
    check(A, c, s)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_one_row_sees_values_that_another_must_not(A, dtype):
    """Largest finite values and keys in places that only some rows read: their size reaches nobody else's precision."""
    c = case(dtype, b=1, sq=150, sk=256, hq=4, hkv=2, d=64, keep=2, nb=5)
    s = make(c, 49)
    s["blocks"][..., 0] = 0
    s["blocks"][..., 1] = torch.arange(150, device="cuda") % 3
    want, bound = ref.attention(s["q"], s["k"], s["v"], s["blocks"], 64, True, 0.125, None, None, s["table"], s["edges"], s["dout"])
    top = torch.finfo(DT[dtype]).max
    k, v = s["k"].clone(), s["v"].clone()
    k[0, 140:150], v[0, 140:150] = -top, top      # block 2
    v[0, 150:160] = -top
    out, lse = A.block_attention(s["q"], k, v, s["blocks"], **kw(c, s))
    dq = A.block_attention_grad(s["dout"], s["q"], k, v, out, lse, s["blocks"], **kw(c, s))[0]
    i = torch.arange(150, device="cuda")
    free = ~((i % 3 == 2) & (i + 106 >= 140))
    for got, name in ((out, "out"), (dq, "dq")):
        near(got[0, free], want[name][0, free], bound[name][0, free], name)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nb", [0, 9])
def test_padded_batches_without_a_mask(A, dtype, nb):
    """Both directions, lengths of their own, more queries than keys among them."""
    c = case(dtype, b=5, sq=77, sk=300, hq=6, hkv=2, d=72, keep=4, causal=False, nb=nb, q_lens=[77, 0, 1, 40, 77], k_lens=[300, 200, 1, 64, 0])
    check(A, c, make(c, 50))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("low", [float("-inf"), -1e4])
@pytest.mark.parametrize("sq,sk,hq,hkv", [(150, 200, 4, 2), (4, 700, 4, 1), (1, 5000, 2, 1)])
def test_buckets_that_mask(A, dtype, low, sq, sk, hq, hkv):
    """A bias of -infinity, or of -10000, keeps far keys out, and near ones for another head."""
    c = case(dtype, sq=sq, sk=sk, hq=hq, hkv=hkv, d=64, keep=-(-sk // 64), nb=4, all=True)
    s = make(c, 51)
    s["edges"] = torch.tensor([-sk + 70, -90, -3], dtype=torch.int32, device="cuda")
    s["table"][0] = low
    s["table"][3, 1] = low
    check(A, c, s)
