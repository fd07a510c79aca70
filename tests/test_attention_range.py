"""Block-sparse attention and the relative bias at the ends of their types' and sizes' ranges."""
import math

import pytest
import torch

import attention_ref as ref
from test_attention import A, DT, case, check, kw, make, near  # noqa: F401

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
